// Rows that a team of lanes holds in registers: who holds which entries, sums over a team, and the sum of what groups of rows
// leave for each column.
#pragma once

#include "lane_ops.h"
#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

struct Team {
    int lanes, vecs;                        // 0 lanes: the row is not held
};

// Of a lane's vectors the last alone may lie behind the row.
__host__ Team team_that_fits(int64_t nv, int64_t lanes, int vecs) {
    return nv > (vecs - 1) * lanes && nv <= vecs * lanes ? Team{(int)lanes, vecs} : Team{0, 0};
}

int64_t vectors_of(int dtype, int64_t hidden) {
    const int64_t vec = dtype == MRL_F32 ? 4 : 8;
    return hidden < vec ? 0 : (hidden + vec - 1) / vec;
}

// Where lane `tl` of a team finds its vector q, and how many entries of its last one are others'.
template <int kVecs, int kVec>
struct Columns {
    int first, step, last, skip;
    __device__ __forceinline__ Columns(int tl, int lanes, int hidden) {
        const int at = (tl + (kVecs - 1) * lanes) * kVec;
        first = tl * kVec;
        step = lanes * kVec;
        last = at < hidden - kVec ? at : hidden - kVec;
        skip = at >= hidden ? kVec : at - last;
    }
    __device__ __forceinline__ int at(int q) const { return q < kVecs - 1 ? first + q * step : last; }
    // entry i of vector q is this lane's
    __device__ __forceinline__ bool own(int q, int i) const { return q < kVecs - 1 || i >= skip; }
};

// Sums of two values over a team, in all of its lanes.  `lds`: an entry per wavefront, not in use since the last barrier but
// one.  Every thread of the workgroup calls it.
__device__ __forceinline__ float2 team_sum2(float a, float b, int lanes, float2* lds) {
    a = mrl::lanes_sum<4>(a);
    b = mrl::lanes_sum<4>(b);
    if (lanes == 16) return make_float2(a, b);
    a = (mrl::lane_value(a, 0) + mrl::lane_value(a, 16)) + (mrl::lane_value(a, 32) + mrl::lane_value(a, 48));
    b = (mrl::lane_value(b, 0) + mrl::lane_value(b, 16)) + (mrl::lane_value(b, 32) + mrl::lane_value(b, 48));
    if (lanes == 64) return make_float2(a, b);
    lds[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    // the team's wavefronts' sums, one in each of 16 lanes
    const int waves = lanes >> 6, first = (threadIdx.x >> 6) / waves * waves, w = threadIdx.x & 15;
    const float2 s = w < waves ? lds[first + w] : make_float2(0.f, 0.f);
    return make_float2(mrl::lanes_sum<4>(s.x), mrl::lanes_sum<4>(s.y));
}

// Sums of the groups' sums, `stride` entries apart (of 455 groups of 3 584 columns: 5 us): 32 columns a workgroup, 32 lanes a column that each take every 32nd group.
template <int WDT>
__global__ __launch_bounds__(1024) void norm_part_sum_kernel(const float* __restrict__ part, int64_t stride, int n_parts, int64_t hidden,
                                                             typename Elem<WDT>::T* __restrict__ dweight,
                                                             typename Elem<WDT>::T* __restrict__ dbias) {
    __shared__ float lds[32][33];
    typename Elem<WDT>::T* out = blockIdx.y == 0 ? dweight : dbias;
    if (!out) return;
    const int c = threadIdx.x & 31, slice = threadIdx.x >> 5;
    const int64_t j = (int64_t)blockIdx.x * 32 + c;
    const float* p = part + blockIdx.y * hidden + (j < hidden ? j : hidden - 1);
    float s = 0.f;
    for (int g = slice; g < n_parts; g += 16 * 32) {    // sixteen on their way at a time
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int k = g + i * 32;
            v[i] = p[(int64_t)(k < n_parts ? k : slice) * stride];
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) s += g + i * 32 < n_parts ? v[i] : 0.f;
    }
    lds[slice][c] = s;
    __syncthreads();
    // a wavefront joins the slices of two columns
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    s = mrl::lanes_sum<4>(lds[lane & 31][2 * wave + (lane >> 5)]);
    s += __shfl_xor(s, 16, 64);
    const int64_t column = (int64_t)blockIdx.x * 32 + 2 * wave + (lane >> 5);
    if ((lane & 31) == 0 && column < hidden) Elem<WDT>::store(out + column, s);
}

template <int N>
struct Int {
    static constexpr int value = N;
};

template <typename F>
void with_vecs(int vecs, F launch) {
    switch (vecs) {
        case 1: return launch(Int<1>());
        case 2: return launch(Int<2>());
        case 3: return launch(Int<3>());
        default: return launch(Int<4>());
    }
}

}  // namespace
