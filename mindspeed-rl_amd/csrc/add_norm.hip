// RMS norm with the residual's addition, and with an output in 8 bits, for gfx950.
//
//   h = x + residual, rounded to the residual's type;  r = (mean_j h_j^2 + eps)^(-1/2),  n_j = h_j r,  y_j = n_j w_j
//   d_j = dh_j + r (g_j - n_j mean_i(g_i n_i)),  g_j = dy_j w_j;  dx = dresidual = d, each rounded to its type;  dw_j = sum_rows dy_j n_j
//   8 bits: s = max(max |y| * (1/448), 2^-126) over the row or over 128 entries,  q = e4m3(y / s)
//
// What is normalised is h as it is stored: the next layer's residual, this norm and its backward see one value, and the call
// gives what an addition and a norm behind it give.  Sums are held in fp32.
//
// Both passes are bound by memory: the forward reads two tensors and writes two, the backward reads three and writes one (two, where the
// stream is wider than the rows).  32 768 x 4 096 bf16: forward 171 us (6.3 TB/s), backward with the weight's gradient 177 (6.1), to e4m3 by
// rows 149, by blocks 152 (6.2); 32 768 x 3 584 bf16 beside an fp32 stream 227 (6.2) and 310 (6.1), to e4m3 205.  (Here and below: calls that
// follow each other in a replayed graph.)
#include "lane_ops.h"
#include "mrl_internal.h"
#include "norm_rows.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

constexpr int kBlock = 256;
constexpr int kColumnSlabs = 256;           // most partial sums of a column
constexpr float kMost = 448.f;              // of e4m3
constexpr float kLeast = 1.17549435e-38f;   // 2^-126: what a scale does not go below

__device__ __forceinline__ float block_sum(float a, float* lds) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) a += __shfl_xor(a, off, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

// Of the bits of |y|: larger than those of any number are an infinity's, and NaN's beyond.
__device__ __forceinline__ uint32_t block_most(uint32_t a, uint32_t* lds) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) a = max(a, (uint32_t)__shfl_xor((int)a, off, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    return max(max(lds[0], lds[1]), max(lds[2], lds[3]));
}

__device__ __forceinline__ float scale_of(uint32_t most) {
    const float s = __uint_as_float(most) * (1.f / kMost);
    return s < kLeast ? kLeast : s;         // NaN stays
}

// Quotients by a scale: y * (1 / s) and a correction by what it leaves of y, which makes it the nearest number to y / s (the
// reciprocal is, and the rest is exact from |y| = 2^-103 on; below, the last bit may be another).  -0 stays, and numbers under an infinite scale are 0.  us, by the
// reciprocal alone / so / by the compiler's division: 32 768 x 4 096 bf16 without a residual 67 / 70 / 91, with one 148 / 150 / 150.
struct Quotient {
    float s, inv;
    __device__ __forceinline__ explicit Quotient(float scale) : s(scale), inv(1.f / scale) {
        if (inv == 0.f) s = 0.f;
    }
    __device__ __forceinline__ float of(float y) const {
        const float q = mrl::mul_rn(y, inv);
        return __builtin_fmaf(-__builtin_fmaf(q, s, -y), inv, q);
    }
};

__device__ __forceinline__ uint8_t code_of(float x) { return (uint8_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false); }

struct FwdArgs {
    const void *x, *residual, *weight;
    void *h, *y;                            // y: the codes where there is `scale`
    float *rstd, *scale;
    int64_t x_stride, residual_stride, n_rows;
    int32_t hidden, block, wide_weight;     // block 0: a scale a row
    float eps;
};

template <int DT>
__device__ __forceinline__ float weight_at(const void* w, int wide, int j) {
    return wide ? ((const float*)w)[j] : Elem<DT>::load((const typename Elem<DT>::T*)w + j);
}

// ------------------------------------------------------------------------------------ rows of any width
// Rows that registers do not hold, or shorter than a vector: a workgroup a row, an entry a thread at a time, read again for every sum
// (from the caches).  4 096 x 40 960 bf16: forward 628 us (2.1 TB/s), backward 961; 100 000 x 7 74 and 117.
template <int DT, int RT>
__global__ __launch_bounds__(kBlock) void add_norm_fwd_kernel(FwdArgs a) {
    using T = typename Elem<DT>::T;
    using R = typename Elem<RT>::T;
    __shared__ float lds[4];
    __shared__ uint32_t mlds[4];
    const int64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    const R* res = a.residual ? (const R*)a.residual + row * a.residual_stride : nullptr;
    R* h = (R*)a.h + row * a.hidden;
    const auto at = [&](int j) { return res ? Elem<RT>::load(h + j) : Elem<DT>::load(x + j); };
    float ss = 0.f;
    for (int j = threadIdx.x; j < a.hidden; j += kBlock) {
        if (res) Elem<RT>::store(h + j, Elem<DT>::load(x + j) + Elem<RT>::load(res + j));
        const float z = at(j);              // what this thread has just written
        ss += z * z;
    }
    const float r = 1.f / sqrtf(block_sum(ss, lds) / (float)a.hidden + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = r;
    const auto value = [&](int j) { return at(j) * r * weight_at<DT>(a.weight, a.wide_weight, j); };
    if (!a.scale) {
        for (int j = threadIdx.x; j < a.hidden; j += kBlock) Elem<DT>::store((T*)a.y + row * a.hidden + j, value(j));
        return;
    }
    uint8_t* q = (uint8_t*)a.y + row * a.hidden;
    if (!a.block) {
        uint32_t most = 0;
        for (int j = threadIdx.x; j < a.hidden; j += kBlock) most = max(most, __float_as_uint(fabsf(value(j))));
        const float s = scale_of(block_most(most, mlds));
        const Quotient by(s);
        if (threadIdx.x == 0) a.scale[row] = s;
        for (int j = threadIdx.x; j < a.hidden; j += kBlock) q[j] = code_of(by.of(value(j)));
        return;
    }
    // a block is two entries of a wavefront's lanes
    const int blocks = a.hidden / 128, lane = threadIdx.x & 63;
    for (int b = threadIdx.x >> 6; b < blocks; b += kBlock / 64) {
        float v[2];
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = b * 128 + i * 64 + lane;      // of h, written by another thread
            float z = Elem<DT>::load(x + j);
            if (res) {
                R t;
                Elem<RT>::store(&t, z + Elem<RT>::load(res + j));
                z = Elem<RT>::load(&t);
            }
            v[i] = z * r * weight_at<DT>(a.weight, a.wide_weight, j);
            most = max(most, __float_as_uint(fabsf(v[i])));
        }
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, 64));
        const float s = scale_of(most);
        const Quotient by(s);
        if (lane == 0) a.scale[row * blocks + b] = s;
#pragma unroll
        for (int i = 0; i < 2; ++i) q[b * 128 + i * 64 + lane] = code_of(by.of(v[i]));
    }
}

struct BwdArgs {
    const void *dy, *dh, *h, *weight;
    const float* rstd;
    void *dx, *dresidual, *dweight;
    float* part;
    int64_t dy_stride, dh_stride, n_rows;
    int32_t hidden, wide_weight;
};

template <int DT, int RT>
__global__ __launch_bounds__(kBlock) void add_norm_bwd_kernel(BwdArgs a) {
    using T = typename Elem<DT>::T;
    using R = typename Elem<RT>::T;
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    const T* dy = (const T*)a.dy + row * a.dy_stride;
    const R* h = (const R*)a.h + row * a.hidden;
    const R* dh = a.dh ? (const R*)a.dh + row * a.dh_stride : nullptr;
    const float r = a.rstd[row];
    float gn = 0.f;
    for (int j = threadIdx.x; j < a.hidden; j += kBlock)
        gn += Elem<DT>::load(dy + j) * weight_at<DT>(a.weight, a.wide_weight, j) * (Elem<RT>::load(h + j) * r);
    const float c = block_sum(gn, lds) / (float)a.hidden;
    for (int j = threadIdx.x; j < a.hidden; j += kBlock) {
        const float g = Elem<DT>::load(dy + j) * weight_at<DT>(a.weight, a.wide_weight, j);
        const float d = r * (g - Elem<RT>::load(h + j) * r * c) + (dh ? Elem<RT>::load(dh + j) : 0.f);
        if (a.dx) Elem<DT>::store((T*)a.dx + row * a.hidden + j, d);
        if (a.dresidual) Elem<RT>::store((R*)a.dresidual + row * a.hidden + j, d);
    }
}

// Partial sums of the columns: a column a thread, a slab of rows per workgroup in y.
template <int DT, int RT>
__global__ __launch_bounds__(kBlock) void add_norm_columns_kernel(BwdArgs a, int64_t slab_rows) {
    const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (j >= a.hidden) return;
    const int64_t lo = (int64_t)blockIdx.y * slab_rows, hi = lo + slab_rows < a.n_rows ? lo + slab_rows : a.n_rows;
    float dw = 0.f;
    for (int64_t row = lo; row < hi; ++row)
        dw += Elem<DT>::load((const typename Elem<DT>::T*)a.dy + row * a.dy_stride + j) *
              (Elem<RT>::load((const typename Elem<RT>::T*)a.h + row * a.hidden + j) * a.rstd[row]);
    a.part[(int64_t)blockIdx.y * a.hidden + j] = dw;
}

// ------------------------------------------------------------------------------------ rows in registers
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_anywhere __attribute__((aligned(2)));

// kN entries as they were loaded: a vector of 16 bytes, half of one beside a wider stream, or two of an fp32 weight.
template <int DT, int kN>
struct Raw {
    static constexpr int kVec = Elem<DT>::kVec, kParts = kN / kVec;
    static constexpr bool kHalf = kN < kVec;
    using T = typename Elem<DT>::T;
    u32x4 v[kHalf ? 1 : kParts];
    template <bool kStream>
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (kHalf) {
            const u32x2_anywhere* from = (const u32x2_anywhere*)p;
            const u32x2 t = kStream ? __builtin_nontemporal_load(from) : *from;
            v[0] = mrl::make_u32x4(t.x, t.y, 0u, 0u);
        } else {
#pragma unroll
            for (int i = 0; i < kParts; ++i) v[i] = kStream ? mrl::Vec<DT>::load_nt(p + i * kVec) : mrl::Vec<DT>::load(p + i * kVec);
        }
    }
    template <bool kStream>
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (kHalf) {
            u32x2_anywhere* to = (u32x2_anywhere*)p;
            const u32x2 t = {v[0].x, v[0].y};
            if (kStream) __builtin_nontemporal_store(t, to);
            else *to = t;
        } else {
#pragma unroll
            for (int i = 0; i < kParts; ++i) {
                if (kStream) mrl::Vec<DT>::store_nt(p + i * kVec, v[i]);
                else mrl::Vec<DT>::store(p + i * kVec, v[i]);
            }
        }
    }
    __device__ __forceinline__ void unpack(float (&z)[kN]) const {
#pragma unroll
        for (int i = 0; i < (kHalf ? 1 : kParts); ++i) {
            float t[kVec];
            Elem<DT>::unpack(v[i], t);
#pragma unroll
            for (int j = 0; j < (kHalf ? kN : kVec); ++j) z[i * kVec + j] = t[j];
        }
    }
    __device__ __forceinline__ void pack(const float (&z)[kN]) {
#pragma unroll
        for (int i = 0; i < (kHalf ? 1 : kParts); ++i) {
            float t[kVec] = {};
#pragma unroll
            for (int j = 0; j < (kHalf ? kN : kVec); ++j) t[j] = z[i * kVec + j];
            v[i] = Elem<DT>::pack(t);
        }
    }
};

template <bool kStream, int kN>
__device__ __forceinline__ void store_codes(uint8_t* p, const float (&z)[kN]) {
    typedef uint32_t Words __attribute__((ext_vector_type(kN / 4)));
    typedef Words WordsAnywhere __attribute__((aligned(1)));
    Words c;
#pragma unroll
    for (int w = 0; w < kN / 4; ++w) {
        int t = __builtin_amdgcn_cvt_pk_fp8_f32(z[4 * w], z[4 * w + 1], 0, false);
        c[w] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(z[4 * w + 2], z[4 * w + 3], t, true);
    }
    if (kStream) __builtin_nontemporal_store(c, (WordsAnywhere*)p);
    else *(WordsAnywhere*)p = c;
}

__device__ __forceinline__ uint32_t lanes_most(uint32_t x) {    // over 16 lanes
    x = max(x, mrl::lane_partner_bits<0>(x));
    x = max(x, mrl::lane_partner_bits<1>(x));
    x = max(x, mrl::lane_partner_bits<2>(x));
    return max(x, mrl::lane_partner_bits<3>(x));
}

// Over a team, in all of its lanes, as team_sum2.
__device__ __forceinline__ uint32_t team_most(uint32_t x, int lanes, uint32_t* lds) {
    x = lanes_most(x);
    if (lanes == 16) return x;
    x = max(x, (uint32_t)__shfl_xor((int)x, 16, 64));
    x = max(x, (uint32_t)__shfl_xor((int)x, 32, 64));
    if (lanes == 64) return x;
    lds[threadIdx.x >> 6] = x;
    __syncthreads();
    const int waves = lanes >> 6, first = (threadIdx.x >> 6) / waves * waves, w = threadIdx.x & 15;
    return lanes_most(w < waves ? lds[first + w] : 0u);
}

// A team a row, kVecs vectors of the stream's type a lane, each row read once.  The last vector of a row that is not whole vectors overlaps the one in
// front of it; what a lane holds twice over is left out of its sums and written twice with the same bits.
template <int DT, int RT, int WDT, int kVecs, bool kRes, bool kFp8, bool kStream>
__global__ __launch_bounds__(1024) void add_norm_fwd_rows_kernel(FwdArgs a, int lanes) {
    using T = typename Elem<DT>::T;
    using R = typename Elem<RT>::T;
    constexpr int kVec = Elem<RT>::kVec;
    __shared__ float2 lds[16];
    __shared__ uint32_t most_lds[16];
    const int team = threadIdx.x / lanes, tl = threadIdx.x - team * lanes;
    const int64_t wanted = (int64_t)blockIdx.x * (blockDim.x / lanes) + team;
    const bool live = wanted < a.n_rows;
    const int64_t row = live ? wanted : a.n_rows - 1;
    const Columns<kVecs, kVec> col(tl, lanes, a.hidden);
    Raw<DT, kVec> x[kVecs];
    Raw<RT, kVec> h[kVecs];
    Raw<WDT, kVec> w[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) x[q].template load<kStream>((const T*)a.x + row * a.x_stride + col.at(q));
    if (kRes) {
#pragma unroll
        for (int q = 0; q < kVecs; ++q) h[q].template load<kStream>((const R*)a.residual + row * a.residual_stride + col.at(q));
    }
#pragma unroll
    for (int q = 0; q < kVecs; ++q) w[q].template load<false>((const typename Elem<WDT>::T*)a.weight + col.at(q));
    const auto value = [&](int q, float (&z)[kVec]) {
        if (kRes) h[q].unpack(z);
        else x[q].unpack(z);
    };
    float ss = 0.f;
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        float z[kVec];
        if (kRes) {
            float t[kVec];
            x[q].unpack(z);
            h[q].unpack(t);
#pragma unroll
            for (int i = 0; i < kVec; ++i) z[i] += t[i];
            h[q].pack(z);
        }
        value(q, z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) ss += col.own(q, i) ? z[i] * z[i] : 0.f;
    }
    const float r = 1.f / sqrtf(team_sum2(ss, 0.f, lanes, lds).x * (1.f / (float)a.hidden) + a.eps);
    Quotient by(1.f);
    if (kFp8 && !a.block) {
        uint32_t most = 0;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec], wf[kVec];
            value(q, z);
            w[q].unpack(wf);
#pragma unroll
            for (int i = 0; i < kVec; ++i) most = max(most, __float_as_uint(fabsf(z[i] * r * wf[i])));
        }
        const float s = scale_of(team_most(most, lanes, most_lds));
        by = Quotient(s);
        if (live && tl == 0) a.scale[row] = s;
    }
    if (!live) return;
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        const int64_t at = row * a.hidden + col.at(q);
        if (kRes) h[q].template store<kStream>((R*)a.h + at);
        float z[kVec], wf[kVec];
        value(q, z);
        w[q].unpack(wf);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = z[i] * r * wf[i];
        if (!kFp8) {
            Raw<DT, kVec> y;
            y.pack(z);
            y.template store<kStream>((T*)a.y + at);
            continue;
        }
        if (a.block) {                      // of whole blocks: 16 lanes, or 32 of fp32, a block
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < kVec; ++i) most = max(most, __float_as_uint(fabsf(z[i])));
            most = lanes_most(most);
            if (kVec == 4) most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
            const float s = scale_of(most);
            by = Quotient(s);
            if (q == kVecs - 1 && col.skip) continue;       // lanes behind the row
            if ((tl & (128 / kVec - 1)) == 0) a.scale[at / 128] = s;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = by.of(z[i]);
        store_codes<kStream>((uint8_t*)a.y + at, z);
    }
    if (a.rstd && tl == 0) a.rstd[row] = r;
}

// The backward in one pass: workgroups stay and take rows in turn, a team a row, and hold the sums over their rows of the lane's
// columns in registers; the workgroup's sums go to part[group][hidden].
constexpr int kBwdBlock = 512;              // threads of a workgroup that holds several teams
// Most workgroups: two on each of 256 CUs (32 768 x 3 584 bf16 156 us, by 768 183, by 1 024 171).
constexpr int kBwdGroups = 512;
constexpr int64_t kBwdManyVecs = 8 << 20;   // 128 MiB of rows

template <int DT, int RT, int WDT, int kVecs, int kBlockMost, bool kDh, bool kStream>
__global__ __launch_bounds__(kBlockMost) void add_norm_bwd_rows_kernel(BwdArgs a, int lanes, void* __restrict__ dweight) {
    using T = typename Elem<DT>::T;
    using R = typename Elem<RT>::T;
    constexpr int kVec = Elem<RT>::kVec;
    constexpr bool kOne = kBlockMost > kBwdBlock;       // the team is the workgroup
    constexpr bool kAhead = kVecs == 1 || (kVecs == 2 && !kOne);   // the next row is requested before this one is summed
    extern __shared__ float columns[];                  // [kVecs * kVec][lanes] sums on their way between teams
    __shared__ float2 lds[2][16];
    const int teams = kOne ? 1 : blockDim.x / lanes, team = kOne ? 0 : threadIdx.x / lanes;
    const int tl = threadIdx.x - team * lanes, hidden = a.hidden;
    const Columns<kVecs, kVec> col(tl, lanes, hidden);
    const float inv = 1.f / (float)hidden;
    float dw[kVecs][kVec] = {};
    Raw<WDT, kVec> w[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) w[q].template load<false>((const typename Elem<WDT>::T*)a.weight + col.at(q));
    const int64_t step = (int64_t)gridDim.x * teams;
    Raw<RT, kVec> hn[kVecs], un[kVecs];
    Raw<DT, kVec> gn[kVecs];
    float rn;
    const auto request = [&](int64_t wanted) {
        const int64_t row = wanted < a.n_rows ? wanted : a.n_rows - 1;
        rn = a.rstd[row];
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            hn[q].template load<kStream>((const R*)a.h + row * hidden + col.at(q));
            gn[q].template load<kStream>((const T*)a.dy + row * a.dy_stride + col.at(q));
        }
        if (kDh) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q) un[q].template load<kStream>((const R*)a.dh + row * a.dh_stride + col.at(q));
        }
    };
    if (kAhead) request((int64_t)blockIdx.x * teams + team);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * teams; base < a.n_rows; base += step, turn ^= 1) {
        // teams behind the last row do that row again, without its share of the columns' sums
        const bool counts = kOne || base + team < a.n_rows;
        const int64_t row = counts ? base + team : a.n_rows - 1;
        if (!kAhead) request(row);
        Raw<RT, kVec> h[kVecs], u[kVecs];
        Raw<DT, kVec> g[kVecs];
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            h[q] = hn[q];
            g[q] = gn[q];
            if (kDh) u[q] = un[q];
        }
        const float r = rn;
        if (kAhead) request(base + team + step);
        float sgn = 0.f;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec], gf[kVec], wf[kVec];
            h[q].unpack(z);
            g[q].unpack(gf);
            w[q].unpack(wf);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float own = col.own(q, i) ? gf[i] : 0.f, n = z[i] * r;
                dw[q][i] += (counts ? own : 0.f) * n;
                sgn += own * wf[i] * n;
            }
        }
        const float c = team_sum2(sgn, 0.f, lanes, lds[turn]).x * inv;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec], gf[kVec], wf[kVec], uf[kVec] = {};
            h[q].unpack(z);
            g[q].unpack(gf);
            w[q].unpack(wf);
            if (kDh) u[q].unpack(uf);
#pragma unroll
            for (int i = 0; i < kVec; ++i) z[i] = r * (gf[i] * wf[i] - z[i] * r * c) + uf[i];
            const int64_t at = row * hidden + col.at(q);
            if (a.dx) {
                Raw<DT, kVec> d;
                d.pack(z);
                d.template store<kStream>((T*)a.dx + at);
            }
            if (a.dresidual) {
                Raw<RT, kVec> d;
                d.pack(z);
                d.template store<kStream>((R*)a.dresidual + at);
            }
        }
    }
    if (!a.part && !dweight) return;
    // the workgroup's sums: teams of a wavefront by lane exchange, then one after the other through LDS
    const bool paired = !kOne && lanes < 64;
    const int turns = paired ? blockDim.x >> 6 : teams, mine = paired ? threadIdx.x >> 6 : team;
    const bool holds = !paired || (threadIdx.x & 63) < 16;
    if (paired) {
#pragma unroll
        for (int q = 0; q < kVecs; ++q)
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                dw[q][i] += __shfl_xor(dw[q][i], 16, 64);
                dw[q][i] += __shfl_xor(dw[q][i], 32, 64);
            }
    }
    float* out = a.part ? a.part + (int64_t)blockIdx.x * hidden : nullptr;
    typename Elem<WDT>::T* vec = (typename Elem<WDT>::T*)dweight;       // the sums themselves, of the only workgroup
    for (int t = 0; t < turns; ++t) {
        if (t == mine && holds) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    float* at = columns + (q * kVec + i) * lanes + tl;          // a lane's place is the same for every team
                    const float s = dw[q][i] + (!kOne && t > 0 ? *at : 0.f);
                    if (t < turns - 1) *at = s;
                    else if (col.own(q, i) && out) out[col.at(q) + i] = s;
                    else if (col.own(q, i)) Elem<WDT>::store(vec + col.at(q) + i, s);
                }
        }
        if (!kOne) __syncthreads();
    }
}

// As many wavefronts as `vecs` vectors a lane make, or more vectors where 16 of them are not enough.
Team team_of_waves(int64_t nv, int vecs) {
    for (; vecs <= 4; ++vecs) {
        const int64_t lanes = (nv + 64 * vecs - 1) / (64 * vecs) * 64;
        if (lanes <= 1024) return team_that_fits(nv, lanes, (int)((nv + lanes - 1) / lanes));
    }
    return {0, 0};
}

// Teams of 16 lanes hold up to 32 vectors, without a residual 64 (us, 16 lanes / a wavefront: 65 536 x 256 bf16 25.6 / 31.6, 512
// 49.0 / 45.3, to e4m3 without a residual 20.4 / 28.1).  Longer rows: two vectors of each of x and the residual are on a lane's way, or four
// of x alone (us, one / two / four: 32 768 x 4 096 bf16 173 / 171 / 176, to e4m3 by blocks (their codes through the caches) 155 / 158 /
// 158, without a residual 117 / 84 / 70).
Team fwd_team_of(int rtype, int64_t hidden, int block, bool residual) {
    const int64_t nv = vectors_of(rtype, hidden);
    if (nv == 0) return {0, 0};
    if (nv <= (residual ? 32 : 64) && !(block && rtype == MRL_F32)) return team_that_fits(nv, 16, (int)((nv + 15) / 16));
    return team_of_waves(nv, residual ? 2 : 4);
}

// One vector a lane, the next row requested ahead, by 16 lanes where they hold the row (us, 16 lanes / a wavefront: 65 536 x 128 bf16
// 18.3 / 28.0, 256 by two vectors a lane 42.6 / 32.7).  Two (ahead as well) for much data where teams of one fill a workgroup of 512 threads by one
// or two and the second vector leaves few lanes idle: a sixteenth of 16 bits, none of fp32.  us, one / two, by MiB of rows: bf16, 256 MiB: 1 600 wide 177 / 186,
// 1 792 181 / 185, 1 920 189 / 185, 2 000 193 / 187, 2 048 190 / 181, 4 000 197 / 185, 4 096 193 / 181, workgroups of other sizes 1 536 175 / 185,
// 3 584 177 / 181, 5 120 183 / 188, four teams 1 024 189 / 195; fp32: 1 000 192 / 196, 1 024 188 / 184, 2 000 193 / 194, 2 048 188 / 184.  By data: 2 048
// bf16 64 MiB 52 / 56, 96 76 / 76, 128 96 / 96, 160 122 / 116, 512 412 / 351; 2 000 128 98 / 100, 160 125 / 121.  Rows that 1 024 lanes do not hold so:
// two or, of fp32, four a lane, not ahead.
Team bwd_team_of(int rtype, int64_t n_rows, int64_t hidden) {
    const int64_t nv = vectors_of(rtype, hidden);
    if (nv == 0) return {0, 0};
    if (nv <= 16) return team_that_fits(nv, 16, 1);
    const int64_t one = (nv + 63) / 64 * 64;
    if ((one == kBwdBlock / 2 || one == kBwdBlock) && (one - nv) * 16 <= (rtype == MRL_F32 ? 0 : one) && n_rows * nv >= kBwdManyVecs)
        return team_that_fits(nv, one / 2, 2);
    for (int vecs = 1; vecs <= (rtype == MRL_F32 ? 4 : 2); vecs *= 2) {
        const int64_t lanes = (nv + 64 * vecs - 1) / (64 * vecs) * 64;
        if (lanes <= 1024) return team_that_fits(nv, lanes, vecs);
    }
    return {0, 0};
}

// Threads and number of the backward's workgroups.
int bwd_block(const Team& team) { return team.lanes > kBwdBlock ? team.lanes : kBwdBlock / team.lanes * team.lanes; }

int bwd_groups(const Team& team, int64_t n_rows) {
    const int teams = bwd_block(team) / team.lanes;
    const int64_t turns = (n_rows + teams - 1) / teams, fit = team.lanes > kBwdBlock ? kBwdGroups / 2 : kBwdGroups;
    const int64_t each = (turns + fit - 1) / fit;       // and no more workgroups than take as long
    return (int)((turns + each - 1) / each);
}

int64_t slab_rows_of(int64_t n_rows) {
    const int64_t rows = (n_rows + kColumnSlabs - 1) / kColumnSlabs;
    return rows < 16 ? 16 : rows;
}

// Threads of a workgroup of the forward's, and how many of them the rows take.
int fwd_block(const Team& team) { return team.lanes > kBlock ? team.lanes : team.lanes > 0 ? kBlock / team.lanes * team.lanes : kBlock; }

int64_t fwd_groups(const Team& team, int64_t n_rows) {
    const int64_t teams = team.lanes > 0 ? fwd_block(team) / team.lanes : 1;
    return (n_rows + teams - 1) / teams;
}

// Rows go past the caches where more bytes are read and written than the memory-side cache keeps for what comes next (us, through /
// past, forward and backward, bf16: 65 536 x 128 (67 MB) 11.4 and 18.5 / 13.7 and 19.3; 16 384 x 1 024 (134 MB) 25.2 and 31.6 / 23.2 and
// 29.4; 32 768 x 1 343 (352 MB) 72.1 and 71.2 / 69.0 and 67.9; 32 768 x 4 096 (1 GB) 183 and 202 / 171 and 177).
constexpr int64_t kCached = 96 << 20;

bool past_caches(int dtype, int rtype, int64_t entries) {
    return entries * 2 * (mrl::float_dtype_bytes(dtype) + mrl::float_dtype_bytes(rtype)) > kCached;
}

// launch(weight's type) for the rows' type or fp32.
template <int DT, typename F>
void with_weight(int wide, F launch) {
    if constexpr (DT == MRL_F32) launch(Int<MRL_F32>());
    else if (wide) launch(Int<MRL_F32>());
    else launch(Int<DT>());
}

template <typename F>
void with_flag(bool flag, F launch) {
    if (flag) launch(Int<1>());
    else launch(Int<0>());
}

template <int DT, int RT>
void launch_fwd(const FwdArgs& a, hipStream_t stream) {
    const Team team = fwd_team_of(RT, a.hidden, a.block, a.residual != nullptr);
    const dim3 grid((unsigned)fwd_groups(team, a.n_rows)), block(fwd_block(team));
    if (team.lanes == 0) {
        hipLaunchKernelGGL((add_norm_fwd_kernel<DT, RT>), grid, block, 0, stream, a);
        return;
    }
    const bool past = past_caches(DT, RT, a.n_rows * a.hidden);
    const auto launch = [&](auto wdt, auto vecs, auto res, auto fp8, auto nt) {
        hipLaunchKernelGGL((add_norm_fwd_rows_kernel<DT, RT, decltype(wdt)::value, decltype(vecs)::value, decltype(res)::value != 0,
                                                     decltype(fp8)::value != 0, decltype(nt)::value != 0>),
                           grid, block, 0, stream, a, team.lanes);
    };
    with_weight<DT>(a.wide_weight, [&](auto wdt) {
        with_vecs(team.vecs, [&](auto vecs) {
            with_flag(past, [&](auto nt) {
                if (!a.scale) launch(wdt, vecs, Int<1>(), Int<0>(), nt);
                else if (a.residual) launch(wdt, vecs, Int<1>(), Int<1>(), nt);
                else if constexpr (DT == RT) launch(wdt, vecs, Int<0>(), Int<1>(), nt);
            });
        });
    });
}

template <int DT, int RT>
void launch_bwd(const BwdArgs& a, hipStream_t stream) {
    const Team team = bwd_team_of(RT, a.n_rows, a.hidden);
    const auto sum_parts = [&](int n_parts) {
        with_weight<DT>(a.wide_weight, [&](auto wdt) {
            constexpr int WDT = decltype(wdt)::value;
            hipLaunchKernelGGL((norm_part_sum_kernel<WDT>), dim3((unsigned)((a.hidden + 31) / 32)), dim3(1024), 0, stream, a.part,
                               (int64_t)a.hidden, n_parts, (int64_t)a.hidden, (typename Elem<WDT>::T*)a.dweight, (typename Elem<WDT>::T*)nullptr);
        });
    };
    if (team.lanes > 0 && a.n_rows > 0 && (a.dx || a.dresidual)) {
        const int groups = bwd_groups(team, a.n_rows), block = bwd_block(team);
        const bool past = past_caches(DT, RT, a.n_rows * a.hidden);
        BwdArgs b = a;
        if (!a.dweight || groups == 1) b.part = nullptr;
        const size_t lds = a.dweight && block > team.lanes ? (size_t)team.lanes * team.vecs * Elem<RT>::kVec * 4 : 0;
        const auto launch = [&](auto wdt, auto vecs, auto most, auto dh, auto nt) {
            hipLaunchKernelGGL((add_norm_bwd_rows_kernel<DT, RT, decltype(wdt)::value, decltype(vecs)::value, decltype(most)::value,
                                                         decltype(dh)::value != 0, decltype(nt)::value != 0>),
                               dim3((unsigned)groups), dim3(block), lds, stream, b, team.lanes, groups > 1 ? nullptr : a.dweight);
        };
        with_weight<DT>(a.wide_weight, [&](auto wdt) {
            with_flag(a.dh != nullptr, [&](auto dh) {
                with_flag(past, [&](auto nt) {
                    if constexpr (RT == MRL_F32) {
                        if (team.vecs == 4) return launch(wdt, Int<4>(), Int<1024>(), dh, nt);
                    }
                    if (team.vecs == 2 && team.lanes > kBwdBlock) launch(wdt, Int<2>(), Int<1024>(), dh, nt);
                    else if (team.vecs == 2) launch(wdt, Int<2>(), Int<kBwdBlock>(), dh, nt);
                    else if (team.lanes > kBwdBlock) launch(wdt, Int<1>(), Int<1024>(), dh, nt);
                    else launch(wdt, Int<1>(), Int<kBwdBlock>(), dh, nt);
                });
            });
        });
        if (a.dweight && groups > 1) sum_parts(groups);
        return;
    }
    if ((a.dx || a.dresidual) && a.n_rows > 0)
        hipLaunchKernelGGL((add_norm_bwd_kernel<DT, RT>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, stream, a);
    if (!a.dweight) return;
    const int64_t slab = slab_rows_of(a.n_rows);
    const int n_slabs = (int)((a.n_rows + slab - 1) / slab);
    if (n_slabs > 0)
        hipLaunchKernelGGL((add_norm_columns_kernel<DT, RT>), dim3((unsigned)((a.hidden + kBlock - 1) / kBlock), (unsigned)n_slabs), dim3(kBlock), 0,
                           stream, a, slab);
    sum_parts(n_slabs);
}

// The instance for the types of the rows and of the residual stream: the rows' type or fp32.
template <typename A>
void dispatch(int dtype, int rtype, const A& a, hipStream_t stream) {
    const auto go = [&](auto launch) { launch(a, stream); };
    constexpr bool kFwd = __is_same(A, FwdArgs);
#define MRL_TYPES(DT, RT)                                                                     \
    go([](const A& args, hipStream_t s) {                                                     \
        if constexpr (kFwd) launch_fwd<DT, RT>(args, s);                                      \
        else launch_bwd<DT, RT>(args, s);                                                     \
    })
    if (dtype == MRL_F32) MRL_TYPES(MRL_F32, MRL_F32);
    else if (dtype == MRL_BF16 && rtype == MRL_F32) MRL_TYPES(MRL_BF16, MRL_F32);
    else if (dtype == MRL_BF16) MRL_TYPES(MRL_BF16, MRL_BF16);
    else if (rtype == MRL_F32) MRL_TYPES(MRL_F16, MRL_F32);
    else MRL_TYPES(MRL_F16, MRL_F16);
#undef MRL_TYPES
}

int check_sizes(const char* fn, int dtype, int rtype, int wdtype, int64_t n_rows, int64_t hidden) {
    MRL_REQUIRE(mrl::float_dtype_bytes(dtype) != 0, MRL_ERR_UNSUPPORTED, "%s: dtype %d (want F32, BF16 or F16)", fn, dtype);
    MRL_REQUIRE(rtype == dtype || rtype == MRL_F32, MRL_ERR_UNSUPPORTED, "%s: residual dtype %d (want the rows' or F32)", fn, rtype);
    MRL_REQUIRE(wdtype == dtype || wdtype == MRL_F32, MRL_ERR_UNSUPPORTED, "%s: weight dtype %d (want the rows' or F32)", fn, wdtype);
    MRL_REQUIRE(n_rows >= 0 && hidden >= 1, MRL_ERR_INVALID_ARG, "%s: n_rows=%lld hidden=%lld", fn, (long long)n_rows,
                (long long)hidden);
    MRL_REQUIRE(hidden <= MRL_NORM_MAX_HIDDEN && n_rows <= 0x7fffffffLL && mrl::launch_fits(n_rows, kBlock), MRL_ERR_UNSUPPORTED,
                "%s: n_rows=%lld hidden=%lld (hidden at most %d, fewer than 2^24 rows)", fn, (long long)n_rows, (long long)hidden,
                MRL_NORM_MAX_HIDDEN);
    return MRL_OK;
}

int check_fwd(const char* fn, int dtype, int rtype, int wdtype, const FwdArgs& a, int64_t hidden) {
    const int rc = check_sizes(fn, dtype, rtype, wdtype, a.n_rows, hidden);
    if (rc != MRL_OK) return rc;
    const Team team = fwd_team_of(rtype, hidden, a.block, a.residual != nullptr);
    MRL_REQUIRE(mrl::launch_fits(fwd_groups(team, a.n_rows), fwd_block(team)), MRL_ERR_UNSUPPORTED,
                "%s: n_rows=%lld of hidden=%lld (2^32 threads hold fewer, up to 1024 for a row)", fn, (long long)a.n_rows, (long long)hidden);
    MRL_REQUIRE((a.x_stride >= hidden && (!a.residual || a.residual_stride >= hidden)) || a.n_rows <= 1, MRL_ERR_INVALID_ARG,
                "%s: strides %lld and %lld below hidden=%lld", fn, (long long)a.x_stride, (long long)a.residual_stride, (long long)hidden);
    MRL_REQUIRE(a.eps > 0.f && a.eps <= 3.0e38f, MRL_ERR_INVALID_ARG, "%s: eps=%g (want a positive, finite number)", fn, (double)a.eps);
    if (a.n_rows == 0) return MRL_OK;
    MRL_REQUIRE(a.x && a.weight && a.y && (a.h != nullptr) == (a.residual != nullptr), MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const size_t es = mrl::float_dtype_bytes(dtype), rs = mrl::float_dtype_bytes(rtype), ws = mrl::float_dtype_bytes(wdtype);
    MRL_REQUIRE(mrl::aligned(a.x, es) && mrl::aligned(a.residual, rs) && mrl::aligned(a.h, rs) && mrl::aligned(a.weight, ws) &&
                    mrl::aligned(a.y, a.scale ? 1 : es) && mrl::aligned(a.rstd, 4) && mrl::aligned(a.scale, 4),
                MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    return MRL_OK;
}

}  // namespace

extern "C" int mrl_add_norm_fwd(const void* x, int dtype, int64_t x_stride, const void* residual, int residual_dtype,
                                int64_t residual_stride, int64_t n_rows, int64_t hidden, const void* weight, int weight_dtype,
                                float eps, void* h, void* y, float* rstd, void* stream) {
    const char* fn = "mrl_add_norm_fwd";
    const FwdArgs a = {x, residual, weight, h, y, rstd, nullptr, x_stride, residual_stride, n_rows, (int32_t)hidden, 0,
                       weight_dtype == MRL_F32, eps};
    const int rc = check_fwd(fn, dtype, residual_dtype, weight_dtype, a, hidden);
    if (rc != MRL_OK || n_rows == 0) return rc;
    MRL_REQUIRE(residual, MRL_ERR_INVALID_ARG, "%s: NULL residual", fn);
    dispatch(dtype, residual_dtype, a, mrl::as_stream(stream));
    return mrl::check_launch(fn);
}

extern "C" int mrl_norm_fp8_fwd(const void* x, int dtype, int64_t x_stride, const void* residual, int residual_dtype,
                                int64_t residual_stride, int64_t n_rows, int64_t hidden, const void* weight, int weight_dtype,
                                float eps, int64_t block, void* h, void* q, float* scale, void* stream) {
    const char* fn = "mrl_norm_fp8_fwd";
    const FwdArgs a = {x, residual, weight, h, q, nullptr, scale, x_stride, residual_stride, n_rows, (int32_t)hidden, (int32_t)block,
                       weight_dtype == MRL_F32, eps};
    MRL_REQUIRE(block == 0 || block == 128, MRL_ERR_UNSUPPORTED, "%s: block=%lld (want 0, a row, or 128)", fn, (long long)block);
    MRL_REQUIRE(block == 0 || hidden % 128 == 0, MRL_ERR_UNSUPPORTED, "%s: hidden=%lld is not whole blocks of 128", fn, (long long)hidden);
    const int rc = check_fwd(fn, dtype, residual ? residual_dtype : dtype, weight_dtype, a, hidden);
    if (rc != MRL_OK || n_rows == 0) return rc;
    MRL_REQUIRE(scale, MRL_ERR_INVALID_ARG, "%s: NULL scale", fn);
    dispatch(dtype, residual ? residual_dtype : dtype, a, mrl::as_stream(stream));
    return mrl::check_launch(fn);
}

extern "C" int64_t mrl_add_norm_bwd_workspace_bytes(int64_t n_rows, int64_t hidden) {
    if (n_rows <= 0 || hidden <= 0 || n_rows > 0x7fffffffLL || !mrl::launch_fits(n_rows, kBlock) || hidden > MRL_NORM_MAX_HIDDEN) return 0;
    // a sum of a column for each workgroup of the one pass or each slab of rows: neither are more than the rows
    static_assert(kColumnSlabs <= kBwdGroups, "a place for every slab");
    return (n_rows < kBwdGroups ? n_rows : kBwdGroups) * hidden * 4;
}

extern "C" int mrl_add_norm_bwd(const void* dy, int64_t dy_stride, const void* dh, int64_t dh_stride, const void* h,
                                int residual_dtype, int dtype, int64_t n_rows, int64_t hidden, const void* weight, int weight_dtype,
                                const float* rstd, void* dx, void* dresidual, void* dweight, void* workspace,
                                int64_t workspace_bytes, void* stream) {
    const char* fn = "mrl_add_norm_bwd";
    const int rc = check_sizes(fn, dtype, residual_dtype, weight_dtype, n_rows, hidden);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE((dy_stride >= hidden && (!dh || dh_stride >= hidden)) || n_rows <= 1, MRL_ERR_INVALID_ARG,
                "%s: strides %lld and %lld below hidden=%lld", fn, (long long)dy_stride, (long long)dh_stride, (long long)hidden);
    MRL_REQUIRE(n_rows == 0 || (dy && h && weight && rstd), MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const int64_t need = dweight ? mrl_add_norm_bwd_workspace_bytes(n_rows, hidden) : 0;
    MRL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MRL_ERR_INVALID_ARG, "%s: workspace of %lld bytes (want %lld)",
                fn, (long long)workspace_bytes, (long long)need);
    const size_t es = mrl::float_dtype_bytes(dtype), rs = mrl::float_dtype_bytes(residual_dtype), ws = mrl::float_dtype_bytes(weight_dtype);
    MRL_REQUIRE(mrl::aligned(dy, es) && mrl::aligned(dh, rs) && mrl::aligned(h, rs) && mrl::aligned(weight, ws) && mrl::aligned(dx, es) &&
                    mrl::aligned(dresidual, rs) && mrl::aligned(dweight, ws) && mrl::aligned(rstd, 4) && mrl::aligned(workspace, 16),
                MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    if (n_rows == 0 && !dweight) return MRL_OK;
    const BwdArgs a = {dy, dh, h, weight, rstd, dx, dresidual, dweight, (float*)workspace, dy_stride, dh_stride, n_rows,
                       (int32_t)hidden, weight_dtype == MRL_F32};
    dispatch(dtype, residual_dtype, a, mrl::as_stream(stream));
    return mrl::check_launch(fn);
}
