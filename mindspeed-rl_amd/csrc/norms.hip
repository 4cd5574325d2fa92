// Layer norm and RMS norm of hidden states for gfx950, forward and backward.
//
//   layer:  mu = mean_j x_j,  r = (mean_j (x_j - mu)^2 + eps)^(-1/2),  n_j = (x_j - mu) r,  y_j = n_j w_j + b_j
//   RMS:    the same without mu and b
//   dx_j = r (g_j - c - n_j mean_i(g_i n_i)),  g_j = dy_j w_j,  c = mean_i g_i (RMS: 0)
//   dw_j = sum_rows dy_j n_j,  db_j = sum_rows dy_j
//
// Everything is held in fp32 and rounded once, to the output's type.  Both passes are bound by memory: the forward reads and
// writes a row once, the backward reads two and writes one.  32 768 x 3 584 bf16 RMS: forward 78 us (6.0 TB/s), backward
// with the weight's gradient 122 us (5.8 TB/s; 114 without); 65 536 x 5 120: 226 and 348 us.  Layer norm with all its gradients:
// 82 and 128 us.  (Here and below: calls that follow each other in a replayed graph.)
#include "lane_ops.h"
#include "mrl_internal.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kWideBlock = 1024;            // of rows that no team holds
constexpr int kColumnSlabs = 256;           // most partial sums of a column

// ------------------------------------------------------------------------------------ rows of any width
// Rows longer than registers hold, or shorter than a vector: a workgroup a row, read again for every sum (from the caches:
// a row is 4 MB at most), in vectors by 1 024 threads.  2 048 x 40 960 bf16 layer norm: forward 102 us (3.3 TB/s of what
// has to move; 264 by 256 threads an entry at a time), dx alone 127, backward 227.

// Sums of two values over the workgroup, the same in every thread.
__device__ __forceinline__ float2 block_sum2(float a, float b, float2* lds) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        a += __shfl_xor(a, off, 64);
        b += __shfl_xor(b, off, 64);
    }
    __syncthreads();                        // what an earlier call left has been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = make_float2(a, b);
    __syncthreads();
    float2 s = lds[0];
#pragma unroll
    for (int w = 1; w < kWideBlock / 64; ++w) {
        s.x += lds[w].x;
        s.y += lds[w].y;
    }
    return s;
}

// body(j) for the row's whole vectors, rest(j) for the entries behind them.
template <int kVec, typename Body, typename Rest>
__device__ __forceinline__ void over_row(int64_t hidden, Body body, Rest rest) {
    const int64_t whole = hidden / kVec * kVec;
    for (int64_t j = (int64_t)threadIdx.x * kVec; j < whole; j += (int64_t)kWideBlock * kVec) body(j);
    if (whole + threadIdx.x < hidden) rest(whole + threadIdx.x);
}

template <int DT>
__device__ __forceinline__ void load_row(const typename Elem<DT>::T* p, float (&z)[Elem<DT>::kVec]) {
    Elem<DT>::unpack(mrl::Vec<DT>::load(p), z);
}

template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kWideBlock) void norm_fwd_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                              int64_t hidden, const typename Elem<WDT>::T* __restrict__ weight,
                                                              const typename Elem<WDT>::T* __restrict__ bias, float eps,
                                                              typename Elem<DT>::T* __restrict__ y, float* __restrict__ mean,
                                                              float* __restrict__ rstd) {
    constexpr int kVec = Elem<DT>::kVec;
    __shared__ float2 lds[kWideBlock / 64];
    const int64_t row = blockIdx.x;
    const typename Elem<DT>::T* xr = x + row * x_stride;
    typename Elem<DT>::T* yr = y + row * hidden;
    float mu = 0.f;
    if (kLayer) {
        float s = 0.f;
        over_row<kVec>(hidden, [&](int64_t j) {
            float z[kVec];
            load_row<DT>(xr + j, z);
#pragma unroll
            for (int i = 0; i < kVec; ++i) s += z[i];
        }, [&](int64_t j) { s += Elem<DT>::load(xr + j); });
        mu = block_sum2(s, 0.f, lds).x / (float)hidden;
    }
    float ss = 0.f;
    over_row<kVec>(hidden, [&](int64_t j) {
        float z[kVec];
        load_row<DT>(xr + j, z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) ss += (z[i] - mu) * (z[i] - mu);
    }, [&](int64_t j) { ss += (Elem<DT>::load(xr + j) - mu) * (Elem<DT>::load(xr + j) - mu); });
    const float r = 1.f / sqrtf(block_sum2(ss, 0.f, lds).x / (float)hidden + eps);
    over_row<kVec>(hidden, [&](int64_t j) {
        float z[kVec], w[kVec], b[kVec] = {};
        load_row<DT>(xr + j, z);
        mrl::load_floats<WDT>(weight + j, w);
        if (kLayer && bias) mrl::load_floats<WDT>(bias + j, b);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = (z[i] - mu) * r * w[i] + b[i];
        mrl::Vec<DT>::store(yr + j, Elem<DT>::pack(z));
    }, [&](int64_t j) {
        const float b = kLayer && bias ? Elem<WDT>::load(bias + j) : 0.f;
        Elem<DT>::store(yr + j, (Elem<DT>::load(xr + j) - mu) * r * Elem<WDT>::load(weight + j) + b);
    });
    if (threadIdx.x == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = r;
    }
}

template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kWideBlock) void norm_dx_kernel(const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
                                                             const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                             int64_t hidden, const typename Elem<WDT>::T* __restrict__ weight,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             typename Elem<DT>::T* __restrict__ dx) {
    constexpr int kVec = Elem<DT>::kVec;
    __shared__ float2 lds[kWideBlock / 64];
    const int64_t row = blockIdx.x;
    const float mu = kLayer ? mean[row] : 0.f, r = rstd[row];
    const typename Elem<DT>::T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
    typename Elem<DT>::T* dxr = dx + row * hidden;
    float sg = 0.f, sgn = 0.f;
    const auto add = [&](float z, float g, float w) {
        sg += g * w;
        sgn += g * w * ((z - mu) * r);
    };
    over_row<kVec>(hidden, [&](int64_t j) {
        float z[kVec], g[kVec], w[kVec];
        load_row<DT>(xr + j, z);
        load_row<DT>(dyr + j, g);
        mrl::load_floats<WDT>(weight + j, w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) add(z[i], g[i], w[i]);
    }, [&](int64_t j) { add(Elem<DT>::load(xr + j), Elem<DT>::load(dyr + j), Elem<WDT>::load(weight + j)); });
    const float2 s = block_sum2(sg, sgn, lds);
    const float c = kLayer ? s.x / (float)hidden : 0.f, cn = s.y / (float)hidden;
    const auto slope = [&](float z, float g, float w) { return r * (g * w - c - (z - mu) * r * cn); };
    over_row<kVec>(hidden, [&](int64_t j) {
        float z[kVec], g[kVec], w[kVec];
        load_row<DT>(xr + j, z);
        load_row<DT>(dyr + j, g);
        mrl::load_floats<WDT>(weight + j, w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = slope(z[i], g[i], w[i]);
        mrl::Vec<DT>::store(dxr + j, Elem<DT>::pack(z));
    }, [&](int64_t j) {
        Elem<DT>::store(dxr + j, slope(Elem<DT>::load(xr + j), Elem<DT>::load(dyr + j), Elem<WDT>::load(weight + j)));
    });
}

// Rows shorter than a vector: a thread a row.  100 000 x 7 bf16 layer norm: forward 6.4 us, a workgroup a row 91.
template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kBlock) void norm_fwd_narrow_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                                 int64_t n_rows, int hidden,
                                                                 const typename Elem<WDT>::T* __restrict__ weight,
                                                                 const typename Elem<WDT>::T* __restrict__ bias, float eps,
                                                                 typename Elem<DT>::T* __restrict__ y, float* __restrict__ mean,
                                                                 float* __restrict__ rstd) {
    const int64_t row = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (row >= n_rows) return;
    const typename Elem<DT>::T* xr = x + row * x_stride;
    float mu = 0.f, ss = 0.f;
    if (kLayer) {
        for (int j = 0; j < hidden; ++j) mu += Elem<DT>::load(xr + j);
        mu /= (float)hidden;
    }
    for (int j = 0; j < hidden; ++j) ss += (Elem<DT>::load(xr + j) - mu) * (Elem<DT>::load(xr + j) - mu);
    const float r = 1.f / sqrtf(ss / (float)hidden + eps);
    for (int j = 0; j < hidden; ++j) {
        const float b = kLayer && bias ? Elem<WDT>::load(bias + j) : 0.f;
        Elem<DT>::store(y + row * hidden + j, (Elem<DT>::load(xr + j) - mu) * r * Elem<WDT>::load(weight + j) + b);
    }
    if (mean) mean[row] = mu;
    if (rstd) rstd[row] = r;
}

template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kBlock) void norm_dx_narrow_kernel(const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
                                                                const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                                int64_t n_rows, int hidden,
                                                                const typename Elem<WDT>::T* __restrict__ weight,
                                                                const float* __restrict__ mean, const float* __restrict__ rstd,
                                                                typename Elem<DT>::T* __restrict__ dx) {
    const int64_t row = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (row >= n_rows) return;
    const typename Elem<DT>::T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
    const float mu = kLayer ? mean[row] : 0.f, r = rstd[row];
    float c = 0.f, cn = 0.f;
    for (int j = 0; j < hidden; ++j) {
        const float g = Elem<DT>::load(dyr + j) * Elem<WDT>::load(weight + j);
        c += kLayer ? g : 0.f;
        cn += g * ((Elem<DT>::load(xr + j) - mu) * r);
    }
    c /= (float)hidden;
    cn /= (float)hidden;
    for (int j = 0; j < hidden; ++j) {
        const float g = Elem<DT>::load(dyr + j) * Elem<WDT>::load(weight + j);
        Elem<DT>::store(dx + row * hidden + j, r * (g - c - (Elem<DT>::load(xr + j) - mu) * r * cn));
    }
}

// Partial sums of the columns, of such rows or where nothing else is asked for: kCols columns a thread (a vector, the last of
// which ends with the row, or one), a slab of rows per workgroup in y.  4 096 x 28 672 bf16: 123 us with the sum of the slabs (3.8 TB/s).
template <int DT, bool kLayer, int kCols>
__global__ __launch_bounds__(kBlock) void norm_columns_kernel(const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
                                                              const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                              int64_t n_rows, int64_t hidden, int64_t slab_rows,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              float* __restrict__ part) {
    const int64_t want = ((int64_t)blockIdx.x * kBlock + threadIdx.x) * kCols;
    if (want >= hidden) return;
    const int64_t j = want < hidden - kCols ? want : hidden - kCols;
    const int64_t lo = (int64_t)blockIdx.y * slab_rows, hi = lo + slab_rows < n_rows ? lo + slab_rows : n_rows;
    float dw[kCols] = {}, db[kCols] = {};
#pragma unroll 4
    for (int64_t row = lo; row < hi; ++row) {
        float z[kCols], g[kCols];
        if constexpr (kCols == 1) {
            z[0] = Elem<DT>::load(x + row * x_stride + j);
            g[0] = Elem<DT>::load(dy + row * dy_stride + j);
        } else {
            load_row<DT>(x + row * x_stride + j, z);
            load_row<DT>(dy + row * dy_stride + j, g);
        }
        const float mu = kLayer ? mean[row] : 0.f, r = rstd[row];
#pragma unroll
        for (int i = 0; i < kCols; ++i) {
            dw[i] += g[i] * ((z[i] - mu) * r);
            db[i] += g[i];
        }
    }
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
        part[((int64_t)blockIdx.y * 2) * hidden + j + i] = dw[i];
        part[((int64_t)blockIdx.y * 2 + 1) * hidden + j + i] = db[i];
    }
}

// ------------------------------------------------------------------------------------ rows in registers
// A team of 16 lanes (rows of up to 64 vectors: 65 536 x 256 bf16 13 us, by a wavefront each 24; of 56 vectors 27 and 27) or of
// whole wavefronts holds a row, kVecs vectors of 16 bytes a lane, so that every row is read
// once.  The last vector of a row that is not whole vectors ends where the row ends and overlaps the one in front of it; lanes
// behind it hold it again.  Entries that a lane holds twice over are left out of its sums (`skip` of them, from the front)
// and written twice with the same bits, so that no access hides behind a branch: around a branch the compiler cannot count
// what is on its way, and every wait would be one for all of it.
struct Team {
    int lanes, vecs;                        // 0 lanes: the row is not held
};

// Rows of whole lines that wavefronts hold go past the caches (kStream): nobody reads a line's other half later.  Through them,
// 32 768 x 3 584 bf16: forward 84 us for 78, backward 138 for 122; 16 384 x 4 096 fp32 154 for 134.  Rows that share lines
// with their neighbours, and the small ones of 16 lanes, go through.

// Of a lane's vectors the last alone may lie behind the row.
__host__ Team team_that_fits(int64_t nv, int64_t lanes, int vecs) {
    return nv > (vecs - 1) * lanes && nv <= vecs * lanes ? Team{(int)lanes, vecs} : Team{0, 0};
}

constexpr int kMaxVecs = 4;

int64_t vectors_of(int dtype, int64_t hidden) {
    const int64_t vec = dtype == MRL_F32 ? 4 : 8;
    return hidden < vec ? 0 : (hidden + vec - 1) / vec;
}

Team team_of(int dtype, int64_t hidden) {
    const int64_t nv = vectors_of(dtype, hidden);
    if (nv == 0) return {0, 0};
    if (nv <= 64) return team_that_fits(nv, 16, (int)((nv + 15) / 16));
    for (int lanes = 64; lanes <= 1024; lanes *= 2)
        if (nv <= (int64_t)lanes * kMaxVecs) return team_that_fits(nv, lanes, (int)((nv + lanes - 1) / lanes));
    return {0, 0};
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

template <int DT, int WDT, bool kLayer, int kVecs, bool kStream>
__global__ __launch_bounds__(1024) void norm_fwd_rows_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                             int64_t n_rows, int hidden, int lanes,
                                                             const typename Elem<WDT>::T* __restrict__ weight,
                                                             const typename Elem<WDT>::T* __restrict__ bias, float eps,
                                                             typename Elem<DT>::T* __restrict__ y, float* __restrict__ mean,
                                                             float* __restrict__ rstd) {
    constexpr int kVec = Elem<DT>::kVec;
    __shared__ float2 lds[2][16];
    const int tl = threadIdx.x & (lanes - 1);
    const int64_t wanted = (int64_t)blockIdx.x * (blockDim.x / lanes) + threadIdx.x / lanes;
    const bool live = wanted < n_rows;
    const int64_t row = live ? wanted : n_rows - 1;
    const typename Elem<DT>::T* xr = x + row * x_stride;
    typename Elem<DT>::T* yr = y + row * hidden;
    const Columns<kVecs, kVec> col(tl, lanes, hidden);
    u32x4 v[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) v[q] = kStream ? mrl::Vec<DT>::load_nt(xr + col.at(q)) : mrl::Vec<DT>::load(xr + col.at(q));
    const float inv = 1.f / (float)hidden;
    float mu = 0.f;
    if (kLayer) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec];
            Elem<DT>::unpack(v[q], z);
#pragma unroll
            for (int i = 0; i < kVec; ++i) s += col.own(q, i) ? z[i] : 0.f;
        }
        mu = team_sum2(s, 0.f, lanes, lds[0]).x * inv;
    }
    float ss = 0.f;
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        float z[kVec];
        Elem<DT>::unpack(v[q], z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const float d = z[i] - mu;
            ss += col.own(q, i) ? d * d : 0.f;
        }
    }
    const float r = 1.f / sqrtf(team_sum2(ss, 0.f, lanes, lds[1]).x * inv + eps);
    if (!live) return;
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        float z[kVec], w[kVec];
        Elem<DT>::unpack(v[q], z);
        mrl::load_floats<WDT>(weight + col.at(q), w);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = (z[i] - mu) * r * w[i];
        if (kLayer && bias) {
            mrl::load_floats<WDT>(bias + col.at(q), w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) z[i] += w[i];
        }
        if (kStream) mrl::Vec<DT>::store_nt(yr + col.at(q), Elem<DT>::pack(z));
        else mrl::Vec<DT>::store(yr + col.at(q), Elem<DT>::pack(z));
    }
    if (tl == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = r;
    }
}

// The backward in one pass: workgroups stay and take rows in turn, a team a row, and hold the sums over their rows of the
// lane's columns in registers; the workgroup's sums go to part[group][2][hidden] (dw, db).  The next row's entries are on
// their way while this one's are summed.  The weight stays in registers: a load of it behind the request for the next
// row would wait for that as well.
constexpr int kBwdBlock = 512;              // threads of a workgroup that holds several teams
constexpr int kBwdGroups = 512;             // most workgroups: two on each of 256 CUs
constexpr int64_t kBwdManyVecs = 4 << 20;   // 64 MiB of rows

template <int DT, int WDT, bool kLayer, int kVecs, int kBlockMost, bool kStream>
__global__ __launch_bounds__(kBlockMost) void norm_bwd_rows_kernel(
    const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride, const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
    int64_t n_rows, int hidden, int lanes, const typename Elem<WDT>::T* __restrict__ weight, const float* __restrict__ mean,
    const float* __restrict__ rstd, typename Elem<DT>::T* __restrict__ dx, float* __restrict__ part,
    typename Elem<WDT>::T* __restrict__ dweight, typename Elem<WDT>::T* __restrict__ dbias) {
    constexpr int kVec = Elem<DT>::kVec, kWVec = Elem<WDT>::kVec;
    constexpr bool kOne = kBlockMost > kBwdBlock;       // the team is the workgroup
    constexpr bool kAhead = kVecs == 1;                 // the next row is requested before this one is summed
    extern __shared__ float columns[];                  // [kVecs * kVec][lanes] sums on their way between teams
    __shared__ float2 lds[2][16];
    const int teams = kOne ? 1 : blockDim.x / lanes, team = kOne ? 0 : threadIdx.x / lanes;
    const int tl = threadIdx.x - team * lanes;
    const Columns<kVecs, kVec> col(tl, lanes, hidden);
    const float inv = 1.f / (float)hidden;
    float dw[kVecs][kVec] = {}, db[kVecs][kVec] = {};
    u32x4 wv[kVecs][kVec / kWVec];
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
#pragma unroll
        for (int p = 0; p < kVec / kWVec; ++p) wv[q][p] = mrl::Vec<WDT>::load(weight + col.at(q) + p * kWVec);
    const auto unpack_weight = [&](int q, float (&w)[kVec]) {
#pragma unroll
        for (int p = 0; p < kVec / kWVec; ++p) {
            float t[kWVec];
            Elem<WDT>::unpack(wv[q][p], t);
#pragma unroll
            for (int i = 0; i < kWVec; ++i) w[p * kWVec + i] = t[i];
        }
    };
    const int64_t step = (int64_t)gridDim.x * teams;
    u32x4 xn[kVecs], gn[kVecs];
    float mun, rn;
    const auto request = [&](int64_t wanted) {
        const int64_t row = wanted < n_rows ? wanted : n_rows - 1;
        const typename Elem<DT>::T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
        mun = kLayer ? mean[row] : 0.f;
        rn = rstd[row];
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            xn[q] = kStream ? mrl::Vec<DT>::load_nt(xr + col.at(q)) : mrl::Vec<DT>::load(xr + col.at(q));
            gn[q] = kStream ? mrl::Vec<DT>::load_nt(dyr + col.at(q)) : mrl::Vec<DT>::load(dyr + col.at(q));
        }
    };
    if (kAhead) request((int64_t)blockIdx.x * teams + team);
    int turn = 0;
    for (int64_t base = (int64_t)blockIdx.x * teams; base < n_rows; base += step, turn ^= 1) {
        // teams behind the last row do that row again, without its share of the columns' sums
        const bool counts = kOne || base + team < n_rows;
        const int64_t row = counts ? base + team : n_rows - 1;
        if (!kAhead) request(row);
        u32x4 xv[kVecs], gv[kVecs];
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            xv[q] = xn[q];
            gv[q] = gn[q];
        }
        const float mu = mun, r = rn;
        if (kAhead) request(base + team + step);
        float sg = 0.f, sgn = 0.f;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec], g[kVec], w[kVec];
            Elem<DT>::unpack(xv[q], z);
            Elem<DT>::unpack(gv[q], g);
            unpack_weight(q, w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                const float own = col.own(q, i) ? g[i] : 0.f, n = (z[i] - mu) * r;
                const float add = counts ? own : 0.f;
                dw[q][i] += add * n;
                if (kLayer) db[q][i] += add;
                sg += own * w[i];
                sgn += own * w[i] * n;
            }
        }
        const float2 sums = team_sum2(sg, sgn, lanes, lds[turn]);
        const float c = kLayer ? sums.x * inv : 0.f, cn = sums.y * inv;
        typename Elem<DT>::T* dxr = dx + row * hidden;
#pragma unroll
        for (int q = 0; q < kVecs; ++q) {
            float z[kVec], g[kVec], w[kVec];
            Elem<DT>::unpack(xv[q], z);
            Elem<DT>::unpack(gv[q], g);
            unpack_weight(q, w);
#pragma unroll
            for (int i = 0; i < kVec; ++i) z[i] = r * (g[i] * w[i] - c - (z[i] - mu) * r * cn);
            if (kStream) mrl::Vec<DT>::store_nt(dxr + col.at(q), Elem<DT>::pack(z));
            else mrl::Vec<DT>::store(dxr + col.at(q), Elem<DT>::pack(z));
        }
    }
    if (!part && !dweight && !dbias) return;
    // the workgroup's sums: teams of a wavefront by lane exchange, then one after the other through LDS
    const bool paired = !kOne && lanes < 64;
    const int turns = paired ? blockDim.x >> 6 : teams, mine = paired ? threadIdx.x >> 6 : team;
    const bool holds = !paired || (threadIdx.x & 63) < 16;
#pragma unroll
    for (int b = 0; b < (kLayer ? 2 : 1); ++b) {
        if (paired) {
#pragma unroll
            for (int q = 0; q < kVecs; ++q)
#pragma unroll
                for (int i = 0; i < kVec; ++i) {
                    float& s = b ? db[q][i] : dw[q][i];
                    s += __shfl_xor(s, 16, 64);
                    s += __shfl_xor(s, 32, 64);
                }
        }
        float* out = part ? part + ((int64_t)blockIdx.x * 2 + b) * hidden : nullptr;
        typename Elem<WDT>::T* vec = b ? dbias : dweight;       // the sums themselves, of the only workgroup
        for (int t = 0; t < turns; ++t) {
            if (t == mine && holds) {
#pragma unroll
                for (int q = 0; q < kVecs; ++q) {
                    float s[kVec];
#pragma unroll
                    for (int i = 0; i < kVec; ++i) {
                        float* at = columns + (q * kVec + i) * lanes + tl;      // a lane's place is the same for every team
                        s[i] = (b ? db[q][i] : dw[q][i]) + (!kOne && t > 0 ? *at : 0.f);
                        if (t < turns - 1) *at = s[i];
                    }
                    if (t < turns - 1) continue;
                    if (!out) {
#pragma unroll
                        for (int i = 0; i < kVec; ++i)
                            if (vec && col.own(q, i)) Elem<WDT>::store(vec + col.at(q) + i, s[i]);
                    } else if (q < kVecs - 1 || col.skip == 0) {
#pragma unroll
                        for (int p = 0; p < kVec; p += 4)
                            mrl::Vec<MRL_F32>::store(out + col.at(q) + p, mrl::make_u32x4(__float_as_uint(s[p]),
                                                     __float_as_uint(s[p + 1]), __float_as_uint(s[p + 2]), __float_as_uint(s[p + 3])));
                    } else {
#pragma unroll
                        for (int i = 0; i < kVec; ++i)
                            if (i >= col.skip) out[col.last + i] = s[i];
                    }
                }
            }
            if (!kOne) __syncthreads();
        }
    }
}

// Sums of the groups' sums (of 455 groups of 3 584 columns: 5 us): 32 columns a workgroup, 32 lanes a column that each take every 32nd group.
template <int WDT>
__global__ __launch_bounds__(1024) void norm_part_sum_kernel(const float* __restrict__ part, int n_parts, int64_t hidden,
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
            v[i] = p[(int64_t)(k < n_parts ? k : slice) * 2 * hidden];
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

int64_t slab_rows_of(int64_t n_rows) {
    const int64_t rows = (n_rows + kColumnSlabs - 1) / kColumnSlabs;
    return rows < 16 ? 16 : rows;
}

// The backward's teams hold twice the entries, and the sums of the columns besides: one or two vectors a lane.  Two, where the
// next row is not requested ahead, are better served by the memory (us, one / two: 32 768 x 3 584 bf16 139 / 122, 65 536 x
// 5 120 381 / 348, 65 536 x 2 048 147 / 136); of little data, where what follows the rows counts, one (9 477 x 1 343 fp16
// 26 / 29, 2 500 x 1 024 fp32 14.7 / 15.7).  Rows of more than 2 048 vectors take four of fp32 (8 192 x 16 000 281 us, by the
// kernels for any width 648); of 16 bits, eight entries each, four do not fit the registers (4 096 x 28 672 521 us, by
// those kernels 298).
Team bwd_team_of(int dtype, int64_t n_rows, int64_t hidden) {
    const int64_t nv = vectors_of(dtype, hidden);
    if (nv == 0) return {0, 0};
    if (nv <= 32) return team_that_fits(nv, 16, (int)((nv + 15) / 16));
    const bool two = nv > 256 || (nv > 128 && n_rows * nv >= kBwdManyVecs);
    for (int vecs = two ? 2 : 1; vecs <= (dtype == MRL_F32 ? 4 : 2); vecs *= 2) {
        const int64_t waves = (nv + 64 * vecs - 1) / (64 * vecs);
        if (waves <= 16) return team_that_fits(nv, waves * 64, vecs);
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

struct FwdArgs {
    const void *x, *weight, *bias;
    void* y;
    float *mean, *rstd;
    int64_t n_rows, hidden, x_stride;
    float eps;
    hipStream_t stream;
};

template <int DT, int WDT, bool kLayer>
void launch_fwd(const FwdArgs& a) {
    using T = typename Elem<DT>::T;
    using W = typename Elem<WDT>::T;
    const Team team = team_of(DT, a.hidden);
    if (team.lanes > 0) {
        const int block = team.lanes > 256 ? team.lanes : 256, teams = block / team.lanes;
        const dim3 grid((unsigned)((a.n_rows + teams - 1) / teams));
        const auto launch = [&](auto vecs, auto stream) {
            hipLaunchKernelGGL((norm_fwd_rows_kernel<DT, WDT, kLayer, decltype(vecs)::value, decltype(stream)::value != 0>), grid,
                               dim3(block), 0, a.stream, (const T*)a.x, a.x_stride, a.n_rows, (int)a.hidden, team.lanes,
                               (const W*)a.weight, (const W*)a.bias, a.eps, (T*)a.y, a.mean, a.rstd);
        };
        if (team.lanes >= 64 && a.hidden * (int64_t)sizeof(T) % 128 == 0) with_vecs(team.vecs, [&](auto v) { launch(v, Int<1>()); });
        else with_vecs(team.vecs, [&](auto v) { launch(v, Int<0>()); });
        return;
    }
    if (a.hidden < Elem<DT>::kVec) {
        hipLaunchKernelGGL((norm_fwd_narrow_kernel<DT, WDT, kLayer>), dim3((unsigned)((a.n_rows + kBlock - 1) / kBlock)), dim3(kBlock),
                           0, a.stream, (const T*)a.x, a.x_stride, a.n_rows, (int)a.hidden, (const W*)a.weight, (const W*)a.bias,
                           a.eps, (T*)a.y, a.mean, a.rstd);
        return;
    }
    hipLaunchKernelGGL((norm_fwd_kernel<DT, WDT, kLayer>), dim3((unsigned)a.n_rows), dim3(kWideBlock), 0, a.stream, (const T*)a.x,
                       a.x_stride, a.hidden, (const W*)a.weight, (const W*)a.bias, a.eps, (T*)a.y, a.mean, a.rstd);
}

struct BwdArgs {
    const void *dy, *x, *weight;
    const float *mean, *rstd;
    void *dx, *dweight, *dbias;
    float* part;
    int64_t n_rows, hidden, dy_stride, x_stride;
    hipStream_t stream;
};

template <int DT, int WDT, bool kLayer>
void launch_bwd(const BwdArgs& a) {
    using T = typename Elem<DT>::T;
    using W = typename Elem<WDT>::T;
    const Team team = bwd_team_of(DT, a.n_rows, a.hidden);
    const auto sum_parts = [&](int n_parts, void* dweight, void* dbias) {
        hipLaunchKernelGGL((norm_part_sum_kernel<WDT>), dim3((unsigned)((a.hidden + 31) / 32), dbias ? 2 : 1), dim3(1024), 0,
                           a.stream, a.part, n_parts, a.hidden, (W*)dweight, (W*)dbias);
    };
    const bool narrow = a.hidden < Elem<DT>::kVec;
    const auto sum_columns = [&](void* dweight, void* dbias) {
        const int64_t slab = slab_rows_of(a.n_rows);
        const int n_slabs = (int)((a.n_rows + slab - 1) / slab);
        const auto columns_kernel = [&](auto cols) {
            constexpr int kCols = decltype(cols)::value;
            const int64_t threads = (a.hidden + kCols - 1) / kCols;
            hipLaunchKernelGGL((norm_columns_kernel<DT, kLayer, kCols>), dim3((unsigned)((threads + kBlock - 1) / kBlock), (unsigned)n_slabs),
                               dim3(kBlock), 0, a.stream, (const T*)a.dy, a.dy_stride, (const T*)a.x, a.x_stride, a.n_rows, a.hidden, slab,
                               a.mean, a.rstd, a.part);
        };
        if (n_slabs > 0 && narrow) columns_kernel(Int<1>());
        else if (n_slabs > 0) columns_kernel(Int<Elem<DT>::kVec>());
        sum_parts(n_slabs, dweight, dbias);
    };
    if (team.lanes > 0 && a.n_rows > 0 && a.dx) {
        // the one pass sums dy for layer norm alone: an RMS norm has no bias, so registers and adds for one would serve
        // nobody but a caller who adds a bias behind it, and that one's dbias comes from a pass over the columns
        void* const dbias = kLayer ? a.dbias : nullptr;
        const bool sums = a.dweight || dbias;
        const int groups = bwd_groups(team, a.n_rows);
        const auto launch = [&](auto vecs, auto most, auto stream) {
            const int block = bwd_block(team);
            const size_t lds = sums && block > team.lanes ? (size_t)team.lanes * team.vecs * Elem<DT>::kVec * 4 : 0;
            hipLaunchKernelGGL((norm_bwd_rows_kernel<DT, WDT, kLayer, decltype(vecs)::value, decltype(most)::value,
                                                     decltype(stream)::value != 0>),
                               dim3((unsigned)groups), dim3(block), lds, a.stream,
                               (const T*)a.dy, a.dy_stride, (const T*)a.x, a.x_stride, a.n_rows, (int)a.hidden, team.lanes,
                               (const W*)a.weight, a.mean, a.rstd, (T*)a.dx, sums && groups > 1 ? a.part : nullptr,
                               groups > 1 ? (W*)nullptr : (W*)a.dweight, groups > 1 ? (W*)nullptr : (W*)dbias);
        };
        const auto launch_block = [&](auto stream) {
            if constexpr (DT == MRL_F32) {
                if (team.vecs == 4) return launch(Int<4>(), Int<1024>(), stream);
            }
            if (team.vecs == 2 && team.lanes > kBwdBlock) launch(Int<2>(), Int<1024>(), stream);
            else if (team.vecs == 2) launch(Int<2>(), Int<kBwdBlock>(), stream);
            else if (team.lanes > kBwdBlock) launch(Int<1>(), Int<1024>(), stream);
            else launch(Int<1>(), Int<kBwdBlock>(), stream);
        };
        if (team.lanes >= 64 && a.hidden * (int64_t)sizeof(T) % 128 == 0) launch_block(Int<1>());
        else launch_block(Int<0>());
        if (sums && groups > 1) sum_parts(groups, a.dweight, dbias);
        if (a.dbias && !dbias) sum_columns(nullptr, a.dbias);
        return;
    }
    if (a.dx && a.n_rows > 0 && narrow)
        hipLaunchKernelGGL((norm_dx_narrow_kernel<DT, WDT, kLayer>), dim3((unsigned)((a.n_rows + kBlock - 1) / kBlock)), dim3(kBlock), 0,
                           a.stream, (const T*)a.dy, a.dy_stride, (const T*)a.x, a.x_stride, a.n_rows, (int)a.hidden,
                           (const W*)a.weight, a.mean, a.rstd, (T*)a.dx);
    else if (a.dx && a.n_rows > 0)
        hipLaunchKernelGGL((norm_dx_kernel<DT, WDT, kLayer>), dim3((unsigned)a.n_rows), dim3(kWideBlock), 0, a.stream, (const T*)a.dy,
                           a.dy_stride, (const T*)a.x, a.x_stride, a.hidden, (const W*)a.weight, a.mean, a.rstd, (T*)a.dx);
    if (a.dweight || a.dbias) sum_columns(a.dweight, a.dbias);
}

// The instance of a launch for the types of rows and vectors: vectors have the rows' type or fp32.
template <bool kLayer>
void dispatch(int dtype, int wdtype, const FwdArgs& a) {
    if (dtype == MRL_F32) launch_fwd<MRL_F32, MRL_F32, kLayer>(a);
    else if (dtype == MRL_BF16 && wdtype == MRL_F32) launch_fwd<MRL_BF16, MRL_F32, kLayer>(a);
    else if (dtype == MRL_BF16) launch_fwd<MRL_BF16, MRL_BF16, kLayer>(a);
    else if (wdtype == MRL_F32) launch_fwd<MRL_F16, MRL_F32, kLayer>(a);
    else launch_fwd<MRL_F16, MRL_F16, kLayer>(a);
}

template <bool kLayer>
void dispatch(int dtype, int wdtype, const BwdArgs& a) {
    if (dtype == MRL_F32) launch_bwd<MRL_F32, MRL_F32, kLayer>(a);
    else if (dtype == MRL_BF16 && wdtype == MRL_F32) launch_bwd<MRL_BF16, MRL_F32, kLayer>(a);
    else if (dtype == MRL_BF16) launch_bwd<MRL_BF16, MRL_BF16, kLayer>(a);
    else if (wdtype == MRL_F32) launch_bwd<MRL_F16, MRL_F32, kLayer>(a);
    else launch_bwd<MRL_F16, MRL_F16, kLayer>(a);
}

// Whether the launch that gives every row a team can hold them (the backward's stays within it).
bool fwd_fits(int dtype, int64_t n_rows, int64_t hidden) {
    const Team team = team_of(dtype, hidden);
    const int64_t lanes = team.lanes > 0 ? team.lanes : vectors_of(dtype, hidden) == 0 ? 1 : kWideBlock;
    const int64_t teams = lanes < 256 ? 256 / lanes : 1;
    return n_rows <= 0x7fffffffLL && mrl::launch_fits((n_rows + teams - 1) / teams, lanes < 256 ? 256 : lanes);
}

int check_sizes(const char* fn, int dtype, int wdtype, int64_t n_rows, int64_t hidden) {
    MRL_REQUIRE(mrl::float_dtype_bytes(dtype) != 0, MRL_ERR_UNSUPPORTED, "%s: dtype %d (want F32, BF16 or F16)", fn, dtype);
    MRL_REQUIRE(wdtype == dtype || wdtype == MRL_F32, MRL_ERR_UNSUPPORTED, "%s: weight dtype %d (want the rows' or F32)", fn,
                wdtype);
    MRL_REQUIRE(n_rows >= 0 && hidden >= 1, MRL_ERR_INVALID_ARG, "%s: n_rows=%lld hidden=%lld", fn, (long long)n_rows,
                (long long)hidden);
    MRL_REQUIRE(hidden <= MRL_NORM_MAX_HIDDEN && fwd_fits(dtype, n_rows, hidden), MRL_ERR_UNSUPPORTED,
                "%s: n_rows=%lld hidden=%lld (hidden at most %d, and fewer rows: 2^32 threads hold at most one each)", fn,
                (long long)n_rows, (long long)hidden, MRL_NORM_MAX_HIDDEN);
    return MRL_OK;
}

}  // namespace

extern "C" int mrl_norm_fwd(const void* x, int dtype, int64_t n_rows, int64_t hidden, int64_t row_stride, const void* weight,
                            const void* bias, int weight_dtype, int subtract_mean, float eps, void* y, float* mean, float* rstd,
                            void* stream) {
    const char* fn = "mrl_norm_fwd";
    const int rc = check_sizes(fn, dtype, weight_dtype, n_rows, hidden);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE(row_stride >= hidden || n_rows <= 1, MRL_ERR_INVALID_ARG, "%s: row_stride=%lld below hidden=%lld", fn,
                (long long)row_stride, (long long)hidden);
    MRL_REQUIRE(eps > 0.f && eps <= 3.0e38f, MRL_ERR_INVALID_ARG, "%s: eps=%g (want a positive, finite number)", fn, (double)eps);
    MRL_REQUIRE(subtract_mean || bias == nullptr, MRL_ERR_INVALID_ARG, "%s: a bias without subtract_mean", fn);
    if (n_rows == 0) return MRL_OK;
    MRL_REQUIRE(x && weight && y, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const size_t es = mrl::float_dtype_bytes(dtype), ws = mrl::float_dtype_bytes(weight_dtype);
    MRL_REQUIRE(mrl::aligned(x, es) && mrl::aligned(y, es) && mrl::aligned(weight, ws) && mrl::aligned(bias, ws) &&
                    mrl::aligned(mean, 4) && mrl::aligned(rstd, 4),
                MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    const FwdArgs a = {x, weight, bias, y, mean, rstd, n_rows, hidden, row_stride, eps, mrl::as_stream(stream)};
    if (subtract_mean) dispatch<true>(dtype, weight_dtype, a);
    else dispatch<false>(dtype, weight_dtype, a);
    return mrl::check_launch(fn);
}

extern "C" int64_t mrl_norm_bwd_workspace_bytes(int64_t n_rows, int64_t hidden) {
    if (n_rows <= 0 || hidden <= 0 || n_rows > 0x7fffffffLL || hidden > MRL_NORM_MAX_HIDDEN) return 0;
    // two sums of a column for each workgroup of the one pass or each slab of rows: neither are more than the rows
    static_assert(kColumnSlabs <= kBwdGroups, "a place for every slab");
    return (n_rows < kBwdGroups ? n_rows : kBwdGroups) * 2 * hidden * 4;
}

extern "C" int mrl_norm_bwd(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, int dtype, int64_t n_rows,
                            int64_t hidden, const void* weight, int weight_dtype, const float* mean, const float* rstd, void* dx,
                            void* dweight, void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "mrl_norm_bwd";
    const int rc = check_sizes(fn, dtype, weight_dtype, n_rows, hidden);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE((dy_stride >= hidden && x_stride >= hidden) || n_rows <= 1, MRL_ERR_INVALID_ARG,
                "%s: strides %lld and %lld below hidden=%lld", fn, (long long)dy_stride, (long long)x_stride, (long long)hidden);
    MRL_REQUIRE(n_rows == 0 || (dy && x && weight && rstd), MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const int64_t need = dweight || dbias ? mrl_norm_bwd_workspace_bytes(n_rows, hidden) : 0;
    MRL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MRL_ERR_INVALID_ARG, "%s: workspace of %lld bytes (want %lld)",
                fn, (long long)workspace_bytes, (long long)need);
    const size_t es = mrl::float_dtype_bytes(dtype), ws = mrl::float_dtype_bytes(weight_dtype);
    MRL_REQUIRE(mrl::aligned(dy, es) && mrl::aligned(x, es) && mrl::aligned(dx, es) && mrl::aligned(weight, ws) &&
                    mrl::aligned(dweight, ws) && mrl::aligned(dbias, ws) && mrl::aligned(mean, 4) && mrl::aligned(rstd, 4) &&
                    mrl::aligned(workspace, 16),
                MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    if (n_rows == 0 && !dweight && !dbias) return MRL_OK;
    const BwdArgs a = {dy, x, weight, mean, rstd, dx, dweight, dbias, (float*)workspace, n_rows, hidden, dy_stride, x_stride,
                       mrl::as_stream(stream)};
    if (mean) dispatch<true>(dtype, weight_dtype, a);
    else dispatch<false>(dtype, weight_dtype, a);
    return mrl::check_launch(fn);
}
