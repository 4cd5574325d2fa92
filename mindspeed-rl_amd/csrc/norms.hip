// Layer norm and RMS norm of hidden states for gfx950, forward and backward.
//
//   layer:  mu = mean_j x_j,  r = (mean_j (x_j - mu)^2 + eps)^(-1/2),  n_j = (x_j - mu) r,  y_j = n_j w_j + b_j
//   RMS:    the same without mu and b
//   dx_j = r (g_j - c - n_j mean_i(g_i n_i)),  g_j = dy_j w_j,  c = mean_i g_i (RMS: 0)
//   dw_j = sum_rows dy_j n_j,  db_j = sum_rows dy_j
//
// Everything is held in fp32 and rounded once, to the output's type.  Both passes are bound by memory.
#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
constexpr int kColumnSlabs = 256;           // most partial sums of a column

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
    for (int w = 1; w < kWaves; ++w) {
        s.x += lds[w].x;
        s.y += lds[w].y;
    }
    return s;
}

template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kBlock) void norm_fwd_kernel(const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                          int64_t hidden, const typename Elem<WDT>::T* __restrict__ weight,
                                                          const typename Elem<WDT>::T* __restrict__ bias, float eps,
                                                          typename Elem<DT>::T* __restrict__ y, float* __restrict__ mean,
                                                          float* __restrict__ rstd) {
    __shared__ float2 lds[kWaves];
    const int64_t row = blockIdx.x;
    const typename Elem<DT>::T* xr = x + row * x_stride;
    float mu = 0.f;
    if (kLayer) {
        float s = 0.f;
        for (int64_t j = threadIdx.x; j < hidden; j += kBlock) s += Elem<DT>::load(xr + j);
        mu = block_sum2(s, 0.f, lds).x / (float)hidden;
    }
    float ss = 0.f;
    for (int64_t j = threadIdx.x; j < hidden; j += kBlock) {
        const float d = Elem<DT>::load(xr + j) - mu;
        ss += d * d;
    }
    const float r = 1.f / sqrtf(block_sum2(ss, 0.f, lds).x / (float)hidden + eps);
    for (int64_t j = threadIdx.x; j < hidden; j += kBlock) {
        float v = (Elem<DT>::load(xr + j) - mu) * r * Elem<WDT>::load(weight + j);
        if (kLayer && bias) v += Elem<WDT>::load(bias + j);
        Elem<DT>::store(y + row * hidden + j, v);
    }
    if (threadIdx.x == 0) {
        if (mean) mean[row] = mu;
        if (rstd) rstd[row] = r;
    }
}

template <int DT, int WDT, bool kLayer>
__global__ __launch_bounds__(kBlock) void norm_dx_kernel(const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
                                                         const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                         int64_t hidden, const typename Elem<WDT>::T* __restrict__ weight,
                                                         const float* __restrict__ mean, const float* __restrict__ rstd,
                                                         typename Elem<DT>::T* __restrict__ dx) {
    __shared__ float2 lds[kWaves];
    const int64_t row = blockIdx.x;
    const float mu = kLayer ? mean[row] : 0.f, r = rstd[row];
    const typename Elem<DT>::T *xr = x + row * x_stride, *dyr = dy + row * dy_stride;
    float sg = 0.f, sgn = 0.f;
    for (int64_t j = threadIdx.x; j < hidden; j += kBlock) {
        const float g = Elem<DT>::load(dyr + j) * Elem<WDT>::load(weight + j);
        sg += g;
        sgn += g * ((Elem<DT>::load(xr + j) - mu) * r);
    }
    const float2 s = block_sum2(sg, sgn, lds);
    const float c = kLayer ? s.x / (float)hidden : 0.f, cn = s.y / (float)hidden;
    for (int64_t j = threadIdx.x; j < hidden; j += kBlock) {
        const float g = Elem<DT>::load(dyr + j) * Elem<WDT>::load(weight + j);
        Elem<DT>::store(dx + row * hidden + j, r * (g - c - (Elem<DT>::load(xr + j) - mu) * r * cn));
    }
}

// Partial sums of the columns: a thread per column, a slab of rows per workgroup in y.
template <int DT, bool kLayer>
__global__ __launch_bounds__(kBlock) void norm_columns_kernel(const typename Elem<DT>::T* __restrict__ dy, int64_t dy_stride,
                                                              const typename Elem<DT>::T* __restrict__ x, int64_t x_stride,
                                                              int64_t n_rows, int64_t hidden, int64_t slab_rows,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              float* __restrict__ part) {
    const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (j >= hidden) return;
    const int64_t lo = (int64_t)blockIdx.y * slab_rows, hi = lo + slab_rows < n_rows ? lo + slab_rows : n_rows;
    float dw = 0.f, db = 0.f;
    for (int64_t row = lo; row < hi; ++row) {
        const float g = Elem<DT>::load(dy + row * dy_stride + j);
        dw += g * ((Elem<DT>::load(x + row * x_stride + j) - (kLayer ? mean[row] : 0.f)) * rstd[row]);
        db += g;
    }
    part[((int64_t)blockIdx.y * 2) * hidden + j] = dw;
    part[((int64_t)blockIdx.y * 2 + 1) * hidden + j] = db;
}

template <int WDT>
__global__ __launch_bounds__(kBlock) void norm_columns_finish_kernel(const float* __restrict__ part, int n_slabs, int64_t hidden,
                                                                     typename Elem<WDT>::T* __restrict__ dweight,
                                                                     typename Elem<WDT>::T* __restrict__ dbias) {
    const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (j >= hidden) return;
    float dw = 0.f, db = 0.f;
    for (int s = 0; s < n_slabs; ++s) {
        dw += part[((int64_t)s * 2) * hidden + j];
        db += part[((int64_t)s * 2 + 1) * hidden + j];
    }
    if (dweight) Elem<WDT>::store(dweight + j, dw);
    if (dbias) Elem<WDT>::store(dbias + j, db);
}

int64_t slab_rows_of(int64_t n_rows) {
    const int64_t rows = (n_rows + kColumnSlabs - 1) / kColumnSlabs;
    return rows < 16 ? 16 : rows;
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
    hipLaunchKernelGGL((norm_fwd_kernel<DT, WDT, kLayer>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, a.stream, (const T*)a.x,
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
    if (a.dx && a.n_rows > 0)
        hipLaunchKernelGGL((norm_dx_kernel<DT, WDT, kLayer>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, a.stream, (const T*)a.dy,
                           a.dy_stride, (const T*)a.x, a.x_stride, a.hidden, (const W*)a.weight, a.mean, a.rstd, (T*)a.dx);
    if (!a.dweight && !a.dbias) return;
    const unsigned columns = (unsigned)((a.hidden + kBlock - 1) / kBlock);
    const int64_t slab = slab_rows_of(a.n_rows);
    const int n_slabs = (int)((a.n_rows + slab - 1) / slab);
    if (n_slabs > 0)
        hipLaunchKernelGGL((norm_columns_kernel<DT, kLayer>), dim3(columns, (unsigned)n_slabs), dim3(kBlock), 0, a.stream,
                           (const T*)a.dy, a.dy_stride, (const T*)a.x, a.x_stride, a.n_rows, a.hidden, slab, a.mean, a.rstd,
                           a.part);
    hipLaunchKernelGGL((norm_columns_finish_kernel<WDT>), dim3(columns), dim3(kBlock), 0, a.stream, a.part, n_slabs, a.hidden,
                       (W*)a.dweight, (W*)a.dbias);
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

int check_sizes(const char* fn, int dtype, int wdtype, int64_t n_rows, int64_t hidden) {
    MRL_REQUIRE(mrl::float_dtype_bytes(dtype) != 0, MRL_ERR_UNSUPPORTED, "%s: dtype %d (want F32, BF16 or F16)", fn, dtype);
    MRL_REQUIRE(wdtype == dtype || wdtype == MRL_F32, MRL_ERR_UNSUPPORTED, "%s: weight dtype %d (want the rows' or F32)", fn,
                wdtype);
    MRL_REQUIRE(n_rows >= 0 && hidden >= 1, MRL_ERR_INVALID_ARG, "%s: n_rows=%lld hidden=%lld", fn, (long long)n_rows,
                (long long)hidden);
    MRL_REQUIRE(n_rows <= 0x7fffffffLL && hidden <= MRL_NORM_MAX_HIDDEN, MRL_ERR_UNSUPPORTED,
                "%s: n_rows=%lld hidden=%lld (at most 2^31 - 1 and %d)", fn, (long long)n_rows, (long long)hidden,
                MRL_NORM_MAX_HIDDEN);
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
    const int64_t slab = slab_rows_of(n_rows);
    return (n_rows + slab - 1) / slab * 2 * hidden * 4;
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
