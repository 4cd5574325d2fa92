// RMS norm with the residual's addition, and with an output in 8 bits, for gfx950.
//
//   h = x + residual, rounded to the residual's type;  r = (mean_j h_j^2 + eps)^(-1/2),  n_j = h_j r,  y_j = n_j w_j
//   d_j = dh_j + r (g_j - n_j mean_i(g_i n_i)),  g_j = dy_j w_j;  dx = dresidual = d, each rounded to its type;  dw_j = sum_rows dy_j n_j
//   8 bits: s = max(max |y| / 448, 2^-126) over the row or over 128 entries,  q = e4m3(y / s)
//
// What is normalised is h as it is stored: the next layer's residual, this norm and its backward see one value, and the call
// gives what an addition and a norm behind it give.  Sums are held in fp32.
#include "lane_ops.h"
#include "mrl_internal.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

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

// A workgroup a row.
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
        const float s = scale_of(block_most(most, mlds)), inv = 1.f / s;
        if (threadIdx.x == 0) a.scale[row] = s;
        for (int j = threadIdx.x; j < a.hidden; j += kBlock) q[j] = code_of(value(j) * inv);
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
        const float s = scale_of(most), inv = 1.f / s;
        if (lane == 0) a.scale[row * blocks + b] = s;
#pragma unroll
        for (int i = 0; i < 2; ++i) q[b * 128 + i * 64 + lane] = code_of(v[i] * inv);
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

template <int WDT>
__global__ __launch_bounds__(kBlock) void add_norm_part_sum_kernel(const float* __restrict__ part, int n_parts, int64_t hidden,
                                                                   typename Elem<WDT>::T* __restrict__ dweight) {
    const int64_t j = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (j >= hidden) return;
    float s = 0.f;
    for (int g = 0; g < n_parts; ++g) s += part[(int64_t)g * hidden + j];
    Elem<WDT>::store(dweight + j, s);
}

int64_t slab_rows_of(int64_t n_rows) {
    const int64_t rows = (n_rows + kColumnSlabs - 1) / kColumnSlabs;
    return rows < 16 ? 16 : rows;
}

template <int DT, int RT>
void launch_fwd(const FwdArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((add_norm_fwd_kernel<DT, RT>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, stream, a);
}

template <int DT, int RT>
void launch_bwd(const BwdArgs& a, hipStream_t stream) {
    if ((a.dx || a.dresidual) && a.n_rows > 0)
        hipLaunchKernelGGL((add_norm_bwd_kernel<DT, RT>), dim3((unsigned)a.n_rows), dim3(kBlock), 0, stream, a);
    if (!a.dweight) return;
    const int64_t slab = slab_rows_of(a.n_rows);
    const int n_slabs = (int)((a.n_rows + slab - 1) / slab);
    const unsigned groups = (unsigned)((a.hidden + kBlock - 1) / kBlock);
    if (n_slabs > 0) hipLaunchKernelGGL((add_norm_columns_kernel<DT, RT>), dim3(groups, (unsigned)n_slabs), dim3(kBlock), 0, stream, a, slab);
    if (a.wide_weight)
        hipLaunchKernelGGL((add_norm_part_sum_kernel<MRL_F32>), dim3(groups), dim3(kBlock), 0, stream, a.part, n_slabs, a.hidden, (float*)a.dweight);
    else
        hipLaunchKernelGGL((add_norm_part_sum_kernel<DT>), dim3(groups), dim3(kBlock), 0, stream, a.part, n_slabs, a.hidden,
                           (typename Elem<DT>::T*)a.dweight);
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
    const int rc = check_fwd(fn, dtype, residual_dtype, weight_dtype, a, hidden);
    if (rc != MRL_OK || n_rows == 0) return rc;
    MRL_REQUIRE(scale, MRL_ERR_INVALID_ARG, "%s: NULL scale", fn);
    dispatch(dtype, residual_dtype, a, mrl::as_stream(stream));
    return mrl::check_launch(fn);
}

extern "C" int64_t mrl_add_norm_bwd_workspace_bytes(int64_t n_rows, int64_t hidden) {
    if (n_rows <= 0 || hidden <= 0 || n_rows > 0x7fffffffLL || !mrl::launch_fits(n_rows, kBlock) || hidden > MRL_NORM_MAX_HIDDEN) return 0;
    return (n_rows < kColumnSlabs ? n_rows : kColumnSlabs) * hidden * 4;
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
