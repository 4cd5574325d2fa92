// The global norm of a list of gradients and clipping by it, for gfx950.
//
//   norm = sqrt(sum over all entries of all tensors of g^2),  factor = min(1, max_norm / (norm + 1e-6)),  out = g * factor
//
// Squares and their sums are held in 64 bits: no gradient that fp32 or bf16 holds overflows them, and the order of the sum
// does not show in the norm's fp32 bits but for a tie.  The list travels in the kernel's arguments, so a captured graph
// holds it, and nothing is copied to the device.
#include <algorithm>

#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kTable = 112;                 // tensors of a launch: 4 KB of arguments
constexpr int64_t kChunk = 8192;            // entries that a workgroup takes at a time
constexpr int kMaxPartials = MRL_GRAD_NORM_PARTIALS;

struct Part {
    const void* data;
    void* out;
    int64_t n;
    int32_t last_chunk;                     // chunks of this tensor and the ones in front of it
    int16_t dtype, out_dtype;
};

struct Table {
    Part part[kTable];
    int32_t n_parts, n_chunks;
};

__device__ __forceinline__ float load_as(const void* p, int dtype, int64_t i) {
    if (dtype == MRL_F32) return Elem<MRL_F32>::load((const float*)p + i);
    if (dtype == MRL_BF16) return Elem<MRL_BF16>::load((const uint16_t*)p + i);
    return Elem<MRL_F16>::load((const uint16_t*)p + i);
}

__device__ __forceinline__ void store_as(void* p, int dtype, int64_t i, float v) {
    if (dtype == MRL_F32) Elem<MRL_F32>::store((float*)p + i, v);
    else if (dtype == MRL_BF16) Elem<MRL_BF16>::store((uint16_t*)p + i, v);
    else Elem<MRL_F16>::store((uint16_t*)p + i, v);
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = lds[0];
#pragma unroll
    for (int w = 1; w < kBlock / 64; ++w) s += lds[w];
    return s;
}

__global__ __launch_bounds__(kBlock) void grad_squares_kernel(Table t, double* __restrict__ partial) {
    __shared__ double lds[kBlock / 64];
    double acc = 0.0;
    int k = 0;
    for (int c = blockIdx.x; c < t.n_chunks; c += gridDim.x) {
        while (c >= t.part[k].last_chunk) ++k;
        const int first = k == 0 ? 0 : t.part[k - 1].last_chunk;
        const int64_t lo = (int64_t)(c - first) * kChunk;
        const int64_t hi = lo + kChunk < t.part[k].n ? lo + kChunk : t.part[k].n;
        for (int64_t i = lo + threadIdx.x; i < hi; i += kBlock) {
            const double g = (double)load_as(t.part[k].data, t.part[k].dtype, i);
            acc += g * g;
        }
    }
    const double s = block_sum(acc, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double lds[kBlock / 64];
    double acc = 0.0;
    for (int i = threadIdx.x; i < n; i += kBlock) acc += partial[i];
    const double s = block_sum(acc, lds);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// fp32 as a caller would form it from the norm that is handed out; NaN (a norm that is none) stays NaN
__device__ __forceinline__ float clip_factor(float norm, float max_norm) {
    const float f = max_norm / (norm + 1e-6f);
    return f > 1.f ? 1.f : f;
}

__global__ __launch_bounds__(kBlock) void grad_scale_kernel(Table t, const float* __restrict__ norm, float max_norm) {
    const float f = clip_factor(*norm, max_norm);
    int k = 0;
    for (int c = blockIdx.x; c < t.n_chunks; c += gridDim.x) {
        while (c >= t.part[k].last_chunk) ++k;
        const Part& p = t.part[k];
        if (f == 1.f && p.out == p.data) continue;
        const int64_t lo = (int64_t)(c - (k == 0 ? 0 : t.part[k - 1].last_chunk)) * kChunk;
        const int64_t hi = lo + kChunk < p.n ? lo + kChunk : p.n;
        for (int64_t i = lo + threadIdx.x; i < hi; i += kBlock)
            store_as(p.out, p.out_dtype, i, load_as(p.data, p.dtype, i) * f);
    }
}

int64_t chunks_of(int64_t n) { return (n + kChunk - 1) / kChunk; }

// The launches of a list: tables of at most kTable tensors that are not empty and 2^30 chunks; `launch(table)` for each.
template <typename F>
void for_tables(const mrl_grad* grads, int64_t n, F launch) {
    Table t;
    t.n_parts = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i < n; ++i) {
        if (grads[i].n == 0) continue;
        chunks += chunks_of(grads[i].n);
        t.part[t.n_parts++] = {grads[i].data, grads[i].out, grads[i].n, (int32_t)chunks, (int16_t)grads[i].dtype,
                               (int16_t)grads[i].out_dtype};
        if (t.n_parts == kTable) {
            t.n_chunks = (int32_t)chunks;
            launch(t);
            t.n_parts = 0;
            chunks = 0;
        }
    }
    if (t.n_parts > 0) {
        t.n_chunks = (int32_t)chunks;
        launch(t);
    }
}

int check_grads(const char* fn, const mrl_grad* grads, int64_t n, bool with_out) {
    MRL_REQUIRE(n >= 0 && (n == 0 || grads), MRL_ERR_INVALID_ARG, "%s: n_grads=%lld", fn, (long long)n);
    MRL_REQUIRE(n <= MRL_GRAD_TENSORS, MRL_ERR_UNSUPPORTED, "%s: %lld tensors (at most %d)", fn, (long long)n, MRL_GRAD_TENSORS);
    for (int64_t i = 0; i < n; ++i) {
        const mrl_grad& g = grads[i];
        const size_t es = mrl::float_dtype_bytes(g.dtype), os = mrl::float_dtype_bytes(g.out_dtype);
        MRL_REQUIRE(es != 0, MRL_ERR_UNSUPPORTED, "%s: tensor %lld: dtype %d (want F32, BF16 or F16)", fn, (long long)i, g.dtype);
        MRL_REQUIRE(g.n >= 0, MRL_ERR_INVALID_ARG, "%s: tensor %lld: n=%lld", fn, (long long)i, (long long)g.n);
        MRL_REQUIRE(g.n <= (1LL << 33), MRL_ERR_UNSUPPORTED, "%s: tensor %lld: n=%lld (at most 2^33)", fn, (long long)i,
                    (long long)g.n);
        MRL_REQUIRE(g.n == 0 || g.data, MRL_ERR_INVALID_ARG, "%s: tensor %lld: NULL pointer", fn, (long long)i);
        MRL_REQUIRE(mrl::aligned(g.data, es), MRL_ERR_MISALIGNED, "%s: tensor %lld: misaligned", fn, (long long)i);
        if (!with_out) continue;
        MRL_REQUIRE(os != 0 && (g.out_dtype == g.dtype || g.out_dtype == MRL_F32), MRL_ERR_UNSUPPORTED,
                    "%s: tensor %lld: out dtype %d (want the gradient's or F32)", fn, (long long)i, g.out_dtype);
        MRL_REQUIRE(g.n == 0 || g.out, MRL_ERR_INVALID_ARG, "%s: tensor %lld: NULL out", fn, (long long)i);
        MRL_REQUIRE(mrl::aligned(g.out, os), MRL_ERR_MISALIGNED, "%s: tensor %lld: misaligned out", fn, (long long)i);
        MRL_REQUIRE(g.n == 0 || g.out != g.data || g.out_dtype == g.dtype, MRL_ERR_INVALID_ARG, "%s: tensor %lld: in place at another dtype",
                    fn, (long long)i);
    }
    return MRL_OK;
}

// What is written meets nothing else that is read or written: a tensor given twice would be scaled twice.
int check_overlap(const char* fn, const mrl_grad* grads, int64_t n) {
    uint32_t order[2 * MRL_GRAD_TENSORS];
    int64_t m = 0;
    const auto begin = [&](uint32_t r) { return (uintptr_t)(r & 1 ? grads[r >> 1].out : grads[r >> 1].data); };
    const auto end = [&](uint32_t r) {
        const mrl_grad& g = grads[r >> 1];
        return begin(r) + (uintptr_t)g.n * mrl::float_dtype_bytes(r & 1 ? g.out_dtype : g.dtype);
    };
    for (int64_t i = 0; i < n; ++i) {
        if (grads[i].n == 0) continue;
        order[m++] = (uint32_t)(2 * i + 1);
        if (grads[i].out != grads[i].data) order[m++] = (uint32_t)(2 * i);
    }
    std::sort(order, order + m, [&](uint32_t a, uint32_t b) { return begin(a) != begin(b) ? begin(a) < begin(b) : a < b; });
    // the furthest ends so far of everything and of what is written
    uintptr_t all = 0, written = 0;
    for (int64_t q = 0; q < m; ++q) {
        const uint32_t r = order[q];
        MRL_REQUIRE(begin(r) >= ((r & 1) ? all : written), MRL_ERR_INVALID_ARG,
                    "%s: tensor %lld shares memory with another that is written", fn, (long long)(r >> 1));
        all = std::max(all, end(r));
        if (r & 1) written = std::max(written, end(r));
    }
    return MRL_OK;
}

// Squares of all tables into the workspace; the number of partial sums.  A launch has as many workgroups as its share of
// the entries, so that there are at most kMaxPartials of them (and one for each launch).
int launch_squares(const mrl_grad* grads, int64_t n, double* partial, hipStream_t s) {
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) total += chunks_of(grads[i].n);
    const int64_t per = (total + kMaxPartials / 2 - 1) / (kMaxPartials / 2);
    int used = 0;
    for_tables(grads, n, [&](const Table& t) {
        const int groups = (int)((t.n_chunks + per - 1) / per);
        hipLaunchKernelGGL(grad_squares_kernel, dim3((unsigned)groups), dim3(kBlock), 0, s, t, partial + used);
        used += groups;
    });
    return used;
}

}  // namespace

extern "C" int mrl_grad_norm(const mrl_grad* grads, int64_t n_grads, float* norm, double* workspace, void* stream) {
    const char* fn = "mrl_grad_norm";
    const int rc = check_grads(fn, grads, n_grads, false);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE(norm && workspace, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(mrl::aligned(norm, 4) && mrl::aligned(workspace, 8), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    hipStream_t s = mrl::as_stream(stream);
    const int used = launch_squares(grads, n_grads, workspace, s);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, s, workspace, used, norm);
    return mrl::check_launch(fn);
}

extern "C" int mrl_grad_clip(const mrl_grad* grads, int64_t n_grads, float max_norm, float* norm, double* workspace,
                             void* stream) {
    const char* fn = "mrl_grad_clip";
    int rc = check_grads(fn, grads, n_grads, true);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE(max_norm >= 0.f, MRL_ERR_INVALID_ARG, "%s: max_norm=%g", fn, (double)max_norm);
    MRL_REQUIRE(norm && workspace, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(mrl::aligned(norm, 4) && mrl::aligned(workspace, 8), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    rc = check_overlap(fn, grads, n_grads);
    if (rc != MRL_OK) return rc;
    hipStream_t s = mrl::as_stream(stream);
    const int used = launch_squares(grads, n_grads, workspace, s);
    hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, s, workspace, used, norm);
    for_tables(grads, n_grads, [&](const Table& t) {
        const int groups = t.n_chunks < 4096 ? t.n_chunks : 4096;
        hipLaunchKernelGGL(grad_scale_kernel, dim3((unsigned)groups), dim3(kBlock), 0, s, t, norm, max_norm);
    });
    return mrl::check_launch(fn);
}
