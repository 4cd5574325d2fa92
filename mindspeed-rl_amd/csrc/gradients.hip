// The global norm of a list of gradients and clipping by it, for gfx950.
//
//   norm = sqrt(sum over all entries of all tensors of g^2),  factor = min(1, max_norm / (norm + 1e-6)),  out = g * factor
//
// Squares and their sums are held in 64 bits: no gradient that fp32 or bf16 holds overflows them, and the order of the sum
// does not show in the norm's fp32 bits but for a tie.  The list travels in the kernel's arguments, so a captured graph
// holds it, and nothing is copied to the device.
//
// Bound by memory.  1.4 GB: the norm 214 us (6.5 TB/s), clipped into other tensors 658 us (2.8 GB and the second read: 6.4 TB/s), bf16
// into fp32 880, in place 703; where the norm is within the bound nothing is written (205).  200 MB: 35, 92, 122, 96 us.  (Here and
// below: bf16, calls that follow each other in a replayed graph.)
#include <algorithm>

#include "lane_ops.h"
#include "mrl_internal.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kTable = 112;                 // tensors of a launch: 4 KB of arguments
constexpr int kSumVecs = 4;                 // vectors of 16 bytes that a thread has on its way where squares are summed
constexpr int kScaleVecs = 1;               // ... and where gradients are scaled: 1.4 GB of bf16 into fp32 880 us, by four 974
constexpr int64_t kCached = 256 << 20;      // bytes that the memory-side cache holds

constexpr int chunk_bytes(int vecs) { return kBlock * vecs * 16; }  // of a tensor that a workgroup takes at a time
constexpr int kMaxPartials = MRL_GRAD_NORM_PARTIALS;
constexpr int kGroups = 2048;               // workgroups of a list: eight on each of 256 CUs
constexpr int64_t kMostGroups = (1LL << 24) - 1;    // of a launch, which holds fewer than 2^32 threads

struct Part {
    const void* data;
    void* out;
    int64_t n;
    int64_t end_chunk;                      // chunks of this tensor and the ones in front of it
};

// Tensors of one type, and of one type of their outputs.
struct Table {
    Part part[kTable];
    int32_t n_parts, n_chunks;
    int32_t in_place;                       // all of them
};

// A chunk of the table: its tensor, its first byte there and how many it has.
struct Place {
    int part, bytes;
    int64_t first;
};

__device__ __forceinline__ int part_of(const int32_t* ends, int chunk) {       // as many tensors end at or in front of it
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_readfirstlane(__popcll(__ballot(ends[lane] <= chunk)) + __popcll(__ballot(ends[64 + lane] <= chunk)));
}

template <int DT, int kVecs>
__device__ __forceinline__ Place place_of(const Table& t, const int32_t* ends, int chunk) {
    constexpr int kChunk = chunk_bytes(kVecs);
    Place c;
    c.part = part_of(ends, chunk);
    c.first = (chunk - (c.part == 0 ? 0 : t.part[c.part - 1].end_chunk)) * kChunk;
    const int64_t left = t.part[c.part].n * (int64_t)sizeof(typename Elem<DT>::T) - c.first;
    c.bytes = left < kChunk ? (int)left : kChunk;
    return c;
}

template <bool kStream>
__device__ __forceinline__ u32x4 load_16(const char* p) {
    const mrl::u32x4_anywhere* v = (const mrl::u32x4_anywhere*)p;
    return kStream ? __builtin_nontemporal_load(v) : *v;
}

// Its bytes as raw vectors.  Vectors behind the tensor's end are zeros, of one that the end cuts the entries behind it.
template <int kVecs, bool kStream>
__device__ __forceinline__ void load_chunk(const Table& t, const Place& c, u32x4 (&v)[kVecs]) {
    const char* from = (const char*)t.part[c.part].data + c.first;
    if (c.bytes == chunk_bytes(kVecs)) {
#pragma unroll
        for (int q = 0; q < kVecs; ++q) v[q] = load_16<kStream>(from + (q * kBlock + threadIdx.x) * 16);
        return;
    }
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        const int at = (q * kBlock + threadIdx.x) * 16;
        v[q] = mrl::make_u32x4(0u, 0u, 0u, 0u);
        if (at + 16 <= c.bytes) {
            v[q] = load_16<kStream>(from + at);
        } else if (at < c.bytes) {
            uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (at + 2 * i < c.bytes) w[i >> 1] |= (uint32_t)*(const uint16_t*)(from + at + 2 * i) << (16 * (i & 1));
            v[q] = mrl::make_u32x4(w[0], w[1], w[2], w[3]);
        }
    }
}

// Where the tensors of the table end, in LDS; 128 entries.
__device__ __forceinline__ void load_ends(const Table& t, int32_t* ends) {
    if (threadIdx.x < 128) ends[threadIdx.x] = (int)threadIdx.x < t.n_parts ? (int32_t)t.part[threadIdx.x].end_chunk : 0x7fffffff;
    __syncthreads();
}

// Sum over the workgroup, the same in every thread.
__device__ __forceinline__ double block_sum(double x, double* lds) {
    x = mrl::lanes_sum<4>(x);
    x = (mrl::lane_value(x, 0) + mrl::lane_value(x, 16)) + (mrl::lane_value(x, 32) + mrl::lane_value(x, 48));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
    __syncthreads();
    double s = lds[0];
#pragma unroll
    for (int w = 1; w < kBlock / 64; ++w) s += lds[w];
    return s;
}

// The sum of squares of a workgroup's chunks, one of which is on its way while the one in front is summed.
template <int DT, bool kStream>
__global__ __launch_bounds__(kBlock, 8) void grad_squares_kernel(Table t, double* __restrict__ partial) {
    __shared__ double lds[kBlock / 64];
    __shared__ int32_t ends[128];
    load_ends(t, ends);
    double acc = 0.0;
    u32x4 next[kSumVecs];
    load_chunk<kSumVecs, kStream>(t, place_of<DT, kSumVecs>(t, ends, blockIdx.x), next);
    for (int c = blockIdx.x; c < t.n_chunks; c += gridDim.x) {
        u32x4 v[kSumVecs];
#pragma unroll
        for (int q = 0; q < kSumVecs; ++q) v[q] = next[q];
        if (c + (int)gridDim.x < t.n_chunks) load_chunk<kSumVecs, kStream>(t, place_of<DT, kSumVecs>(t, ends, c + gridDim.x), next);
#pragma unroll
        for (int q = 0; q < kSumVecs; ++q) {
            float z[Elem<DT>::kVec];
            Elem<DT>::unpack(v[q], z);
#pragma unroll
            for (int i = 0; i < Elem<DT>::kVec; ++i) acc = __builtin_fma((double)z[i], (double)z[i], acc);
        }
    }
    const double s = block_sum(acc, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// The norm from the workgroups' sums, in every thread.
__device__ __forceinline__ float norm_of(const double* partial, int n, double* lds) {
    double acc = 0.0;
    for (int i0 = threadIdx.x; i0 < n; i0 += kBlock * 8) {
        double v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = partial[i0 + i * kBlock < n ? i0 + i * kBlock : 0];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc += i0 + i * kBlock < n ? v[i] : 0.0;
    }
    return (float)sqrt(block_sum(acc, lds));
}

__global__ __launch_bounds__(kBlock) void grad_norm_kernel(const double* __restrict__ partial, int n, float* __restrict__ norm) {
    __shared__ double lds[kBlock / 64];
    const float v = norm_of(partial, n, lds);
    if (threadIdx.x == 0) *norm = v;
}

template <int DT>
__device__ __forceinline__ void scale_chunk(const Table& t, const Place& c, float f) {
    constexpr int kVec = Elem<DT>::kVec, kVecs = kScaleVecs;
    u32x4 v[kVecs];
    load_chunk<kVecs, true>(t, c, v);
    typename Elem<DT>::T* to = (typename Elem<DT>::T*)((char*)t.part[c.part].out + c.first);
    const int n = c.bytes / (16 / kVec);
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        const int at = (q * kBlock + threadIdx.x) * kVec;
        float z[kVec];
        Elem<DT>::unpack(v[q], z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] *= f;
        if (at + kVec <= n) {
            mrl::Vec<DT>::store_nt(to + at, Elem<DT>::pack(z));
        } else {
#pragma unroll
            for (int i = 0; i < kVec; ++i)
                if (at + i < n) Elem<DT>::store(to + at + i, z[i]);
        }
    }
}

// To fp32: a lane reads 8 bytes and writes 16, so that what a wavefront writes at a time lies together.
template <int DT>
__device__ __forceinline__ void widen_chunk(const Table& t, const Place& c, float f) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    typedef u32x2 u32x2_anywhere __attribute__((aligned(2)));
    constexpr int kUnits = 2 * kScaleVecs;
    const char* from = (const char*)t.part[c.part].data + c.first;
    float* to = (float*)t.part[c.part].out + c.first / 2;
    u32x2 v[kUnits] = {};
    if (c.bytes >= 8) {
#pragma unroll
        for (int q = 0; q < kUnits; ++q) {
            const int at = (q * kBlock + threadIdx.x) * 8;
            v[q] = __builtin_nontemporal_load((const u32x2_anywhere*)(from + (at + 8 <= c.bytes ? at : 0)));
        }
    }
#pragma unroll
    for (int q = 0; q < kUnits; ++q) {
        const int at = (q * kBlock + threadIdx.x) * 8;
        if (at + 8 <= c.bytes) {
            float z[8];
            Elem<DT>::unpack(mrl::make_u32x4(v[q].x, v[q].y, 0u, 0u), z);
            mrl::Vec<MRL_F32>::store_nt(to + at / 2, mrl::make_u32x4(__float_as_uint(z[0] * f), __float_as_uint(z[1] * f),
                                                                     __float_as_uint(z[2] * f), __float_as_uint(z[3] * f)));
        } else {
            for (int i = at; i < c.bytes; i += 2) to[i / 2] = Elem<DT>::load((const uint16_t*)(from + i)) * f;
        }
    }
}

// The norm comes from the partial sums, formed by every workgroup for itself, or from where a launch in front left it
// (n_partial == 0); the factor in fp32, as a caller would form it from the norm that is handed out (NaN, of a norm that
// is none, stays NaN).
template <int DT, int OT>
__global__ __launch_bounds__(kBlock, 8) void grad_scale_kernel(Table t, const double* __restrict__ partial, int n_partial,
                                                               float* norm, float max_norm, int write_norm) {
    __shared__ double lds[kBlock / 64];
    __shared__ int32_t ends[128];
    const float total = n_partial > 0 ? norm_of(partial, n_partial, lds) : *norm;
    if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
    const float quotient = max_norm / (total + 1e-6f), f = quotient > 1.f ? 1.f : quotient;
    if (f == 1.f && t.in_place) return;
    load_ends(t, ends);
    for (int c = blockIdx.x; c < t.n_chunks; c += gridDim.x) {
        const Place at = place_of<DT, kScaleVecs>(t, ends, c);
        if constexpr (DT == OT) scale_chunk<DT>(t, at, f);
        else widen_chunk<DT>(t, at, f);
    }
}

int64_t bytes_of(const mrl_grad& g) { return g.n * mrl::float_dtype_bytes(g.dtype); }

int64_t chunks_of(const mrl_grad& g, int vecs) { return (bytes_of(g) + chunk_bytes(vecs) - 1) / chunk_bytes(vecs); }

// The launches of a list for the tensors of a kind - type, type of the output (-1: any), whether in place (-1: either) - that
// are not empty: launch(table) for each at most kTable of them.
template <typename F>
void for_tables(const mrl_grad* grads, int64_t n, int vecs, int dtype, int out_dtype, int in_place, F launch) {
    Table t;
    t.n_parts = 0;
    t.in_place = in_place;
    int64_t chunks = 0;
    for (int64_t i = 0; i < n; ++i) {
        const mrl_grad& g = grads[i];
        if (g.n == 0 || g.dtype != dtype || (out_dtype >= 0 && g.out_dtype != out_dtype) ||
            (in_place >= 0 && (g.out == g.data) != (in_place != 0)))
            continue;
        chunks += chunks_of(g, vecs);
        t.part[t.n_parts++] = {g.data, g.out, g.n, chunks};
        t.n_chunks = (int32_t)chunks;
        if (t.n_parts == kTable) {
            launch(t);
            t.n_parts = 0;
            chunks = 0;
        }
    }
    if (t.n_parts > 0) launch(t);
}

int check_grads(const char* fn, const mrl_grad* grads, int64_t n, bool with_out) {
    MRL_REQUIRE(n >= 0 && (n == 0 || grads), MRL_ERR_INVALID_ARG, "%s: n_grads=%lld", fn, (long long)n);
    static_assert(kGroups + MRL_GRAD_TENSORS / kTable + 3 <= kMaxPartials, "a partial sum for every workgroup");
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

// Chunks that each workgroup takes: as many as make kGroups of them for the list (and one more at most for each launch).
int64_t chunks_each(const mrl_grad* grads, int64_t n, int vecs) {
    int64_t total = 0;
    for (int64_t i = 0; i < n; ++i) total += chunks_of(grads[i], vecs);
    return (total + kGroups - 1) / kGroups;
}

// Squares of all tensors into the workspace; the number of partial sums.  A list that is read again and that the
// memory-side cache holds is left there, anything else goes past it (us, left / past: clipping 200 MB 92 / 103; the norm of
// 1.4 GB 240 / 214).
int launch_squares(const mrl_grad* grads, int64_t n, bool read_again, double* partial, hipStream_t s) {
    const int64_t each = chunks_each(grads, n, kSumVecs);
    int64_t bytes = 0;
    for (int64_t i = 0; i < n; ++i) bytes += bytes_of(grads[i]);
    const bool stream = !read_again || bytes > kCached;
    int used = 0;
    const auto launch = [&](const Table& t, auto through, auto past) {
        const int groups = (int)((t.n_chunks + each - 1) / each);
        hipLaunchKernelGGL(stream ? past : through, dim3((unsigned)groups), dim3(kBlock), 0, s, t, partial + used);
        used += groups;
    };
    for_tables(grads, n, kSumVecs, MRL_BF16, -1, -1,
               [&](const Table& t) { launch(t, grad_squares_kernel<MRL_BF16, false>, grad_squares_kernel<MRL_BF16, true>); });
    for_tables(grads, n, kSumVecs, MRL_F16, -1, -1,
               [&](const Table& t) { launch(t, grad_squares_kernel<MRL_F16, false>, grad_squares_kernel<MRL_F16, true>); });
    for_tables(grads, n, kSumVecs, MRL_F32, -1, -1,
               [&](const Table& t) { launch(t, grad_squares_kernel<MRL_F32, false>, grad_squares_kernel<MRL_F32, true>); });
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
    const int used = launch_squares(grads, n_grads, false, workspace, s);
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
    const int used = launch_squares(grads, n_grads, true, workspace, s);
    const int64_t each = chunks_each(grads, n_grads, kScaleVecs);
    // Lists of more chunks than workgroups fit: those that go elsewhere take a workgroup a chunk, which the memory serves
    // best (1.4 GB 658 us; by workgroups that stay 723), and a launch in front forms the norm for them; in place the workgroups
    // stay, half as many (1.4 GB 703 us, all of them 734), for there may be nothing to do: a workgroup a chunk takes 655, but 278
    // instead of 205 where nothing is.  Of shorter lists every workgroup forms it (1 MB into fp32 7.3 us; with the launch 8.7).
    const bool alone = used == 0 || each > 1;
    if (alone) hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(kBlock), 0, s, workspace, used, norm);
    int write_norm = alone ? 0 : 1;
    const auto launch = [&](const Table& t, auto kernel) {
        const int64_t groups = t.in_place ? (t.n_chunks + 2 * each - 1) / (2 * each) : t.n_chunks < kMostGroups ? t.n_chunks : kMostGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(kBlock), 0, s, t, workspace, alone ? 0 : used, norm, max_norm,
                           write_norm);
        write_norm = 0;
    };
    for (int in_place = 0; in_place < 2; ++in_place) {
        for_tables(grads, n_grads, kScaleVecs, MRL_BF16, MRL_BF16, in_place, [&](const Table& t) { launch(t, grad_scale_kernel<MRL_BF16, MRL_BF16>); });
        for_tables(grads, n_grads, kScaleVecs, MRL_F16, MRL_F16, in_place, [&](const Table& t) { launch(t, grad_scale_kernel<MRL_F16, MRL_F16>); });
        for_tables(grads, n_grads, kScaleVecs, MRL_F32, MRL_F32, in_place, [&](const Table& t) { launch(t, grad_scale_kernel<MRL_F32, MRL_F32>); });
    }
    for_tables(grads, n_grads, kScaleVecs, MRL_BF16, MRL_F32, 0, [&](const Table& t) { launch(t, grad_scale_kernel<MRL_BF16, MRL_F32>); });
    for_tables(grads, n_grads, kScaleVecs, MRL_F16, MRL_F32, 0, [&](const Table& t) { launch(t, grad_scale_kernel<MRL_F16, MRL_F32>); });
    return mrl::check_launch(fn);
}
