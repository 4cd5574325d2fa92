// Token table for gfx950: rows of a [vocab, hidden] table, and the table's gradient by sorted tokens.
//
//   out_t = scale * table[id_t - start]                      (zeros where id_t - start is outside [0, vocab))
//   dtable_v = (dtable_v +) scale * sum_{t: id_t - start = v} dy_t
//
// The gradient's tokens are sorted by row, stably, by a radix sort of two or three digits; sums are then taken along the
// sorted list, in its order, in fp32, by workgroups of equal shares of it, and what crosses a share is joined afterwards:
// the same tokens give the same bits, a row that many tokens name is summed by many workgroups, and every row is rounded
// once.  Bound by memory, and by the sort's few launches where tokens are few.
#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kSortBlock = 512;             // threads of the sort's workgroups, as many as a digit has values
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kDigits = 512;
constexpr int kDigitBits = 9;
constexpr int kSortGroups = 128;            // most workgroups of a sort pass
constexpr int kShares = 2048;               // most shares of the sorted list
constexpr int kMinShare = 32;

// the row that a token names, `vocab` where it is outside
__device__ __forceinline__ int32_t row_of(const void* ids, int dtype, int64_t t, int64_t start, int64_t vocab) {
    const int64_t id = dtype == MRL_I64 ? reinterpret_cast<const int64_t*>(ids)[t] : (int64_t) reinterpret_cast<const int32_t*>(ids)[t];
    // start is at least 0, so a negative id cannot wrap into the table
    return id >= start && id - start < vocab ? (int32_t)(id - start) : (int32_t)vocab;
}

template <int DT>
__global__ __launch_bounds__(kBlock) void lookup_kernel(const void* __restrict__ ids, int ids_dtype, int64_t start,
                                                        const typename Elem<DT>::T* __restrict__ table, int64_t vocab,
                                                        int64_t hidden, float scale, typename Elem<DT>::T* __restrict__ out) {
    const int64_t t = blockIdx.x;
    const int32_t row = row_of(ids, ids_dtype, t, start, vocab);
    for (int64_t j = threadIdx.x; j < hidden; j += kBlock)
        Elem<DT>::store(out + t * hidden + j, row < vocab ? Elem<DT>::load(table + row * hidden + j) * scale : 0.f);
}

// ------------------------------------------------------------------------------------ sort
struct SortPlan {
    int passes, bits, groups;               // digits, their width, workgroups of a pass
    int64_t per_group;                      // tokens of a workgroup
};

__host__ SortPlan sort_plan(int64_t n_tokens, int64_t vocab) {
    int key_bits = 1;
    while ((vocab >> key_bits) != 0) ++key_bits;                    // keys are 0 .. vocab
    SortPlan p;
    p.passes = (key_bits + kDigitBits - 1) / kDigitBits;
    p.bits = (key_bits + p.passes - 1) / p.passes;
    p.per_group = (n_tokens + kSortGroups - 1) / kSortGroups;
    p.per_group = (p.per_group + kSortBlock - 1) / kSortBlock * kSortBlock;
    p.groups = (int)((n_tokens + p.per_group - 1) / p.per_group);
    return p;
}

// counts[group][digit] of the first digit, and zeros in those of the later passes.
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens,
                                                                int64_t start, int64_t vocab, SortPlan p,
                                                                int32_t* __restrict__ counts) {
    __shared__ int32_t hist[kDigits];
    hist[threadIdx.x] = 0;
    __syncthreads();
    const int64_t lo = blockIdx.x * p.per_group, hi = lo + p.per_group < n_tokens ? lo + p.per_group : n_tokens;
    const int32_t mask = (1 << p.bits) - 1;
    for (int64_t t = lo + threadIdx.x; t < hi; t += kSortBlock)
        atomicAdd(&hist[row_of(ids, ids_dtype, t, start, vocab) & mask], 1);
    __syncthreads();
    const int64_t at = (int64_t)blockIdx.x * kDigits + threadIdx.x, matrix = (int64_t)kSortGroups * kDigits;
    counts[at] = hist[threadIdx.x];
    for (int q = 1; q < p.passes; ++q) counts[q * matrix + at] = 0;
}

// One stable pass: a workgroup's tokens, in order, behind those of the workgroups in front of it.  Each wavefront takes a
// contiguous part of them; lanes of equal digit find each other by ballots.  Counts the next digit where the tokens land.
template <bool kFirst>
__global__ __launch_bounds__(kSortBlock) void sort_pass_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens,
                                                               int64_t start, int64_t vocab, SortPlan p, int pass,
                                                               const int32_t* __restrict__ keys_in,
                                                               const int32_t* __restrict__ tokens_in,
                                                               int32_t* __restrict__ keys_out, int32_t* __restrict__ tokens_out,
                                                               const int32_t* __restrict__ counts,
                                                               int32_t* __restrict__ next_counts) {
    __shared__ int32_t place[kSortWaves][kDigits];
    __shared__ int32_t wave_sum[kSortWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t mask = (1 << p.bits) - 1;
    const int shift = pass * p.bits;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) place[w][tid] = 0;
    // this digit's tokens altogether, and in the workgroups in front of this one
    int32_t total = 0, before = 0;
    for (int g = 0; g < p.groups; ++g) {
        const int32_t c = counts[g * kDigits + tid];
        total += c;
        if (g < (int)blockIdx.x) before += c;
    }
    int32_t incl = total;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
    }
    if (lane == 63) wave_sum[wave] = incl;
    __syncthreads();
    int32_t base = incl - total + before;
    for (int w = 0; w < wave; ++w) base += wave_sum[w];

    const int64_t lo = blockIdx.x * p.per_group, hi = lo + p.per_group < n_tokens ? lo + p.per_group : n_tokens;
    const int64_t per_wave = p.per_group / kSortWaves;             // whole wavefronts: per_group is whole workgroups
    const int64_t w_lo = lo + wave * per_wave, w_hi = w_lo + per_wave < hi ? w_lo + per_wave : hi;
    const auto key_at = [&](int64_t t) { return kFirst ? row_of(ids, ids_dtype, t, start, vocab) : keys_in[t]; };
    for (int64_t t = w_lo + lane; t < w_hi; t += 64) atomicAdd(&place[wave][(key_at(t) >> shift) & mask], 1);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        const int32_t c = place[w][tid];
        place[w][tid] = base;
        base += c;
    }
    __syncthreads();
    volatile int32_t* mine = place[wave];
    for (int64_t t0 = w_lo; t0 < w_hi; t0 += 64) {
        const int64_t t = t0 + lane;
        const bool active = t < w_hi;
        const int32_t key = active ? key_at(t) : 0;
        const int32_t digit = (key >> shift) & mask;
        uint64_t same = __ballot(active);
        for (int b = 0; b < p.bits; ++b) {
            const uint64_t set = __ballot((digit >> b) & 1);
            same &= ((digit >> b) & 1) ? set : ~set;
        }
        const int rank = __popcll(same & ((1ull << lane) - 1));
        const int32_t at = mine[digit] + rank;
        __builtin_amdgcn_wave_barrier();
        if (active) {
            if ((same >> lane) == 1ull) mine[digit] = at + 1;      // the last lane of this digit
            keys_out[at] = key;
            tokens_out[at] = kFirst ? (int32_t)t : tokens_in[t];
            if (next_counts) atomicAdd(&next_counts[(int64_t)(at / p.per_group) * kDigits + ((key >> (shift + p.bits)) & mask)], 1);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// ------------------------------------------------------------------------------------ sums
struct Sums {
    const int32_t *keys, *tokens;           // sorted
    float* part;                            // [share][2][hidden]: of a run from the share in front, of one that goes on behind
    int64_t n_tokens, hidden, share;
    int32_t vocab;
    float scale;
};

template <int GT, bool kAdd>
__device__ __forceinline__ void put(typename Elem<GT>::T* at, float sum, float scale) {
    Elem<GT>::store(at, kAdd ? Elem<GT>::load(at) + sum * scale : sum * scale);
}

// A share of the sorted list, a thread for a column.
template <int DT, int GT, bool kAdd>
__global__ __launch_bounds__(kBlock) void sum_kernel(Sums s, const typename Elem<DT>::T* __restrict__ dy,
                                                     typename Elem<GT>::T* __restrict__ dtable) {
    const int64_t j = (int64_t)blockIdx.y * kBlock + threadIdx.x;
    if (j >= s.hidden) return;
    const int64_t begin = blockIdx.x * s.share, end = begin + s.share < s.n_tokens ? begin + s.share : s.n_tokens;
    const int32_t prev = begin > 0 ? s.keys[begin - 1] : -1, next = end < s.n_tokens ? s.keys[end] : -1;
    for (int64_t p = begin; p < end;) {
        const int64_t first = p;
        const int32_t key = s.keys[p];
        if (key >= s.vocab) break;                                  // so are all behind it
        float acc = 0.f;
        do acc += Elem<DT>::load(dy + (int64_t)s.tokens[p] * s.hidden + j);
        while (++p < end && s.keys[p] == key);
        if (first == begin && prev == key) s.part[(blockIdx.x * 2ll) * s.hidden + j] = acc;
        else if (p == end && next == key) s.part[(blockIdx.x * 2ll + 1) * s.hidden + j] = acc;
        else put<GT, kAdd>(dtable + key * s.hidden + j, acc, s.scale);
    }
}

// The runs that cross shares: the share that one begins in adds up its parts.
template <int GT, bool kAdd>
__global__ __launch_bounds__(kBlock) void join_kernel(Sums s, typename Elem<GT>::T* __restrict__ dtable) {
    const int64_t j = (int64_t)blockIdx.y * kBlock + threadIdx.x;
    const int64_t begin = blockIdx.x * s.share, end = begin + s.share;
    if (end >= s.n_tokens) return;
    const int32_t key = s.keys[end - 1];
    if (key >= s.vocab || s.keys[end] != key) return;
    if (begin > 0 && s.keys[begin - 1] == key) return;              // begun further in front
    int64_t lo = end, hi = s.n_tokens;                              // the run's last token is in [lo, hi)
    while (hi - lo > 1) {
        const int64_t mid = (lo + hi) >> 1;
        if (s.keys[mid] == key) lo = mid; else hi = mid;
    }
    if (j >= s.hidden) return;
    float acc = s.part[(blockIdx.x * 2ll + 1) * s.hidden + j];
    for (int64_t g = blockIdx.x + 1ll; g <= lo / s.share; ++g) acc += s.part[g * 2 * s.hidden + j];
    put<GT, kAdd>(dtable + key * s.hidden + j, acc, s.scale);
}

template <int GT>
__global__ __launch_bounds__(kBlock) void zero_kernel(typename Elem<GT>::T* __restrict__ p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x; i < n; i += (int64_t)gridDim.x * kBlock) p[i] = 0;
}

// ------------------------------------------------------------------------------------ host
int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t share_of(int64_t n_tokens) {
    const int64_t s = (n_tokens + kShares - 1) / kShares;
    return s < kMinShare ? kMinShare : s;
}

struct Workspace {
    int64_t keys[2], tokens[2], counts, part, bytes;
};

Workspace workspace_of(int64_t n_tokens, int64_t vocab, int64_t hidden) {
    const SortPlan p = sort_plan(n_tokens, vocab);
    Workspace w;
    int64_t at = 0;
    for (int q = 0; q < 2; ++q) {
        w.keys[q] = at;
        at += round16(4 * n_tokens);
        w.tokens[q] = at;
        at += round16(4 * n_tokens);
    }
    w.counts = at;
    at += (int64_t)p.passes * kSortGroups * kDigits * 4;
    w.part = at;
    const int64_t share = share_of(n_tokens);
    at += (n_tokens + share - 1) / share * 2 * hidden * 4;
    w.bytes = at;
    return w;
}

int check_sizes(const char* fn, const void* ids, int ids_dtype, int64_t n_tokens, int64_t start, int dtype, int64_t vocab,
                int64_t hidden, float scale) {
    MRL_REQUIRE(mrl::int_dtype_bytes(ids_dtype) != 0, MRL_ERR_UNSUPPORTED, "%s: ids dtype %d (want I32 or I64)", fn, ids_dtype);
    MRL_REQUIRE(mrl::float_dtype_bytes(dtype) != 0, MRL_ERR_UNSUPPORTED, "%s: dtype %d (want F32, BF16 or F16)", fn, dtype);
    MRL_REQUIRE(n_tokens >= 0 && start >= 0 && vocab >= 1 && hidden >= 1, MRL_ERR_INVALID_ARG,
                "%s: n_tokens=%lld vocab_start=%lld vocab=%lld hidden=%lld", fn, (long long)n_tokens, (long long)start,
                (long long)vocab, (long long)hidden);
    MRL_REQUIRE(n_tokens <= 0x7fffffffLL && vocab < 0x7fffffffLL && hidden <= MRL_NORM_MAX_HIDDEN, MRL_ERR_UNSUPPORTED,
                "%s: n_tokens=%lld vocab=%lld hidden=%lld (at most 2^31 - 1, 2^31 - 2 and %d)", fn, (long long)n_tokens,
                (long long)vocab, (long long)hidden, MRL_NORM_MAX_HIDDEN);
    MRL_REQUIRE(scale - scale == 0.f, MRL_ERR_INVALID_ARG, "%s: scale=%g", fn, (double)scale);
    MRL_REQUIRE(n_tokens == 0 || ids, MRL_ERR_INVALID_ARG, "%s: NULL ids", fn);
    MRL_REQUIRE(mrl::aligned(ids, mrl::int_dtype_bytes(ids_dtype)), MRL_ERR_MISALIGNED, "%s: misaligned ids", fn);
    return MRL_OK;
}

template <int DT, int GT, bool kAdd>
void launch_sums(const Sums& s, const void* dy, void* dtable, hipStream_t stream) {
    using G = typename Elem<GT>::T;
    const unsigned columns = (unsigned)((s.hidden + kBlock - 1) / kBlock);
    const unsigned shares = (unsigned)((s.n_tokens + s.share - 1) / s.share);
    hipLaunchKernelGGL((sum_kernel<DT, GT, kAdd>), dim3(shares, columns), dim3(kBlock), 0, stream, s,
                       (const typename Elem<DT>::T*)dy, (G*)dtable);
    hipLaunchKernelGGL((join_kernel<GT, kAdd>), dim3(shares, columns), dim3(kBlock), 0, stream, s, (G*)dtable);
}

template <int DT, int GT>
void launch_sums(bool add, const Sums& s, const void* dy, void* dtable, hipStream_t stream) {
    if (add) launch_sums<DT, GT, true>(s, dy, dtable, stream);
    else launch_sums<DT, GT, false>(s, dy, dtable, stream);
}

}  // namespace

extern "C" int mrl_embedding_fwd(const void* ids, int ids_dtype, int64_t n_tokens, int64_t vocab_start, const void* table,
                                 int dtype, int64_t vocab, int64_t hidden, float scale, void* out, void* stream) {
    const char* fn = "mrl_embedding_fwd";
    const int rc = check_sizes(fn, ids, ids_dtype, n_tokens, vocab_start, dtype, vocab, hidden, scale);
    if (rc != MRL_OK || n_tokens == 0) return rc;
    MRL_REQUIRE(table && out, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const size_t es = mrl::float_dtype_bytes(dtype);
    MRL_REQUIRE(mrl::aligned(table, es) && mrl::aligned(out, es), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    const dim3 grid((unsigned)n_tokens), block(kBlock);
    hipStream_t s = mrl::as_stream(stream);
    if (dtype == MRL_F32)
        hipLaunchKernelGGL((lookup_kernel<MRL_F32>), grid, block, 0, s, ids, ids_dtype, vocab_start, (const float*)table, vocab,
                           hidden, scale, (float*)out);
    else if (dtype == MRL_BF16)
        hipLaunchKernelGGL((lookup_kernel<MRL_BF16>), grid, block, 0, s, ids, ids_dtype, vocab_start, (const uint16_t*)table, vocab,
                           hidden, scale, (uint16_t*)out);
    else
        hipLaunchKernelGGL((lookup_kernel<MRL_F16>), grid, block, 0, s, ids, ids_dtype, vocab_start, (const uint16_t*)table, vocab,
                           hidden, scale, (uint16_t*)out);
    return mrl::check_launch(fn);
}

extern "C" int64_t mrl_embedding_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab, int64_t hidden) {
    if (n_tokens <= 0 || vocab <= 0 || hidden <= 0 || n_tokens > 0x7fffffffLL || vocab >= 0x7fffffffLL ||
        hidden > MRL_NORM_MAX_HIDDEN)
        return 0;
    return workspace_of(n_tokens, vocab, hidden).bytes;
}

extern "C" int mrl_embedding_bwd(const void* ids, int ids_dtype, int64_t n_tokens, int64_t vocab_start, const void* dy, int dtype,
                                 int64_t vocab, int64_t hidden, float scale, void* dtable, int dtable_dtype, int accumulate,
                                 void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "mrl_embedding_bwd";
    const int rc = check_sizes(fn, ids, ids_dtype, n_tokens, vocab_start, dtype, vocab, hidden, scale);
    if (rc != MRL_OK) return rc;
    MRL_REQUIRE(dtable_dtype == dtype || dtable_dtype == MRL_F32, MRL_ERR_UNSUPPORTED,
                "%s: dtable dtype %d (want the gradient's or F32)", fn, dtable_dtype);
    MRL_REQUIRE(dtable && (dy || n_tokens == 0), MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    const int64_t need = mrl_embedding_bwd_workspace_bytes(n_tokens, vocab, hidden);
    MRL_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), MRL_ERR_INVALID_ARG, "%s: workspace of %lld bytes (want %lld)",
                fn, (long long)workspace_bytes, (long long)need);
    MRL_REQUIRE(mrl::aligned(dy, mrl::float_dtype_bytes(dtype)) && mrl::aligned(dtable, mrl::float_dtype_bytes(dtable_dtype)) &&
                    mrl::aligned(workspace, 16),
                MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    hipStream_t s = mrl::as_stream(stream);
    if (!accumulate) {
        const int64_t n = vocab * hidden;
        const int64_t blocks = (n + kBlock * 16 - 1) / (kBlock * 16);
        const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536)), block(kBlock);
        if (dtable_dtype == MRL_F32) hipLaunchKernelGGL((zero_kernel<MRL_F32>), grid, block, 0, s, (float*)dtable, n);
        else hipLaunchKernelGGL((zero_kernel<MRL_BF16>), grid, block, 0, s, (uint16_t*)dtable, n);
    }
    if (n_tokens == 0) return mrl::check_launch(fn);
    const Workspace w = workspace_of(n_tokens, vocab, hidden);
    const SortPlan p = sort_plan(n_tokens, vocab);
    char* base = (char*)workspace;
    int32_t *keys[2], *tokens[2];
    for (int q = 0; q < 2; ++q) {
        keys[q] = (int32_t*)(base + w.keys[q]);
        tokens[q] = (int32_t*)(base + w.tokens[q]);
    }
    int32_t* counts = (int32_t*)(base + w.counts);
    const dim3 grid((unsigned)p.groups), block(kSortBlock);
    hipLaunchKernelGGL(sort_count_kernel, grid, block, 0, s, ids, ids_dtype, n_tokens, vocab_start, vocab, p, counts);
    for (int q = 0; q < p.passes; ++q) {
        const int to = q & 1, from = to ^ 1;
        int32_t* here = counts + (int64_t)q * kSortGroups * kDigits;
        int32_t* next = q + 1 < p.passes ? here + (int64_t)kSortGroups * kDigits : nullptr;
        if (q == 0)
            hipLaunchKernelGGL((sort_pass_kernel<true>), grid, block, 0, s, ids, ids_dtype, n_tokens, vocab_start, vocab, p, q,
                               (const int32_t*)nullptr, (const int32_t*)nullptr, keys[to], tokens[to], here, next);
        else
            hipLaunchKernelGGL((sort_pass_kernel<false>), grid, block, 0, s, ids, ids_dtype, n_tokens, vocab_start, vocab, p, q,
                               keys[from], tokens[from], keys[to], tokens[to], here, next);
    }
    const int sorted = (p.passes - 1) & 1;
    const Sums sums = {keys[sorted], tokens[sorted], (float*)(base + w.part), n_tokens, hidden, share_of(n_tokens),
                       (int32_t)vocab, scale};
    const bool add = accumulate != 0;
    if (dtype == MRL_F32) launch_sums<MRL_F32, MRL_F32>(add, sums, dy, dtable, s);
    else if (dtype == MRL_BF16 && dtable_dtype == MRL_F32) launch_sums<MRL_BF16, MRL_F32>(add, sums, dy, dtable, s);
    else if (dtype == MRL_BF16) launch_sums<MRL_BF16, MRL_BF16>(add, sums, dy, dtable, s);
    else if (dtable_dtype == MRL_F32) launch_sums<MRL_F16, MRL_F32>(add, sums, dy, dtable, s);
    else launch_sums<MRL_F16, MRL_F16>(add, sums, dy, dtable, s);
    return mrl::check_launch(fn);
}
