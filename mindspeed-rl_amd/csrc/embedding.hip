// Token table for gfx950: rows of a [vocab, hidden] table, and the table's gradient by sorted tokens.
//
//   out_t = scale * table[id_t - start]                      (zeros where id_t - start is outside [0, vocab))
//   dtable_v = (dtable_v +) scale * sum_{t: id_t - start = v} dy_t
//
// The gradient's tokens are sorted by row, stably, by a radix sort of digits of up to 9 bits (two for 152 064 rows); sums are
// then taken along the sorted list, in its order, in fp32, by workgroups of equal shares of it, and what crosses a share is
// joined afterwards: the same tokens give the same bits, a row that many tokens name is summed by many workgroups, and
// every row is rounded once.  Bound by memory, and by the sort's few launches where tokens are few.
//
// 32 768 tokens of 12 242 rows of 152 064 x 3 584 bf16: lookup 57 us (5.7 TB/s), gradient 257 us (1.1 GB of zeros, 235 MB read:
// 5.2 TB/s), added to fp32 141 us.  64 tokens: 8, 175 (6.2 TB/s) and 15 us.  (Here and below: calls that follow each other in a
// replayed graph.)
#include "lane_ops.h"
#include "mrl_internal.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kSortBlock = 512;             // threads of the sort's workgroups, as many as a digit has values
constexpr int kSortWaves = kSortBlock / 64;
constexpr int kDigits = 512;
constexpr int kDigitBits = 9;
constexpr int kSortGroups = 128;            // most workgroups of a sort pass
constexpr int kShares = 4096;               // most shares of the sorted list
constexpr int kMinShare = 8;
constexpr int kFewTokens = 2048;            // that one workgroup sorts in its LDS: 500 tokens 18 us in all, 2 000 23; by passes 25, 26
constexpr int64_t kMostTokens = 1LL << 26;  // of a call, and one more
constexpr int64_t kLaunchTokens = kMostTokens - kBlock / 64;        // with a wavefront each, as many as a launch holds

// the row that a token names, `vocab` where it is outside
__device__ __forceinline__ int32_t row_of(const void* ids, int dtype, int64_t t, int64_t start, int64_t vocab) {
    const int64_t id = dtype == MRL_I64 ? reinterpret_cast<const int64_t*>(ids)[t] : (int64_t) reinterpret_cast<const int32_t*>(ids)[t];
    // start is at least 0, so a negative id cannot wrap into the table
    return id >= start && id - start < vocab ? (int32_t)(id - start) : (int32_t)vocab;
}

// Rows shorter than a vector: a thread an entry.
template <int DT>
__global__ __launch_bounds__(kBlock) void lookup_narrow_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens,
                                                               int64_t start, const typename Elem<DT>::T* __restrict__ table,
                                                               int64_t vocab, int hidden, float scale,
                                                               typename Elem<DT>::T* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= n_tokens * hidden) return;
    const int64_t t = i / hidden, row = row_of(ids, ids_dtype, t, start, vocab);
    Elem<DT>::store(out + i, row < vocab ? Elem<DT>::load(table + row * hidden + (i - t * hidden)) * scale : 0.f);
}

// A wavefront a token and kVecs vectors a lane, all on their way together; a row that is not whole vectors ends with one that
// overlaps the one in front of it, and lanes behind the row write that again: the same bits.  Table rows are read through
// the caches (tokens repeat), what is written goes past them (57 us at the size above; through them 68).
template <int DT, int kVecs>
__global__ __launch_bounds__(kBlock) void lookup_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens, int64_t start,
                                                        const typename Elem<DT>::T* __restrict__ table, int64_t vocab,
                                                        int hidden, float scale, typename Elem<DT>::T* __restrict__ out) {
    constexpr int kVec = Elem<DT>::kVec;
    const int lane = threadIdx.x & 63;
    const int64_t t = (int64_t)blockIdx.x * (kBlock / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (t >= n_tokens) return;
    const int64_t row = row_of(ids, ids_dtype, t, start, vocab);
    const bool inside = row < vocab;
    const typename Elem<DT>::T* from = table + (inside ? row : 0) * hidden;
    typename Elem<DT>::T* to = out + t * hidden;
    const int first = ((int)blockIdx.y * kVecs * 64 + lane) * kVec, most = hidden - kVec;
    u32x4 v[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        const int j = first + q * 64 * kVec;
        v[q] = mrl::Vec<DT>::load(from + (j < most ? j : most));
    }
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
        const int j = first + q * 64 * kVec;
        float z[kVec];
        Elem<DT>::unpack(v[q], z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) z[i] = inside ? z[i] * scale : 0.f;
        mrl::Vec<DT>::store_nt(to + (j < most ? j : most), Elem<DT>::pack(z));
    }
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

// Zeros for the gradient's rows that no token names: workgroups behind the sort's, which is bound by latency and leaves the
// memory to them.  Rows that are named are written later.  Spread over the sort's launches, 32 768 tokens of 152 064 x 3 584
// bf16 take 257 us; all behind the first 274.
struct Fill {
    char* at;                               // 2-byte aligned at least
    int64_t bytes;                          // this launch's part
};

constexpr int kFillVecs = 1;                // vectors a thread
constexpr int64_t kFillBytes = (int64_t)kSortBlock * kFillVecs * 16;

__device__ __forceinline__ void fill_part(const Fill& f, int64_t block) {
    const u32x4 zero = mrl::make_u32x4(0u, 0u, 0u, 0u);
    const int64_t lo = block * kFillBytes;
#pragma unroll
    for (int q = 0; q < kFillVecs; ++q) {
        const int64_t at = lo + ((int64_t)q * kSortBlock + threadIdx.x) * 16;
        if (at + 16 <= f.bytes) *(mrl::u32x4_anywhere*)(f.at + at) = zero;
        else
            for (int64_t i = at; i < f.bytes; i += 2) *(uint16_t*)(f.at + i) = 0;
    }
}

// counts[group][digit] of the first digit, and zeros in those of the later passes.
__global__ __launch_bounds__(kSortBlock) void sort_count_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens,
                                                                int64_t start, int64_t vocab, SortPlan p,
                                                                int32_t* __restrict__ counts, Fill fill) {
    __shared__ int32_t hist[kDigits];
    if ((int)blockIdx.x >= p.groups) return fill_part(fill, blockIdx.x - p.groups);
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

// The steps of a stable pass by a workgroup over its tokens [lo, hi), of which each wavefront takes `per_wave` in a row.
// `place[wave][digit]` counts at first and then says where the next token of the digit goes.
struct Placing {
    int32_t (*place)[kDigits];
    int64_t w_lo, w_hi;
    int bits, shift;

    __device__ __forceinline__ void clear() const {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) place[w][threadIdx.x] = 0;
    }
    template <typename Key>
    __device__ __forceinline__ void count(Key key_at) const {
        for (int64_t t = w_lo + (threadIdx.x & 63); t < w_hi; t += 64)
            atomicAdd(&place[threadIdx.x >> 6][(key_at(t) >> shift) & ((1 << bits) - 1)], 1);
    }
    // thread d: where the workgroup's first token of digit d goes
    __device__ __forceinline__ void start(int32_t base) const {
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            const int32_t c = place[w][threadIdx.x];
            place[w][threadIdx.x] = base;
            base += c;
        }
    }
    // put(t, key, at, same) for every token, in order within the wavefront: lanes of equal digit (`same`) find each other by
    // ballots.
    template <typename Key, typename Put>
    __device__ __forceinline__ void run(Key key_at, Put put) const {
        const int lane = threadIdx.x & 63;
        volatile int32_t* mine = place[threadIdx.x >> 6];
        for (int64_t t0 = w_lo; t0 < w_hi; t0 += 64) {
            const int64_t t = t0 + lane;
            const bool active = t < w_hi;
            const int32_t key = active ? key_at(t) : 0;
            const int32_t digit = (key >> shift) & ((1 << bits) - 1);
            uint64_t same = __ballot(active);
            for (int b = 0; b < bits; ++b) {
                const uint64_t set = __ballot((digit >> b) & 1);
                same &= ((digit >> b) & 1) ? set : ~set;
            }
            const int32_t at = mine[digit] + __popcll(same & ((1ull << lane) - 1));
            __builtin_amdgcn_wave_barrier();
            if (active) {
                if ((same >> lane) == 1ull) mine[digit] = at + 1;   // the last lane of this digit
                put(t, key, at, same);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
};

// Sum of the values of the threads in front of this one.  `lds`: an entry per wavefront; a barrier inside.
__device__ __forceinline__ int32_t sum_in_front(int32_t x, int32_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t incl = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int32_t o = __shfl_up(incl, off, 64);
        if (lane >= off) incl += o;
    }
    if (lane == 63) lds[wave] = incl;
    __syncthreads();
    int32_t before = incl - x;
    for (int w = 0; w < wave; ++w) before += lds[w];
    return before;
}

// One stable pass: a workgroup's tokens, in order, behind those of the workgroups in front of it.  Counts the next digit
// where the tokens land.
template <bool kFirst>
__global__ __launch_bounds__(kSortBlock) void sort_pass_kernel(const void* __restrict__ ids, int ids_dtype, int64_t n_tokens,
                                                               int64_t start, int64_t vocab, SortPlan p, int pass,
                                                               const int32_t* __restrict__ keys_in,
                                                               const int32_t* __restrict__ tokens_in,
                                                               int32_t* __restrict__ keys_out, int32_t* __restrict__ tokens_out,
                                                               const int32_t* __restrict__ counts,
                                                               int32_t* __restrict__ next_counts, Fill fill) {
    if ((int)blockIdx.x >= p.groups) return fill_part(fill, blockIdx.x - p.groups);
    __shared__ int32_t place[kSortWaves][kDigits];
    __shared__ int32_t wave_sum[kSortWaves];
    const int tid = threadIdx.x;
    const int64_t lo = blockIdx.x * p.per_group, hi = lo + p.per_group < n_tokens ? lo + p.per_group : n_tokens;
    const int64_t per_wave = p.per_group / kSortWaves;             // whole wavefronts: per_group is whole workgroups
    const int64_t w_lo = lo + (tid >> 6) * per_wave;
    const Placing step = {place, w_lo, w_lo + per_wave < hi ? w_lo + per_wave : hi, p.bits, pass * p.bits};
    const auto key_at = [&](int64_t t) { return kFirst ? row_of(ids, ids_dtype, t, start, vocab) : keys_in[t]; };
    step.clear();
    // this digit's tokens altogether, and in the workgroups in front of this one
    int32_t total = 0, before = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 16) {         // sixteen on their way at a time
        int32_t c[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) c[i] = counts[(g0 + i < p.groups ? g0 + i : 0) * kDigits + tid];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            total += g0 + i < p.groups ? c[i] : 0;
            before += g0 + i < (int)blockIdx.x ? c[i] : 0;
        }
    }
    const int32_t base = sum_in_front(total, wave_sum) + before;   // its barrier: `place` is cleared
    step.count(key_at);
    __syncthreads();
    step.start(base);
    __syncthreads();
    const uint32_t per_group = (uint32_t)p.per_group;
    step.run(key_at, [&](int64_t t, int32_t key, int32_t at, uint64_t same) {
        keys_out[at] = key;
        tokens_out[at] = kFirst ? (int32_t)t : tokens_in[t];
        if (!next_counts) return;
        // lanes that count what the first lane of their digit counts leave it to that: a token that is everywhere would
        // have every lane add to one counter (49 152 tokens, most of two kinds: 15 us a pass without)
        const uint32_t counter = (uint32_t)at / per_group * kDigits + ((key >> (step.shift + p.bits)) & ((1 << p.bits) - 1));
        const int first = __ffsll((unsigned long long)same) - 1;
        const bool with_first = counter == (uint32_t)__shfl((int)counter, first, 64);
        const uint64_t counted = same & __ballot(with_first);
        if ((int)(threadIdx.x & 63) == first) atomicAdd(&next_counts[counter], __popcll(counted));
        else if (!with_first) atomicAdd(&next_counts[counter], 1);
    });
}

// All passes in one launch, for as many tokens as a workgroup holds.
__global__ __launch_bounds__(kSortBlock) void sort_few_kernel(const void* __restrict__ ids, int ids_dtype, int n_tokens, int64_t start,
                                                              int64_t vocab, SortPlan p, int32_t* __restrict__ keys_out,
                                                              int32_t* __restrict__ tokens_out, Fill fill) {
    if (blockIdx.x >= 1) return fill_part(fill, blockIdx.x - 1);
    __shared__ int32_t place[kSortWaves][kDigits];
    __shared__ int32_t wave_sum[kSortWaves];
    __shared__ int32_t keys[2][kFewTokens];
    __shared__ uint16_t tokens[2][kFewTokens];
    const int tid = threadIdx.x;
    for (int t = tid; t < n_tokens; t += kSortBlock) {
        keys[0][t] = row_of(ids, ids_dtype, t, start, vocab);
        tokens[0][t] = (uint16_t)t;
    }
    const int per_wave = ((n_tokens + kSortBlock - 1) / kSortBlock) * 64, w_lo = (tid >> 6) * per_wave;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int from = pass & 1, to = from ^ 1;
        const bool last = pass == p.passes - 1;
        const Placing step = {place, w_lo, w_lo + per_wave < n_tokens ? w_lo + per_wave : n_tokens, p.bits, pass * p.bits};
        const auto key_at = [&](int64_t t) { return keys[from][t]; };
        step.clear();
        __syncthreads();                                // the tokens of the step in front are in their places, too
        step.count(key_at);
        __syncthreads();
        int32_t total = 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) total += place[w][tid];
        step.start(sum_in_front(total, wave_sum));
        __syncthreads();
        step.run(key_at, [&](int64_t t, int32_t key, int32_t at, uint64_t) {
            if (last) {
                keys_out[at] = key;
                tokens_out[at] = tokens[from][t];
            } else {
                keys[to][at] = key;
                tokens[to][at] = tokens[from][t];
            }
        });
        __syncthreads();
    }
}

// ------------------------------------------------------------------------------------ sums
// The sorted list in equal shares, a workgroup each; part[share][2][hidden] holds the sum of a run that the share in front
// began, and that of one which goes on behind this share.
struct Sums {
    float* part;
    int64_t n_tokens, hidden, share;
    int32_t vocab;
    float scale;
};

// Rows shorter than a vector: a thread a column.
template <int DT, int GT, bool kAdd>
__global__ __launch_bounds__(64) void sum_narrow_kernel(Sums s, const int32_t* __restrict__ keys, const int32_t* __restrict__ tokens,
                                                        const typename Elem<DT>::T* __restrict__ dy,
                                                        typename Elem<GT>::T* __restrict__ dtable) {
    const int64_t j = threadIdx.x;
    if (j >= s.hidden) return;
    const int64_t begin = blockIdx.x * s.share, end = begin + s.share < s.n_tokens ? begin + s.share : s.n_tokens;
    const int32_t prev = begin > 0 ? keys[begin - 1] : -1, next = end < s.n_tokens ? keys[end] : -1;
    for (int64_t p = begin; p < end;) {
        const int64_t first = p;
        const int32_t key = keys[p];
        if (key >= s.vocab) break;                                  // so are all behind it
        float acc = 0.f;
        do acc += Elem<DT>::load(dy + (int64_t)tokens[p] * s.hidden + j);
        while (++p < end && keys[p] == key);
        typename Elem<GT>::T* at = dtable + key * s.hidden + j;
        if (first == begin && prev == key) s.part[(blockIdx.x * 2ll) * s.hidden + j] = acc;
        else if (p == end && next == key) s.part[(blockIdx.x * 2ll + 1) * s.hidden + j] = acc;
        else Elem<GT>::store(at, kAdd ? Elem<GT>::load(at) + acc * s.scale : acc * s.scale);
    }
}

// kVec columns of a row: written, or added to what is there.  Entries in front of `skip` are another lane's.
template <int GT, int kVec, bool kAdd>
__device__ __forceinline__ void put_columns(typename Elem<GT>::T* at, const float (&acc)[kVec], float scale, int skip) {
    constexpr int kGVec = Elem<GT>::kVec;
    if (skip != 0) {
#pragma unroll
        for (int i = 0; i < kVec; ++i)
            if (i >= skip) Elem<GT>::store(at + i, kAdd ? Elem<GT>::load(at + i) + acc[i] * scale : acc[i] * scale);
        return;
    }
#pragma unroll
    for (int p = 0; p < kVec / kGVec; ++p) {
        float z[kGVec] = {};
        if (kAdd) Elem<GT>::unpack(mrl::Vec<GT>::load(at + p * kGVec), z);
#pragma unroll
        for (int i = 0; i < kGVec; ++i) z[i] = kAdd ? z[i] + acc[p * kGVec + i] * scale : acc[p * kGVec + i] * scale;
        mrl::Vec<GT>::store(at + p * kGVec, Elem<GT>::pack(z));
    }
}

constexpr int kSumBlock = 512;              // most lanes of a share
constexpr int kSumRows = 4;                 // rows of a batch, of which one is summed and one on its way

// A lane a vector of columns; the tokens of the share one after the other.  32 768 x 3 584 bf16 with 11 937 rows written: 67 us
// (4.8 TB/s).  What a row waits for is its own load, so the list's next 64 tokens lie in the wavefront's lanes.
template <int DT, int GT, bool kAdd>
__global__ __launch_bounds__(kSumBlock) void sum_kernel(Sums s, const int32_t* __restrict__ keys, const int32_t* __restrict__ tokens,
                                                        const typename Elem<DT>::T* __restrict__ dy,
                                                        typename Elem<GT>::T* __restrict__ dtable) {
    constexpr int kVec = Elem<DT>::kVec;
    const int64_t begin = blockIdx.x * s.share, end = begin + s.share < s.n_tokens ? begin + s.share : s.n_tokens;
    int32_t key = keys[begin];
    if (key >= s.vocab) return;                                     // so are all behind it
    const int64_t want = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * kVec;
    const int64_t col = want < s.hidden - kVec ? want : s.hidden - kVec;
    const int skip = want >= s.hidden ? kVec : (int)(want - col);
    const int32_t next = end < s.n_tokens ? keys[end] : -1;
    bool from_front = begin > 0 && keys[begin - 1] == key;
    float acc[kVec] = {};
    const auto finish = [&](bool goes_on) {
        if (from_front || goes_on) {
            float* to = s.part + (blockIdx.x * 2ll + (from_front ? 0 : 1)) * s.hidden + col;
#pragma unroll
            for (int p = 0; p < kVec; p += 4)                       // overlapping entries are the same bits
                mrl::Vec<MRL_F32>::store(to + p, mrl::make_u32x4(__float_as_uint(acc[p]), __float_as_uint(acc[p + 1]),
                                                                 __float_as_uint(acc[p + 2]), __float_as_uint(acc[p + 3])));
        } else {
            put_columns<GT, kVec, kAdd>(dtable + key * s.hidden + col, acc, s.scale, skip);
        }
    };
    int32_t kn[kSumRows];
    u32x4 vn[kSumRows];
    for (int64_t block = begin; block < end; block += 64) {
        const int lane = threadIdx.x & 63, n = end - block < 64 ? (int)(end - block) : 64;
        const int64_t mine = block + (lane < n ? lane : n - 1);
        const int32_t lane_key = keys[mine], lane_token = tokens[mine];
        const auto request = [&](int p) {
#pragma unroll
            for (int i = 0; i < kSumRows; ++i) {
                const int at = p + i < n ? p + i : n - 1;
                kn[i] = __builtin_amdgcn_readlane(lane_key, at);
                vn[i] = mrl::Vec<DT>::load_nt(dy + (int64_t)__builtin_amdgcn_readlane(lane_token, at) * s.hidden + col);
            }
        };
        request(0);
        for (int p = 0; p < n; p += kSumRows) {
            int32_t k[kSumRows];
            u32x4 v[kSumRows];
#pragma unroll
            for (int i = 0; i < kSumRows; ++i) {
                k[i] = kn[i];
                v[i] = vn[i];
            }
            request(p + kSumRows);
#pragma unroll
            for (int i = 0; i < kSumRows; ++i) {
                if (p + i >= n) break;
                if (k[i] != key) {
                    finish(false);
                    key = k[i];
                    if (key >= s.vocab) return;
                    from_front = false;
#pragma unroll
                    for (int c = 0; c < kVec; ++c) acc[c] = 0.f;
                }
                float z[kVec];
                Elem<DT>::unpack(v[i], z);
#pragma unroll
                for (int c = 0; c < kVec; ++c) acc[c] += z[c];
            }
        }
    }
    finish(next == key);
}

constexpr int kJoinWaves = 8;
constexpr int kJoinShares = 2 * kJoinWaves; // shares of a workgroup for short runs
constexpr int kJoinShort = 16;              // shares of a run that a wavefront joins alone
constexpr int kJoinAhead = 16;              // parts that a wavefront has on its way
static_assert(kShares <= 64 * 64, "two steps find where a run ends");

// kCols columns of a lane: one, or four with one access for all of them.
template <int kCols>
struct Few {
    float v[kCols];
    static __device__ __forceinline__ Few load(const float* p) {
        Few f;
        if constexpr (kCols == 1) f.v[0] = *p;
        else mrl_vocab::Elem<MRL_F32>::unpack(mrl::Vec<MRL_F32>::load(p), f.v);
        return f;
    }
    __device__ __forceinline__ void add(const Few& o, bool counts) {
#pragma unroll
        for (int i = 0; i < kCols; ++i) v[i] += counts ? o.v[i] : 0.f;
    }
};

// Runs that cross shares.
struct Runs {
    const int32_t* keys;
    int64_t n_tokens, share;
    int32_t vocab;

    // whether the run of `key`, which is in a share in front of share g, goes on there
    __device__ __forceinline__ bool goes_on(int64_t g, int32_t key) const {
        const int64_t first = g * share;
        const int32_t k = keys[first < n_tokens ? first : 0];
        return (first < n_tokens) & (k == key);
    }
    // whether a run that begins in share g goes on in share g + n
    __device__ __forceinline__ bool begins(int64_t g, int n, int32_t* key) const {
        const bool last = (g + 1) * share >= n_tokens;
        const int32_t k = keys[last ? 0 : (g + 1) * share - 1], front = keys[g > 0 && !last ? g * share - 1 : 0];
        *key = k;
        return !last & (k < vocab) & (g == 0 || front != k) & goes_on(g + n, k);
    }
};

// A lane's columns of a row; a row that is not whole lanes ends with one that overlaps the one in front of it.
template <int GT, bool kAdd, int kCols>
struct JoinedColumns {
    const Sums& s;
    typename Elem<GT>::T* dtable;
    int64_t col;
    int skip;

    __device__ __forceinline__ JoinedColumns(const Sums& s, typename Elem<GT>::T* dtable, int64_t tile) : s(s), dtable(dtable) {
        const int64_t want = (tile * 64 + (threadIdx.x & 63)) * kCols;
        col = want < s.hidden - kCols ? want : s.hidden - kCols;
        skip = want >= s.hidden ? kCols : (int)(want - col);
    }
    __device__ __forceinline__ Few<kCols> part(int64_t share, int slot) const {
        return Few<kCols>::load(s.part + (share * 2 + slot) * s.hidden + col);
    }
    __device__ __forceinline__ void put(int32_t key, const Few<kCols>& sum) const {
        typename Elem<GT>::T* at = dtable + key * s.hidden + col;
#pragma unroll
        for (int i = 0; i < kCols; ++i)
            if (i >= skip) Elem<GT>::store(at + i, kAdd ? Elem<GT>::load(at + i) + sum.v[i] * s.scale : sum.v[i] * s.scale);
    }
};

// Long runs by workgroups of a tile of 64 columns and 64 shares, whose wavefronts take every kJoinWaves-th part; short ones by
// a wavefront each of workgroups of 64 kCols columns and kJoinShares shares.  Joins of 32 768 x 3 584 bf16: 10 us; of 49 152 x
// 2 048 added to fp32, most tokens of two kinds: 13.
template <int GT, bool kAdd, int kCols>
__global__ __launch_bounds__(kJoinWaves * 64) void join_kernel(Sums s, const int32_t* __restrict__ keys, int long_tiles,
                                                               int64_t long_groups, int tiles,
                                                               typename Elem<GT>::T* __restrict__ dtable) {
    __shared__ float lds[kJoinWaves][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Runs runs = {keys, s.n_tokens, s.share, s.vocab};
    int32_t my_key;
    if (blockIdx.x < long_groups) {
        const JoinedColumns<GT, kAdd, 1> row(s, dtable, blockIdx.x % long_tiles);
        const int64_t base = (int64_t)(blockIdx.x / long_tiles) * 64;
        for (uint64_t todo = __ballot(runs.begins(base + lane, kJoinShort, &my_key)); todo != 0; todo &= todo - 1) {   // the same in every wavefront
            const int from = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)todo) - 1);
            const int64_t share = base + from;
            const int32_t key = __shfl(my_key, from, 64);
            // the last share that it goes on in: in steps of 64 shares (64 of them are more than kShares), then one by one
            int64_t last = share + kJoinShort;
            last += 64 * __popcll(__ballot(runs.goes_on(last + 64 * (lane + 1), key)));
            last += __popcll(__ballot(runs.goes_on(last + 1 + lane, key)));
            Few<1> sum = {};
            for (int64_t g = share + wave; g <= last; g += kJoinWaves * kJoinAhead) {
                Few<1> v[kJoinAhead];
#pragma unroll
                for (int i = 0; i < kJoinAhead; ++i) {
                    const int64_t p = g + i * kJoinWaves <= last ? g + i * kJoinWaves : last;
                    v[i] = row.part(p, p == share ? 1 : 0);
                }
#pragma unroll
                for (int i = 0; i < kJoinAhead; ++i) sum.add(v[i], g + i * kJoinWaves <= last);
            }
            lds[wave][lane] = sum.v[0];
            __syncthreads();
            if (wave == 0) {
#pragma unroll
                for (int w = 1; w < kJoinWaves; ++w) sum.v[0] += lds[w][lane];
                row.put(key, sum);
            }
            __syncthreads();
        }
        return;
    }
    const int64_t group = blockIdx.x - long_groups;
    const JoinedColumns<GT, kAdd, kCols> row(s, dtable, group % tiles);
    // half a wavefront a share, a lane for each share that its run may go on in
    const int64_t base = group / tiles * kJoinShares + wave * 2;
    const int ahead = (lane & 31) + 1;
    const uint64_t on = __ballot(runs.begins(base + (lane >> 5), ahead, &my_key) & (ahead <= kJoinShort));
    for (int h = 0; h < 2; ++h) {
        const int n = __popc((uint32_t)(on >> (32 * h)));           // sorted: none of them but the first ones
        if (n == 0 || n == kJoinShort) continue;
        const int64_t share = base + h;
        Few<kCols> sum = row.part(share, 1);
        for (int i0 = 1; i0 <= n; i0 += 5) {
            Few<kCols> v[5];
#pragma unroll
            for (int i = 0; i < 5; ++i) v[i] = row.part(share + (i0 + i <= n ? i0 + i : n), 0);
#pragma unroll
            for (int i = 0; i < 5; ++i) sum.add(v[i], i0 + i <= n);
        }
        row.put(__builtin_amdgcn_readlane(my_key, 32 * h), sum);
    }
}

// ------------------------------------------------------------------------------------ host
template <int N>
struct Int {
    static constexpr int value = N;
};

int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t share_of(int64_t n_tokens, int64_t hidden) {
    // as many as 256 CUs hold at a time, 32 wavefronts each, with a vector of eight entries a lane and at most 8 to a share
    const int64_t waves = (hidden + 64 * 8 - 1) / (64 * 8), fit = 256 * (32 / (waves < 8 ? waves : 8));
    const int64_t most = fit < kShares ? fit : kShares;
    const int64_t s = (n_tokens + most - 1) / most;
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
    const int64_t share = share_of(n_tokens, hidden);
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
    MRL_REQUIRE(n_tokens < kMostTokens && vocab < 0x7fffffffLL && hidden <= MRL_NORM_MAX_HIDDEN, MRL_ERR_UNSUPPORTED,
                "%s: n_tokens=%lld vocab=%lld hidden=%lld (at most 2^26 - 1, 2^31 - 2 and %d)", fn, (long long)n_tokens,
                (long long)vocab, (long long)hidden, MRL_NORM_MAX_HIDDEN);
    MRL_REQUIRE(scale - scale == 0.f, MRL_ERR_INVALID_ARG, "%s: scale=%g", fn, (double)scale);
    MRL_REQUIRE(n_tokens == 0 || ids, MRL_ERR_INVALID_ARG, "%s: NULL ids", fn);
    MRL_REQUIRE(mrl::aligned(ids, mrl::int_dtype_bytes(ids_dtype)), MRL_ERR_MISALIGNED, "%s: misaligned ids", fn);
    return MRL_OK;
}

template <int DT, int GT, bool kAdd>
void launch_sums(const Sums& s, const int32_t* keys, const int32_t* tokens, const void* dy, void* dtable, hipStream_t stream) {
    using T = typename Elem<DT>::T;
    using G = typename Elem<GT>::T;
    const int64_t shares = (s.n_tokens + s.share - 1) / s.share, nv = (s.hidden + Elem<DT>::kVec - 1) / Elem<DT>::kVec;
    if (s.hidden < Elem<DT>::kVec) {
        hipLaunchKernelGGL((sum_narrow_kernel<DT, GT, kAdd>), dim3((unsigned)shares), dim3(64), 0, stream, s, keys, tokens,
                           (const T*)dy, (G*)dtable);
    } else {
        const int64_t block = nv < kSumBlock ? (nv + 63) / 64 * 64 : kSumBlock;
        hipLaunchKernelGGL((sum_kernel<DT, GT, kAdd>), dim3((unsigned)shares, (unsigned)((nv + block - 1) / block)),
                           dim3((unsigned)block), 0, stream, s, keys, tokens, (const T*)dy, (G*)dtable);
    }
    if (shares <= 1) return;
    const auto join = [&](auto cols) {
        constexpr int kCols = decltype(cols)::value;
        const int64_t tiles = (s.hidden + 64 * kCols - 1) / (64 * kCols), long_tiles = (s.hidden + 63) / 64;
        // runs of more shares than kJoinShort take as many, and one
        const int64_t long_groups = shares > kJoinShort ? long_tiles * ((shares + 63) / 64) : 0;
        const int64_t groups = long_groups + tiles * ((shares + kJoinShares - 1) / kJoinShares);
        hipLaunchKernelGGL((join_kernel<GT, kAdd, kCols>), dim3((unsigned)groups), dim3(kJoinWaves * 64), 0, stream, s, keys,
                           (int)long_tiles, long_groups, (int)tiles, (G*)dtable);
    };
    // 32 768 x 3 584 added: four columns 141 us, one 146; rows of fewer columns than a wavefront's four leave lanes idle (16 384 x 64
    // 34.5 either way)
    if (s.hidden >= 256) join(Int<4>());
    else join(Int<1>());
}

template <int DT, int GT>
void launch_sums(bool add, const Sums& s, const int32_t* keys, const int32_t* tokens, const void* dy, void* dtable,
                 hipStream_t stream) {
    if (add) launch_sums<DT, GT, true>(s, keys, tokens, dy, dtable, stream);
    else launch_sums<DT, GT, false>(s, keys, tokens, dy, dtable, stream);
}

// The part of a fill that launch `k` of `n` takes, in whole workgroups.
Fill fill_share(void* dtable, int64_t bytes, int k, int n) {
    const int64_t blocks = (bytes + kFillBytes - 1) / kFillBytes;
    const int64_t lo = blocks * k / n * kFillBytes, hi = k == n - 1 ? bytes : blocks * (k + 1) / n * kFillBytes;
    return {(char*)dtable + lo, hi - lo};
}

int64_t fill_blocks(const Fill& f) { return (f.bytes + kFillBytes - 1) / kFillBytes; }

template <int DT>
void launch_lookup(const void* ids, int ids_dtype, int64_t n_tokens, int64_t start, const void* table, int64_t vocab,
                   int64_t hidden, float scale, void* out, hipStream_t stream) {
    using T = typename Elem<DT>::T;
    if (hidden < Elem<DT>::kVec) {
        hipLaunchKernelGGL((lookup_narrow_kernel<DT>), dim3((unsigned)((n_tokens * hidden + kBlock - 1) / kBlock)), dim3(kBlock), 0,
                           stream, ids, ids_dtype, n_tokens, start, (const T*)table, vocab, (int)hidden, scale, (T*)out);
        return;
    }
    const int64_t waves = (hidden + Elem<DT>::kVec * 64 - 1) / (Elem<DT>::kVec * 64);       // of a row, a vector a lane
    const auto launch = [&](auto vecs) {
        constexpr int kVecs = decltype(vecs)::value;
        const dim3 grid((unsigned)((n_tokens + kBlock / 64 - 1) / (kBlock / 64)), (unsigned)((waves + kVecs - 1) / kVecs));
        hipLaunchKernelGGL((lookup_kernel<DT, kVecs>), grid, dim3(kBlock), 0, stream, ids, ids_dtype, n_tokens, start,
                           (const T*)table, vocab, (int)hidden, scale, (T*)out);
    };
    // Few tokens are spread over the chip.  Of many, a lane takes as many vectors as divide the row's, so that none reads over:
    // 32 768 x 3 584 bf16 57 us, one vector 76; 9 477 x 1 343 fp16 8.5, by four 9.8; 32 768 x 2 560 bf16 38.7, by four 40.9.
    if (n_tokens * waves <= 4096 || waves == 1) launch(Int<1>());
    else if (waves % 7 == 0) launch(Int<7>());
    else if (waves % 5 == 0) launch(Int<5>());
    else if (waves % 3 == 0) launch(Int<3>());
    else if (waves % 4 == 0) launch(Int<4>());
    else if (waves % 2 == 0) launch(Int<2>());
    else launch(Int<4>());
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
    hipStream_t s = mrl::as_stream(stream);
    for (int64_t t = 0; t < n_tokens; t += kLaunchTokens) {         // a second launch for the last three tokens of the most
        const int64_t n = n_tokens - t < kLaunchTokens ? n_tokens - t : kLaunchTokens;
        const void* some = (const char*)ids + t * mrl::int_dtype_bytes(ids_dtype);
        void* to = (char*)out + t * hidden * (int64_t)es;
        if (dtype == MRL_F32) launch_lookup<MRL_F32>(some, ids_dtype, n, vocab_start, table, vocab, hidden, scale, to, s);
        else if (dtype == MRL_BF16) launch_lookup<MRL_BF16>(some, ids_dtype, n, vocab_start, table, vocab, hidden, scale, to, s);
        else launch_lookup<MRL_F16>(some, ids_dtype, n, vocab_start, table, vocab, hidden, scale, to, s);
    }
    return mrl::check_launch(fn);
}

extern "C" int64_t mrl_embedding_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab, int64_t hidden) {
    if (n_tokens <= 0 || vocab <= 0 || hidden <= 0 || n_tokens >= kMostTokens || vocab >= 0x7fffffffLL ||
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
    const int64_t fill_bytes = accumulate ? 0 : vocab * hidden * (int64_t)mrl::float_dtype_bytes(dtable_dtype);
    MRL_REQUIRE(mrl::launch_fits(kSortGroups + fill_blocks({nullptr, fill_bytes}), kSortBlock), MRL_ERR_UNSUPPORTED,
                "%s: vocab=%lld hidden=%lld (a whole gradient of fewer than 2^36 - 2^21 bytes)", fn, (long long)vocab, (long long)hidden);
    if (n_tokens == 0) {
        if (fill_bytes == 0) return MRL_OK;
        const Fill f = {(char*)dtable, fill_bytes};
        hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)fill_blocks(f)), dim3(kSortBlock), 0, s, (const void*)nullptr, ids_dtype, 0, 0, 1,
                           SortPlan{1, 1, 0, kSortBlock}, (int32_t*)nullptr, f);
        return mrl::check_launch(fn);
    }
    const Workspace w = workspace_of(n_tokens, vocab, hidden);
    const SortPlan p = sort_plan(n_tokens, vocab);
    char* base = (char*)workspace;
    int32_t *keys[2], *tokens[2];
    for (int q = 0; q < 2; ++q) {
        keys[q] = (int32_t*)(base + w.keys[q]);
        tokens[q] = (int32_t*)(base + w.tokens[q]);
    }
    int32_t* counts = (int32_t*)(base + w.counts);
    const dim3 block(kSortBlock);
    if (n_tokens <= kFewTokens) {
        const Fill f = {(char*)dtable, fill_bytes};
        const int to = (p.passes - 1) & 1;
        hipLaunchKernelGGL(sort_few_kernel, dim3((unsigned)(1 + fill_blocks(f))), block, 0, s, ids, ids_dtype, (int)n_tokens, vocab_start, vocab, p,
                           keys[to], tokens[to], f);
    }
    const Fill f0 = fill_share(dtable, fill_bytes, 0, p.passes + 1);
    if (n_tokens > kFewTokens)
        hipLaunchKernelGGL(sort_count_kernel, dim3((unsigned)(p.groups + fill_blocks(f0))), block, 0, s, ids, ids_dtype, n_tokens,
                           vocab_start, vocab, p, counts, f0);
    for (int q = 0; n_tokens > kFewTokens && q < p.passes; ++q) {
        const int to = q & 1, from = to ^ 1;
        int32_t* here = counts + (int64_t)q * kSortGroups * kDigits;
        int32_t* next = q + 1 < p.passes ? here + (int64_t)kSortGroups * kDigits : nullptr;
        const Fill f = fill_share(dtable, fill_bytes, q + 1, p.passes + 1);
        const dim3 grid((unsigned)(p.groups + fill_blocks(f)));
        if (q == 0)
            hipLaunchKernelGGL((sort_pass_kernel<true>), grid, block, 0, s, ids, ids_dtype, n_tokens, vocab_start, vocab, p, q,
                               (const int32_t*)nullptr, (const int32_t*)nullptr, keys[to], tokens[to], here, next, f);
        else
            hipLaunchKernelGGL((sort_pass_kernel<false>), grid, block, 0, s, ids, ids_dtype, n_tokens, vocab_start, vocab, p, q,
                               keys[from], tokens[from], keys[to], tokens[to], here, next, f);
    }
    const int sorted = (p.passes - 1) & 1;
    const Sums sums = {(float*)(base + w.part), n_tokens, hidden, share_of(n_tokens, hidden), (int32_t)vocab, scale};
    const int32_t *sk = keys[sorted], *st = tokens[sorted];
    const bool add = accumulate != 0;
    if (dtype == MRL_F32) launch_sums<MRL_F32, MRL_F32>(add, sums, sk, st, dy, dtable, s);
    else if (dtype == MRL_BF16 && dtable_dtype == MRL_F32) launch_sums<MRL_BF16, MRL_F32>(add, sums, sk, st, dy, dtable, s);
    else if (dtype == MRL_BF16) launch_sums<MRL_BF16, MRL_BF16>(add, sums, sk, st, dy, dtable, s);
    else if (dtable_dtype == MRL_F32) launch_sums<MRL_F16, MRL_F32>(add, sums, sk, st, dy, dtable, s);
    else launch_sums<MRL_F16, MRL_F16>(add, sums, sk, st, dy, dtable, s);
    return mrl::check_launch(fn);
}
