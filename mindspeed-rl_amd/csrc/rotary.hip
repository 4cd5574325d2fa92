// Rotary positions of queries and keys for gfx950.
//
//   (a, b) -> scale (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i],  i = 0 .. part/2 - 1
//   pairs: entries i and i + part/2 of the turned part of a head, or 2i and 2i + 1 (interleaved); the gradient turns back, by -t
//
// The angle is formed in 64 bits, in turns, and its whole turns are taken off there: at position 2^20 fp32 would be off by 0.06.
// What is left of it is at most an eighth of a turn off a quarter; sine and cosine of that are their Taylor series in fp32 (terms to x^9 and
// x^10: what is cut off is below 3e-9).  Entries are turned in fp32 and rounded once.
//
// Bound by memory: 32 768 tokens of 32 bf16 heads of 128 (537 MB) 90 us (6.0 TB/s), either layout; heads that end inside lines 4.6 to
// 5.5 TB/s (28 and 4 bf16 heads of 72 56 us; the counters show every byte written to memory once, so it is not lines that go there twice), of 66
// 3.3 (47 us).  65 536 tokens of 2 heads of 64: 10 us.  (Here and below: calls that follow each other in a replayed graph.)
#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256, kBlockLog = 8;
// Units of a lane on their way at a time (us, two / four: 32 768 tokens of 32 bf16 heads of 128, there and back, 188 / 178).
constexpr int kUnits = 4;
// Bytes read and written that the memory-side cache holds; more go past the caches, where all stretches are whole lines (us, through /
// past: 32 768 tokens of 32 bf16 heads of 128 98.8 / 89.6, of 64 fp32 98.0 / 88.1; of 128 with 64 turned 98.0 / 105.9, of 96 75.9 / 89.7; 9 477 of 17
// fp16 heads of 192, 124 MB, 24.7 / 32.6).
constexpr int64_t kCached = 256 << 20;

struct Side {                               // queries or keys
    const void* x;
    void* out;                              // [tokens, heads, dim], dense
    int64_t outer, inner, head;             // strides of x
    int32_t heads, dim, start, units;       // units of a head: turned ones, then copied ones
    int32_t front, copied;                  // vectors in front of the turned part, and of all that is copied
};

struct Args {
    Side side[2];
    const void* positions;
    int64_t pos_outer, pos_inner;
    const double* inv_freq;
    int32_t n_tokens, n_inner, part, turned, pos_wide, interleaved, splits, lanes_log;
    float scale, sign;
};

// 2, 4, 8 or 16 bytes at any entry's address.
template <int kBytes>
struct Bits {
    typedef uint32_t V __attribute__((ext_vector_type(kBytes / 4)));
    typedef V At __attribute__((aligned(2)));
};
template <>
struct Bits<2> {
    typedef uint16_t V, At;
};
template <>
struct Bits<4> {
    typedef uint32_t V;
    typedef uint32_t At __attribute__((aligned(2)));
};

// kN entries as they lie in memory.
template <int DT, int kN>
struct Pack {
    using E = Elem<DT>;
    static constexpr int kBytes = kN * sizeof(typename E::T);
    using B = Bits<kBytes>;
    typename B::V v;
    template <bool kStream>
    __device__ __forceinline__ void load(const typename E::T* p) {
        const typename B::At* from = (const typename B::At*)p;
        v = kStream ? __builtin_nontemporal_load(from) : *from;
    }
    template <bool kStream>
    __device__ __forceinline__ void store(typename E::T* p) const {
        typename B::At* to = (typename B::At*)p;
        if (kStream) __builtin_nontemporal_store(v, to);
        else *to = v;
    }
    __device__ __forceinline__ void unpack(float (&z)[kN]) const {
        u32x4 w = mrl::make_u32x4(0u, 0u, 0u, 0u);
        if constexpr (kBytes <= 4) {
            w[0] = v;
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) w[i] = v[i];
        }
        float t[E::kVec];
        E::unpack(w, t);
#pragma unroll
        for (int i = 0; i < kN; ++i) z[i] = t[i];
    }
    __device__ __forceinline__ void pack(const float (&z)[kN]) {
        float t[E::kVec] = {};
#pragma unroll
        for (int i = 0; i < kN; ++i) t[i] = z[i];
        const u32x4 w = E::pack(t);
        if constexpr (kBytes <= 4) {
            v = (typename B::V)w[0];
        } else {
#pragma unroll
            for (int i = 0; i < kBytes / 4; ++i) v[i] = w[i];
        }
    }
};

// scale * cos and sign * scale * sin of 2 pi t.
__device__ __forceinline__ float2 turn_of(double t, float scale, float sign) {
    t = 4.0 * (t - rint(t));
    const double n = rint(t);
    const float x = (float)(t - n) * 1.57079632679489662f, x2 = x * x;
    const float s = x + x * x2 * (-1.f / 6 + x2 * (1.f / 120 + x2 * (-1.f / 5040 + x2 * (1.f / 362880))));
    const float c = 1.f + x2 * (-0.5f + x2 * (1.f / 24 + x2 * (-1.f / 720 + x2 * (1.f / 40320 + x2 * (-1.f / 3628800)))));
    const int q = (int)n & 3;               // quarters
    const float cq = q & 1 ? s : c, sq = q & 1 ? c : s;
    return make_float2(q == 1 || q == 2 ? -cq * scale : cq * scale, (q >= 2 ? -sq : sq) * sign * scale);
}

// A unit is two vectors of kN entries of a head.  Halves: the same place in both.  Interleaved: a vector of each half of the
// vectors, so that what the lanes take at a time lies together.  Copied entries the same.  The last vector of a stretch that is not whole
// vectors ends where the stretch ends and overlaps the one in front of it: what lies in both is written twice with the same bits.
//
// A token's units are dealt to a wavefront, four to a lane on their way at a time (kBatch; or to `splits` wavefronts, of few tokens), or, where
// there are no more than 64, one to each of 2^lanes_log lanes.  While they are on their way the sines and cosines of the token's pairs
// are formed, once, and put into LDS.
template <int DT, int kN, bool kInterleaved, bool kStream, int kBatch>
__global__ __launch_bounds__(kBlock) void rotary_kernel(Args a) {
    using T = typename Elem<DT>::T;
    constexpr bool kWave = kBatch > 1, kSide = kInterleaved && kN > 1;     // pairs lie side by side in a vector
    extern __shared__ float2 turns[];       // (cosine, sine) of a token's pairs, after one another
    const int pairs = a.part / 2;
    int lane, lanes, slot, base;
    uint32_t token;
    if (kWave) {
        const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), item = blockIdx.x * (kBlock / 64) + wave;
        lane = threadIdx.x & 63;
        lanes = 64;
        slot = wave;
        token = item / (uint32_t)a.splits;
        base = (int)(item - token * a.splits) * 64;
    } else {
        lanes = 1 << a.lanes_log;
        lane = threadIdx.x & (lanes - 1);
        slot = threadIdx.x >> a.lanes_log;
        token = (blockIdx.x << (kBlockLog - a.lanes_log)) + slot;
        base = 0;
    }
    if (token >= (uint32_t)a.n_tokens) return;          // no barrier follows
    float2* turn_at = turns + slot * pairs;
    const uint32_t outer = token / (uint32_t)a.n_inner, inner = token - outer * (uint32_t)a.n_inner;
    // what the angles take is requested in front of the entries: a wait for a load is one for those in front of it
    const int64_t place = outer * a.pos_outer + inner * a.pos_inner;
    const double position = a.pos_wide ? (double)((const int64_t*)a.positions)[place] : (double)((const int32_t*)a.positions)[place];
    const double frequency = a.inv_freq[lane < pairs ? lane : 0];
    const T* from0 = (const T*)a.side[0].x + ((int64_t)outer * a.side[0].outer + (int64_t)inner * a.side[0].inner);
    const T* from1 = (const T*)a.side[1].x + ((int64_t)outer * a.side[1].outer + (int64_t)inner * a.side[1].inner);
    T* to0 = (T*)a.side[0].out + (int64_t)token * (a.side[0].heads * a.side[0].dim);
    T* to1 = (T*)a.side[1].out + (int64_t)token * (a.side[1].heads * a.side[1].dim);
    const int first = a.side[0].heads * a.side[0].units, all = first + a.side[1].heads * a.side[1].units;
    const int step = 64 * a.splits;
    Pack<DT, kN> va[kBatch], vb[kBatch];
    int one[kBatch], two[kBatch], pair[kBatch], pair2[kBatch];              // pair < 0: copied
    const auto request = [&](int base) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int wanted = base + q * step + lane, idx = wanted < all ? wanted : all - 1;
            const bool second = idx >= first;
            const int n = second ? idx - first : idx, units = second ? a.side[1].units : a.side[0].units;
            const int head = (int)((unsigned)n / (unsigned)units), unit = n - head * units;
            const int dim = second ? a.side[1].dim : a.side[0].dim, start = second ? a.side[1].start : a.side[0].start;
            const int front = second ? a.side[1].front : a.side[0].front, copied = second ? a.side[1].copied : a.side[0].copied;
            const bool turn = unit < a.turned;
            int t1, t2;
            if (kSide) {
                t1 = min(unit * kN, a.part - kN);
                t2 = min((unit + a.turned) * kN, a.part - kN);
                pair[q] = t1 >> 1;
                pair2[q] = t2 >> 1;
            } else {
                const int at = min(unit * kN, pairs - kN);
                t1 = kInterleaved ? 2 * at : at;
                t2 = kInterleaved ? 2 * at + 1 : at + pairs;
                pair[q] = pair2[q] = at;
            }
            const int c1 = unit - a.turned, c2 = min(c1 + (copied + 1) / 2, copied - 1), behind = dim - kN;
            const auto copy = [&](int c) { return c < front ? min(c * kN, start - kN) : min(start + a.part + (c - front) * kN, behind); };
            t1 = turn ? start + t1 : copy(c1);
            t2 = turn ? start + t2 : copy(c2);
            pair[q] = turn ? pair[q] : -1;
            const T* x = (second ? from1 : from0) + head * (second ? a.side[1].head : a.side[0].head);
            one[q] = head * dim + t1;
            two[q] = head * dim + t2;
            va[q].template load<kStream>(x + t1);
            vb[q].template load<kStream>(x + t2);
        }
    };
    if (base >= all) return;
    request(base);
    for (int i = lane; i < pairs; i += lanes) {
        const double f = i < lanes ? frequency : a.inv_freq[i];
        turn_at[i] = turn_of(position * (f * 0.15915494309189533577), a.scale, a.sign);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    while (true) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const bool turn = pair[q] >= 0;
            const float2* t1 = turn_at + (turn ? pair[q] : 0);
            const float2* t2 = turn_at + (turn ? pair2[q] : 0);
            float za[kN], zb[kN], ya[kN], yb[kN];
            va[q].unpack(za);
            vb[q].unpack(zb);
            if constexpr (kSide) {
#pragma unroll
                for (int i = 0; i < kN; i += 2) {
                    const float2 s = t1[i / 2], u = t2[i / 2];
                    ya[i] = za[i] * s.x - za[i + 1] * s.y;
                    ya[i + 1] = za[i + 1] * s.x + za[i] * s.y;
                    yb[i] = zb[i] * u.x - zb[i + 1] * u.y;
                    yb[i + 1] = zb[i + 1] * u.x + zb[i] * u.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < kN; ++i) {
                    const float2 s = t1[i];
                    ya[i] = za[i] * s.x - zb[i] * s.y;
                    yb[i] = zb[i] * s.x + za[i] * s.y;
                }
            }
            Pack<DT, kN> pa, pb;
            pa.pack(ya);
            pb.pack(yb);
            pa.v = turn ? pa.v : va[q].v;   // what is copied keeps its bits
            pb.v = turn ? pb.v : vb[q].v;
            const int idx = base + q * step + lane;
            if (idx < all) {
                T* out = idx >= first ? to1 : to0;
                pa.template store<kStream>(out + one[q]);
                pb.template store<kStream>(out + two[q]);
            }
        }
        base += kBatch * step;
        if (base >= all) return;
        request(base);
    }
}

int check_grid(int64_t groups, const Args& a) {
    MRL_REQUIRE(mrl::launch_fits(groups, kBlock), MRL_ERR_UNSUPPORTED,
                "mrl_rotary: %d tokens (2^32 threads hold fewer, a wavefront for one of more than 32 units)", a.n_tokens);
    return MRL_OK;
}

template <int DT, int kN, bool kInterleaved>
int launch(Args a, hipStream_t stream) {
    constexpr bool kSide = kInterleaved && kN > 1;
    const auto vectors = [](int n) { return (n + kN - 1) / kN; };
    a.turned = kSide ? (vectors(a.part) + 1) / 2 : vectors(a.part / 2);
    int64_t units = 0, entries = 0;
    for (Side& s : a.side) {
        s.front = vectors(s.start);
        s.copied = s.front + vectors(s.dim - a.part - s.start);
        s.units = s.heads ? a.turned + (s.copied + 1) / 2 : 1;
        units += (int64_t)s.heads * s.units;
        entries += (int64_t)a.n_tokens * s.heads * s.dim;
    }
    constexpr int kLine = 128 / sizeof(typename Elem<DT>::T);
    bool past = 2 * entries * (int64_t)sizeof(typename Elem<DT>::T) > kCached && a.part % (2 * kLine) == 0;
    for (const Side& s : a.side) past = past && s.dim % kLine == 0 && s.start % kLine == 0;
    a.splits = 1;
    // several tokens a wavefront (us, a token / several: 65 536 tokens of 2 bf16 heads of 64 46.7 / 9.8, of 8 of 128 59.1 / 45.9)
    if (units <= 64) {
        while ((1 << a.lanes_log) < units) ++a.lanes_log;
        const int teams = kBlock >> a.lanes_log;
        const int64_t groups = ((int64_t)a.n_tokens + teams - 1) / teams;
        const int rc = check_grid(groups, a);
        if (rc != MRL_OK) return rc;
        const dim3 grid((unsigned)groups);
        const size_t lds = (size_t)teams * (a.part / 2) * sizeof(float2);
        if (past) hipLaunchKernelGGL((rotary_kernel<DT, kN, kInterleaved, true, 1>), grid, dim3(kBlock), lds, stream, a);
        else hipLaunchKernelGGL((rotary_kernel<DT, kN, kInterleaved, false, 1>), grid, dim3(kBlock), lds, stream, a);
        return MRL_OK;
    }
    // few tokens by several wavefronts each (us, one / several: 64 tokens of 64 bf16 heads of 128 6.1 / 3.6, 256 of 32 4.5 / 3.8, 1 024 5.8 / 5.6)
    while (a.n_tokens * a.splits < 2048 && units > a.splits * 64) a.splits *= 2;
    const int waves = kBlock / 64;
    const int64_t groups = ((int64_t)a.n_tokens * a.splits + waves - 1) / waves;
    const int rc = check_grid(groups, a);
    if (rc != MRL_OK) return rc;
    const dim3 grid((unsigned)groups);
    const size_t lds = (size_t)waves * (a.part / 2) * sizeof(float2);
    if (past) hipLaunchKernelGGL((rotary_kernel<DT, kN, kInterleaved, true, kUnits>), grid, dim3(kBlock), lds, stream, a);
    else hipLaunchKernelGGL((rotary_kernel<DT, kN, kInterleaved, false, kUnits>), grid, dim3(kBlock), lds, stream, a);
    return MRL_OK;
}

// The widest vectors that no stretch of a head is shorter than: a half of the turned part (interleaved: the part), what lies
// in front of it and behind.
template <int DT, int kN>
int launch_widest(const Args& a, hipStream_t stream) {
    bool fits = (a.interleaved ? a.part : a.part / 2) >= kN;
    for (const Side& s : a.side) {
        const int behind = s.dim - a.part - s.start;
        if (s.heads) fits = fits && (s.start == 0 || s.start >= kN) && (behind == 0 || behind >= kN);
    }
    if constexpr (kN > 1) {
        if (!fits) return launch_widest<DT, kN / 2>(a, stream);
    }
    return a.interleaved ? launch<DT, kN, true>(a, stream) : launch<DT, kN, false>(a, stream);
}

}  // namespace

extern "C" int mrl_rotary(const mrl_rotary_side* q, const mrl_rotary_side* k, int dtype, const void* positions, int positions_dtype,
                          int64_t pos_outer, int64_t pos_inner, int64_t n_outer, int64_t n_inner, const double* inv_freq,
                          int64_t part, int interleaved, float scale, int back, void* stream) {
    const char* fn = "mrl_rotary";
    const size_t es = mrl::float_dtype_bytes(dtype);
    MRL_REQUIRE(es != 0, MRL_ERR_UNSUPPORTED, "%s: dtype %d (want F32, BF16 or F16)", fn, dtype);
    const size_t ps = mrl::int_dtype_bytes(positions_dtype);
    MRL_REQUIRE(ps != 0, MRL_ERR_UNSUPPORTED, "%s: positions dtype %d (want I32 or I64)", fn, positions_dtype);
    MRL_REQUIRE(q, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(n_outer >= 0 && n_inner >= 0, MRL_ERR_INVALID_ARG, "%s: n_outer=%lld n_inner=%lld", fn, (long long)n_outer, (long long)n_inner);
    MRL_REQUIRE(part >= 2 && part % 2 == 0, MRL_ERR_INVALID_ARG, "%s: part=%lld (want an even number from 2 on)", fn, (long long)part);
    MRL_REQUIRE(part <= MRL_ROTARY_MAX_PART, MRL_ERR_UNSUPPORTED, "%s: part=%lld (at most %d)", fn, (long long)part, MRL_ROTARY_MAX_PART);
    MRL_REQUIRE(n_outer == 0 || n_inner <= ((1LL << 26) - 1) / n_outer, MRL_ERR_UNSUPPORTED, "%s: %lld x %lld tokens (fewer than 2^26)",
                fn, (long long)n_outer, (long long)n_inner);
    MRL_REQUIRE(scale - scale == 0.f, MRL_ERR_INVALID_ARG, "%s: scale=%g", fn, (double)scale);
    Args a = {};
    a.n_tokens = (int32_t)(n_outer * n_inner);
    for (int i = 0; i < 2; ++i) {
        const mrl_rotary_side* s = i ? k : q;
        if (!s) continue;
        MRL_REQUIRE(s->heads >= 1 && s->dim >= part && s->start >= 0 && s->start <= s->dim - part, MRL_ERR_INVALID_ARG,
                    "%s: %lld heads of %lld entries, the part from %lld on", fn, (long long)s->heads, (long long)s->dim, (long long)s->start);
        MRL_REQUIRE(s->dim <= MRL_ROTARY_MAX_ROW / s->heads, MRL_ERR_UNSUPPORTED, "%s: %lld heads of %lld entries (at most %d in a token)",
                    fn, (long long)s->heads, (long long)s->dim, MRL_ROTARY_MAX_ROW);
        MRL_REQUIRE(a.n_tokens == 0 || (s->x && s->out), MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
        MRL_REQUIRE(mrl::aligned(s->x, es) && mrl::aligned(s->out, es), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
        a.side[i] = {s->x, s->out, s->stride_outer, s->stride_inner, s->stride_head, (int32_t)s->heads, (int32_t)s->dim,
                     (int32_t)s->start, 0, 0, 0};
    }
    if (a.n_tokens == 0) return MRL_OK;
    MRL_REQUIRE(positions && inv_freq, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(mrl::aligned(positions, ps) && mrl::aligned(inv_freq, 8), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    a.positions = positions;
    a.pos_outer = pos_outer;
    a.pos_inner = pos_inner;
    a.inv_freq = inv_freq;
    a.n_inner = (int32_t)n_inner;
    a.part = (int32_t)part;
    a.pos_wide = positions_dtype == MRL_I64;
    a.interleaved = interleaved != 0;
    a.scale = scale;
    a.sign = back ? -1.f : 1.f;
    hipStream_t s = mrl::as_stream(stream);
    const int rc = dtype == MRL_F32 ? launch_widest<MRL_F32, 4>(a, s)
                   : dtype == MRL_BF16 ? launch_widest<MRL_BF16, 8>(a, s)
                                       : launch_widest<MRL_F16, 8>(a, s);
    return rc != MRL_OK ? rc : mrl::check_launch(fn);
}
