// Rotary positions of queries and keys for gfx950.
//
//   (a, b) -> scale (a cos t - b sin t, b cos t + a sin t),  t = position * inv_freq[i],  i = 0 .. part/2 - 1
//   pairs: entries i and i + part/2 of the turned part of a head, or 2i and 2i + 1 (interleaved); the gradient turns back, by -t
//
// The angle is formed in 64 bits, in turns, and its whole turns are taken off there: at position 2^20 fp32 would be off by 0.06.
// What is left of it is at most an eighth of a turn off a quarter; sine and cosine of that are their Taylor series in fp32 (terms to x^9 and
// x^10: what is cut off is below 3e-9).  Entries are turned in fp32 and rounded once.
#include "mrl_internal.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / 64;
// Units of a lane on their way at a time (us, two / four: 32 768 tokens of 32 bf16 heads of 128, there and back, 188 / 178).
constexpr int kBatch = 4;
// Bytes read and written that the memory-side cache holds; more go past the caches (us, through / past: the same 196 / 178, 9 477 tokens
// of 17 fp16 heads of 192 24.7 / 32.6).
constexpr int64_t kCached = 256 << 20;

struct Side {                               // queries or keys
    const void* x;
    void* out;                              // [tokens, heads, dim], dense
    int64_t outer, inner, head;             // strides of x
    int32_t heads, dim, start;
    int32_t units, copied;                  // units of a head: pairs, then what is copied, so many entries each
};

struct Args {
    Side side[2];
    const void* positions;
    int64_t pos_outer, pos_inner;
    const double* inv_freq;
    int32_t n_tokens, n_inner, part, pos_wide, interleaved, splits;
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

// A wavefront takes a token, or one of `splits` shares of its units.  A unit is kN pairs, or two vectors of kN entries (one, where
// the layout has it so) that are copied.  Four units a lane are on their way while the sines and cosines of the token's pairs are
// formed, once, a pair a lane, and put into LDS.
template <int DT, int kN, bool kInterleaved, bool kStream>
__global__ __launch_bounds__(kBlock) void rotary_kernel(Args a) {
    using T = typename Elem<DT>::T;
    extern __shared__ float4 turns[];       // cosines, sines: a wavefront's
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pairs = a.part / 2;
    const uint32_t item = blockIdx.x * kWaves + wave, token = item / a.splits;
    if (token >= (uint32_t)a.n_tokens) return;          // no barrier follows
    float* cosines = (float*)turns + wave * 2 * pairs;
    float* sines = cosines + pairs;
    const uint32_t outer = token / (uint32_t)a.n_inner, inner = token - outer * (uint32_t)a.n_inner;
    // what the angles take is requested in front of the entries: a wait for a load is one for those in front of it
    const int64_t place = outer * a.pos_outer + inner * a.pos_inner;
    const double position = a.pos_wide ? (double)((const int64_t*)a.positions)[place] : (double)((const int32_t*)a.positions)[place];
    const double frequency = a.inv_freq[lane < pairs ? lane : 0];
    const T* from0 = (const T*)a.side[0].x + ((int64_t)outer * a.side[0].outer + (int64_t)inner * a.side[0].inner);
    const T* from1 = (const T*)a.side[1].x + ((int64_t)outer * a.side[1].outer + (int64_t)inner * a.side[1].inner);
    T* to0 = (T*)a.side[0].out + (int64_t)token * (a.side[0].heads * a.side[0].dim);
    T* to1 = (T*)a.side[1].out + (int64_t)token * (a.side[1].heads * a.side[1].dim);
    const int turned = pairs / kN;
    const int first = a.side[0].heads * a.side[0].units, all = first + a.side[1].heads * a.side[1].units;
    const int step = 64 * a.splits;
    Pack<DT, kN> va[kBatch], vb[kBatch];
    int at[kBatch], two[kBatch], unit[kBatch];
    const auto request = [&](int base) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const int wanted = base + q * step + lane, idx = wanted < all ? wanted : all - 1;
            const bool second = idx >= first;
            const int n = second ? idx - first : idx, units = second ? a.side[1].units : a.side[0].units;
            const int head = (int)((unsigned)n / (unsigned)units), start = second ? a.side[1].start : a.side[0].start;
            unit[q] = n - head * units;
            const bool turn = unit[q] < turned;
            const int copied = second ? a.side[1].copied : a.side[0].copied;
            int copy = (unit[q] - turned) * copied;
            copy += copy >= start ? a.part : 0;
            const int one = turn ? start + unit[q] * (kInterleaved ? 2 * kN : kN) : copy;
            two[q] = turn ? (kInterleaved ? kN : pairs) : copied - kN;
            const T* x = (second ? from1 : from0) + head * (second ? a.side[1].head : a.side[0].head) + one;
            at[q] = head * (second ? a.side[1].dim : a.side[0].dim) + one;
            va[q].template load<kStream>(x);
            vb[q].template load<kStream>(x + two[q]);
        }
    };
    int base = (int)(item - token * a.splits) * 64;
    if (base >= all) return;
    request(base);
    for (int i = lane; i < pairs; i += 64) {
        const double f = i < 64 ? frequency : a.inv_freq[i];
        const float2 cs = turn_of(position * (f * 0.15915494309189533577), a.scale, a.sign);
        cosines[i] = cs.x;
        sines[i] = cs.y;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    while (true) {
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
            const bool turn = unit[q] < turned;
            const int pair = turn ? unit[q] * kN : 0;
            float z[2 * kN], y[2 * kN], c[kN], sn[kN], za[kN], zb[kN];
            if constexpr (kN >= 4) {
#pragma unroll
                for (int i = 0; i < kN; i += 4) {
                    *(float4*)(c + i) = *(const float4*)(cosines + pair + i);
                    *(float4*)(sn + i) = *(const float4*)(sines + pair + i);
                }
            } else {
#pragma unroll
                for (int i = 0; i < kN; ++i) {
                    c[i] = cosines[pair + i];
                    sn[i] = sines[pair + i];
                }
            }
            va[q].unpack(za);
            vb[q].unpack(zb);
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                z[i] = za[i];
                z[kN + i] = zb[i];
            }
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int p = kInterleaved ? 2 * i : i, r = kInterleaved ? 2 * i + 1 : kN + i;
                y[p] = z[p] * c[i] - z[r] * sn[i];
                y[r] = z[r] * c[i] + z[p] * sn[i];
            }
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                za[i] = y[i];
                zb[i] = y[kN + i];
            }
            Pack<DT, kN> ya, yb;
            ya.pack(za);
            yb.pack(zb);
            ya.v = turn ? ya.v : va[q].v;   // what is copied keeps its bits
            yb.v = turn ? yb.v : vb[q].v;
            const int idx = base + q * step + lane;
            if (idx < all) {
                T* out = (idx >= first ? to1 : to0) + at[q];
                ya.template store<kStream>(out);
                yb.template store<kStream>(out + two[q]);
            }
        }
        base += kBatch * step;
        if (base >= all) return;
        request(base);
    }
}

template <int DT, int kN>
void launch(Args a, hipStream_t stream) {
    const int turned = a.part / 2 / kN;
    int64_t units = 0;
    for (Side& s : a.side) {
        s.copied = s.start % (2 * kN) == 0 && (s.dim - a.part) % (2 * kN) == 0 ? 2 * kN : kN;
        s.units = s.heads ? turned + (s.dim - a.part) / s.copied : 1;
        units += (int64_t)s.heads * s.units;
    }
    a.splits = 1;
    while (a.n_tokens * a.splits < 2048 && units > a.splits * 64) a.splits *= 2;
    const unsigned groups = (unsigned)((a.n_tokens * a.splits + kWaves - 1) / kWaves);
    const size_t lds = kWaves * a.part * sizeof(float);
    int64_t entries = 0;
    for (const Side& s : a.side) entries += (int64_t)a.n_tokens * s.heads * s.dim;
    const auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3(groups), dim3(kBlock), lds, stream, a); };
    if (2 * entries * (int64_t)sizeof(typename Elem<DT>::T) <= kCached) {
        if (a.interleaved) go(rotary_kernel<DT, kN, true, false>);
        else go(rotary_kernel<DT, kN, false, false>);
    } else {
        if (a.interleaved) go(rotary_kernel<DT, kN, true, true>);
        else go(rotary_kernel<DT, kN, false, true>);
    }
}

template <int DT>
void dispatch(const Args& a, hipStream_t stream) {
    constexpr int kMost = Elem<DT>::kVec;
    // whole vectors of the turned halves, of what is copied in front of them and behind
    int fits = a.part / 2;
    for (const Side& s : a.side)
        if (s.heads) fits |= s.start | (s.dim - a.part);
    if (fits % kMost == 0) return launch<DT, kMost>(a, stream);
    if (fits % 4 == 0) return launch<DT, 4>(a, stream);
    if (fits % 2 == 0) return launch<DT, 2>(a, stream);
    launch<DT, 1>(a, stream);
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
                     (int32_t)s->start, 0, 0};
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
    if (dtype == MRL_F32) dispatch<MRL_F32>(a, s);
    else if (dtype == MRL_BF16) dispatch<MRL_BF16>(a, s);
    else dispatch<MRL_F16>(a, s);
    return mrl::check_launch(fn);
}
