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

struct Side {                               // queries or keys
    const void* x;
    void* out;                              // [tokens, heads, dim], dense
    int64_t outer, inner, head;             // strides of x
    int32_t heads, dim, start, units;       // units of a head: pairs, then what is copied
};

struct Args {
    Side side[2];
    const void* positions;
    int64_t pos_outer, pos_inner;
    const double* inv_freq;
    int64_t n_tokens, n_inner;
    int32_t part, pos_wide, interleaved, splits;
    float scale, sign;
};

// kN entries as they lie in memory.
template <typename T, int kN>
struct Pack {
    T v[kN];
};
template <typename T, int kN>
__device__ __forceinline__ Pack<T, kN> load_pack(const T* p) {
    Pack<T, kN> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int kN>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, kN>& v) {
    __builtin_memcpy(p, &v, sizeof(v));
}

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

// A wavefront takes a token, or one of `splits` shares of its units; the sines and cosines of the token's pairs are formed
// once, a pair a lane, and lie in LDS.
template <int DT, int kN>
__global__ __launch_bounds__(kBlock) void rotary_kernel(Args a) {
    using T = typename Elem<DT>::T;
    extern __shared__ float turns[];        // cosines, sines: a wavefront's
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, pairs = a.part / 2;
    const int64_t item = (int64_t)blockIdx.x * kWaves + wave;
    const int64_t token = item / a.splits;
    float* cosines = turns + wave * 2 * pairs;
    float* sines = cosines + pairs;
    const bool live = token < a.n_tokens;
    const int64_t outer = live ? token / a.n_inner : 0, inner = live ? token - outer * a.n_inner : 0;
    if (live) {
        const int64_t at = outer * a.pos_outer + inner * a.pos_inner;
        const double position = a.pos_wide ? (double)((const int64_t*)a.positions)[at] : (double)((const int32_t*)a.positions)[at];
        for (int i = lane; i < pairs; i += 64) {
            const float2 cs = turn_of(position * (a.inv_freq[i] * 0.15915494309189533577), a.scale, a.sign);
            cosines[i] = cs.x;
            sines[i] = cs.y;
        }
    }
    __syncthreads();
    if (!live) return;
    const int turned = pairs / kN;
    const int first = a.side[0].heads * a.side[0].units, all = first + a.side[1].heads * a.side[1].units;
    for (int idx = (int)(item - token * a.splits) * 64 + lane; idx < all; idx += 64 * a.splits) {
        const Side& s = a.side[idx >= first];
        const int at = idx >= first ? idx - first : idx;
        const int head = (int)((unsigned)at / (unsigned)s.units), unit = at - head * s.units;
        const T* x = (const T*)s.x + outer * s.outer + inner * s.inner + head * s.head;
        T* out = (T*)s.out + (token * s.heads + head) * s.dim;
        if (unit >= turned) {
            int j = (unit - turned) * kN;
            if (j >= s.start) j += a.part;
            store_pack<T, kN>(out + j, load_pack<T, kN>(x + j));
            continue;
        }
        const int one = s.start + (a.interleaved ? unit * 2 * kN : unit * kN), two = one + (a.interleaved ? kN : pairs);
        Pack<T, kN> va = load_pack<T, kN>(x + one), vb = load_pack<T, kN>(x + two);
        float z[2 * kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            z[i] = Elem<DT>::load(&va.v[i]);
            z[kN + i] = Elem<DT>::load(&vb.v[i]);
        }
        float y[2 * kN];
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const float c = cosines[unit * kN + i], sn = sines[unit * kN + i];
            const int p = a.interleaved ? 2 * i : i, q = a.interleaved ? 2 * i + 1 : kN + i;
            y[p] = z[p] * c - z[q] * sn;
            y[q] = z[q] * c + z[p] * sn;
        }
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            Elem<DT>::store(&va.v[i], y[i]);
            Elem<DT>::store(&vb.v[i], y[kN + i]);
        }
        store_pack<T, kN>(out + one, va);
        store_pack<T, kN>(out + two, vb);
    }
}

template <int DT, int kN>
void launch(Args a, hipStream_t stream) {
    const int turned = a.part / 2 / kN;
    int64_t units = 0;
    for (Side& s : a.side) {
        s.units = s.heads ? turned + (s.dim - a.part) / kN : 1;
        units += (int64_t)s.heads * s.units;
    }
    a.splits = 1;
    while (a.n_tokens * a.splits < 2048 && units > a.splits * 64) a.splits *= 2;
    const int64_t items = a.n_tokens * a.splits;
    hipLaunchKernelGGL((rotary_kernel<DT, kN>), dim3((unsigned)((items + kWaves - 1) / kWaves)), dim3(kBlock),
                       kWaves * a.part * sizeof(float), stream, a);
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
    a.n_tokens = n_outer * n_inner;
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
                     (int32_t)s->start, 0};
    }
    if (a.n_tokens == 0) return MRL_OK;
    MRL_REQUIRE(positions && inv_freq, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(mrl::aligned(positions, ps) && mrl::aligned(inv_freq, 8), MRL_ERR_MISALIGNED, "%s: misaligned buffer", fn);
    a.positions = positions;
    a.pos_outer = pos_outer;
    a.pos_inner = pos_inner;
    a.inv_freq = inv_freq;
    a.n_inner = n_inner;
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
