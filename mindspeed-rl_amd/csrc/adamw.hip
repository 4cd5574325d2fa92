// A step of AdamW over a list of tensors for gfx950, clipped on the way, with moments in 32 or in 8 bits.
//
//   g' = g min(1, max_norm / (norm + 1e-6)),  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - m / (sqrt(v) / sqrt(1 - b2^t) + eps) lr / (1 - b1^t)
//
// Everything is held in fp32 (the powers of the betas in 64 bits) and the operations that lead to the moments are rounded one by
// one, so that their bits do not depend on how the compiler joins them.  fp32 main weights are where there are any what p is, and the
// parameter is p rounded.
//
// 8 bits: 128 entries of a tensor in a row share an fp32 scale s = max(max |x| * (1/448), 2^-126), x being m and sqrt(v) (whose
// range is half of v's in its logarithm), and are held as e4m3 codes of x / s (x times 1 / s, two roundings).  Moments change by less than half a step of such a
// code from one update to the next, and rounding to the nearest would leave them where they are, so a value goes up or down by a
// dither u in [0, 1), floor(|x / s| / step + u): the mean of what is held, m or sqrt(v), moves as it should.  v is the square of what is
// held, and every update adds the dither's variance to it: with gradients that differ from update to update it is too large by about half of a code's relative step (independent
// normal ones: 2.5 % at b2 = 0.95, 5 % at 0.999), and sqrt(v) spreads by such a step.  u is the hash of the step's number and
// the entry's place, the same for both moments; the same call gives the same bits.  A sqrt(v) above zero keeps at least
// the least code, so that no m is divided by eps alone because its v was lost.
#include <algorithm>
#include <memory>
#include <new>

#include "lane_ops.h"
#include "mrl_internal.h"
#include "vector_access.h"
#include "vocab_common.h"

namespace {

using mrl_vocab::Elem;

// A lane takes four entries, so that what a wavefront reads or writes of an fp32 tensor at a time lies together, and a workgroup
// one chunk, after which it ends: the memory serves small workgroups that come and go best.  All of it goes past the caches.  us,
// 719 M bf16 parameters with fp32 gradients, main weights and moments (21.6 GB, 6.1 TB/s) by 64, 128, 256 threads 3 655, 3 560, 3 813;
// 449 M with bf16 gradients and moments in 8 bits (7.2 GB, 6.2 TB/s) 1 187, 1 173, 1 171, 42 M of fp32 that lie off the lines 157, 136, 126;
// eight entries a lane 4 226 (1 344), through the caches 4 001 (1 300).
constexpr int kUnit = 4;                    // entries of a lane: 32 lanes a block of 128
constexpr int block_of(bool small) { return small ? 256 : 128; }
constexpr int chunk_of(bool small) { return block_of(small) * kUnit; }     // entries of a workgroup
constexpr int kTable = 54;                  // tensors of a launch: 4 KB of arguments
constexpr int64_t kMostGroups = (1LL << 24) - 1;    // of a launch, which holds fewer than 2^32 threads
constexpr float kMost = 448.f;              // of e4m3
constexpr float kLeastCode = 0.001953125f;  // 2^-9
constexpr float kLeastScale = 1.17549435e-38f;      // 2^-126

struct Part {
    void* param;
    const void* grad;
    float* master;
    void *m, *v;
    float *m_scale, *v_scale;
    int64_t n;
    int64_t end_chunk;                      // chunks of this tensor and the ones in front of it
};

struct Table {
    Part part[kTable];
    int32_t n_parts, n_chunks;
};

// What the step's number sets, for all workgroups.
struct Coefs {
    float factor, decay, rate, second;
    uint32_t key;
};

struct Constants {
    float b1, rest1, b2, rest2, eps;
};

__global__ void adamw_prepare_kernel(int64_t* step, double lr, const float* lr_at, double b1, double b2, double weight_decay,
                                     const float* norm, float max_norm, Coefs* out) {
    const int64_t t = *step + 1;
    if (lr_at) lr = (double)*lr_at;
    Coefs c;
    // max_norm times the reciprocal, each rounded: the bits that torch gives a number over a tensor, its own clipping's among them.  The
    // moments' codes go up or down by less than a rounding, and a caller who forms the factor there is to find the same ones.
    const float quotient = norm ? mrl::mul_rn(1.f / (*norm + 1e-6f), max_norm) : 1.f;
    c.factor = quotient > 1.f ? 1.f : quotient;         // NaN, of a norm that is none, stays NaN
    c.decay = (float)(1.0 - lr * weight_decay);
    c.rate = (float)(lr / (1.0 - pow(b1, (double)t)));
    c.second = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    c.key = (uint32_t)t * 0x9E3779B9u;
    *out = c;
    *step = t;
}

// 16 bits for the even and 16 for the odd entry of a pair: what multiplications and shifts mix of its number and the step's.  Shifts and constants are those of
// a published 32-bit mixer, which Chris Wellons found by a search for little bias.
__device__ __forceinline__ uint32_t dither(uint32_t pair, uint32_t key) {
    uint32_t x = pair ^ key;
    x = (x ^ (x >> 16)) * 0x7feb352du;
    x = (x ^ (x >> 15)) * 0x846ca68bu;
    return x ^ (x >> 16);
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_anywhere __attribute__((aligned(2)));
typedef uint32_t u32_anywhere __attribute__((aligned(1)));

// A lane's entries as they lie in memory.  kWhole: all of them are the tensor's, and a load is one instruction that nothing waits for
// before the values are asked for; else `valid` of them are, zeros stand behind them, and they are loaded one by one.
template <int DT>
struct Unit {
    using T = typename Elem<DT>::T;
    u32x4 v;
    template <bool kWhole>
    __device__ __forceinline__ void load(const void* base, int64_t at, int valid) {
        const T* p = (const T*)base + at;
        if constexpr (!kWhole) {
            float z[kUnit];
#pragma unroll
            for (int i = 0; i < kUnit; ++i) z[i] = i < valid ? Elem<DT>::load(p + i) : 0.f;
            put(z);
        } else if constexpr (DT == MRL_F32) {
            v = mrl::Vec<DT>::load_nt(p);
        } else {
            const u32x2 t = __builtin_nontemporal_load((const u32x2_anywhere*)p);
            v = mrl::make_u32x4(t.x, t.y, 0u, 0u);
        }
    }
    template <bool kWhole>
    __device__ __forceinline__ void store(void* base, int64_t at, int valid) const {
        T* p = (T*)base + at;
        if constexpr (!kWhole) {
            float z[kUnit];
            get(z);
#pragma unroll
            for (int i = 0; i < kUnit; ++i)
                if (i < valid) Elem<DT>::store(p + i, z[i]);
        } else if constexpr (DT == MRL_F32) {
            mrl::Vec<DT>::store_nt(p, v);
        } else {
            const u32x2 t = {v.x, v.y};
            __builtin_nontemporal_store(t, (u32x2_anywhere*)p);
        }
    }
    __device__ __forceinline__ void get(float (&z)[kUnit]) const {
        float t[Elem<DT>::kVec];
        Elem<DT>::unpack(v, t);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) z[i] = t[i];
    }
    __device__ __forceinline__ void put(const float (&z)[kUnit]) {
        float t[Elem<DT>::kVec] = {};
#pragma unroll
        for (int i = 0; i < kUnit; ++i) t[i] = z[i];
        v = Elem<DT>::pack(t);
    }
};

template <bool kWhole>
__device__ __forceinline__ uint32_t load_codes(const void* base, int64_t at, int valid) {
    const uint8_t* p = (const uint8_t*)base + at;
    if (kWhole) return __builtin_nontemporal_load((const u32_anywhere*)p);
    uint32_t c = 0;
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
        if (i < valid) c |= (uint32_t)p[i] << (8 * i);
    return c;
}

template <bool kWhole>
__device__ __forceinline__ void store_codes(void* base, int64_t at, int valid, uint32_t c) {
    uint8_t* p = (uint8_t*)base + at;
    if (kWhole) {
        __builtin_nontemporal_store(c, (u32_anywhere*)p);
        return;
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
        if (i < valid) p[i] = (uint8_t)(c >> (8 * i));
}

__device__ __forceinline__ void values_of(uint32_t c, float scale, float (&z)[kUnit]) {
    const mrl_vocab::floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
    z[0] = mrl::mul_rn(lo[0], scale);
    z[1] = mrl::mul_rn(lo[1], scale);
    z[2] = mrl::mul_rn(hi[0], scale);
    z[3] = mrl::mul_rn(hi[1], scale);
}

// The scale of the 32 lanes of a block, from the largest |z|, by its bits: an infinity's lie above all numbers', NaN's above those.
__device__ __forceinline__ float block_scale(const float (&z)[kUnit]) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kUnit; ++i) most = max(most, __float_as_uint(fabsf(z[i])));
    most = max(most, mrl::lane_partner_bits<0>(most));
    most = max(most, mrl::lane_partner_bits<1>(most));
    most = max(most, mrl::lane_partner_bits<2>(most));
    most = max(most, mrl::lane_partner_bits<3>(most));
    most = max(most, (uint32_t)__shfl_xor((int)most, 16, 64));
    const float s = mrl::mul_rn(__uint_as_float(most), 1.f / kMost);
    return s < kLeastScale ? kLeastScale : s;
}

// floor(|x| / step + u) steps of x's binade, x = z / scale: what the conversion instruction does with the dither in the upper bits.
template <bool kRoot>
__device__ __forceinline__ uint32_t codes_of(const float (&z)[kUnit], float scale, const uint32_t (&bits)[kUnit / 2]) {
    const float inv = 1.f / scale;
    float x[kUnit];
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        float t = mrl::mul_rn(z[i], inv);
        t = t > kMost ? kMost : t;          // NaN stays
        if (kRoot) t = z[i] > 0.f && t < kLeastCode ? kLeastCode : t;
        else t = t < -kMost ? -kMost : t;
        x[i] = t;
    }
    int c = 0;
    c = __builtin_amdgcn_cvt_sr_fp8_f32(x[0], (int)(bits[0] << 16), c, 0);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(x[1], (int)(bits[0] & 0xffff0000u), c, 1);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(x[2], (int)(bits[1] << 16), c, 2);
    c = __builtin_amdgcn_cvt_sr_fp8_f32(x[3], (int)(bits[1] & 0xffff0000u), c, 3);
    return (uint32_t)c;
}

// A lane's share of a chunk: entries from `at` on.
template <int PT, int GT, bool kMaster, bool kSmall, bool kWhole>
__device__ __forceinline__ void step_unit(const Part& p, int64_t at, const Coefs& c, const Constants& k) {
    const int64_t left = p.n - at;
    const int valid = kWhole || left >= kUnit ? kUnit : left > 0 ? (int)left : 0;
    constexpr int kWT = kMaster ? MRL_F32 : PT;
    void* const weights = kMaster ? (void*)p.master : p.param;
    Unit<GT> gu;
    Unit<kWT> wu;
    Unit<MRL_F32> mu, vu;
    uint32_t mc, vc;
    // A lane behind the tensor's end has no block to ask: other lanes write the scales of theirs meanwhile, and what is not finite there
    // would reach the block that this one shares its reductions with.
    const bool holds = kWhole || valid > 0;
    float ms = 0.f, vs = 0.f;
    gu.template load<kWhole>(p.grad, at, valid);
    wu.template load<kWhole>(weights, at, valid);
    if (kSmall) {
        mc = load_codes<kWhole>(p.m, at, valid);
        vc = load_codes<kWhole>(p.v, at, valid);
        if (holds) {
            ms = p.m_scale[at / 128];
            vs = p.v_scale[at / 128];
        }
    } else {
        mu.template load<kWhole>(p.m, at, valid);
        vu.template load<kWhole>(p.v, at, valid);
    }
    float g[kUnit], w[kUnit], m[kUnit], v[kUnit], root[kUnit];
    gu.get(g);
    wu.get(w);
    if (kSmall) {
        values_of(mc, ms, m);
        values_of(vc, vs, v);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = mrl::mul_rn(v[i], v[i]);
    } else {
        mu.get(m);
        vu.get(v);
    }
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
        g[i] = mrl::mul_rn(g[i], c.factor);
        m[i] = mrl::add_rn(mrl::mul_rn(m[i], k.b1), mrl::mul_rn(g[i], k.rest1));
        v[i] = mrl::add_rn(mrl::mul_rn(v[i], k.b2), mrl::mul_rn(mrl::mul_rn(g[i], g[i]), k.rest2));
        root[i] = sqrtf(v[i]);
        w[i] = w[i] * c.decay - m[i] / (root[i] * c.second + k.eps) * c.rate;
    }
    wu.put(w);
    wu.template store<kWhole>(weights, at, valid);
    if (kMaster) {
        Unit<PT> pu;
        pu.put(w);
        pu.template store<kWhole>(p.param, at, valid);
    }
    if (kSmall) {
        uint32_t bits[kUnit / 2];
#pragma unroll
        for (int i = 0; i < kUnit / 2; ++i) bits[i] = dither((uint32_t)(at / 2) + i, c.key);
        ms = block_scale(m);
        vs = block_scale(root);
        store_codes<kWhole>(p.m, at, valid, codes_of<false>(m, ms, bits));
        store_codes<kWhole>(p.v, at, valid, codes_of<true>(root, vs, bits));
        if (holds && (threadIdx.x & 31) == 0) {
            p.m_scale[at / 128] = ms;
            p.v_scale[at / 128] = vs;
        }
    } else {
        mu.put(m);
        vu.put(v);
        mu.template store<kWhole>(p.m, at, valid);
        vu.template store<kWhole>(p.v, at, valid);
    }
}

template <int PT, int GT, bool kMaster, bool kSmall>
__global__ __launch_bounds__(block_of(kSmall)) void adamw_kernel(Table t, const Coefs* __restrict__ coefs, Constants k) {
    constexpr int kChunk = chunk_of(kSmall);
    __shared__ int32_t ends[64];
    if (threadIdx.x < 64) ends[threadIdx.x] = (int)threadIdx.x < t.n_parts ? (int32_t)t.part[threadIdx.x].end_chunk : 0x7fffffff;
    __syncthreads();
    const Coefs c = *coefs;
    for (int chunk = blockIdx.x; chunk < t.n_chunks; chunk += gridDim.x) {
        // as many tensors end at or in front of it
        const int part = __builtin_amdgcn_readfirstlane(__popcll(__ballot(ends[threadIdx.x & 63] <= chunk)));
        const Part& p = t.part[part];
        const int64_t first = (chunk - (part == 0 ? 0 : t.part[part - 1].end_chunk)) * kChunk, at = first + threadIdx.x * kUnit;
        // every wavefront of it decides alike
        if (first + kChunk <= p.n) step_unit<PT, GT, kMaster, kSmall, true>(p, at, c, k);
        else step_unit<PT, GT, kMaster, kSmall, false>(p, at, c, k);
    }
}

// The launches of a list for the tensors of a kind that are not empty: launch(table) for each at most kTable of them.
template <typename F>
void for_tables(const mrl_adamw_tensor* list, int64_t n, int chunk, int dtype, int grad_dtype, bool master, F launch) {
    Table t;
    t.n_parts = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i < n; ++i) {
        const mrl_adamw_tensor& p = list[i];
        if (p.n == 0 || p.dtype != dtype || p.grad_dtype != grad_dtype || (p.master != nullptr) != master) continue;
        chunks += (p.n + chunk - 1) / chunk;
        t.part[t.n_parts++] = {p.param, p.grad, (float*)p.master, p.exp_avg, p.exp_avg_sq, p.exp_avg_scale, p.exp_avg_sq_scale, p.n, chunks};
        t.n_chunks = (int32_t)chunks;
        if (t.n_parts == kTable) {
            launch(t);
            t.n_parts = 0;
            chunks = 0;
        }
    }
    if (t.n_parts > 0) launch(t);
}

int check_tensor(const char* fn, long long i, const mrl_adamw_tensor& p, int bits) {
    const size_t es = mrl::float_dtype_bytes(p.dtype), gs = mrl::float_dtype_bytes(p.grad_dtype), ms = bits == 8 ? 1 : 4;
    MRL_REQUIRE(es != 0, MRL_ERR_UNSUPPORTED, "%s: tensor %lld: dtype %d (want F32, BF16 or F16)", fn, i, p.dtype);
    MRL_REQUIRE(gs != 0 && (p.grad_dtype == p.dtype || p.grad_dtype == MRL_F32), MRL_ERR_UNSUPPORTED,
                "%s: tensor %lld: gradient dtype %d (want the parameter's or F32)", fn, i, p.grad_dtype);
    MRL_REQUIRE(p.n >= 0, MRL_ERR_INVALID_ARG, "%s: tensor %lld: n=%lld", fn, i, (long long)p.n);
    MRL_REQUIRE(p.n <= (1LL << 33), MRL_ERR_UNSUPPORTED, "%s: tensor %lld: n=%lld (at most 2^33)", fn, i, (long long)p.n);
    MRL_REQUIRE(!p.master || p.dtype != MRL_F32, MRL_ERR_INVALID_ARG, "%s: tensor %lld: main weights beside an F32 parameter", fn, i);
    MRL_REQUIRE(p.n == 0 || (p.param && p.grad && p.exp_avg && p.exp_avg_sq && (bits == 32 || (p.exp_avg_scale && p.exp_avg_sq_scale))),
                MRL_ERR_INVALID_ARG, "%s: tensor %lld: NULL pointer", fn, i);
    MRL_REQUIRE(mrl::aligned(p.param, es) && mrl::aligned(p.grad, gs) && mrl::aligned(p.master, 4) && mrl::aligned(p.exp_avg, ms) &&
                    mrl::aligned(p.exp_avg_sq, ms) && mrl::aligned(p.exp_avg_scale, 4) && mrl::aligned(p.exp_avg_sq_scale, 4),
                MRL_ERR_MISALIGNED, "%s: tensor %lld: misaligned", fn, i);
    return MRL_OK;
}

// What is written meets nothing else that is read or written: a parameter given twice would take two steps.
int check_overlap(const char* fn, const mrl_adamw_tensor* list, int64_t n, int bits, const int64_t* step, const float* norm,
                  const float* lr, const float* workspace) {
    struct Range {
        uintptr_t begin, end;
        int32_t tensor;
        bool written;
    };
    const std::unique_ptr<Range[]> all(new (std::nothrow) Range[n * 7 + 4]);
    MRL_REQUIRE(all, MRL_ERR_UNSUPPORTED, "%s: no host memory to look %lld tensors over", fn, (long long)n);
    int64_t count = 0;
    const auto add = [&](const void* p, int64_t bytes, int64_t i, bool written) {
        if (p && bytes > 0) all[count++] = {(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, (int32_t)i, written};
    };
    for (int64_t i = 0; i < n; ++i) {
        const mrl_adamw_tensor& p = list[i];
        const int64_t moment = bits == 8 ? p.n : 4 * p.n, scales = bits == 8 ? (p.n + 127) / 128 * 4 : 0;
        add(p.param, p.n * mrl::float_dtype_bytes(p.dtype), i, true);
        add(p.grad, p.n * mrl::float_dtype_bytes(p.grad_dtype), i, false);
        add(p.master, p.n * 4, i, true);
        add(p.exp_avg, moment, i, true);
        add(p.exp_avg_sq, moment, i, true);
        add(p.exp_avg_scale, scales, i, true);
        add(p.exp_avg_sq_scale, scales, i, true);
    }
    add(step, 8, -1, true);
    add(norm, 4, -1, false);
    add(lr, 4, -1, false);
    add(workspace, MRL_ADAMW_WORKSPACE_BYTES, -1, true);
    std::sort(all.get(), all.get() + count, [](const Range& a, const Range& b) { return a.begin < b.begin; });
    // the furthest ends so far of everything and of what is written
    uintptr_t reach = 0, written = 0;
    for (int64_t q = 0; q < count; ++q) {
        const Range& r = all[q];
        MRL_REQUIRE(r.begin >= (r.written ? reach : written), MRL_ERR_INVALID_ARG, "%s: tensor %d shares memory with another that is written",
                    fn, r.tensor);
        reach = std::max(reach, r.end);
        if (r.written) written = std::max(written, r.end);
    }
    return MRL_OK;
}

}  // namespace

extern "C" int mrl_adamw_step(const mrl_adamw_tensor* tensors, int64_t n_tensors, int bits, int64_t* step, double lr,
                              const float* lr_at, double beta1, double beta2, double eps, double weight_decay, const float* grad_norm,
                              float max_norm, void* workspace, void* stream) {
    const char* fn = "mrl_adamw_step";
    MRL_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || tensors), MRL_ERR_INVALID_ARG, "%s: n_tensors=%lld", fn, (long long)n_tensors);
    MRL_REQUIRE(n_tensors <= MRL_GRAD_TENSORS, MRL_ERR_UNSUPPORTED, "%s: %lld tensors (at most %d)", fn, (long long)n_tensors, MRL_GRAD_TENSORS);
    MRL_REQUIRE(bits == 32 || bits == 8, MRL_ERR_UNSUPPORTED, "%s: bits=%d (want 32 or 8)", fn, bits);
    const auto number = [](double x) { return x >= 0.0 && x <= 3.0e38; };
    MRL_REQUIRE((lr_at || number(lr)) && number(weight_decay) && number(eps) && eps > 0.0 && (float)eps > 0.f, MRL_ERR_INVALID_ARG,
                "%s: lr=%g eps=%g weight_decay=%g", fn, lr, eps, weight_decay);
    MRL_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0, MRL_ERR_INVALID_ARG, "%s: betas %g and %g (want [0, 1))", fn,
                beta1, beta2);
    MRL_REQUIRE(!grad_norm || max_norm >= 0.f, MRL_ERR_INVALID_ARG, "%s: max_norm=%g", fn, (double)max_norm);
    MRL_REQUIRE(step && workspace, MRL_ERR_INVALID_ARG, "%s: NULL pointer", fn);
    MRL_REQUIRE(mrl::aligned(step, 8) && mrl::aligned(lr_at, 4) && mrl::aligned(grad_norm, 4) && mrl::aligned(workspace, 16), MRL_ERR_MISALIGNED,
                "%s: misaligned buffer", fn);
    for (int64_t i = 0; i < n_tensors; ++i) {
        const int rc = check_tensor(fn, (long long)i, tensors[i], bits);
        if (rc != MRL_OK) return rc;
    }
    const int rc = check_overlap(fn, tensors, n_tensors, bits, step, grad_norm, lr_at, (const float*)workspace);
    if (rc != MRL_OK) return rc;
    hipStream_t s = mrl::as_stream(stream);
    Coefs* coefs = (Coefs*)workspace;
    static_assert(sizeof(Coefs) <= MRL_ADAMW_WORKSPACE_BYTES, "the workspace holds them");
    hipLaunchKernelGGL(adamw_prepare_kernel, dim3(1), dim3(1), 0, s, step, lr, lr_at, beta1, beta2, weight_decay, grad_norm, max_norm, coefs);
    const Constants k = {(float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps};
    const auto launch = [&](const Table& t, auto kernel) {
        const int64_t groups = t.n_chunks < kMostGroups ? t.n_chunks : kMostGroups;
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(block_of(bits == 8)), 0, s, t, coefs, k);
    };
#define MRL_KIND(DT, GT, MASTER)                                                                                     \
    for_tables(tensors, n_tensors, chunk_of(bits == 8), DT, GT, MASTER, [&](const Table& t) {                                             \
        bits == 8 ? launch(t, adamw_kernel<DT, GT, MASTER, true>) : launch(t, adamw_kernel<DT, GT, MASTER, false>);  \
    })
    MRL_KIND(MRL_F32, MRL_F32, false);
    MRL_KIND(MRL_BF16, MRL_BF16, false);
    MRL_KIND(MRL_BF16, MRL_BF16, true);
    MRL_KIND(MRL_BF16, MRL_F32, false);
    MRL_KIND(MRL_BF16, MRL_F32, true);
    MRL_KIND(MRL_F16, MRL_F16, false);
    MRL_KIND(MRL_F16, MRL_F16, true);
    MRL_KIND(MRL_F16, MRL_F32, false);
    MRL_KIND(MRL_F16, MRL_F32, true);
#undef MRL_KIND
    return mrl::check_launch(fn);
}
