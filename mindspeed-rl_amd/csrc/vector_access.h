// 16 bytes of a row at any element's address.  gfx950 serves global accesses of 16 bytes at any byte; an access that
// crosses a 128-byte line takes a second request.
#pragma once

#include "mrl_internal.h"
#include "vocab_common.h"

namespace mrl {

typedef u32x4 u32x4_anywhere __attribute__((aligned(2)));

template <int DT>
struct Vec {
    using E = mrl_vocab::Elem<DT>;
    using T = typename E::T;
    static constexpr int kVec = E::kVec;
    using At = u32x4_anywhere;
    static __device__ __forceinline__ u32x4 load(const T* p) { return *(const At*)p; }
    static __device__ __forceinline__ u32x4 load_nt(const T* p) { return __builtin_nontemporal_load((const At*)p); }
    static __device__ __forceinline__ void store(T* p, const u32x4& v) { *(At*)p = v; }
    static __device__ __forceinline__ void store_nt(T* p, const u32x4& v) { __builtin_nontemporal_store(v, (At*)p); }
};

// kN entries of a vector of another type than the rows', as floats: as many loads as they take.
template <int DT, int kN>
__device__ __forceinline__ void load_floats(const typename mrl_vocab::Elem<DT>::T* p, float (&out)[kN]) {
    constexpr int kVec = mrl_vocab::Elem<DT>::kVec;
    static_assert(kN % kVec == 0, "whole vectors");
#pragma unroll
    for (int q = 0; q < kN / kVec; ++q) {
        float z[kVec];
        mrl_vocab::Elem<DT>::unpack(Vec<DT>::load(p + q * kVec), z);
#pragma unroll
        for (int i = 0; i < kVec; ++i) out[q * kVec + i] = z[i];
    }
}

}  // namespace mrl
