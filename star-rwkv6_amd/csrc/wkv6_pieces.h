// Pieces of a few elements between memory and registers, at any element's address, for the kernels that go through dense arrays of any length.
#pragma once
#include "wkv6_common.h"

#include <type_traits>

namespace wkv6 {
namespace {

// kEach (4 or 8) elements as they sit in memory, at any element's address; the last ones of a tensor one by one.  S: 4-, 2- or 1-byte elements.
template <typename S, int kEach> struct Piece {
    static constexpr int kWords = kEach * sizeof(S) / 4, kAtOnce = kWords < 4 ? kWords : 4;
    typedef uint32_t vec __attribute__((ext_vector_type(kAtOnce), aligned(sizeof(S))));
    uint32_t r[kWords];
    template <bool kPast> __device__ __forceinline__ void load(const S *p, int n) {
        if (n >= kEach) {
#pragma unroll
            for (int k = 0; k < kWords / kAtOnce; ++k) {
                const vec *at = reinterpret_cast<const vec *>(p) + k;
                vec v;
                if (kPast) v = __builtin_nontemporal_load(at);
                else v = *at;
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) r[k * kAtOnce + i] = v[i];
            }
            return;
        }
        const auto *bits = reinterpret_cast<const unsigned_of *>(p);
#pragma unroll
        for (int i = 0; i < kWords; ++i) r[i] = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (e < n) r[e * (int)sizeof(S) / 4] |= (uint32_t)bits[e] << (e * 8 * (int)sizeof(S) % 32);
    }
    template <bool kPast> __device__ __forceinline__ void store(S *p, int n) const {
        if (n >= kEach) {
#pragma unroll
            for (int k = 0; k < kWords / kAtOnce; ++k) {
                vec *at = reinterpret_cast<vec *>(p) + k;
                vec v;
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) v[i] = r[k * kAtOnce + i];
                if (kPast) __builtin_nontemporal_store(v, at);
                else *at = v;
            }
            return;
        }
        auto *bits = reinterpret_cast<unsigned_of *>(p);
#pragma unroll
        for (int e = 0; e < kEach; ++e)
            if (e < n) bits[e] = (unsigned_of)(r[e * (int)sizeof(S) / 4] >> (e * 8 * (int)sizeof(S) % 32));
    }
    typedef std::conditional_t<sizeof(S) == 4, uint32_t, std::conditional_t<sizeof(S) == 2, uint16_t, uint8_t>> unsigned_of;
};

template <int kEach> __device__ __forceinline__ void unpack(const Piece<float, kEach> &b, float (&o)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) o[i] = __uint_as_float(b.r[i]);
}
template <int kEach> __device__ __forceinline__ void unpack(const Piece<bf16_t, kEach> &b, float (&o)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) o[2 * i] = __uint_as_float(b.r[i] << 16), o[2 * i + 1] = __uint_as_float(b.r[i] & 0xffff0000u);
}
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
template <int kEach> __device__ __forceinline__ void unpack(const Piece<f16_t, kEach> &b, float (&o)[kEach]) {
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) {
        const h2 h = __builtin_bit_cast(h2, b.r[i]);
        o[2 * i] = (float)h[0], o[2 * i + 1] = (float)h[1];
    }
}
template <int kEach> __device__ __forceinline__ void unpack(const Piece<uint8_t, kEach> &b, float (&o)[kEach]) {   // float8
    typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < kEach / 4; ++i) {
        const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.r[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.r[i], true);
        o[4 * i] = lo[0], o[4 * i + 1] = lo[1], o[4 * i + 2] = hi[0], o[4 * i + 3] = hi[1];
    }
}
template <int kEach> __device__ __forceinline__ void pack(const float (&v)[kEach], Piece<float, kEach> &b) {
#pragma unroll
    for (int i = 0; i < kEach; ++i) b.r[i] = __float_as_uint(v[i]);
}
template <int kEach> __device__ __forceinline__ void pack(const float (&v)[kEach], Piece<bf16_t, kEach> &b) {
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) b.r[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
}
template <int kEach> __device__ __forceinline__ void pack(const float (&v)[kEach], Piece<f16_t, kEach> &b) {
#pragma unroll
    for (int i = 0; i < kEach / 2; ++i) b.r[i] = __builtin_bit_cast(uint32_t, (h2){to_f16(v[2 * i]), to_f16(v[2 * i + 1])});
}

}  // namespace
}  // namespace wkv6
