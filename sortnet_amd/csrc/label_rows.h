// Rows of values: element types, 16-byte loads and stores, sums over lanes.
#pragma once
#include "common.h"
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

namespace sd {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int64_t kCached = 256ll << 20;    // bytes of the last-level cache

// 16 bytes of a row at an element's own alignment: rows of an odd number of classes start anywhere, and gfx950 loads and stores
// such vectors whole.
template <class T> struct Elem;
template <> struct Elem<float> {
    static constexpr int kVec = 4;
    struct __attribute__((packed, aligned(4))) Pack { u32x4 v; };
    static __device__ __forceinline__ float get(float v) { return v; }
    static __device__ __forceinline__ float put(float v) { return v; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[4]) {
        #pragma unroll
        for (int i = 0; i < 4; i++) f[i] = __uint_as_float(v[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        u32x4 v;
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = __float_as_uint(f[i]);
        return v;
    }
    static __device__ __forceinline__ u32x4 splat(float v) { const uint32_t w = __float_as_uint(v); return u32x4{w, w, w, w}; }
};
struct bf16 { uint16_t bits; };
template <> struct Elem<bf16> {
    static constexpr int kVec = 8;
    struct __attribute__((packed, aligned(2))) Pack { u32x4 v; };
    static __device__ __forceinline__ float get(bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }
    static __device__ __forceinline__ uint16_t bits(float v) { const __bf16 h = (__bf16)v; return __builtin_bit_cast(uint16_t, h); }
    static __device__ __forceinline__ bf16 put(float v) { return bf16{bits(v)}; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
        #pragma unroll
        for (int i = 0; i < 4; i++) {
            f[2 * i] = __uint_as_float(v[i] << 16);
            f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 v;
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (uint32_t)bits(f[2 * i]) | (uint32_t)bits(f[2 * i + 1]) << 16;
        return v;
    }
    static __device__ __forceinline__ u32x4 splat(bf16 v) { const uint32_t w = v.bits | (uint32_t)v.bits << 16; return u32x4{w, w, w, w}; }
};
struct fp16 { uint16_t bits; };
template <> struct Elem<fp16> {
    static constexpr int kVec = 8;
    struct __attribute__((packed, aligned(2))) Pack { u32x4 v; };
    static __device__ __forceinline__ float half(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }
    static __device__ __forceinline__ float get(fp16 v) { return half(v.bits); }
    static __device__ __forceinline__ uint16_t bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ fp16 put(float v) { return fp16{bits(v)}; }
    static __device__ __forceinline__ void unpack(u32x4 v, float (&f)[8]) {
        #pragma unroll
        for (int i = 0; i < 4; i++) { f[2 * i] = half(v[i] & 0xffffu); f[2 * i + 1] = half(v[i] >> 16); }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 v;
        #pragma unroll
        for (int i = 0; i < 4; i++) v[i] = (uint32_t)bits(f[2 * i]) | (uint32_t)bits(f[2 * i + 1]) << 16;
        return v;
    }
    static __device__ __forceinline__ u32x4 splat(fp16 v) { const uint32_t w = v.bits | (uint32_t)v.bits << 16; return u32x4{w, w, w, w}; }
};

template <class T> __device__ __forceinline__ u32x4 load16(const T* p) { return reinterpret_cast<const typename Elem<T>::Pack*>(p)->v; }
template <class T> __device__ __forceinline__ void store16(T* p, u32x4 v) { reinterpret_cast<typename Elem<T>::Pack*>(p)->v = v; }
// the same for what is not read again soon, past the caches
template <class T> __device__ __forceinline__ u32x4 stream16(const T* p) { return __builtin_nontemporal_load(&reinterpret_cast<const typename Elem<T>::Pack*>(p)->v); }
template <class T> __device__ __forceinline__ void put_stream16(T* p, u32x4 v) { __builtin_nontemporal_store(v, &reinterpret_cast<typename Elem<T>::Pack*>(p)->v); }

// One step of adding up (or the like) the lanes of a wavefront in groups of 2, 4, .. 64: v of this lane and of its partner, which are then in the
// same group.  Every lane of a group of the step before holds the same value, so a mirrored half will do for an exchanged one: rows of 16 by
// DPP, wider groups by gfx950's swaps, a few clocks each where a permutation through LDS is about 60.
template <int STEP, class Op> __device__ __forceinline__ uint32_t lanes_step(uint32_t v, Op op) {
    if constexpr (STEP == 0) return op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));           // neighbours
    else if constexpr (STEP == 1) return op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));      // pairs of a quad
    else if constexpr (STEP == 2) return op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));     // halves of 8
    else if constexpr (STEP == 3) return op(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false));     // halves of 16
    else if constexpr (STEP == 4) { const auto p = __builtin_amdgcn_permlane16_swap(v, v, false, false); return op(p[0], p[1]); }
    else { const auto p = __builtin_amdgcn_permlane32_swap(v, v, false, false); return op(p[0], p[1]); }
}
template <int STEP> __device__ __forceinline__ double lanes_add(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    uint32_t lo[2], hi[2];
    lanes_step<STEP>((uint32_t)bits, [&](uint32_t a, uint32_t b) { lo[0] = a; lo[1] = b; return 0u; });
    lanes_step<STEP>((uint32_t)(bits >> 32), [&](uint32_t a, uint32_t b) { hi[0] = a; hi[1] = b; return 0u; });
    return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
template <int STEP> __device__ __forceinline__ float lanes_max(float v) {
    return __uint_as_float(lanes_step<STEP>(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }));
}
// over groups of 2^shift lanes (the same shift in all of them, each group whole or not there at all)
__device__ __forceinline__ double group_total(double v, int shift) {
    if (shift > 0) v = lanes_add<0>(v);
    if (shift > 1) v = lanes_add<1>(v);
    if (shift > 2) v = lanes_add<2>(v);
    if (shift > 3) v = lanes_add<3>(v);
    if (shift > 4) v = lanes_add<4>(v);
    if (shift > 5) v = lanes_add<5>(v);
    return v;
}
__device__ __forceinline__ float group_max(float v, int shift) {
    if (shift > 0) v = lanes_max<0>(v);
    if (shift > 1) v = lanes_max<1>(v);
    if (shift > 2) v = lanes_max<2>(v);
    if (shift > 3) v = lanes_max<3>(v);
    if (shift > 4) v = lanes_max<4>(v);
    if (shift > 5) v = lanes_max<5>(v);
    return v;
}

// calls f with a null pointer of the element type that `dtype` names; false for none
template <class F> bool with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case SD_FLOAT32: f((float*)nullptr); return true;
        case SD_BFLOAT16: f((bf16*)nullptr); return true;
        case SD_FLOAT16: f((fp16*)nullptr); return true;
    }
    return false;
}

}  // namespace sd
