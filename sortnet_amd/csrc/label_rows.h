// Rows of logits: element types, 16-byte loads and the exponentials of their softmax.
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
    static __device__ __forceinline__ float exp(float v) { return expf(v); }
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
    // results are rounded to 8 bits: the hardware's exp2 of a rounded argument is exact enough (|v| 2^-24 relative)
    static __device__ __forceinline__ float exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
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
    static __device__ __forceinline__ float exp(float v) { return __builtin_amdgcn_exp2f(v * 1.44269504f); }
};

template <class T> __device__ __forceinline__ u32x4 load16(const T* p) { return reinterpret_cast<const typename Elem<T>::Pack*>(p)->v; }
template <class T> __device__ __forceinline__ void store16(T* p, u32x4 v) { reinterpret_cast<typename Elem<T>::Pack*>(p)->v = v; }
// the same for what is not read again soon, past the caches
template <class T> __device__ __forceinline__ u32x4 stream16(const T* p) { return __builtin_nontemporal_load(&reinterpret_cast<const typename Elem<T>::Pack*>(p)->v); }
template <class T> __device__ __forceinline__ void put_stream16(T* p, u32x4 v) { __builtin_nontemporal_store(v, &reinterpret_cast<typename Elem<T>::Pack*>(p)->v); }

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
