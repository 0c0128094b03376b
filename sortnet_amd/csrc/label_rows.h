// Rows of values: element types, 16-byte loads and stores, sums over lanes.
#pragma once
#include <cfloat>
#include <type_traits>
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
        for (int i = 0; i < 4; i++) v[i] = both(f[2 * i], f[2 * i + 1]);
        return v;
    }
    // (two at once: one conversion instead of two, a shift and an or)
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t both(float low, float high) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{low, high}), bf16x2)); }
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
        for (int i = 0; i < 4; i++) v[i] = both(f[2 * i], f[2 * i + 1]);
        return v;
    }
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 fp16x2 __attribute__((ext_vector_type(2)));
    static __device__ __forceinline__ uint32_t both(float low, float high) { return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{low, high}), fp16x2)); }
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

// where row r of logits begins whose rows lie `outer_stride` apart in blocks of `inner` rows that lie `inner_stride` apart
template <class T, class R> __device__ __forceinline__ const T* row_start(const R& a, int64_t r) {
    const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
    return static_cast<const T*>(a.logits) + o * a.outer_stride + i * a.inner_stride;
}

__device__ __forceinline__ double wave_total(double v) { return group_total(v, 6); }

__device__ __forceinline__ float finite(float top) { return fmaxf(top, -FLT_MAX); }

// exp of a difference to the largest value of a row (or of a part of it): the hardware's exp2 of v log2(e), 1 for 0, so that a row's largest
// term is exact.  log2(e) is the sum of two numbers (both positive: -inf stays -inf): of one it would be off by 1.3e-8 of v to one side, which the sum
// over a row and the sum over an answer's rows add up.  As it is the product is rounded once, off by up to |v| 2^-24 of the result to either side,
// and the hardware's exp2 by up to 1.4 2^-24, 0.06 2^-24 below on average (measured over 2^24 values a binade; expf 0.04).
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(fmaf(v, 1.44269504f, v * 1.92596299e-8f)); }

// Sums of a row: exponentials of a few vectors in pairs, in 32 bits, and these sums in 64 (an addition to a sum in 32 bits that has the
// largest value, 1, in it is off by up to 6e-8, and there are hundreds of them).
template <int N> __device__ __forceinline__ float tree(const float (&f)[N]) {
    float s[N];
    #pragma unroll
    for (int i = 0; i < N; i++) s[i] = f[i];
    #pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        #pragma unroll
        for (int i = 0; i < o; i++) s[i] += s[i + o];
    }
    return s[0];
}

// A short row, which 2^shift lanes of a wavefront hold in registers, NV vectors each.
// The last vector of a row of at least one ends with the row and overlaps the one before it; a shorter row is one vector, padded with -inf.
template <class T, int NV> struct HeldRow {
    static constexpr int V = Elem<T>::kVec;
    u32x4 v[NV];
    int n, vecs, lane, shift;

    __device__ __forceinline__ int index(int k) const { return lane + (k << shift); }
    __device__ __forceinline__ int column(int i) const { return i * V + V <= n ? i * V : n - V; }     // (n >= V)

    __device__ __forceinline__ void load(const T* p) {
        if (n >= V) {
            #pragma unroll
            for (int k = 0; k < NV; k++)
                if (index(k) < vecs) v[k] = load16(p + column(index(k)));
        } else if (lane == 0) {
            float f[V];
            #pragma unroll
            for (int i = 0; i < V; i++) f[i] = i < n ? Elem<T>::get(p[i]) : -INFINITY;
            v[0] = Elem<T>::pack(f);
        }
    }
    // What was derived from the vectors before is derived again afterwards: kept, it would be twice their registers.
    __device__ __forceinline__ void again() {
        #pragma unroll
        for (int k = 0; k < NV; k++) asm("" : "+v"(v[k]));
    }
};

// zeros in a row of a gradient, by a whole workgroup
template <class T> __device__ __forceinline__ void clear_row(T* q, int n, int threads) {
    constexpr int V = Elem<T>::kVec;
    const int full = n / V;
    for (int i = threadIdx.x; i < full; i += threads) put_stream16(q + i * V, u32x4{0u, 0u, 0u, 0u});
    for (int j = full * V + threadIdx.x; j < n; j += threads) q[j] = T{};
}

// Whether this workgroup is the last to have stored its part, which its first work-item did before; the parts of all are then
// visible to it.  The counter is the call's own and was cleared by the kernel before this one.
__device__ __forceinline__ bool last_workgroup(uint32_t* ticket) {
    __shared__ int last;
    if (threadIdx.x == 0) {
        __threadfence();
        last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        __threadfence();
    }
    __syncthreads();
    return last != 0;
}

__device__ __forceinline__ double published(const double* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void publish(double* p, double v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// calls f with a null pointer of the element type that `dtype` names; false for none
template <class F> bool with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case SD_FLOAT32: f((float*)nullptr); return true;
        case SD_BFLOAT16: f((bf16*)nullptr); return true;
        case SD_FLOAT16: f((fp16*)nullptr); return true;
    }
    return false;
}

// rows of logits without labels (sd_logit_rows)
struct LogitRows {
    const void* logits;
    int64_t rows, classes, outer_stride, inner_stride;
    uint32_t inner;
};

inline int check_logits(const sd_logit_rows* in, const char* who, LogitRows* a) {
    SD_REQUIRE(in, "%s: null rows", who);
    SD_REQUIRE(in->dtype == SD_FLOAT32 || in->dtype == SD_BFLOAT16 || in->dtype == SD_FLOAT16, "%s: dtype=%d is none of SD_FLOAT32, SD_BFLOAT16, SD_FLOAT16", who, in->dtype);
    SD_REQUIRE(in->rows > 0 && in->rows < (1ll << 31), "%s: rows=%lld outside 1..2^31-1", who, (long long)in->rows);
    SD_REQUIRE(in->classes > 0 && in->classes < (1ll << 31), "%s: classes=%lld outside 1..2^31-1", who, (long long)in->classes);
    SD_REQUIRE(in->inner > 0 && in->rows % in->inner == 0 && in->inner < (1ll << 31), "%s: inner=%lld does not divide rows=%lld", who, (long long)in->inner, (long long)in->rows);
    SD_REQUIRE(in->logits, "%s: null logits", who);
    SD_REQUIRE((reinterpret_cast<uintptr_t>(in->logits) & (in->dtype == SD_FLOAT32 ? 3 : 1)) == 0, "%s: logits are not aligned to their type", who);
    *a = LogitRows{in->logits, in->rows, in->classes, in->outer_stride, in->inner_stride, (uint32_t)in->inner};
    return SD_OK;
}

constexpr int64_t kMostBlocks = 1 << 22;
inline unsigned blocks_for(int64_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }
inline int vec_of(int dtype) { return dtype == SD_FLOAT32 ? 4 : 8; }

constexpr int kHeld = 8;            // 16-byte vectors of a short row that a lane holds, at most
constexpr int kHeldLong = 16 * 1024;    // and of a long row that a workgroup holds
constexpr int kShortBlocks = 4096;      // workgroups of short rows, at most

// Lanes of a wavefront that hold a row together (as a power of two) and vectors that each holds; shift = -1: a row is read by whole workgroups.
// Many rows want few lanes with several vectors each (fewer steps to add up lanes per row), few rows one vector per lane.
struct Group { int shift, vectors; };
inline Group group_of(int64_t rows, int64_t classes, int vec) {
    const int64_t vecs = (classes + vec - 1) / vec;
    if (vecs > 64 * kHeld) return {-1, 0};
    int shift = 0;
    while (shift < 6 && (1 << shift) < vecs) shift++;
    int vectors = 1;
    while ((int64_t)vectors << shift < vecs) vectors *= 2;
    while (vectors < 4 && shift > 0 && (rows << shift) > (1 << 16)) { shift--; vectors *= 2; }
    return {shift, vectors};
}

template <class F> void with_vectors(int vectors, F&& f) {
    switch (vectors) {
        case 1: f(std::integral_constant<int, 1>()); return;
        case 2: f(std::integral_constant<int, 2>()); return;
        case 4: f(std::integral_constant<int, 4>()); return;
        default: f(std::integral_constant<int, kHeld>()); return;
    }
}

// Parts of a long row: so many that there are kWholeRows workgroups (2.75 for each compute unit), none with less than one vector per work-item.
// With 2048: 2000 x 50001 bf16 35.8 us whole, in two parts 38.2; 1000 x 131072 43.6 and 48.2; 1030 x 131072 fp32 90.3 and 86.8.
constexpr int64_t kWholeRows = 704;
inline int row_splits(int64_t rows, int64_t classes, int vec) {
    const int64_t want = (kWholeRows + rows - 1) / rows, most = (classes + 256 * vec - 1) / (256 * vec);
    return (int)(want < most ? want : most);
}

// Rows that would be read in parts: where a workgroup can hold a row it is read whole, which spares the launch that joins the parts:
// 128 x 8192 bf16 6.8 -> 4.4 us, 512 x 16384 8.6 -> 5.4, 512 x 32000 11.9 -> 9.3.  Rows for a workgroup of 512, of which fewer run at once: 256 x 50001
// 10.4 -> 9.0, but 16 rows 7.1 -> 8.4 and 1024 21.2 -> 26.0.
inline bool one_launch(int64_t rows, int64_t classes, int vec) {
    const int64_t vecs = (classes + vec - 1) / vec;
    return rows < kWholeRows && (vecs <= 16 * 256 || (vecs <= 16 * 512 && rows >= 32 && rows <= 512));
}

inline int64_t part_of(int64_t classes, int splits, int vec) {
    const int64_t step = 256 * vec, n = (classes + splits - 1) / splits;
    return (n + step - 1) / step * step;
}

inline unsigned short_blocks(int64_t rows, int per) {
    const int64_t n = (rows + per - 1) / per;
    return (unsigned)(n < kShortBlocks ? n : kShortBlocks);
}

// Launches of kernels whose workgroups do one thing each: at most 2^20 of them at a time (a grid of 2^32 work-items would be too large).
template <class F> inline void in_slices(int64_t blocks, F&& f) {
    for (int64_t from = 0; from < blocks; from += 1 << 20) f(from, (unsigned)(blocks - from < 1 << 20 ? blocks - from : 1 << 20));
}

}  // namespace sd
