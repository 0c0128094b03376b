// Dropout whose mask is never stored: value i of a tensor (row-major) is kept where a 16-bit field of the counter RNG lies below
// round(65536 q), and is then multiplied by the reciprocal of that probability.  The backward is the same kernel on the gradient, and a
// call with the same seed makes the same mask again.
// One word serves two neighbouring values: pair j = i / 2 stands at column j mod 2^15 of row j / 2^15; the word is mixed with two keys of
// its row, so that the words of two rows of a mask are no shifted copies of each other (one key of 32 bits leaves 2^32 sequences that
// overlap).  Rows of two masks are the same where both keys are: with x = seed ^ c and m = c ^ d, c and d being the streams' constants, where
// (x + n) ^ m = (x ^ m) + n for a distance of n rows, and that holds where x and x + n differ in no bit of m below 2^31.  Seeds that
// count up are spread so that this is so for no n below 2^17 (functional.dropout_seed).
// Bound by the bytes.  Results are stored past the caches (2^26 values bf16 90 -> 78 us for two tensors in turn).
#include <cmath>
#include <type_traits>
#include "label_rows.h"

namespace sd {

struct DropArgs {
    const void* x[3];
    void* y[3];
    int64_t n;
    const int64_t* seeds;   // the seed's low 32 bits on the device, or null: `seed`
    uint32_t seed, limit;
    float scale;
};

__device__ __forceinline__ uint32_t drop_word(uint32_t key, uint32_t other, uint32_t col) { return rng_mix(rng_word(key, col) ^ other); }

// A workgroup takes 256 vectors of 16 bytes of each of COUNT tensors; these lie in one row of the generator, so the two keys are the
// workgroup's.  (Several vectors per work-item on their way lost: 2^27 values bf16, two tensors in turn, 173 us, four vectors 184.)
template <class T, int COUNT> __global__ void __launch_bounds__(256) dropout_kernel(DropArgs a) {
    constexpr int V = Elem<T>::kVec, kStep = 256 * V;
    static_assert(65536 % kStep == 0, "a step within one row of the generator");
    const uint32_t seed = a.seeds ? (uint32_t)*a.seeds : a.seed;
    const int at = (int)threadIdx.x * V;
    for (int64_t base = (int64_t)blockIdx.x * kStep; base < a.n; base += (int64_t)gridDim.x * kStep) {
        const bool whole = base + at + V <= a.n;
        u32x4 v[COUNT];
        #pragma unroll
        for (int t = 0; t < COUNT; t++)
            if (whole) v[t] = load16(static_cast<const T*>(a.x[t]) + base + at);
        const uint32_t row = (uint32_t)(base >> 16), col = (uint32_t)(base & 0xffff) >> 1;
        const uint32_t key = rng_row_key(seed, 5u, row), other = rng_row_key(seed, 6u, row);
        bool keep[V];
        #pragma unroll
        for (int k = 0; k < V / 2; k++) {
            const uint32_t w = drop_word(key, other, col + at / 2 + k);
            keep[2 * k] = (w & 0xffffu) < a.limit;
            keep[2 * k + 1] = (w >> 16) < a.limit;
        }
        #pragma unroll
        for (int t = 0; t < COUNT; t++) {
            const T* x = static_cast<const T*>(a.x[t]) + base + at;
            T* y = static_cast<T*>(a.y[t]) + base + at;
            if (whole) {
                float f[V];
                Elem<T>::unpack(v[t], f);
                #pragma unroll
                for (int k = 0; k < V; k++) f[k] = keep[k] ? f[k] * a.scale : 0.f;
                put_stream16(y, Elem<T>::pack(f));
            } else {
                #pragma unroll
                for (int k = 0; k < V; k++)
                    if (base + at + k < a.n) y[k] = keep[k] ? Elem<T>::put(Elem<T>::get(x[k]) * a.scale) : T{};
            }
        }
    }
}

template <class T, int COUNT> void launch_dropout(const DropArgs& a, hipStream_t stream) {
    const int64_t step = 256 * Elem<T>::kVec, want = (a.n + step - 1) / step;
    hipLaunchKernelGGL((dropout_kernel<T, COUNT>), dim3((unsigned)(want < (1 << 22) ? want : (1 << 22))), dim3(256), 0, stream, a);
}

}  // namespace sd

using namespace sd;

extern "C" int sd_dropout(const void* x0, const void* x1, const void* x2, int dtype, int64_t n, double q, uint32_t seed, const int64_t* seed_on_device,
                          void* y0, void* y1, void* y2, sd_stream_t stream) {
    sd::CallGuard call_guard;
    SD_REQUIRE(q >= 0.0 && q <= 1.0, "dropout: keep probability q=%g outside 0..1", q);
    SD_REQUIRE(n >= 0 && n < (1ll << 48), "dropout: %lld values", (long long)n);
    DropArgs a{{nullptr, nullptr, nullptr}, {nullptr, nullptr, nullptr}, n, seed_on_device, seed, (uint32_t)std::floor(q * 65536.0 + 0.5), 0.f};
    a.scale = a.limit ? (float)(65536.0 / a.limit) : 0.f;
    const void* const xs[3] = {x0, x1, x2};
    void* const ys[3] = {y0, y1, y2};
    int count = 0;
    for (int k = 0; k < 3; k++) {
        SD_REQUIRE(!xs[k] == !ys[k], "dropout: tensor %d has an input or an output alone", k);
        if (xs[k]) { a.x[count] = xs[k]; a.y[count] = ys[k]; count++; }
    }
    SD_REQUIRE(dtype == SD_FLOAT32 || dtype == SD_BFLOAT16 || dtype == SD_FLOAT16, "dropout: dtype=%d is none of SD_FLOAT32, SD_BFLOAT16, SD_FLOAT16", dtype);
    if (n == 0 || count == 0) return SD_OK;
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (count == 1) launch_dropout<T, 1>(a, s);
        else if (count == 2) launch_dropout<T, 2>(a, s);
        else launch_dropout<T, 3>(a, s);
    });
    return check_launch("dropout_kernel");
}
