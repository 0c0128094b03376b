// Dropout whose mask is never stored: value i of a tensor (row-major) is kept where a 16-bit field of the counter RNG lies below
// round(65536 q), and is then multiplied by the reciprocal of that probability.  The backward is the same kernel on the gradient, and a
// call with the same seed makes the same mask again.
// One word serves two neighbouring values: pair j = i / 2 stands at column j mod 2^15 of row j / 2^15; the word is mixed with two keys of
// its row, so that the words of two rows are no shifted copies of each other (one key of 32 bits leaves 2^32 sequences that overlap).
// Bound by the bytes; the words take about half of the issue slots that the bytes of a 16-bit tensor leave.
#include <cmath>
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

// A work-item takes 8 neighbouring values at a time of each of COUNT tensors.
template <class T, int COUNT> __global__ void __launch_bounds__(256) dropout_kernel(DropArgs a) {
    constexpr int V = Elem<T>::kVec, P = 8 / V;
    const uint32_t seed = a.seeds ? (uint32_t)*a.seeds : a.seed;
    const int64_t eights = (a.n + 7) / 8;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < eights; e += (int64_t)gridDim.x * 256) {
        const int64_t i = e * 8;
        const uint32_t row = (uint32_t)(i >> 16), col = (uint32_t)(i & 0xffff) >> 1;
        const uint32_t key = rng_row_key(seed, 5u, row), other = rng_row_key(seed, 6u, row);
        bool keep[8];
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t w = drop_word(key, other, col + k);
            keep[2 * k] = (w & 0xffffu) < a.limit;
            keep[2 * k + 1] = (w >> 16) < a.limit;
        }
        #pragma unroll
        for (int t = 0; t < COUNT; t++) {
            const T* x = static_cast<const T*>(a.x[t]) + i;
            T* y = static_cast<T*>(a.y[t]) + i;
            if (i + 8 <= a.n) {
                #pragma unroll
                for (int p = 0; p < P; p++) {
                    float f[V];
                    Elem<T>::unpack(load16(x + p * V), f);
                    #pragma unroll
                    for (int k = 0; k < V; k++) f[k] = keep[p * V + k] ? f[k] * a.scale : 0.f;
                    store16(y + p * V, Elem<T>::pack(f));
                }
            } else {
                #pragma unroll
                for (int k = 0; k < 8; k++)
                    if (i + k < a.n) y[k] = keep[k] ? Elem<T>::put(Elem<T>::get(x[k]) * a.scale) : T{};
            }
        }
    }
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
    const int64_t want = ((n + 7) / 8 + 255) / 256;
    const dim3 grid((unsigned)(want < (1 << 20) ? want : (1 << 20)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (count == 1) hipLaunchKernelGGL((dropout_kernel<T, 1>), grid, dim3(256), 0, s, a);
        else if (count == 2) hipLaunchKernelGGL((dropout_kernel<T, 2>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((dropout_kernel<T, 3>), grid, dim3(256), 0, s, a);
    });
    return check_launch("dropout_kernel");
}
