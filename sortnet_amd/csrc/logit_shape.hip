// Logits as they stand when a class is chosen: per row and class v, with n = how often v stands in the row's history,
//   y = z;  where n > 0  y = (z > 0 ? z / repetition : z * repetition) - frequency n - presence;  y += bias[v];  -inf where v is not allowed,
// in 32 bits and in this order, rounded once.  The gradient is 0 where v is not allowed, g / repetition or g * repetition where n > 0, else g.
// Bound by the bytes of the logits in and out.  The counts of a workgroup's columns stand in its LDS, for which it reads the whole history of
// its rows: no scratch, nothing to sort, and any number of repeated classes.
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kShapeCounts = 8192;      // columns whose counts a workgroup holds (32 KiB)
enum { kAll = 0, kFlags = SD_ALLOWED_FLAGS, kBits = SD_ALLOWED_BITS };

struct Shape {
    const void *history, *lengths;
    int64_t length, history_outer, history_inner;
    int wide_history, wide_lengths;             // int64 instead of int32
    const float *repetition_rows, *presence_rows, *frequency_rows;
    float repetition, presence, frequency;
    const float* bias;
    int64_t bias_outer, bias_inner;
    const void* allowed;
    int64_t allowed_outer, allowed_inner;
    const void* grad;                           // backward: what flows into the result, rows one behind the other
    void* out;
    int64_t part;                               // columns of a workgroup, a multiple of 8
    int parts, group;                           // parts of a row, or (with one part) rows of a workgroup
};

struct __attribute__((packed, aligned(1))) Bytes8 { uint32_t lo, hi; };
struct __attribute__((packed, aligned(1))) Bytes4 { uint32_t lo; };

// bit i: column c + i of V columns is allowed (c a multiple of V)
template <int V, int ALLOWED> __device__ __forceinline__ uint32_t allowed_bits(const void* row, int c) {
    if constexpr (ALLOWED == kBits) {
        const uint32_t byte = static_cast<const uint8_t*>(row)[c >> 3];
        return V == 8 ? byte : byte >> (c & 4);
    } else {
        uint32_t bits = 0;
        const uint8_t* p = static_cast<const uint8_t*>(row) + c;
        uint32_t w[V / 4];
        if constexpr (V == 8) { const Bytes8 b = *reinterpret_cast<const Bytes8*>(p); w[0] = b.lo; w[1] = b.hi; }
        else w[0] = reinterpret_cast<const Bytes4*>(p)->lo;
        #pragma unroll
        for (int i = 0; i < V; i++) bits |= (w[i / 4] >> (8 * (i & 3)) & 0xffu) ? 1u << i : 0u;
        return bits;
    }
}

template <int ALLOWED> __device__ __forceinline__ bool allowed_one(const void* row, int c) {
    if constexpr (ALLOWED == kBits) return static_cast<const uint8_t*>(row)[c >> 3] >> (c & 7) & 1;
    else return static_cast<const uint8_t*>(row)[c] != 0;
}

__device__ __forceinline__ float penalised(float z, float n, float repetition, float presence, float frequency) {
    return (z > 0.f ? z / repetition : z * repetition) - frequency * n - presence;
}
__device__ __forceinline__ float penalised_slope(float g, float z, float repetition) { return z > 0.f ? g / repetition : g * repetition; }

template <class T, int ALLOWED, bool HISTORY, bool GRAD> __global__ void __launch_bounds__(256) shape_kernel(LogitRows a, Shape s) {
    constexpr int V = Elem<T>::kVec;
    __shared__ __align__(16) uint32_t counts[HISTORY ? kShapeCounts : 4];
    const int64_t r0 = (int64_t)(blockIdx.x / s.parts) * s.group, c0 = (int64_t)(blockIdx.x % s.parts) * s.part;
    const int rows = (int)(a.rows - r0 < s.group ? a.rows - r0 : s.group);
    const int columns = (int)(a.classes - c0 < s.part ? a.classes - c0 : s.part), width = (columns + 7) & ~7, vecs = (columns + V - 1) / V;
    const auto place = [&](int64_t r, int64_t outer, int64_t inner) {
        const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
        return o * outer + i * inner;
    };
    if (HISTORY) {
        for (int i = threadIdx.x; i < rows * width / 4; i += 256) reinterpret_cast<u32x4*>(counts)[i] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
        for (int i = 0; i < rows; i++) {
            const int64_t r = r0 + i;
            int64_t n = s.length;
            if (s.lengths) {
                const int64_t given = s.wide_lengths ? static_cast<const int64_t*>(s.lengths)[r] : static_cast<const int*>(s.lengths)[r];
                n = given < 0 ? 0 : given < n ? given : n;
            }
            const int64_t at = place(r, s.history_outer, s.history_inner);
            for (int64_t j = threadIdx.x; j < n; j += 256) {
                const int64_t token = s.wide_history ? static_cast<const int64_t*>(s.history)[at + j] : static_cast<const int*>(s.history)[at + j];
                if (token >= c0 && token < c0 + columns) atomicAdd(&counts[i * width + (int)(token - c0)], 1u);
            }
        }
        __syncthreads();
    }
    for (int item = threadIdx.x; item < rows * vecs; item += 256) {
        const int i = item / vecs, c = (item - i * vecs) * V;
        const int64_t r = r0 + i;
        const T* z = row_start<T>(a, r) + c0 + c;
        const T* g = GRAD ? static_cast<const T*>(s.grad) + r * a.classes + c0 + c : nullptr;
        T* q = static_cast<T*>(s.out) + r * a.classes + c0 + c;
        const float* bias = !GRAD && s.bias ? s.bias + place(r, s.bias_outer, s.bias_inner) + c0 + c : nullptr;
        const uint8_t* allowed = ALLOWED == kAll ? nullptr
            : static_cast<const uint8_t*>(s.allowed) + (ALLOWED == kBits ? 4 : 1) * place(r, s.allowed_outer, s.allowed_inner);
        float repetition = 1.f, presence = 0.f, frequency = 0.f;
        if (HISTORY) {
            repetition = s.repetition_rows ? s.repetition_rows[r] : s.repetition;
            presence = s.presence_rows ? s.presence_rows[r] : s.presence;
            frequency = s.frequency_rows ? s.frequency_rows[r] : s.frequency;
        }
        if (c + V <= columns) {
            float f[V];
            Elem<T>::unpack(load16(GRAD ? g : z), f);
            if (HISTORY) {
                uint32_t n[V], any = 0;
                #pragma unroll
                for (int k = 0; k < V; k++) { n[k] = counts[i * width + c + k]; any |= n[k]; }
                if (any) {
                    #pragma unroll
                    for (int k = 0; k < V; k++)
                        if (n[k]) f[k] = GRAD ? penalised_slope(f[k], Elem<T>::get(z[k]), repetition) : penalised(f[k], (float)n[k], repetition, presence, frequency);
                }
            }
            if (!GRAD && bias) {
                #pragma unroll
                for (int k = 0; k < V; k += 4) {
                    float b[4];
                    Elem<float>::unpack(load16(bias + k), b);
                    #pragma unroll
                    for (int m = 0; m < 4; m++) f[k + m] += b[m];
                }
            }
            if (ALLOWED != kAll) {
                const uint32_t bits = allowed_bits<V, ALLOWED == kAll ? kBits : ALLOWED>(allowed, (int)c0 + c);
                #pragma unroll
                for (int k = 0; k < V; k++) f[k] = bits >> k & 1 ? f[k] : GRAD ? 0.f : -INFINITY;
            }
            store16(q, Elem<T>::pack(f));
        } else {
            for (int k = 0; k < columns - c; k++) {
                float f = Elem<T>::get(GRAD ? g[k] : z[k]);
                const uint32_t n = HISTORY ? counts[i * width + c + k] : 0u;
                if (n) f = GRAD ? penalised_slope(f, Elem<T>::get(z[k]), repetition) : penalised(f, (float)n, repetition, presence, frequency);
                if (!GRAD && bias) f += bias[k];
                if (ALLOWED != kAll && !allowed_one<ALLOWED == kAll ? kBits : ALLOWED>(allowed, (int)c0 + c + k)) f = GRAD ? 0.f : -INFINITY;
                q[k] = Elem<T>::put(f);
            }
        }
    }
}

static int shape_logits(const char* who, const sd_logit_rows* in, const sd_constraints* c, const void* grad, void* out, hipStream_t stream) {
    LogitRows a;
    if (int rc = check_logits(in, who, &a)) return rc;
    const uintptr_t odd = in->dtype == SD_FLOAT32 ? 3 : 1;
    SD_REQUIRE(c && out, "%s: null argument", who);
    SD_REQUIRE((reinterpret_cast<uintptr_t>(out) & odd) == 0 && (reinterpret_cast<uintptr_t>(grad) & odd) == 0, "%s: results or gradients are not aligned to their type", who);
    SD_REQUIRE(!c->history || c->history_bytes == 4 || c->history_bytes == 8, "%s: history of %d bytes", who, c->history_bytes);
    SD_REQUIRE(!c->lengths || c->length_bytes == 4 || c->length_bytes == 8, "%s: lengths of %d bytes", who, c->length_bytes);
    SD_REQUIRE(!c->history || (c->history_length >= 0 && c->history_length <= UINT32_MAX), "%s: history_length=%lld outside 0..2^32-1", who, (long long)c->history_length);
    SD_REQUIRE(!c->history || (reinterpret_cast<uintptr_t>(c->history) & (c->history_bytes - 1)) == 0, "%s: the history is not aligned to its type", who);
    SD_REQUIRE(!c->lengths || (reinterpret_cast<uintptr_t>(c->lengths) & (c->length_bytes - 1)) == 0, "%s: lengths are not aligned to their type", who);
    SD_REQUIRE(!c->lengths || c->history, "%s: lengths without a history", who);
    SD_REQUIRE(c->repetition_rows || (c->repetition > 0.0 && c->repetition <= FLT_MAX && (float)c->repetition > 0.f), "%s: repetition=%g must be positive and finite", who, c->repetition);
    SD_REQUIRE(c->presence_rows || (c->presence >= -FLT_MAX && c->presence <= FLT_MAX), "%s: presence=%g must be finite", who, c->presence);
    SD_REQUIRE(c->frequency_rows || (c->frequency >= -FLT_MAX && c->frequency <= FLT_MAX), "%s: frequency=%g must be finite", who, c->frequency);
    SD_REQUIRE(((reinterpret_cast<uintptr_t>(c->repetition_rows) | reinterpret_cast<uintptr_t>(c->presence_rows) | reinterpret_cast<uintptr_t>(c->frequency_rows) |
                 reinterpret_cast<uintptr_t>(c->bias)) & 3) == 0, "%s: penalties or bias are not aligned to their type", who);
    SD_REQUIRE(!c->allowed || c->allowed_kind == kFlags || c->allowed_kind == kBits, "%s: allowed_kind=%d is neither SD_ALLOWED_FLAGS nor SD_ALLOWED_BITS", who, c->allowed_kind);
    SD_REQUIRE(!c->allowed || c->allowed_kind != kBits || (reinterpret_cast<uintptr_t>(c->allowed) & 3) == 0, "%s: allowed is not aligned to its type", who);
    Shape s{};
    const bool history = c->history && c->history_length > 0;
    if (history) {
        s.history = c->history; s.lengths = c->lengths;
        s.length = c->history_length; s.history_outer = c->history_outer; s.history_inner = c->history_inner;
        s.wide_history = c->history_bytes == 8; s.wide_lengths = c->length_bytes == 8;
        s.repetition_rows = c->repetition_rows; s.presence_rows = c->presence_rows; s.frequency_rows = c->frequency_rows;
        s.repetition = (float)c->repetition; s.presence = (float)c->presence; s.frequency = (float)c->frequency;
    }
    s.bias = c->bias; s.bias_outer = c->bias_outer; s.bias_inner = c->bias_inner;
    s.allowed = c->allowed; s.allowed_outer = c->allowed_outer; s.allowed_inner = c->allowed_inner;
    s.grad = grad; s.out = out;
    const int64_t width = (a.classes + 7) / 8 * 8;
    if (width <= kShapeCounts) {
        const int64_t most = kShapeCounts / width, want = (a.rows + 1023) / 1024;
        s.group = (int)(want < most ? want : most);
        s.parts = 1;
        s.part = width;
    } else {
        const int64_t want = (a.classes * a.rows / 1024 + 2047) / 2048 * 2048;
        s.group = 1;
        s.part = want < 2048 ? 2048 : want < kShapeCounts ? want : kShapeCounts;
        s.parts = (int)((a.classes + s.part - 1) / s.part);
    }
    const int64_t blocks = (a.rows + s.group - 1) / s.group * s.parts;
    SD_REQUIRE(blocks < (1ll << 31), "%s: %lld rows of %lld classes are too many for one call", who, (long long)a.rows, (long long)a.classes);
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto launch = [&](auto allowed, auto with_history) {
            if (grad) hipLaunchKernelGGL((shape_kernel<T, allowed.value, with_history.value, true>), dim3((unsigned)blocks), dim3(256), 0, stream, a, s);
            else hipLaunchKernelGGL((shape_kernel<T, allowed.value, with_history.value, false>), dim3((unsigned)blocks), dim3(256), 0, stream, a, s);
        };
        const auto with = [&](auto allowed) { history ? launch(allowed, std::true_type()) : launch(allowed, std::false_type()); };
        if (!s.allowed) with(std::integral_constant<int, kAll>());
        else if (c->allowed_kind == kFlags) with(std::integral_constant<int, kFlags>());
        else with(std::integral_constant<int, kBits>());
    });
    return check_launch("shape_kernel");
}

}  // namespace sd

using namespace sd;

extern "C" int sd_constrain_logits(const sd_logit_rows* rows, const sd_constraints* constraints, void* out, sd_stream_t stream) {
    sd::CallGuard call_guard;
    return shape_logits("constrain_logits", rows, constraints, nullptr, out, static_cast<hipStream_t>(stream));
}

extern "C" int sd_constrain_gradient(const sd_logit_rows* rows, const sd_constraints* constraints, const void* grad_output, void* grad, sd_stream_t stream) {
    sd::CallGuard call_guard;
    SD_REQUIRE(grad_output, "constrain_gradient: null gradient");
    return shape_logits("constrain_gradient", rows, constraints, grad_output, grad, static_cast<hipStream_t>(stream));
}
