// The k largest logits of each row in order (of equal ones the lower class first), their classes, and the log-sum of the others at a temperature:
//   rest = log sum over the classes that are not among the k of exp(z[v] / T)   (-inf where there are none).
// Values are compared by whole numbers in their order (order_of): NaN above all, -0 as 0.  With the class behind it, upside down, every logit
// has a number of its own, so the k largest are the same in every call.
#include <climits>
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kMostTop = SD_MOST_TOP;

__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}

struct Top {
    int k;
    double inverse;         // 1 / temperature
    void* values;
    int* classes;
    float* rest;
};

// exp((v - last) / T), v being at most `last`
__device__ __forceinline__ double share_of(float v, float last, double inverse) {
    return v == last ? (v == -INFINITY ? 0.0 : 1.0) : (double)expf((float)(((double)v - (double)last) * inverse));
}

// A workgroup per row: the k-th largest order bit by bit, each a pass over the row, then the k numbers, then the sum of the others.
template <class T> __global__ void __launch_bounds__(256) top_rows_kernel(LogitRows a, Top o) {
    __shared__ unsigned long long found[kMostTop];
    __shared__ int count, counts[4];
    __shared__ double sums[4];
    const int n = (int)a.classes, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* p = row_start<T>(a, r);
        uint32_t kth = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t least = kth | 1u << bit;
            int c = 0;
            for (int i = threadIdx.x; i < n; i += 256) c += order_of(Elem<T>::get(p[i])) >= least;
            for (int s = 32; s > 0; s >>= 1) c += __shfl_xor(c, s);
            if (lane == 0) counts[wave] = c;
            __syncthreads();
            if (counts[0] + counts[1] + counts[2] + counts[3] >= o.k) kth = least;
            __syncthreads();
        }
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
        const auto number = [&](float v, int i) { return (unsigned long long)order_of(v) << 32 | (uint32_t)~i; };
        for (int i = threadIdx.x; i < n; i += 256) {
            const float v = Elem<T>::get(p[i]);
            if (order_of(v) > kth) found[atomicAdd(&count, 1)] = number(v, i);
        }
        __syncthreads();
        const int above = count;
        // equal ones by class: 256 at a time, each behind those of the lanes and wavefronts before it
        int have = above;
        for (int i0 = 0; i0 < n && have < o.k; i0 += 256) {
            const int i = i0 + threadIdx.x;
            const bool equal = i < n && order_of(Elem<T>::get(p[i])) == kth;
            const unsigned long long lanes = __ballot(equal);
            if (lane == 0) counts[wave] = __popcll(lanes);
            __syncthreads();
            int at = have;
            for (int w = 0; w < wave; w++) at += counts[w];
            at += __popcll(lanes & ((1ull << lane) - 1ull));
            if (equal && at < o.k) found[at] = number(value_of(kth), i);
            have += counts[0] + counts[1] + counts[2] + counts[3];
            __syncthreads();
        }
        __syncthreads();
        __shared__ unsigned long long kth_number;
        if ((int)threadIdx.x < o.k) {
            const unsigned long long mine = found[threadIdx.x];
            int rank = 0;
            for (int j = 0; j < o.k; j++) rank += found[j] > mine;
            const int cls = (int)~(uint32_t)mine;
            static_cast<T*>(o.values)[r * o.k + rank] = p[cls];
            o.classes[r * o.k + rank] = cls;
            if (rank == o.k - 1) kth_number = mine;
        }
        __syncthreads();
        const unsigned long long last = kth_number;
        const float last_value = value_of((uint32_t)(last >> 32));
        double sum = 0.0;
        for (int i = threadIdx.x; i < n; i += 256) {
            const float v = Elem<T>::get(p[i]);
            if (v != v) sum = __builtin_nan("");
            else if (number(v, i) < last) sum += share_of(v, last_value, o.inverse);
        }
        sum = wave_total(sum);
        if (lane == 0) sums[wave] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            sum = sums[0] + sums[1] + sums[2] + sums[3];
            o.rest[r] = sum == 0.0 ? -INFINITY : (float)(log(sum) + (double)last_value * o.inverse);
        }
        __syncthreads();
    }
}

}  // namespace sd

using namespace sd;

extern "C" int64_t sd_top_scratch(const sd_logit_rows* rows, int64_t k) {
    LogitRows a;
    if (check_logits(rows, "top_scratch", &a) != SD_OK) return -1;
    if (k < 1 || k > kMostTop || k > a.classes) { set_error("top_scratch: k=%lld of %lld classes: 1..%d are possible", (long long)k, (long long)a.classes, kMostTop); return -1; }
    return 0;
}

extern "C" int sd_top_logits(const sd_logit_rows* rows, int64_t k, double temperature, void* values, int* classes, float* rest, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    if (int rc = check_logits(rows, "top_logits", &a)) return rc;
    SD_REQUIRE(k >= 1 && k <= kMostTop && k <= a.classes, "top_logits: k=%lld of %lld classes: 1..%d are possible", (long long)k, (long long)a.classes, kMostTop);
    SD_REQUIRE(temperature >= 1e-4 && temperature <= 1e4, "top_logits: temperature=%g outside 1e-4..1e4", temperature);
    SD_REQUIRE(values && classes && rest, "top_logits: null argument");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(values) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0 && ((reinterpret_cast<uintptr_t>(classes) | reinterpret_cast<uintptr_t>(rest)) & 3) == 0,
               "top_logits: results are not aligned to their types");
    (void)scratch;
    const Top o{(int)k, 1.0 / temperature, values, classes, rest};
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        hipLaunchKernelGGL(top_rows_kernel<T>, dim3(blocks_for(a.rows)), dim3(256), 0, static_cast<hipStream_t>(stream), a, o);
    });
    return check_launch("top_rows_kernel");
}
