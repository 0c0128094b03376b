// Distillation from a teacher's top logits.  The teacher gives row r some classes c_j with logits t_j and, as one more outcome, the log-sum `rest` of
// its other logits; the student's row z has the same outcomes.  With a temperature T, in the outcomes' softmaxes
//   q_j ~ exp(t_j / T), q_r ~ exp(rest);   p_j ~ exp(z[c_j] / T), p_r ~ S,   S = sum over the classes that are in no entry of exp(z[v] / T),
// the divergence is D = sum_j q_j (log q_j - log p_j) + q_r (log q_r - log p_r), the loss weight T^2 times the mean of D, and
//   d D / d (z[v] / T) = p_v - sum of the q_j with c_j = v   for a class of an entry,   (p_r - q_r) exp(z[v] / T) / S   for another one.
// S is formed without the entries' classes, not as a difference, so that what the student gives the others keeps its digits however small it is.
// There are few outcomes per row: they are in 64 bits.  Both passes are bound by the bytes of the logits, and by the launches where there are few.
// A class that stands in several entries is one class: it counts once in p and takes the sum of their q.
// All sums have a fixed order: results are the same in every call.
#include <climits>
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kMostEntries = SD_MOST_TOP;   // of a row: one per work-item of a workgroup
constexpr int kVectors = 8;                 // 16-byte vectors of a long row that a work-item holds at a time
static_assert(kMostEntries <= 256, "a work-item per entry");

// The teacher's rows
struct Lists {
    const void *values, *classes;
    const float* rest;
    int k, dtype, wide;         // wide: classes are int64 instead of int32
    __device__ __forceinline__ int64_t cls(int64_t at) const {
        return wide ? static_cast<const int64_t*>(classes)[at] : (int64_t)static_cast<const int*>(classes)[at];
    }
    __device__ __forceinline__ float value(int64_t at) const {
        if (dtype == SD_FLOAT32) return static_cast<const float*>(values)[at];
        if (dtype == SD_BFLOAT16) return Elem<bf16>::get(static_cast<const bf16*>(values)[at]);
        return Elem<fp16>::get(static_cast<const fp16*>(values)[at]);
    }
};

// z / T as an exponent of 2: log2(e) / T is the sum of two positive numbers, the first rounded down (see exp_of)
struct Temper { double inverse; float high, low; };
__device__ __forceinline__ float exp_at(float v, const Temper& t) { return __builtin_amdgcn_exp2f(fmaf(v, t.high, v * t.low)); }
// the same for what is stored in T (see exp_to in label_loss.hip)
template <class T> __device__ __forceinline__ float exp_stored(float v, const Temper& t) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(v * t.high);
    else return exp_at(v, t);
}

struct Outcome {
    float2* stats;              // (largest of the others, (p_r - q_r) / S with S relative to it), what the gradient needs (or null)
    float* entries;             // p_v - sum of q, one for each entry (or null)
    float *divergences, *kept;
    uint32_t* ticket;           // cleared for the kernel of sums behind this one
};

struct Others { float top; double sum; };     // of the classes in no entry: sum of exp((z - top) / T)

// What makes a row count, of one of its entries: 1 for an entry, 2 for one that is not -inf.  A row counts, and is read, that has an entry and an entry or
// a rest above -inf.
__device__ __forceinline__ int says(const Lists& l, int64_t at) { return l.cls(at) < 0 ? 0 : l.value(at) != -INFINITY ? 3 : 1; }

// The end of row r by a group of 2^shift lanes of a wavefront, all of which call it.  repeats: a class may stand in several entries.
// Returns what stats receives.
template <class T> __device__ __forceinline__ float2 finish_row(const LogitRows& a, const Lists& l, const Temper& t, const Outcome& e, int64_t r, Others o, bool repeats,
                                                              int lane, int shift) {
    const int lanes = 1 << shift;
    const T* z = row_start<T>(a, r);
    float most_t = -INFINITY, most_z = -INFINITY, any = 0.f, live = 0.f, bad = 0.f;
    for (int j = lane; j < l.k; j += lanes) {
        const int64_t c = l.cls(r * l.k + j);
        if (c < 0) continue;
        const float v = l.value(r * l.k + j);
        any = 1.f;
        if (v != -INFINITY) live = 1.f;
        most_t = fmaxf(most_t, v);
        if (c >= a.classes || v != v) { bad = 1.f; continue; }
        const float u = Elem<T>::get(z[c]);
        most_z = fmaxf(most_z, u);
        if (u != u) bad = 1.f;
    }
    most_t = group_max(most_t, shift); most_z = group_max(most_z, shift); any = group_max(any, shift); live = group_max(live, shift);
    const double rest = l.rest ? (double)l.rest[r] : -INFINITY;
    if (rest != rest || o.sum != o.sum) bad = 1.f;
    bad = group_max(bad, shift);
    const double am = fmax((double)most_t * t.inverse, rest);
    if (any == 0.f || (live == 0.f && rest == -INFINITY)) {     // (see says)
        if (e.entries)
            for (int j = lane; j < l.k; j += lanes) e.entries[r * l.k + j] = 0.f;
        if (lane == 0) {
            e.divergences[r] = 0.f;
            e.kept[r] = 0.f;
            if (e.stats) e.stats[r] = make_float2(0.f, 0.f);
        }
        return make_float2(0.f, 0.f);
    }
    // the student's logits relative to the largest of all (beside it, however large, the logarithm of a sum keeps its digits)
    const double base = (double)fmaxf(most_z, finite(o.top));
    const auto tempered = [&](float u) { return ((double)u - base) * t.inverse; };
    const double log_s = o.sum > 0.0 ? log(o.sum) + tempered(finite(o.top)) : -INFINITY;
    const double um = fmax(tempered(most_z), log_s);
    // whether an entry before j has its class
    const auto repeated = [&](int j, int64_t c) {
        if (repeats)
            for (int i = 0; i < j; i++)
                if (l.cls(r * l.k + i) == c) return true;
        return false;
    };
    double sum_t = 0.0, sum_z = 0.0;
    for (int j = lane; j < l.k; j += lanes) {
        const int64_t c = l.cls(r * l.k + j);
        if (c < 0 || c >= a.classes) continue;
        sum_t += exp((double)l.value(r * l.k + j) * t.inverse - am);
        if (!repeated(j, c)) sum_z += exp(tempered(Elem<T>::get(z[c])) - um);
    }
    sum_t = group_total(sum_t, shift) + exp(rest - am);
    sum_z = group_total(sum_z, shift) + exp(log_s - um);
    if (bad != 0.f) sum_z = __builtin_nan("");
    const double log_t = log(sum_t), log_z = log(sum_z);
    double divergence = 0.0;
    for (int j = lane; j < l.k; j += lanes) {
        const int64_t c = l.cls(r * l.k + j);
        float slope = 0.f;
        if (c >= 0) {
            const bool inside = c < a.classes;
            const double at = (double)l.value(r * l.k + j) * t.inverse - am - log_t, az = (inside ? tempered(Elem<T>::get(z[c])) : 0.0) - um - log_z;
            double q = exp(at);
            if (q != 0.0) divergence += q * (at - az);
            if (repeats) {      // every entry of a class gets the same slope
                q = 0.0;
                for (int i = 0; i < l.k; i++)
                    if (l.cls(r * l.k + i) == c) q += exp((double)l.value(r * l.k + i) * t.inverse - am - log_t);
            }
            slope = (float)(exp(az) - q);
        }
        if (e.entries) e.entries[r * l.k + j] = slope;
    }
    divergence = group_total(divergence, shift);
    const double at = rest - am - log_t, az = log_s - um - log_z, q = exp(at);
    if (q != 0.0) divergence += q * (at - az);
    const float2 stats = make_float2(finite(o.top), o.sum > 0.0 || bad != 0.f ? (float)((exp(az) - q) / o.sum) : 0.f);
    if (lane == 0) {
        e.divergences[r] = (float)(divergence + (sum_z != sum_z ? sum_z : 0.0));
        e.kept[r] = 1.f;
        if (e.stats) e.stats[r] = stats;
    }
    return stats;
}

// ---- a workgroup reads a row ---------------------------------------------------------------------------------------------------
template <int N> __device__ __forceinline__ void take(const float (&f)[N], float& top, double& sum, const Temper& t) {
    float m = top, g[N];
    #pragma unroll
    for (int i = 0; i < N; i++) m = fmaxf(m, f[i]);
    const float b = finite(m);
    #pragma unroll
    for (int i = 0; i < N; i++) g[i] = exp_at(f[i] - b, t);
    sum = sum * (double)exp_at(finite(top) - b, t) + (double)tree(g);
    top = m;
}

template <class T> __global__ void __launch_bounds__(256) distill_rows_kernel(LogitRows a, Lists l, Temper t, Outcome e) {
    constexpr int V = Elem<T>::kVec, kWords = kVectors * V / 32, kSpan = 256 * kVectors * V;
    __shared__ uint32_t marks[256][kWords];
    __shared__ Others waves[4];
    __shared__ int repeats;
    if (blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T* p = row_start<T>(a, r);
        const int64_t cls = (int)threadIdx.x < l.k ? l.cls(r * l.k + threadIdx.x) : -1;
        if (threadIdx.x == 0) repeats = 0;
        float top = -INFINITY;
        double sum = 0.0;
        const int said = (int)threadIdx.x < l.k ? says(l, r * l.k + threadIdx.x) : 0;
        const bool entry = __syncthreads_or(said & 1), live = __syncthreads_or(said & 2);
        if (entry && (live || (l.rest && l.rest[r] != -INFINITY))) {
            for (int64_t c0 = 0; c0 < a.classes; c0 += kSpan) {
                #pragma unroll
                for (int w = 0; w < kWords; w++) marks[threadIdx.x][w] = 0u;
                __syncthreads();
                if (cls >= c0 && cls < c0 + kSpan && cls < a.classes) {
                    const int at = (int)(cls - c0), vec = at / V, bit = vec / 256 * V + at % V;
                    const uint32_t one = 1u << (bit & 31);
                    if (atomicOr(&marks[vec % 256][bit >> 5], one) & one) repeats = 1;
                }
                __syncthreads();
                #pragma unroll
                for (int k = 0; k < kVectors; k++) {
                    const int64_t c = c0 + (int64_t)(k * 256 + (int)threadIdx.x) * V;
                    float f[V];
                    if (c + V <= a.classes) Elem<T>::unpack(load16(p + c), f);
                    else {
                        #pragma unroll
                        for (int i = 0; i < V; i++) f[i] = c + i < a.classes ? Elem<T>::get(p[c + i]) : -INFINITY;
                    }
                    const uint32_t listed = marks[threadIdx.x][k * V / 32] >> (k * V & 31);
                    #pragma unroll
                    for (int i = 0; i < V; i++) f[i] = listed >> i & 1 ? -INFINITY : f[i];
                    take(f, top, sum, t);
                }
                __syncthreads();
            }
        }
        {   // all work-items' to the first wavefront
            const float m = group_max(top, 6);
            sum = group_total(sum * (double)exp_at(finite(top) - finite(m), t), 6);
            if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = Others{m, sum};
            __syncthreads();
            if (threadIdx.x < 64) {
                Others o{-INFINITY, 0.0};
                for (int w = 0; w < 4; w++) o.top = fmaxf(o.top, waves[w].top);
                for (int w = 0; w < 4; w++) o.sum += waves[w].sum * (double)exp_at(finite(waves[w].top) - finite(o.top), t);
                finish_row<T>(a, l, t, e, r, o, repeats != 0, threadIdx.x, 6);
            }
            __syncthreads();
        }
    }
}

// ---- the loss --------------------------------------------------------------------------------------------------------------------
// loss = weight T^2 mean of the divergences over the rows that count (0 where there are none), scale = weight T / their number
struct Mean { const float *divergences, *kept; int64_t rows; double loss_factor, scale_factor; float *loss, *scale; double* parts; uint32_t* ticket; };
__global__ void __launch_bounds__(1024) distill_mean_kernel(Mean m) {
    __shared__ double waves[16][2];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s[2] = {0.0, 0.0};
    #pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < m.rows; i += (int64_t)gridDim.x * 1024) { s[0] += (double)m.divergences[i]; s[1] += (double)m.kept[i]; }
    #pragma unroll
    for (int k = 0; k < 2; k++) {
        s[k] = wave_total(s[k]);
        if (lane == 0) waves[wave][k] = s[k];
    }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < 2; k++) {
        s[k] = 0.0;
        if (wave == 0) s[k] = wave_total(lane < 16 ? waves[lane][k] : 0.0);
    }
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) {
            publish(m.parts + 2 * blockIdx.x, s[0]);
            publish(m.parts + 2 * blockIdx.x + 1, s[1]);
        }
        if (!last_workgroup(m.ticket) || wave != 0) return;
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            s[k] = 0.0;
            for (int b = lane; b < (int)gridDim.x; b += 64) s[k] += published(m.parts + 2 * b + k);
            s[k] = wave_total(s[k]);
        }
    }
    if (threadIdx.x == 0) {
        const double count = s[1] > 1.0 ? s[1] : 1.0;
        *m.loss = (float)(m.loss_factor * s[0] / count);
        if (m.scale) *m.scale = (float)(m.scale_factor / count);
    }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------------------
struct Slopes { const float2* stats; const float* entries; const float *scale, *scale2; void* grad; };

// A workgroup writes `part` columns of a row, then those of its entries that lie there.
template <class T> __global__ void __launch_bounds__(256) distill_gradient_kernel(LogitRows a, Lists l, Temper t, Slopes g, int splits, int64_t part) {
    constexpr int V = Elem<T>::kVec;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = b / splits, c0 = (b - r * splits) * part, c1 = a.classes - c0 < part ? a.classes : c0 + part;
        const float2 st = g.stats[r];
        const float by = g.scale2 ? *g.scale * *g.scale2 : *g.scale, w = st.y * by;
        const T* src = row_start<T>(a, r);
        T* q = static_cast<T*>(g.grad) + r * a.classes;
        const int64_t full = c1 / V;
        for (int64_t i = c0 / V + threadIdx.x; i < full; i += 256) {
            float f[V];
            if (st.y == 0.f) {
                #pragma unroll
                for (int k = 0; k < V; k++) f[k] = 0.f;
            } else {
                Elem<T>::unpack(load16(src + i * V), f);
                #pragma unroll
                for (int k = 0; k < V; k++) f[k] = exp_stored<T>(f[k] - st.x, t) * w;
            }
            put_stream16(q + i * V, Elem<T>::pack(f));
        }
        for (int64_t j = full * V + threadIdx.x; j < c1; j += 256) q[j] = Elem<T>::put(st.y == 0.f ? 0.f : exp_stored<T>(Elem<T>::get(src[j]) - st.x, t) * w);
        __syncthreads();        // (the entries' values stand where these stood)
        if ((int)threadIdx.x < l.k) {
            const int64_t c = l.cls(r * l.k + threadIdx.x);
            if (c >= c0 && c < c1) q[c] = Elem<T>::put(g.entries[r * l.k + threadIdx.x] * by);
        }
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
namespace {

constexpr int kMeanBlocks = 128;

int check_lists(const sd_top_lists* in, const sd_logit_rows* rows, const char* who, Lists* l) {
    SD_REQUIRE(in && in->values && in->classes, "%s: null lists", who);
    SD_REQUIRE(in->k >= 1 && in->k <= kMostEntries, "%s: k=%lld entries for each row: 1..%d are possible", who, (long long)in->k, kMostEntries);
    SD_REQUIRE(in->dtype == SD_FLOAT32 || in->dtype == SD_BFLOAT16 || in->dtype == SD_FLOAT16, "%s: values of dtype=%d", who, in->dtype);
    SD_REQUIRE(in->class_bytes == 4 || in->class_bytes == 8, "%s: classes of %d bytes", who, in->class_bytes);
    SD_REQUIRE((reinterpret_cast<uintptr_t>(in->values) & (in->dtype == SD_FLOAT32 ? 3 : 1)) == 0 && (reinterpret_cast<uintptr_t>(in->classes) & (in->class_bytes - 1)) == 0 &&
               (reinterpret_cast<uintptr_t>(in->rest) & 3) == 0, "%s: lists are not aligned to their types", who);
    *l = Lists{in->values, in->classes, in->rest, (int)in->k, in->dtype, in->class_bytes == 8};
    return SD_OK;
}

int check_temper(double temperature, double weight, const char* who, Temper* t) {
    SD_REQUIRE(temperature >= 1e-4 && temperature <= 1e4, "%s: temperature=%g outside 1e-4..1e4", who, temperature);
    SD_REQUIRE(weight >= -FLT_MAX && weight <= FLT_MAX, "%s: weight=%g must be finite", who, weight);
    const double by = 1.4426950408889634074 / temperature;
    float high = (float)by;
    if ((double)high >= by) high = nextafterf(high, 0.f);
    *t = Temper{1.0 / temperature, high, (float)(by - (double)high)};
    return SD_OK;
}

}  // namespace

}  // namespace sd

using namespace sd;

// scratch: the ticket, sums of workgroups, a mark for each row that counts
static int64_t distill_floats(int64_t rows) { return 4 + 4 * kMeanBlocks + (rows + 3) / 4 * 4; }

extern "C" int64_t sd_distill_scratch(const sd_logit_rows* rows, int64_t k) {
    LogitRows a;
    if (check_logits(rows, "distill_scratch", &a) != SD_OK) return -1;
    if (k < 1 || k > kMostEntries) { set_error("distill_scratch: k=%lld entries for each row: 1..%d are possible", (long long)k, kMostEntries); return -1; }
    return distill_floats(a.rows);
}

extern "C" int sd_distill_loss(const sd_logit_rows* rows, const sd_top_lists* lists, double temperature, double weight, float* stats, float* entries, float* scale,
                               float* loss, float* divergences, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    Lists l;
    Temper t;
    if (int rc = check_logits(rows, "distill_loss", &a)) return rc;
    if (int rc = check_lists(lists, rows, "distill_loss", &l)) return rc;
    if (int rc = check_temper(temperature, weight, "distill_loss", &t)) return rc;
    SD_REQUIRE(loss && divergences && scratch, "distill_loss: null argument");
    SD_REQUIRE(!stats == !entries && !stats == !scale, "distill_loss: the gradient needs stats, entries and scale");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "distill_loss: stats must be aligned to 8 bytes, scratch to 16");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const Outcome e{reinterpret_cast<float2*>(stats), entries, divergences, scratch + 4 + 4 * kMeanBlocks, reinterpret_cast<uint32_t*>(scratch)};
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        hipLaunchKernelGGL(distill_rows_kernel<T>, dim3(blocks_for(a.rows)), dim3(256), 0, s, a, l, t, e);
    });
    if (int rc = check_launch("distill_rows_kernel")) return rc;
    const int64_t want = (a.rows + 16383) / 16384;
    const Mean m{divergences, e.kept, a.rows, weight * temperature * temperature, weight * temperature, loss, scale, reinterpret_cast<double*>(scratch + 4), e.ticket};
    hipLaunchKernelGGL(distill_mean_kernel, dim3((unsigned)(want < kMeanBlocks ? want : kMeanBlocks)), dim3(1024), 0, s, m);
    return check_launch("distill_mean_kernel");
}

extern "C" int sd_distill_gradient(const sd_logit_rows* rows, const sd_top_lists* lists, double temperature, const float* stats, const float* entries, const float* scale,
                                   const float* scale2, void* grad, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    Lists l;
    Temper t;
    if (int rc = check_logits(rows, "distill_gradient", &a)) return rc;
    if (int rc = check_lists(lists, rows, "distill_gradient", &l)) return rc;
    if (int rc = check_temper(temperature, 1.0, "distill_gradient", &t)) return rc;
    SD_REQUIRE(stats && entries && scale && grad, "distill_gradient: null argument");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (reinterpret_cast<uintptr_t>(grad) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0,
               "distill_gradient: stats must be aligned to 8 bytes, the gradient to its type");
    const Slopes g{reinterpret_cast<const float2*>(stats), entries, scale, scale2, grad};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t part = 256 * vec_of(rows->dtype) * 4;
    const int splits = (int)((a.classes + part - 1) / part);
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        hipLaunchKernelGGL(distill_gradient_kernel<T>, dim3(blocks_for(a.rows * splits)), dim3(256), 0, s, a, l, t, g, splits, part);
    });
    return check_launch("distill_gradient_kernel");
}
