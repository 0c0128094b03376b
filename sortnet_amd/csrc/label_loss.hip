// Losses on the log probability of a label: row r of the logits z has
//   top = max_v z[v], sum = sum_v exp(z[v] - top), lp = z[label] - top - log(sum), and d lp / d z[v] = [v = label] - exp(z[v] - top) / sum.
// A loss is a function of the lp's, so its gradient is weight_r ([v = label] - softmax[v]) with one weight per row; what differs
// from loss to loss is done per row (finish_row) and per answer (the kernels of sums), and the passes over the logits are
// shared.  Both passes are bound by the bytes of the logits, and by the launches where there are few.
// The running maximum starts at -inf and is used as max(., -FLT_MAX), so that a row's leading -inf (classes that are masked out) neither
// make a NaN nor count; a row of nothing else has the log probability NaN, as have rows with +inf or NaN.
// All sums have a fixed order: results are the same in every call.
#include <cfloat>
#include "label_rows.h"

namespace sd {

constexpr int kUnroll = 4;          // 16-byte loads of a work-item that are on their way together
constexpr int kGroupVecs = 8;       // vectors per lane up to which a row is read by (a part of) one wavefront
constexpr int64_t kMostBlocks = 1 << 22;

struct Rows {
    const void* logits;
    const int64_t* labels;
    int64_t rows, classes, outer_stride, inner_stride, ignore;
    uint32_t inner;
};

enum { kValues = 0, kPreference = 1, kPolicy = 2 };

// what happens to a row once its statistics are known
struct Finish {
    int kind;
    float* log_probs;       // values, preference
    float2* stats;          // (top, 1 / sum), what the gradient needs (or null)
    float* weight;          // preference: cleared (rows of no answer keep that), policy: d loss_r / d lp
    float4* terms;          // policy: surrogate, divergence, clipped, kept
    const float *old, *advantage, *ref;
    int64_t advantage_outer, advantage_inner;
    float low, high, kl;
    uint32_t* ticket;       // cleared for the kernel of sums behind this one (or null)
};

template <class T> __device__ __forceinline__ const T* row_start(const Rows& a, int64_t r) {
    const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
    return static_cast<const T*>(a.logits) + o * a.outer_stride + i * a.inner_stride;
}

__device__ __forceinline__ float finite(float top) { return fmaxf(top, -FLT_MAX); }

// (top, sum) of two parts of a row
template <class T> __device__ __forceinline__ void join(float& top, float& sum, float top2, float sum2) {
    const float t = fmaxf(top, top2);
    sum = sum * Elem<T>::exp(finite(top) - finite(t)) + sum2 * Elem<T>::exp(finite(top2) - finite(t));
    top = t;
}

template <class T, int N> __device__ __forceinline__ void take(const float (&f)[N], float& top, float& sum) {
    float t = top;
    #pragma unroll
    for (int i = 0; i < N; i++) t = fmaxf(t, f[i]);
    const float b = finite(t);
    float s = sum * Elem<T>::exp(finite(top) - b);
    #pragma unroll
    for (int i = 0; i < N; i++) s += Elem<T>::exp(f[i] - b);
    top = t;
    sum = s;
}

// (top, sum) of this work-item's share of p[0 .. n), which `lanes` work-items read together
template <class T> __device__ __forceinline__ void scan(const T* p, int64_t n, int lane, int lanes, float& top, float& sum) {
    constexpr int V = Elem<T>::kVec;
    const int64_t full = n / V;
    int64_t i = lane;
    for (; i + (int64_t)(kUnroll - 1) * lanes < full; i += (int64_t)kUnroll * lanes) {
        u32x4 v[kUnroll];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) v[k] = load16(p + (i + (int64_t)k * lanes) * V);
        float f[kUnroll * V];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) Elem<T>::unpack(v[k], reinterpret_cast<float (&)[V]>(f[k * V]));
        take<T>(f, top, sum);
    }
    for (; i < full; i += lanes) {
        float f[V];
        Elem<T>::unpack(load16(p + i * V), f);
        take<T>(f, top, sum);
    }
    for (int64_t j = full * V + lane; j < n; j += lanes) {
        const float f[1] = {Elem<T>::get(p[j])};
        take<T>(f, top, sum);
    }
}

// one work-item per row, with the row's top and sum
template <class T> __device__ void finish_row(const Rows& a, const Finish& e, int64_t r, float top, float sum) {
    const int64_t label = a.labels[r];
    const bool kept = label != a.ignore, known = label >= 0 && label < a.classes;
    float lp = 0.f;
    if (kept) {
        top = finite(top);
        // a label that names no class has no log probability
        lp = known ? Elem<T>::get(row_start<T>(a, r)[label]) - top - logf(sum) : __builtin_nanf("");
    }
    if (e.stats) e.stats[r] = make_float2(top, 1.f / sum);
    if (e.kind != kPolicy) {
        e.log_probs[r] = lp;
        if (e.weight) e.weight[r] = 0.f;
        return;
    }
    float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
    float w = 0.f;
    if (kept) {
        const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
        const float adv = e.advantage[o * e.advantage_outer + i * e.advantage_inner];
        const float ratio = expf(lp - e.old[r]);
        const float held = ratio < e.low ? e.low : ratio > e.high ? e.high : ratio;
        const float free = ratio * adv, bounded = held * adv;
        const bool clipped = bounded < free;
        t.x = -(clipped ? bounded : free);
        t.z = clipped ? 1.f : 0.f;
        t.w = 1.f;
        w = clipped ? 0.f : -free;
        if (e.kl != 0.f) {
            const float apart = e.ref[r] - lp, grown = expm1f(apart);
            t.y = grown - apart;
            w -= e.kl * grown;
        }
    }
    e.terms[r] = t;
    if (e.weight) e.weight[r] = w;
}

// Rows of up to kGroupVecs vectors per lane of a wavefront: 2^shift lanes to a row.
template <class T> __global__ void __launch_bounds__(256) label_rows_kernel(Rows a, Finish e, int shift) {
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    const int lanes = 1 << shift, lane = threadIdx.x & (lanes - 1), per = 256 >> shift;
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += (int64_t)gridDim.x * per) {
        float top = -INFINITY, sum = 0.f;
        if (a.labels[r] != a.ignore) scan(row_start<T>(a, r), a.classes, lane, lanes, top, sum);
        else top = 0.f, sum = 1.f;
        for (int o = lanes >> 1; o > 0; o >>= 1) {
            const float t = __shfl_xor(top, o), s = __shfl_xor(sum, o);
            join<T>(top, sum, t, s);
        }
        if (lane == 0) finish_row<T>(a, e, r, top, sum);
    }
}

// Longer rows: a workgroup per row, or per one of `splits` parts of a row, which then leaves its (top, sum) for join_rows_kernel.
template <class T> __global__ void __launch_bounds__(256) label_long_rows_kernel(Rows a, Finish e, int splits, int64_t part, float2* parts) {
    __shared__ float2 waves[4];
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = splits == 1 ? b : b / splits, c0 = (b - r * splits) * part;
        const int64_t n = a.classes - c0 < part ? a.classes - c0 : part;
        float top = -INFINITY, sum = 0.f;
        const bool kept = a.labels[r] != a.ignore;      // (the whole workgroup's)
        if (kept) {
            scan(row_start<T>(a, r) + c0, n, threadIdx.x, 256, top, sum);
            for (int o = 32; o > 0; o >>= 1) {
                const float t = __shfl_xor(top, o), s = __shfl_xor(sum, o);
                join<T>(top, sum, t, s);
            }
            if (lane == 0) waves[wave] = make_float2(top, sum);
            __syncthreads();
            if (threadIdx.x == 0)
                for (int k = 1; k < 4; k++) join<T>(top, sum, waves[k].x, waves[k].y);
            __syncthreads();
        } else top = 0.f, sum = 1.f;
        if (threadIdx.x == 0) {
            if (splits == 1) finish_row<T>(a, e, r, top, sum);
            else parts[b] = make_float2(top, sum);
        }
    }
}

// a wavefront per row joins the parts of label_long_rows_kernel
template <class T> __global__ void __launch_bounds__(256) join_rows_kernel(Rows a, Finish e, int splits, const float2* parts) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * 4) {
        float top = -INFINITY, sum = 0.f;
        if (a.labels[r] != a.ignore) {
            for (int k = lane; k < splits; k += 64) join<T>(top, sum, parts[r * splits + k].x, parts[r * splits + k].y);
            for (int o = 32; o > 0; o >>= 1) {
                const float t = __shfl_xor(top, o), s = __shfl_xor(sum, o);
                join<T>(top, sum, t, s);
            }
        } else top = 0.f, sum = 1.f;
        if (lane == 0) finish_row<T>(a, e, r, top, sum);
    }
}

// ---- gradient ------------------------------------------------------------------------------------------------------------
struct Gradient {
    const float2* stats;
    const float* weight;
    const float *scale, *scale2;    // one number each that every weight is multiplied by (or null)
    void* grad;                     // rows one behind the other
};

__device__ __forceinline__ float row_weight(const Rows& a, const Gradient& g, int64_t r, int64_t label) {
    if (label == a.ignore) return 0.f;
    if (label < 0 || label >= a.classes) return __builtin_nanf("");
    float w = g.weight[r];
    if (g.scale) w *= *g.scale;
    if (g.scale2) w *= *g.scale2;
    return w;
}

// N values from column c on
template <class T, int N> __device__ __forceinline__ void slopes(float (&f)[N], float2 st, float w, int64_t c, int64_t label) {
    #pragma unroll
    for (int i = 0; i < N; i++) f[i] = -(Elem<T>::exp(f[i] - st.x) * st.y) * w;
    const uint64_t at = (uint64_t)(label - c);
    if (at < N) {
        #pragma unroll
        for (int i = 0; i < N; i++) f[i] += i == (int)at ? w : 0.f;
    }
}

// columns [c0, c1) of a row, c0 a multiple of the vector's length; a row of weight 0 (ignored, clipped, or of no answer) is not read
template <class T> __device__ __forceinline__ void grad_row(const Rows& a, const Gradient& g, int64_t r, int64_t c0, int64_t c1, int lane, int lanes) {
    constexpr int V = Elem<T>::kVec;
    const int64_t label = a.labels[r];
    const float w = row_weight(a, g, r, label);
    const T* src = row_start<T>(a, r);
    T* dst = static_cast<T*>(g.grad) + r * a.classes;
    const int64_t full = c1 / V;
    if (w == 0.f) {
        for (int64_t i = c0 / V + lane; i < full; i += lanes) store16(dst + i * V, u32x4{0u, 0u, 0u, 0u});
        for (int64_t j = full * V + lane; j < c1; j += lanes) dst[j] = T{};
        return;
    }
    const float2 st = g.stats[r];
    int64_t i = c0 / V + lane;
    for (; i + (int64_t)(kUnroll - 1) * lanes < full; i += (int64_t)kUnroll * lanes) {
        u32x4 v[kUnroll];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) v[k] = load16(src + (i + (int64_t)k * lanes) * V);
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const int64_t c = (i + (int64_t)k * lanes) * V;
            float f[V];
            Elem<T>::unpack(v[k], f);
            slopes<T>(f, st, w, c, label);
            store16(dst + c, Elem<T>::pack(f));
        }
    }
    for (; i < full; i += lanes) {
        float f[V];
        Elem<T>::unpack(load16(src + i * V), f);
        slopes<T>(f, st, w, i * V, label);
        store16(dst + i * V, Elem<T>::pack(f));
    }
    for (int64_t j = full * V + lane; j < c1; j += lanes) {
        float f[1] = {Elem<T>::get(src[j])};
        slopes<T>(f, st, w, j, label);
        dst[j] = Elem<T>::put(f[0]);
    }
}

template <class T> __global__ void __launch_bounds__(256) label_gradient_kernel(Rows a, Gradient g, int shift) {
    const int lanes = 1 << shift, lane = threadIdx.x & (lanes - 1), per = 256 >> shift;
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += (int64_t)gridDim.x * per)
        grad_row<T>(a, g, r, 0, a.classes, lane, lanes);
}

template <class T> __global__ void __launch_bounds__(256) label_long_gradient_kernel(Rows a, Gradient g, int splits, int64_t part) {
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = b / splits, c0 = (b - r * splits) * part;
        grad_row<T>(a, g, r, c0, a.classes - c0 < part ? a.classes : c0 + part, threadIdx.x, 256);
    }
}

// ---- sums over rows ---------------------------------------------------------------------------------------------------------
__device__ __forceinline__ double wave_total(double v) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
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

struct Pairs {
    const float *log_probs, *ref;
    const int64_t* labels;
    int64_t ignore, rows, tokens;
    const int *offsets32;           // where the answers start and the last one ends; both null: `tokens` rows to an answer
    const int64_t* offsets64;
    int pairs;
    double beta, smoothing;
    float *weight, *rewards, *loss;
    double* parts;                  // one per workgroup
    uint32_t* ticket;
};

__device__ __forceinline__ int64_t answer_start(const Pairs& a, int64_t k) {
    const int64_t at = a.offsets32 ? a.offsets32[k] : a.offsets64 ? a.offsets64[k] : k * a.tokens;
    return at < 0 ? 0 : at > a.rows ? a.rows : at;
}

// A wavefront per pair: x = beta (chosen - rejected), the sums of lp - ref over the rows of the two answers, in 64 bits; then the
// pair's loss and the weight of its rows.
__global__ void __launch_bounds__(256) preference_kernel(Pairs a) {
    __shared__ double waves[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double loss = 0.0;
    for (int64_t pair = (int64_t)blockIdx.x * 4 + wave; pair < a.pairs; pair += (int64_t)gridDim.x * 4) {
        double reward[2];
        int64_t from[2], until[2];
        #pragma unroll
        for (int k = 0; k < 2; k++) {
            from[k] = answer_start(a, pair + k * (int64_t)a.pairs);
            until[k] = answer_start(a, pair + k * (int64_t)a.pairs + 1);
            double s = 0.0;
            #pragma unroll 4
            for (int64_t r = from[k] + lane; r < until[k]; r += 64)
                if (a.labels[r] != a.ignore) s += (double)(a.log_probs[r] - a.ref[r]);
            reward[k] = a.beta * wave_total(s);
            if (lane == 0) a.rewards[pair + k * (int64_t)a.pairs] = (float)reward[k];
        }
        const double x = reward[0] - reward[1], small = exp(-fabs(x)), tail = log1p(small);
        // -log sigma(x) = max(-x, 0) + log(1 + exp(-|x|))
        double l = (1.0 - a.smoothing) * ((x < 0.0 ? -x : 0.0) + tail);
        if (a.smoothing != 0.0) l += a.smoothing * ((x > 0.0 ? x : 0.0) + tail);
        loss += l;
        const double up = (x < 0.0 ? small : 1.0) / (1.0 + small), down = (x < 0.0 ? 1.0 : small) / (1.0 + small);   // sigma(x), sigma(-x)
        const float slope = (float)(-a.beta / a.pairs * ((1.0 - a.smoothing) * down - a.smoothing * up));
        if (a.weight) {
            #pragma unroll
            for (int k = 0; k < 2; k++)
                for (int64_t r = from[k] + lane; r < until[k]; r += 64)
                    if (a.labels[r] != a.ignore) a.weight[r] = k ? -slope : slope;
        }
    }
    if (lane == 0) waves[wave] = loss;
    __syncthreads();
    if (threadIdx.x == 0) publish(a.parts + blockIdx.x, waves[0] + waves[1] + waves[2] + waves[3]);
    if (!last_workgroup(a.ticket) || wave != 0) return;
    double total = 0.0;
    for (int k = lane; k < (int)gridDim.x; k += 64) total += published(a.parts + k);
    total = wave_total(total);
    if (lane == 0) *a.loss = (float)(total / a.pairs);
}

// Means of the policy's terms over the kept rows (over one where there are none); `scale` = 1 / that number.
__global__ void __launch_bounds__(256) policy_sums_kernel(const float4* terms, int64_t rows, double kl, float* loss, float* stats, float* scale,
                                                          double* parts, uint32_t* ticket) {
    __shared__ double waves[4][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    #pragma unroll 4
    for (int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x; r < rows; r += (int64_t)gridDim.x * 256) {
        const float4 t = terms[r];
        s[0] += t.x; s[1] += t.y; s[2] += t.z; s[3] += t.w;
    }
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        s[k] = wave_total(s[k]);
        if (lane == 0) waves[wave][k] = s[k];
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        #pragma unroll
        for (int k = 0; k < 4; k++) publish(parts + 4 * blockIdx.x + k, waves[0][k] + waves[1][k] + waves[2][k] + waves[3][k]);
    }
    if (!last_workgroup(ticket) || wave != 0) return;
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        s[k] = 0.0;
        for (int b = lane; b < (int)gridDim.x; b += 64) s[k] += published(parts + 4 * b + k);
        s[k] = wave_total(s[k]);
    }
    if (lane == 0) {
        const double count = s[3] > 1.0 ? s[3] : 1.0;
        *loss = (float)((s[0] + kl * s[1]) / count);
        stats[0] = (float)(s[0] / count);
        stats[1] = (float)(s[1] / count);
        stats[2] = (float)(s[2] / count);
        *scale = (float)(1.0 / count);
    }
}

// ---- host -----------------------------------------------------------------------------------------------------------------
namespace {

constexpr int kPairBlocks = 256, kSumBlocks = 128;

int vec_of(int dtype) { return dtype == SD_FLOAT32 ? 4 : 8; }

// lanes of a wavefront that read a row together (as a power of two), or -1: a row is read by whole workgroups
int group_shift(int64_t classes, int vec) {
    const int64_t vecs = (classes + vec - 1) / vec;
    if (vecs > 64 * kGroupVecs) return -1;
    int s = 0;
    while (s < 6 && (1 << s) < vecs) s++;
    return s;
}

// Parts of a long row: so many that there are 2048 workgroups (eight for each compute unit), none with less than one vector per work-item.
int row_splits(int64_t rows, int64_t classes, int vec) {
    const int64_t want = (2048 + rows - 1) / rows, most = (classes + 256 * vec - 1) / (256 * vec);
    return (int)(want < most ? want : most);
}

int64_t part_of(int64_t classes, int splits, int vec) {
    const int64_t step = 256 * vec, n = (classes + splits - 1) / splits;
    return (n + step - 1) / step * step;
}

unsigned blocks_for(int64_t n) { return (unsigned)(n < kMostBlocks ? n : kMostBlocks); }

// scratch of a call: the ticket, sums of workgroups, and then what follows
constexpr int64_t kSumFloats = 4 + 2 * (kPairBlocks > 4 * kSumBlocks ? kPairBlocks : 4 * kSumBlocks);

int check_rows(const sd_label_rows* in, const char* who, Rows* a) {
    SD_REQUIRE(in, "%s: null rows", who);
    SD_REQUIRE(in->dtype == SD_FLOAT32 || in->dtype == SD_BFLOAT16 || in->dtype == SD_FLOAT16, "%s: dtype=%d is none of SD_FLOAT32, SD_BFLOAT16, SD_FLOAT16", who, in->dtype);
    SD_REQUIRE(in->rows > 0 && in->rows < (1ll << 31), "%s: rows=%lld outside 1..2^31-1", who, (long long)in->rows);
    SD_REQUIRE(in->classes > 0 && in->classes < (1ll << 31), "%s: classes=%lld outside 1..2^31-1", who, (long long)in->classes);
    SD_REQUIRE(in->inner > 0 && in->rows % in->inner == 0 && in->inner < (1ll << 31), "%s: inner=%lld does not divide rows=%lld", who, (long long)in->inner, (long long)in->rows);
    SD_REQUIRE(in->logits && in->labels, "%s: null logits or labels", who);
    *a = Rows{in->logits, in->labels, in->rows, in->classes, in->outer_stride, in->inner_stride, in->ignore_index, (uint32_t)in->inner};
    return SD_OK;
}

int64_t split_floats(const sd_label_rows* in) {
    const int vec = vec_of(in->dtype);
    if (group_shift(in->classes, vec) >= 0) return 0;
    const int splits = row_splits(in->rows, in->classes, vec);
    return splits > 1 ? 2 * in->rows * splits : 0;
}

int launch_rows(const sd_label_rows* in, const Rows& a, const Finish& e, float* parts, hipStream_t stream) {
    const int vec = vec_of(in->dtype), shift = group_shift(a.classes, vec);
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (shift >= 0) {
            const int per = 256 >> shift;
            hipLaunchKernelGGL(label_rows_kernel<T>, dim3(blocks_for((a.rows + per - 1) / per)), dim3(256), 0, stream, a, e, shift);
            return;
        }
        int splits = row_splits(a.rows, a.classes, vec);
        const int64_t part = part_of(a.classes, splits, vec);
        splits = (int)((a.classes + part - 1) / part);
        float2* out = reinterpret_cast<float2*>(parts);
        hipLaunchKernelGGL(label_long_rows_kernel<T>, dim3(blocks_for(a.rows * splits)), dim3(256), 0, stream, a, e, splits, part, out);
        if (splits > 1) hipLaunchKernelGGL(join_rows_kernel<T>, dim3(blocks_for((a.rows + 3) / 4)), dim3(256), 0, stream, a, e, splits, out);
    });
    return check_launch("label_rows_kernel");
}

}  // namespace

}  // namespace sd

using namespace sd;

extern "C" int64_t sd_label_scratch(const sd_label_rows* in) {
    Rows a;
    if (check_rows(in, "label_scratch", &a) != SD_OK) return -1;
    return kSumFloats + split_floats(in) + 4 * in->rows;
}

extern "C" int sd_label_log_probs(const sd_label_rows* in, float* log_probs, float* stats, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "label_log_probs", &a)) return rc;
    SD_REQUIRE(log_probs && scratch, "label_log_probs: null output or scratch");
    Finish e{};
    e.kind = kValues;
    e.log_probs = log_probs;
    e.stats = reinterpret_cast<float2*>(stats);
    return launch_rows(in, a, e, scratch + kSumFloats, static_cast<hipStream_t>(stream));
}

extern "C" int sd_preference_loss(const sd_label_rows* in, const float* ref, const void* offsets, int offset_bytes, int64_t tokens, int pairs, double beta, double smoothing,
                                  float* stats, float* weight, float* rewards, float* loss, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "preference_loss", &a)) return rc;
    SD_REQUIRE(ref && rewards && loss && scratch, "preference_loss: null argument");
    SD_REQUIRE(!stats == !weight, "preference_loss: the gradient needs both stats and weight");
    SD_REQUIRE(pairs > 0, "preference_loss: pairs=%d must be positive", pairs);
    SD_REQUIRE(!offsets || offset_bytes == 4 || offset_bytes == 8, "preference_loss: offsets of %d bytes", offset_bytes);
    SD_REQUIRE(offsets || (tokens > 0 && 2 * (int64_t)pairs * tokens == a.rows), "preference_loss: %d pairs of answers of %lld rows are not %lld rows", pairs, (long long)tokens, (long long)a.rows);
    SD_REQUIRE(smoothing >= 0.0 && smoothing < 0.5, "preference_loss: label_smoothing=%g outside 0..0.5", smoothing);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t parts = split_floats(in);
    Finish e{};
    e.kind = kPreference;
    e.log_probs = scratch + kSumFloats + parts;
    e.stats = reinterpret_cast<float2*>(stats);
    e.weight = weight;
    e.ticket = reinterpret_cast<uint32_t*>(scratch);
    if (int rc = launch_rows(in, a, e, scratch + kSumFloats, s)) return rc;
    Pairs p{e.log_probs, ref, a.labels, a.ignore, a.rows, tokens, offset_bytes == 4 ? static_cast<const int*>(offsets) : nullptr,
            offset_bytes == 8 ? static_cast<const int64_t*>(offsets) : nullptr, pairs, beta, smoothing, weight, rewards, loss,
            reinterpret_cast<double*>(scratch + 4), e.ticket};
    const int blocks = (pairs + 3) / 4 < kPairBlocks ? (pairs + 3) / 4 : kPairBlocks;
    hipLaunchKernelGGL(preference_kernel, dim3(blocks), dim3(256), 0, s, p);
    return check_launch("preference_kernel");
}

extern "C" int sd_policy_loss(const sd_label_rows* in, const float* old_log_probs, const float* advantages, int64_t advantage_outer, int64_t advantage_inner,
                              const float* ref, double clip_low, double clip_high, double kl, float* stats, float* weight, float* scale, float* loss, float* means,
                              float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "policy_loss", &a)) return rc;
    SD_REQUIRE(old_log_probs && advantages && scale && loss && means && scratch, "policy_loss: null argument");
    SD_REQUIRE(!stats == !weight, "policy_loss: the gradient needs both stats and weight");
    SD_REQUIRE(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0, "policy_loss: clip=%g, clip_high=%g: need 0 <= clip <= 1 and 0 <= clip_high", clip_low, clip_high);
    SD_REQUIRE(ref || kl == 0.0, "policy_loss: a KL term needs reference log probabilities");
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int64_t parts = split_floats(in);
    Finish e{};
    e.kind = kPolicy;
    e.stats = reinterpret_cast<float2*>(stats);
    e.weight = weight;
    e.terms = reinterpret_cast<float4*>(scratch + kSumFloats);          // (16-byte aligned: before the parts)
    e.old = old_log_probs; e.advantage = advantages; e.ref = ref;
    e.advantage_outer = advantage_outer; e.advantage_inner = advantage_inner;
    e.low = (float)(1.0 - clip_low); e.high = (float)(1.0 + clip_high); e.kl = (float)kl;
    e.ticket = reinterpret_cast<uint32_t*>(scratch);
    if (int rc = launch_rows(in, a, e, scratch + kSumFloats + 4 * a.rows, s)) return rc;
    const int64_t want = (a.rows + 2047) / 2048;
    hipLaunchKernelGGL(policy_sums_kernel, dim3((unsigned)(want < kSumBlocks ? want : kSumBlocks)), dim3(256), 0, s, e.terms, a.rows, kl, loss, means, scale,
                       reinterpret_cast<double*>(scratch + 4), e.ticket);
    return check_launch("policy_sums_kernel");
}

extern "C" int sd_label_gradient(const sd_label_rows* in, const float* stats, const float* weight, const float* scale, const float* scale2, void* grad, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "label_gradient", &a)) return rc;
    SD_REQUIRE(stats && weight && grad, "label_gradient: null argument");
    const Gradient g{reinterpret_cast<const float2*>(stats), weight, scale, scale2, grad};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int vec = vec_of(in->dtype), shift = group_shift(a.classes, vec);
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (shift >= 0) {
            const int per = 256 >> shift;
            hipLaunchKernelGGL(label_gradient_kernel<T>, dim3(blocks_for((a.rows + per - 1) / per)), dim3(256), 0, s, a, g, shift);
            return;
        }
        const int64_t part = 256 * vec * kUnroll;
        const int splits = (int)((a.classes + part - 1) / part);
        hipLaunchKernelGGL(label_long_gradient_kernel<T>, dim3(blocks_for(a.rows * splits)), dim3(256), 0, s, a, g, splits, part);
    });
    return check_launch("label_gradient_kernel");
}
