// Losses on the log probability of a label: row r of the logits z has
//   top = max_v z[v], sum = sum_v exp(z[v] - top), lp = z[label] - top - log(sum), and d lp / d z[v] = [v = label] - exp(z[v] - top) / sum.
// A loss is a function of the lp's, so its gradient is weight_r ([v = label] - softmax[v]) with one weight per row; what differs
// from loss to loss is done per row (finish_row) and per answer (the kernels of sums), and the passes over the logits are
// shared.  Both passes are bound by the bytes of the logits, and by the launches where there are few.
// The running maximum starts at -inf and is used as max(., -FLT_MAX), so that a row's leading -inf (classes that are masked out) neither
// make a NaN nor count; a row of nothing else has the log probability NaN, as have rows with +inf or NaN.
// All sums have a fixed order: results are the same in every call.
#include <cfloat>
#include <climits>
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kUnroll = 4;          // 16-byte loads of a work-item of a long row that are on their way together
constexpr int kHeld = 8;            // 16-byte vectors of a short row that a lane holds, at most
constexpr int kHeldLong = 16 * 1024;    // and of a long row that a workgroup holds
constexpr int64_t kMostBlocks = 1 << 22;
constexpr int kShortBlocks = 4096;      // workgroups of short rows, at most
// Bytes of a FUSED short row from which its gradient is stored past the caches: us with and without, 262144 x 200 fp32 82 / 95,
// 65536 x 1000 bf16 60 / 62; 1048576 x 10 fp32, whose rows share cache lines, 53 / 35.
constexpr int kStreamRow = 512;

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
    float* out;             // values: log probabilities; preference: log probability - ref
    float2* stats;          // (top, 1 / sum), what the gradient needs (or null)
    float* weight;          // preference: cleared (rows of no answer keep that), policy: d loss_r / d lp (or null)
    double* terms;          // policy: sums of surrogate, divergence, clipped and kept rows, four numbers per workgroup or long row
    const float *old, *advantage, *ref;
    int64_t advantage_outer, advantage_inner;
    float low, high, kl;
    uint32_t* ticket;       // cleared for the kernel of sums behind this one (or null)
};

struct Gradient {
    const float2* stats;
    const float* weight;
    const float *scale, *scale2;    // one number each that every weight is multiplied by (or null)
    void* grad;                     // rows one behind the other
    bool unless_one;                // nothing is done where *scale2 is 1
};

template <class T> __device__ __forceinline__ const T* row_start(const Rows& a, int64_t r) {
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
// The same for what is stored in T: one product will do where that has 16 bits, whose half step is 2^-11 of a value at least.  (4096 x 131072 bf16,
// policy with its gradient: 437 us with two everywhere, 425 so, 413 with one in the sums, too.)
template <class T> __device__ __forceinline__ float exp_to(float v) {
    if constexpr (sizeof(T) == 2) return __builtin_amdgcn_exp2f(v * 1.44269504f);
    else return exp_of(v);
}

// ---- a row's end: one work-item per row ------------------------------------------------------------------------------------
// What it needs besides (top, sum), loaded before the row is read, so that the loads run beside it.
struct Given { int64_t label; float at, old, advantage, ref; };

template <class T> __device__ __forceinline__ Given given(const Rows& a, const Finish& e, int64_t r, int64_t label) {
    Given g{label, __builtin_nanf(""), 0.f, 0.f, 0.f};      // a label that names no class has no log probability
    if (label == a.ignore) return g;
    if (label >= 0 && label < a.classes) g.at = Elem<T>::get(row_start<T>(a, r)[label]);
    if (e.kind == kPolicy) {
        const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
        g.advantage = e.advantage[o * e.advantage_outer + i * e.advantage_inner];
        g.old = e.old[r];
    }
    if (e.ref) g.ref = e.ref[r];
    return g;
}

// log of a row's sum to 2e-9: log(2^e m) = e log 2 + 2 artanh t with t = f / (2 + f), f = m - 1, |t| < 0.172, by its power series; t is
// a quotient and its remainder, so that only sums are formed in 64 bits.
// A log probability and its distance from another model's are differences of numbers many times their size; in 32 bits each step of
// them would be off by up to 2.4e-7 where log probabilities lie between 4 and 8, which the mean over a batch shows.
__device__ __forceinline__ double log_of_sum(double sum) {
    const float s = (float)sum;
    if (!(s > 0.f && s < INFINITY)) return (double)logf(s);
    const float past = (float)(sum - (double)s);        // log(s + past) = log(s) + past / s, past being 2^-24 of s
    const uint32_t bits = __float_as_uint(s);
    int e = (int)(bits >> 23) - 127;
    float m = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
    if (m > 1.41421354f) { m *= 0.5f; e++; }
    const float f = m - 1.f, d = 2.f + f, dl = f - (d - 2.f);       // 2 + f = d + dl exactly
    const float r = __builtin_amdgcn_rcpf(d), t = f * r, tl = fmaf(-t, dl, fmaf(-t, d, f)) * r, u = t * t;
    float p = 1.f / 13.f;
    p = fmaf(p, u, 1.f / 11.f); p = fmaf(p, u, 1.f / 9.f); p = fmaf(p, u, 1.f / 7.f); p = fmaf(p, u, 1.f / 5.f); p = fmaf(p, u, 1.f / 3.f);
    return fma((double)e, 0.69314718055994530942, (double)(2.f * t)) + (double)fmaf(2.f, fmaf(t * u, p, tl), past * __builtin_amdgcn_rcpf(s));
}

// exp(a) - 1 - a.  Near 0 that is a^2 / 2 and the difference of two numbers of the size of a: taken by its power series up to |a| = 1/2,
// whose first term left out is 2e-9 of it; beyond, the difference in 64 bits is off by expm1f's error, 6e-7 of the result at 1/2.
__device__ __forceinline__ float excess(double apart, float grown) {
    const float a = (float)apart;
    if (!(fabsf(a) < 0.5f)) return (float)((double)grown - apart);
    float p = 1.f / 181440.f;
    p = fmaf(p, a, 1.f / 20160.f); p = fmaf(p, a, 1.f / 2520.f); p = fmaf(p, a, 1.f / 360.f); p = fmaf(p, a, 1.f / 60.f);
    p = fmaf(p, a, 1.f / 12.f); p = fmaf(p, a, 1.f / 3.f); p = fmaf(p, a, 1.f);
    return 0.5f * a * a * p;
}

struct End { float top, inverse, weight, surrogate, divergence, clipped, kept; };

__device__ __forceinline__ End finish_row(const Rows& a, const Finish& e, int64_t r, const Given& g, float top, double sum) {
    const bool kept = g.label != a.ignore;
    top = finite(top);
    End end{kept ? top : 0.f, 1.f / (float)sum, 0.f, 0.f, 0.f, 0.f, 0.f};
    const double lp = kept ? (double)g.at - (double)top - log_of_sum(sum) : 0.0;
    if (e.stats) e.stats[r] = make_float2(end.top, end.inverse);
    if (e.kind != kPolicy) {
        e.out[r] = kept ? (float)(lp - (double)g.ref) : 0.f;
        if (e.weight) e.weight[r] = 0.f;
        return end;
    }
    if (kept) {
        const float ratio = expf((float)(lp - (double)g.old));
        const float held = ratio < e.low ? e.low : ratio > e.high ? e.high : ratio;
        const float free = ratio * g.advantage, bounded = held * g.advantage;
        const bool clipped = bounded < free;
        end.surrogate = -(clipped ? bounded : free);
        end.clipped = clipped ? 1.f : 0.f;
        end.kept = 1.f;
        end.weight = clipped ? 0.f : -free;
        if (e.kl != 0.f) {
            const double apart = (double)g.ref - lp;
            const float grown = expm1f((float)apart);
            end.divergence = excess(apart, grown);
            end.weight -= e.kl * grown;
        }
    }
    if (e.weight) e.weight[r] = end.weight;
    return end;
}

__device__ __forceinline__ void store_terms(double* to, double surrogate, double divergence, double clipped, double kept) {
    to[0] = surrogate; to[1] = divergence; to[2] = clipped; to[3] = kept;
}

// the weight of a row's gradient
__device__ __forceinline__ float scaled(const Gradient& g, float w) {
    if (g.scale) w *= *g.scale;
    if (g.scale2) w *= *g.scale2;
    return w;
}

__device__ __forceinline__ float row_weight(const Rows& a, const Gradient& g, int64_t r, int64_t label) {
    if (label == a.ignore) return 0.f;
    if (label < 0 || label >= a.classes) return __builtin_nanf("");
    return scaled(g, g.weight[r]);
}

// N values from column c on become their gradients (a label that names no class, whose low half may name one, has w = NaN)
template <class T, int N> __device__ __forceinline__ void slopes(float (&f)[N], float top, float inverse, float w, int c, int label) {
    const float by = -(inverse * w);
    #pragma unroll
    for (int i = 0; i < N; i++) f[i] = exp_to<T>(f[i] - top) * by;
    const uint32_t at = (uint32_t)label - (uint32_t)c;
    if (at < N) {
        #pragma unroll
        for (int i = 0; i < N; i++) f[i] += i == (int)at ? w : 0.f;
    }
}

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

// ---- short rows: 2^shift lanes of a wavefront hold a row in registers, NV vectors each ---------------------------------------
// The last vector of a row of at least one ends with the row and overlaps the one before it; a shorter row is one vector, padded with -inf.
template <class T, int NV> struct Held {
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
    __device__ __forceinline__ float top() const {
        float t = -INFINITY;
        #pragma unroll
        for (int k = 0; k < NV; k++)
            if (index(k) < vecs) {
                float f[V];
                Elem<T>::unpack(v[k], f);
                #pragma unroll
                for (int i = 0; i < V; i++) t = fmaxf(t, f[i]);
            }
        return group_max(t, shift);
    }
    __device__ __forceinline__ double sum(float top) const {
        const float b = finite(top);
        double s = 0.0;
        #pragma unroll
        for (int k = 0; k < NV; k++)
            if (index(k) < vecs) {
                const int past = n >= V ? index(k) * V - column(index(k)) : 0;      // values that the vector before has, too
                float f[V];
                Elem<T>::unpack(v[k], f);
                #pragma unroll
                for (int i = 0; i < V; i++) f[i] = exp_of(f[i] - b);
                if (past > 0) {
                    #pragma unroll
                    for (int i = 0; i < V; i++) f[i] = i < past ? 0.f : f[i];
                }
                s += (double)tree(f);
            }
        return group_total(s, shift);
    }
    // the gradient of weight w; zeros, without a look at the values, where that is 0
    __device__ __forceinline__ void gradient(T* q, float top, float inverse, float w, int label, int stream_from) const {
        #pragma unroll
        for (int k = 0; k < NV; k++)
            if (index(k) < vecs) {
                const int c = n >= V ? column(index(k)) : 0;
                float f[V];
                if (w == 0.f) {
                    #pragma unroll
                    for (int i = 0; i < V; i++) f[i] = 0.f;
                } else {
                    Elem<T>::unpack(v[k], f);
                    slopes<T>(f, top, inverse, w, c, label);
                }
                if (n * (int)sizeof(T) >= stream_from) put_stream16(q + c, Elem<T>::pack(f));
                else if (n >= V) store16(q + c, Elem<T>::pack(f));
                else {
                    #pragma unroll
                    for (int i = 0; i < V; i++)
                        if (i < n) q[i] = Elem<T>::put(f[i]);
                }
            }
    }
};

// FUSED: the gradient leaves with the row (its scale is known before: the reciprocal of the number of rows that count)
template <class T, int NV, bool FUSED> __global__ void __launch_bounds__(256) label_rows_kernel(Rows a, Finish e, Gradient g, int shift) {
    __shared__ double waves[4][4];
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    const int per = 256 >> shift;
    Held<T, NV> row;
    row.n = (int)a.classes; row.shift = shift;
    row.lane = threadIdx.x & ((1 << shift) - 1);
    row.vecs = (row.n + Elem<T>::kVec - 1) / Elem<T>::kVec;
    double terms[4] = {0.0, 0.0, 0.0, 0.0};
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += (int64_t)gridDim.x * per) {
        const int64_t label = a.labels[r];
        Given in{label, 0.f, 0.f, 0.f, 0.f};
        float top = 0.f;
        double sum = 1.0;
        if (label != a.ignore) {
            row.load(row_start<T>(a, r));
            if (row.lane == 0) in = given<T>(a, e, r, label);
            top = row.top();
            row.again();
            sum = row.sum(top);
        }
        End end{};
        if (row.lane == 0) {
            end = finish_row(a, e, r, in, top, sum);
            if (e.terms) { terms[0] += end.surrogate; terms[1] += end.divergence; terms[2] += end.clipped; terms[3] += end.kept; }
        }
        if (FUSED) {
            row.again();
            const int lead = (threadIdx.x & 63) - row.lane;
            const float w = scaled(g, __shfl(end.weight, lead));
            row.gradient(static_cast<T*>(g.grad) + r * a.classes, __shfl(end.top, lead), __shfl(end.inverse, lead), w, (int)label, kStreamRow);
        }
    }
    if (e.terms) {
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            terms[k] = wave_total(terms[k]);
            if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6][k] = terms[k];
        }
        __syncthreads();
        if (threadIdx.x < 4) e.terms[4 * (int64_t)blockIdx.x + threadIdx.x] = waves[0][threadIdx.x] + waves[1][threadIdx.x] + waves[2][threadIdx.x] + waves[3][threadIdx.x];
    }
}

template <class T, int NV> __global__ void __launch_bounds__(256) label_gradient_kernel(Rows a, Gradient g, int shift) {
    if (g.unless_one && *g.scale2 == 1.f) return;
    const int per = 256 >> shift;
    Held<T, NV> row;
    row.n = (int)a.classes; row.shift = shift;
    row.lane = threadIdx.x & ((1 << shift) - 1);
    row.vecs = (row.n + Elem<T>::kVec - 1) / Elem<T>::kVec;
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += (int64_t)gridDim.x * per) {
        const int64_t label = a.labels[r];
        const float w = row_weight(a, g, r, label);
        const float2 st = g.stats[r];
        if (w != 0.f) row.load(row_start<T>(a, r));
        row.gradient(static_cast<T*>(g.grad) + r * a.classes, st.x, st.y, w, (int)label, INT_MAX);
    }
}

// ---- long rows: a workgroup reads a row, or one of its parts ------------------------------------------------------------------
struct Part { float top; double sum; };

// (top, sum) of two parts of a row
__device__ __forceinline__ void join(float& top, double& sum, float top2, double sum2) {
    const float t = fmaxf(top, top2);
    sum = sum * (double)exp_of(finite(top) - finite(t)) + sum2 * (double)exp_of(finite(top2) - finite(t));
    top = t;
}

template <int N> __device__ __forceinline__ void take(float (&f)[N], float& top, double& sum) {
    float t = top;
    #pragma unroll
    for (int i = 0; i < N; i++) t = fmaxf(t, f[i]);
    const float b = finite(t);
    #pragma unroll
    for (int i = 0; i < N; i++) f[i] = exp_of(f[i] - b);
    sum = sum * (double)exp_of(finite(top) - b) + (double)tree(f);
    top = t;
}

// of all lanes of a wavefront
__device__ __forceinline__ void join_wave(float& top, double& sum) {
    const float t = group_max(top, 6);
    sum = group_total(sum * (double)exp_of(finite(top) - finite(t)), 6);
    top = t;
}

// of all work-items of a workgroup, to its first
template <int WAVES> __device__ __forceinline__ void join_workgroup(float& top, double& sum, Part* waves) {
    join_wave(top, sum);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = Part{top, sum};
    __syncthreads();
    if (threadIdx.x < 64) {     // lanes 0 .. WAVES - 1 of each 16 hold the wavefronts' parts
        const Part part = waves[threadIdx.x & (WAVES - 1)];
        top = group_max(part.top, 4);
        sum = group_total((threadIdx.x & 15) < WAVES ? part.sum * (double)exp_of(finite(part.top) - finite(top)) : 0.0, 4);
    }
    __syncthreads();        // (waves is written again)
}

// (top, sum) of this work-item's share of p[0 .. n), which `lanes` work-items read together
template <class T, bool STREAM> __device__ __forceinline__ void scan(const T* p, int64_t n, int lane, int lanes, float& top, double& sum) {
    constexpr int V = Elem<T>::kVec;
    const int64_t full = n / V;
    int64_t i = lane;
    for (; i + (int64_t)(kUnroll - 1) * lanes < full; i += (int64_t)kUnroll * lanes) {
        u32x4 v[kUnroll];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) v[k] = STREAM ? stream16(p + (i + (int64_t)k * lanes) * V) : load16(p + (i + (int64_t)k * lanes) * V);
        float f[kUnroll * V];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) Elem<T>::unpack(v[k], reinterpret_cast<float (&)[V]>(f[k * V]));
        take(f, top, sum);
    }
    for (; i < full; i += lanes) {
        float f[V];
        Elem<T>::unpack(load16(p + i * V), f);
        take(f, top, sum);
    }
    for (int64_t j = full * V + lane; j < n; j += lanes) {
        float f[1] = {Elem<T>::get(p[j])};
        take(f, top, sum);
    }
}

// zeros in a row of a gradient, by a whole workgroup
template <class T> __device__ __forceinline__ void clear_row(T* q, int n, int threads) {
    constexpr int V = Elem<T>::kVec;
    const int full = n / V;
    for (int i = threadIdx.x; i < full; i += threads) put_stream16(q + i * V, u32x4{0u, 0u, 0u, 0u});
    for (int j = full * V + threadIdx.x; j < n; j += threads) q[j] = T{};
}

// columns [c0, c1) of a row, c0 a multiple of the vector's length; a row of weight 0 (ignored, clipped, or of no answer) is not read
template <class T, bool STREAM> __device__ __forceinline__ void grad_row(const T* src, T* dst, float top, float inverse, float w, int label, int64_t c0, int64_t c1, int lane, int lanes) {
    constexpr int V = Elem<T>::kVec;
    const int64_t full = c1 / V;
    if (w == 0.f) {
        for (int64_t i = c0 / V + lane; i < full; i += lanes) put_stream16(dst + i * V, u32x4{0u, 0u, 0u, 0u});
        for (int64_t j = full * V + lane; j < c1; j += lanes) dst[j] = T{};
        return;
    }
    int64_t i = c0 / V + lane;
    for (; i + (int64_t)(kUnroll - 1) * lanes < full; i += (int64_t)kUnroll * lanes) {
        u32x4 v[kUnroll];
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) v[k] = STREAM ? stream16(src + (i + (int64_t)k * lanes) * V) : load16(src + (i + (int64_t)k * lanes) * V);
        #pragma unroll
        for (int k = 0; k < kUnroll; k++) {
            const int64_t c = (i + (int64_t)k * lanes) * V;
            float f[V];
            Elem<T>::unpack(v[k], f);
            slopes<T>(f, top, inverse, w, (int)c, label);
            put_stream16(dst + c, Elem<T>::pack(f));
        }
    }
    for (; i < full; i += lanes) {
        float f[V];
        Elem<T>::unpack(load16(src + i * V), f);
        slopes<T>(f, top, inverse, w, (int)(i * V), label);
        put_stream16(dst + i * V, Elem<T>::pack(f));
    }
    for (int64_t j = full * V + lane; j < c1; j += lanes) {
        float f[1] = {Elem<T>::get(src[j])};
        slopes<T>(f, top, inverse, w, (int)j, label);
        dst[j] = Elem<T>::put(f[0]);
    }
}

// A pass over long rows reads them from the last to the first, the gradient's pass from the first on, so that it finds
// what the last-level cache holds still there; the rows behind them are read past the caches, which leaves these alone and is faster by itself:
// 4096 x 131072 bf16 forward 180 -> 162 us, both passes 541 -> 484.
__host__ __device__ __forceinline__ bool beyond_cache(const Rows& a, int64_t r, int64_t size) { return r * a.classes * size >= kCached; }

__device__ __forceinline__ End finish_long_row(const Rows& a, const Finish& e, int64_t r, const Given& g, float top, double sum) {
    const End end = finish_row(a, e, r, g, top, sum);
    if (e.terms) store_terms(e.terms + 4 * r, end.surrogate, end.divergence, end.clipped, end.kept);
    return end;
}

// A workgroup per row, or per one of `splits` parts of a row, which then leaves its (top, sum) for join_rows_kernel.
template <class T> __global__ void __launch_bounds__(256, 8) label_long_rows_kernel(Rows a, Finish e, int splits, int64_t part, Part* parts) {
    __shared__ Part waves[4];
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t back = splits == 1 ? b : b / splits, s = b - back * splits, r = a.rows - 1 - back, c0 = s * part;
        const int64_t n = a.classes - c0 < part ? a.classes - c0 : part;
        float top = 0.f;
        double sum = 1.0;
        const int64_t label = a.labels[r];
        Given in{label, 0.f, 0.f, 0.f, 0.f};
        if (label != a.ignore) {        // (the whole workgroup's)
            if (threadIdx.x == 0 && splits == 1) in = given<T>(a, e, r, label);
            top = -INFINITY; sum = 0.0;
            if (beyond_cache(a, r, sizeof(T))) scan<T, true>(row_start<T>(a, r) + c0, n, threadIdx.x, 256, top, sum);
            else scan<T, false>(row_start<T>(a, r) + c0, n, threadIdx.x, 256, top, sum);
            join_workgroup<4>(top, sum, waves);
        }
        if (threadIdx.x == 0) {
            if (splits > 1) parts[r * splits + s] = Part{top, sum};
            else finish_long_row(a, e, r, in, top, sum);
        }
    }
}

// The workgroup holds a long row in its registers, at most 16 vectors per work-item.  FUSED: the logits are read once and the gradient leaves
// with the statistics.  FAR: logits that the last-level cache cannot hold are read past it (4096 x 131072 bf16 437 -> 432 us with
// the launches beside it, 4096 x 65536 206 -> 197; 2000 x 50001 fp16, which it holds, 76, past it 95).  (Reading the row again from the caches instead lost: eight rows of 256 KiB
// per compute unit are more than the last level holds, 4096 x 131072 596 us where two passes of their own took 515.)
template <class T, int NV, int THREADS, bool FUSED, bool FAR> __global__ void __launch_bounds__(THREADS, 4) label_held_rows_kernel(Rows a, Finish e, Gradient g) {
    constexpr int V = Elem<T>::kVec, kChunk = (NV == 16 ? 8 : 16) / V;
    __shared__ Part waves[THREADS / 64];
    __shared__ End row_end;
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    const int n = (int)a.classes, full = n / V, rest = full * V + (int)threadIdx.x;     // the values behind the last whole vector: one per work-item
    const T lowest = Elem<T>::put(-INFINITY);
    for (int64_t r = a.rows - 1 - blockIdx.x; r >= 0; r -= gridDim.x) {     // (the producer's last rows may be in the caches)
        const int64_t label = a.labels[r];
        T* q = static_cast<T*>(g.grad) + r * a.classes;
        if (label == a.ignore) {        // (the whole workgroup's)
            if (threadIdx.x == 0) finish_long_row(a, e, r, Given{label, 0.f, 0.f, 0.f, 0.f}, 0.f, 1.0);
            if (FUSED) clear_row(q, n, THREADS);
            continue;
        }
        const T* p = row_start<T>(a, r);
        u32x4 v[NV];
        const u32x4 none = Elem<T>::splat(lowest);
        T last = lowest;
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int i = (int)threadIdx.x + k * THREADS;
            v[k] = none;
            if (i < full) v[k] = FAR ? stream16(p + i * V) : load16(p + i * V);
        }
        if (rest < n) last = p[rest];
        Given in{label, 0.f, 0.f, 0.f, 0.f};
        if (threadIdx.x == 0) in = given<T>(a, e, r, label);
        float top = -INFINITY;
        double sum = 0.0;
        #pragma unroll
        for (int c = 0; c < NV; c += kChunk) {
            float f[kChunk * V];
            #pragma unroll
            for (int k = 0; k < kChunk; k++) Elem<T>::unpack(v[c + k], reinterpret_cast<float (&)[V]>(f[k * V]));
            take(f, top, sum);
        }
        float f1[1] = {Elem<T>::get(last)};
        take(f1, top, sum);
        join_workgroup<THREADS / 64>(top, sum, waves);
        if (threadIdx.x == 0) row_end = finish_long_row(a, e, r, in, top, sum);
        if (!FUSED) continue;
        __syncthreads();
        const End end = row_end;
        __syncthreads();    // (row_end is written again)
        const float w = scaled(g, end.weight);
        if (w == 0.f) { clear_row(q, n, THREADS); continue; }
        // (as in Held::again)
        int item = threadIdx.x;
        asm("" : "+v"(item));
        #pragma unroll
        for (int k = 0; k < NV; k++) asm("" : "+v"(v[k]));
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const int i = item + k * THREADS;
            float f[V];
            Elem<T>::unpack(v[k], f);
            slopes<T>(f, end.top, end.inverse, w, i * V, (int)label);
            if (i < full) put_stream16(q + i * V, Elem<T>::pack(f));
        }
        if (rest < n) {
            float f[1] = {Elem<T>::get(last)};
            slopes<T>(f, end.top, end.inverse, w, rest, (int)label);
            q[rest] = Elem<T>::put(f[0]);
        }
    }
}

// a wavefront per row joins the parts of label_long_rows_kernel
template <class T> __global__ void __launch_bounds__(256) join_rows_kernel(Rows a, Finish e, int splits, const Part* parts) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * 4) {
        const int64_t label = a.labels[r];
        Given in{label, 0.f, 0.f, 0.f, 0.f};
        float top = 0.f;
        double sum = 1.0;
        if (label != a.ignore) {
            if (lane == 0) in = given<T>(a, e, r, label);
            top = -INFINITY; sum = 0.0;
            for (int k = lane; k < splits; k += 64) join(top, sum, parts[r * splits + k].top, parts[r * splits + k].sum);
            join_wave(top, sum);
        }
        if (lane == 0) finish_long_row(a, e, r, in, top, sum);
    }
}

template <class T> __global__ void __launch_bounds__(256) label_long_gradient_kernel(Rows a, Gradient g, int splits, int64_t part) {
    if (g.unless_one && *g.scale2 == 1.f) return;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = b / splits, c0 = (b - r * splits) * part, c1 = a.classes - c0 < part ? a.classes : c0 + part;
        const int64_t label = a.labels[r];
        const float2 st = g.stats[r];
        const float w = row_weight(a, g, r, label);
        T* q = static_cast<T*>(g.grad) + r * a.classes;
        if (beyond_cache(a, r, sizeof(T))) grad_row<T, true>(row_start<T>(a, r), q, st.x, st.y, w, (int)label, c0, c1, threadIdx.x, 256);
        else grad_row<T, false>(row_start<T>(a, r), q, st.x, st.y, w, (int)label, c0, c1, threadIdx.x, 256);
    }
}

// ---- sums over rows ---------------------------------------------------------------------------------------------------------
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
    const float* ratios;            // log probability - ref of each row, 0 where ignored
    int64_t rows, tokens;
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

// WAVES wavefronts per pair: x = beta (chosen - rejected), the sums of lp - ref over the rows of the two answers, in 64 bits; then the
// pair's loss and the weight of its rows.  The workgroups' sums are added in order by the last one.
template <int WAVES> __global__ void __launch_bounds__(256) preference_kernel(Pairs a) {
    __shared__ double waves[4], sums[2][4];
    constexpr int kPairs = 4 / WAVES, kLanes = 64 * WAVES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, item = threadIdx.x & (kLanes - 1);
    double loss = 0.0;
    for (int64_t p0 = (int64_t)blockIdx.x * kPairs; p0 < a.pairs; p0 += (int64_t)gridDim.x * kPairs) {
        const int64_t pair = p0 + wave / WAVES;
        const bool here = pair < a.pairs;
        double s[2] = {0.0, 0.0};
        int64_t from[2] = {0, 0}, until[2] = {0, 0};
        if (here) {
            #pragma unroll
            for (int k = 0; k < 2; k++) {
                from[k] = answer_start(a, pair + k * (int64_t)a.pairs);
                until[k] = answer_start(a, pair + k * (int64_t)a.pairs + 1);
            }
            #pragma unroll
            for (int k = 0; k < 2; k++) {
                #pragma unroll 4
                for (int64_t r = from[k] + item; r < until[k]; r += kLanes) s[k] += (double)a.ratios[r];
            }
        }
        s[0] = wave_total(s[0]); s[1] = wave_total(s[1]);
        if (WAVES > 1) {
            if (lane == 0) { sums[0][wave] = s[0]; sums[1][wave] = s[1]; }
            __syncthreads();
            #pragma unroll
            for (int k = 0; k < 2; k++) s[k] = sums[k][0] + sums[k][1] + sums[k][2] + sums[k][3];
            __syncthreads();
        }
        if (here) {
            const double chosen = a.beta * s[0], rejected = a.beta * s[1];
            const double x = chosen - rejected, small = exp(-fabs(x)), tail = log1p(small);
            // -log sigma(x) = max(-x, 0) + log(1 + exp(-|x|))
            double l = (1.0 - a.smoothing) * ((x < 0.0 ? -x : 0.0) + tail);
            if (a.smoothing != 0.0) l += a.smoothing * ((x > 0.0 ? x : 0.0) + tail);
            if (item == 0) {
                a.rewards[pair] = (float)chosen;
                a.rewards[pair + a.pairs] = (float)rejected;
                loss += l;
            }
            if (a.weight) {
                const double up = (x < 0.0 ? small : 1.0) / (1.0 + small), down = (x < 0.0 ? 1.0 : small) / (1.0 + small);   // sigma(x), sigma(-x)
                const float slope = (float)(-a.beta / a.pairs * ((1.0 - a.smoothing) * down - a.smoothing * up));
                #pragma unroll
                for (int k = 0; k < 2; k++)
                    for (int64_t r = from[k] + item; r < until[k]; r += kLanes) a.weight[r] = k ? -slope : slope;   // (ignored rows have none whatever stands here)
            }
        }
    }
    if (lane == 0) waves[wave] = loss;
    __syncthreads();
    loss = waves[0] + waves[1] + waves[2] + waves[3];
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) publish(a.parts + blockIdx.x, loss);
        if (!last_workgroup(a.ticket) || wave != 0) return;
        loss = 0.0;
        for (int k = lane; k < (int)gridDim.x; k += 64) loss += published(a.parts + k);
        loss = wave_total(loss);
    }
    if (threadIdx.x == 0) *a.loss = (float)(loss / a.pairs);
}

// Means of the policy's terms over the kept rows (over one where there are none); `scale` = 1 / that number (or null: it has been found).
__global__ void __launch_bounds__(1024) policy_sums_kernel(const double* terms, int64_t count, double kl, float* loss, float* stats, float* scale,
                                                          double* parts, uint32_t* ticket) {
    __shared__ double waves[16][4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    #pragma unroll 4
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 1024) {
        const double2 t = reinterpret_cast<const double2*>(terms)[2 * i], u = reinterpret_cast<const double2*>(terms)[2 * i + 1];
        s[0] += t.x; s[1] += t.y; s[2] += u.x; s[3] += u.y;
    }
    #pragma unroll
    for (int k = 0; k < 4; k++) {
        s[k] = wave_total(s[k]);
        if (lane == 0) waves[wave][k] = s[k];
    }
    __syncthreads();
    #pragma unroll
    for (int k = 0; k < 4; k++) s[k] = 0.0;
    if (wave == 0) {
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            s[k] = lane < 16 ? waves[lane][k] : 0.0;
            for (int o = 8; o > 0; o >>= 1) s[k] += __shfl_xor(s[k], o);
        }
    }
    if (gridDim.x > 1) {
        if (threadIdx.x == 0) {
            #pragma unroll
            for (int k = 0; k < 4; k++) publish(parts + 4 * blockIdx.x + k, s[k]);
        }
        if (!last_workgroup(ticket) || wave != 0) return;
        #pragma unroll
        for (int k = 0; k < 4; k++) {
            s[k] = 0.0;
            for (int b = lane; b < (int)gridDim.x; b += 64) s[k] += published(parts + 4 * b + k);
            s[k] = wave_total(s[k]);
        }
    }
    if (threadIdx.x == 0) {
        const double kept = s[3] > 1.0 ? s[3] : 1.0;
        *loss = (float)((s[0] + kl * s[1]) / kept);
        stats[0] = (float)(s[0] / kept);
        stats[1] = (float)(s[1] / kept);
        stats[2] = (float)(s[2] / kept);
        if (scale) *scale = (float)(1.0 / kept);
    }
}

// The number of rows that count, before they are read: of whole labels (one workgroup, or `counts` of several), then of these counts, to `scale` =
// 1 / the number.  Sums of whole numbers: their order does not matter.
template <class N> __global__ void __launch_bounds__(1024) count_rows_kernel(const N* from, int64_t n, int64_t ignore, int* counts, float* scale) {
    __shared__ int waves[16];
    int s = 0;
    #pragma unroll 8
    for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 1024) s += sizeof(N) == 8 ? (from[i] != (N)ignore ? 1 : 0) : (int)from[i];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int k = 1; k < 16; k++) s += waves[k];
    if (counts) counts[blockIdx.x] = s;
    else *scale = (float)(1.0 / (s > 1 ? s : 1));
}

// ---- host -----------------------------------------------------------------------------------------------------------------
namespace {

constexpr int kPairBlocks = 256, kSumBlocks = 128;

int vec_of(int dtype) { return dtype == SD_FLOAT32 ? 4 : 8; }

// Lanes of a wavefront that hold a row together (as a power of two) and vectors that each holds; shift = -1: a row is read by whole workgroups.
// Many rows want few lanes with several vectors each (fewer steps to add up lanes per row), few rows one vector per lane.
struct Group { int shift, vectors; };
Group group_of(int64_t rows, int64_t classes, int vec) {
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
int row_splits(int64_t rows, int64_t classes, int vec) {
    const int64_t want = (kWholeRows + rows - 1) / rows, most = (classes + 256 * vec - 1) / (256 * vec);
    return (int)(want < most ? want : most);
}

// Rows that would be read in parts: where a workgroup can hold a row it is read whole, which spares the launch that joins the parts:
// 128 x 8192 bf16 6.8 -> 4.4 us, 512 x 16384 8.6 -> 5.4, 512 x 32000 11.9 -> 9.3.  Rows for a workgroup of 512, of which fewer run at once: 256 x 50001
// 10.4 -> 9.0, but 16 rows 7.1 -> 8.4 and 1024 21.2 -> 26.0.
bool one_launch(int64_t rows, int64_t classes, int vec) {
    const int64_t vecs = (classes + vec - 1) / vec;
    return rows < kWholeRows && (vecs <= 16 * 256 || (vecs <= 16 * 512 && rows >= 32 && rows <= 512));
}

int64_t part_of(int64_t classes, int splits, int vec) {
    const int64_t step = 256 * vec, n = (classes + splits - 1) / splits;
    return (n + step - 1) / step * step;
}

unsigned short_blocks(int64_t rows, int per) {
    const int64_t n = (rows + per - 1) / per;
    return (unsigned)(n < kShortBlocks ? n : kShortBlocks);
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
    SD_REQUIRE((reinterpret_cast<uintptr_t>(in->logits) & (in->dtype == SD_FLOAT32 ? 3 : 1)) == 0 && (reinterpret_cast<uintptr_t>(in->labels) & 7) == 0,
               "%s: logits or labels are not aligned to their type", who);
    *a = Rows{in->logits, in->labels, in->rows, in->classes, in->outer_stride, in->inner_stride, in->ignore_index, (uint32_t)in->inner};
    return SD_OK;
}

int check_work(const char* who, const float* stats, const float* scratch) {
    SD_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "%s: stats must be aligned to 8 bytes, scratch to 16", who);
    return SD_OK;
}

int64_t split_floats(const sd_label_rows* in) {
    const int vec = vec_of(in->dtype);
    if (group_of(in->rows, in->classes, vec).shift >= 0 || one_launch(in->rows, in->classes, vec)) return 0;
    const int splits = row_splits(in->rows, in->classes, vec);
    return splits > 1 ? (int64_t)(sizeof(Part) / sizeof(float)) * in->rows * splits : 0;
}

// parts of the policy's terms: one per workgroup of short rows, one per long row
int64_t term_count(const sd_label_rows* in) {
    const Group group = group_of(in->rows, in->classes, vec_of(in->dtype));
    return group.shift >= 0 ? short_blocks(in->rows, 256 >> group.shift) : in->rows;
}

// with `g` the rows' gradients, too (rows that a workgroup can hold)
int launch_rows(const sd_label_rows* in, const Rows& a, const Finish& e, const Gradient* g, float* parts, hipStream_t stream) {
    const int vec = vec_of(in->dtype);
    const Group group = group_of(a.rows, a.classes, vec);
    const Gradient grad = g ? *g : Gradient{};
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (group.shift >= 0) {
            const int per = 256 >> group.shift;
            const dim3 grid(short_blocks(a.rows, per));
            with_vectors(group.vectors, [&](auto nv) {
                if (g) hipLaunchKernelGGL((label_rows_kernel<T, nv.value, true>), grid, dim3(256), 0, stream, a, e, grad, group.shift);
                else hipLaunchKernelGGL((label_rows_kernel<T, nv.value, false>), grid, dim3(256), 0, stream, a, e, grad, group.shift);
            });
            return;
        }
        if (g || one_launch(a.rows, a.classes, vec)) {
            const dim3 grid(blocks_for(a.rows));
            const int64_t vecs = (a.classes + vec - 1) / vec;
            const auto held = [&](auto fused, auto far) {
                if (vecs <= 4 * 256) hipLaunchKernelGGL((label_held_rows_kernel<T, 4, 256, fused.value, far.value>), grid, dim3(256), 0, stream, a, e, grad);
                else if (vecs <= 8 * 256) hipLaunchKernelGGL((label_held_rows_kernel<T, 8, 256, fused.value, far.value>), grid, dim3(256), 0, stream, a, e, grad);
                else if (vecs <= 16 * 256) hipLaunchKernelGGL((label_held_rows_kernel<T, 16, 256, fused.value, far.value>), grid, dim3(256), 0, stream, a, e, grad);
                else if (vecs <= 16 * 512) hipLaunchKernelGGL((label_held_rows_kernel<T, 16, 512, fused.value, far.value>), grid, dim3(512), 0, stream, a, e, grad);
                else if constexpr (fused.value) hipLaunchKernelGGL((label_held_rows_kernel<T, 16, 1024, true, far.value>), grid, dim3(1024), 0, stream, a, e, grad);
            };
            if (!g) held(std::false_type(), std::false_type());     // (few rows)
            else if (beyond_cache(a, a.rows, sizeof(T))) held(std::true_type(), std::true_type());
            else held(std::true_type(), std::false_type());
            return;
        }
        int splits = row_splits(a.rows, a.classes, vec);
        const int64_t part = part_of(a.classes, splits, vec);
        splits = (int)((a.classes + part - 1) / part);
        Part* out = reinterpret_cast<Part*>(parts);
        hipLaunchKernelGGL(label_long_rows_kernel<T>, dim3(blocks_for(a.rows * splits)), dim3(256), 0, stream, a, e, splits, part, out);
        if (splits > 1) hipLaunchKernelGGL(join_rows_kernel<T>, dim3(blocks_for((a.rows + 3) / 4)), dim3(256), 0, stream, a, e, splits, out);
    });
    return check_launch("label_rows_kernel");
}

}  // namespace

}  // namespace sd

using namespace sd;

extern "C" int64_t sd_label_scratch(const sd_label_rows* in, int loss) {
    Rows a;
    if (check_rows(in, "label_scratch", &a) != SD_OK) return -1;
    // (the policy's terms are 64-bit numbers, the preferences' rows one float each)
    return (split_floats(in) + (loss ? kSumFloats + 8 * term_count(in) + in->rows : 0) + 3) / 4 * 4;
}

extern "C" int sd_label_log_probs(const sd_label_rows* in, float* log_probs, float* stats, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "label_log_probs", &a)) return rc;
    if (int rc = check_work("label_log_probs", stats, scratch)) return rc;
    SD_REQUIRE(log_probs && (scratch || split_floats(in) == 0), "label_log_probs: null output or scratch");
    Finish e{};
    e.kind = kValues;
    e.out = log_probs;
    e.stats = reinterpret_cast<float2*>(stats);
    return launch_rows(in, a, e, nullptr, scratch, static_cast<hipStream_t>(stream));
}

extern "C" int sd_preference_loss(const sd_label_rows* in, const float* ref, const void* offsets, int offset_bytes, int64_t tokens, int pairs, double beta, double smoothing,
                                  float* stats, float* weight, float* rewards, float* loss, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "preference_loss", &a)) return rc;
    if (int rc = check_work("preference_loss", stats, scratch)) return rc;
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
    e.out = scratch + kSumFloats + parts;
    e.ref = ref;
    e.stats = reinterpret_cast<float2*>(stats);
    e.weight = weight;
    e.ticket = reinterpret_cast<uint32_t*>(scratch);
    if (int rc = launch_rows(in, a, e, nullptr, scratch + kSumFloats, s)) return rc;
    const Pairs p{e.out, a.rows, tokens, offset_bytes == 4 ? static_cast<const int*>(offsets) : nullptr, offset_bytes == 8 ? static_cast<const int64_t*>(offsets) : nullptr,
                  pairs, beta, smoothing, weight, rewards, loss, reinterpret_cast<double*>(scratch + 4), e.ticket};
    // a workgroup per pair where that fills the card no more than once, and answers are long enough for it
    if (pairs <= kPairBlocks && a.rows >= 64 * (int64_t)pairs) hipLaunchKernelGGL(preference_kernel<4>, dim3(pairs), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(preference_kernel<1>, dim3((pairs + 3) / 4 < kPairBlocks ? (pairs + 3) / 4 : kPairBlocks), dim3(256), 0, s, p);
    return check_launch("preference_kernel");
}

// Whether the gradient leaves with the rows: it then costs one reading of the logits less (5.5 TB/s) and a launch more (4 us); a
// workgroup must be able to hold a row, and there must be rows for all compute units.
static bool fused_policy(const sd_label_rows* in) {
    const int vec = vec_of(in->dtype);
    if (in->rows * in->classes * (16 / vec) < (32ll << 20)) return false;
    return group_of(in->rows, in->classes, vec).shift >= 0 || (in->rows >= 512 && in->classes <= kHeldLong * vec);
}

extern "C" int sd_policy_fuses(const sd_label_rows* in) {
    Rows a;
    return check_rows(in, "policy_fuses", &a) == SD_OK && fused_policy(in) ? 1 : 0;
}

extern "C" int sd_policy_loss(const sd_label_rows* in, const float* old_log_probs, const float* advantages, int64_t advantage_outer, int64_t advantage_inner,
                              const float* ref, double clip_low, double clip_high, double kl, float* stats, float* weight, float* scale, void* grad, float* loss,
                              float* means, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "policy_loss", &a)) return rc;
    if (int rc = check_work("policy_loss", stats, scratch)) return rc;
    SD_REQUIRE(old_log_probs && advantages && scale && loss && means && scratch, "policy_loss: null argument");
    SD_REQUIRE(!stats == !weight, "policy_loss: the gradient needs both stats and weight");
    SD_REQUIRE(!grad || stats, "policy_loss: a gradient that leaves with the rows needs stats and weight, too");
    SD_REQUIRE(!grad || fused_policy(in), "policy_loss: the gradient of these rows does not leave with them (sd_policy_fuses)");
    SD_REQUIRE(clip_low >= 0.0 && clip_low <= 1.0 && clip_high >= 0.0, "policy_loss: clip=%g, clip_high=%g: need 0 <= clip <= 1 and 0 <= clip_high", clip_low, clip_high);
    SD_REQUIRE(ref || kl == 0.0, "policy_loss: a KL term needs reference log probabilities");
    hipStream_t s = static_cast<hipStream_t>(stream);
    Finish e{};
    e.kind = kPolicy;
    e.stats = reinterpret_cast<float2*>(stats);
    e.weight = weight;
    const int64_t terms = term_count(in);
    e.terms = reinterpret_cast<double*>(scratch + kSumFloats);          // (16-byte aligned: before the parts)
    e.old = old_log_probs; e.advantage = advantages; e.ref = kl != 0.0 ? ref : nullptr;
    e.advantage_outer = advantage_outer; e.advantage_inner = advantage_inner;
    e.low = (float)(1.0 - clip_low); e.high = (float)(1.0 + clip_high); e.kl = (float)kl;
    e.ticket = reinterpret_cast<uint32_t*>(scratch);
    Gradient g{};
    g.scale = scale; g.grad = grad;
    if (grad) {
        // (the counts' place is the sums', which are written later)
        int* counts = reinterpret_cast<int*>(scratch + 4);
        const int64_t want = (a.rows + 8191) / 8192;
        const int blocks = (int)(want < kSumBlocks ? want : kSumBlocks);
        hipLaunchKernelGGL(count_rows_kernel<int64_t>, dim3(blocks), dim3(1024), 0, s, a.labels, a.rows, a.ignore, blocks > 1 ? counts : nullptr, scale);
        if (blocks > 1) hipLaunchKernelGGL(count_rows_kernel<int>, dim3(1), dim3(1024), 0, s, counts, (int64_t)blocks, (int64_t)0, nullptr, scale);
    }
    if (int rc = launch_rows(in, a, e, grad ? &g : nullptr, scratch + kSumFloats + 8 * terms, s)) return rc;
    const int64_t want = (terms + 16383) / 16384;
    hipLaunchKernelGGL(policy_sums_kernel, dim3((unsigned)(want < kSumBlocks ? want : kSumBlocks)), dim3(1024), 0, s, e.terms, terms, kl, loss, means, grad ? nullptr : scale,
                       reinterpret_cast<double*>(scratch + 4), e.ticket);
    return check_launch("policy_sums_kernel");
}

extern "C" int sd_label_gradient(const sd_label_rows* in, const float* stats, const float* weight, const float* scale, const float* scale2, int unless_one, void* grad,
                                 sd_stream_t stream) {
    sd::CallGuard call_guard;
    Rows a;
    if (int rc = check_rows(in, "label_gradient", &a)) return rc;
    if (int rc = check_work("label_gradient", stats, nullptr)) return rc;
    SD_REQUIRE(stats && weight && grad, "label_gradient: null argument");
    SD_REQUIRE(!unless_one || scale2, "label_gradient: unless_one needs scale2");
    const Gradient g{reinterpret_cast<const float2*>(stats), weight, scale, scale2, grad, unless_one != 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int vec = vec_of(in->dtype);
    const Group group = group_of(a.rows, a.classes, vec);
    // a launch that mostly finds nothing to do has no more workgroups than run at once: each takes time to come and go
    const auto blocks = [&](int64_t n) { return dim3(unless_one && n > 8 * num_cus() ? (unsigned)(8 * num_cus()) : blocks_for(n)); };
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (group.shift >= 0) {
            const int per = 256 >> group.shift;
            with_vectors(group.vectors, [&](auto nv) {
                hipLaunchKernelGGL((label_gradient_kernel<T, nv.value>), blocks((a.rows + per - 1) / per), dim3(256), 0, s, a, g, group.shift);
            });
            return;
        }
        const int64_t part = 256 * vec * kUnroll;
        const int splits = (int)((a.classes + part - 1) / part);
        hipLaunchKernelGGL(label_long_gradient_kernel<T>, blocks(a.rows * splits), dim3(256), 0, s, a, g, splits, part);
    });
    return check_launch("label_gradient_kernel");
}
