// Distillation from a teacher's top logits.  The teacher gives row r some classes c_j with logits t_j and, as one more outcome, the log-sum `rest` of
// its other logits; the student's row z has the same outcomes.  With a temperature T, in the outcomes' softmaxes
//   q_j ~ exp(t_j / T), q_r ~ exp(rest);   p_j ~ exp(z[c_j] / T), p_r ~ S,   S = sum over the classes that are in no entry of exp(z[v] / T),
// the divergence is D = sum_j q_j (log q_j - log p_j) + q_r (log q_r - log p_r), the loss weight T^2 times the mean of D, and
//   d D / d (z[v] / T) = p_v - sum of the q_j with c_j = v   for a class of an entry,   (p_r - q_r) exp(z[v] / T) / S   for another one.
// S is formed without the entries' classes, not as a difference, so that what the student gives the others keeps its digits however small it is.
// There are few outcomes per row: they are in 64 bits, as three sums over the entries (Sums) that need no S, so that what is left when S is there is a few
// numbers per row.  Both passes are bound by the bytes of the logits, and by the launches where there are few.
// A class that stands in several entries counts once in p and takes the sum of their q in the gradient.  D keeps a term for each entry, q_j log q_j, which is below that of
// the merged class by q_j log(q / q_j): merging them would cost each row a search among its entries for what the logits do not change.
// All sums have a fixed order: results are the same in every call.
#include "label_rows.h"

namespace sd {

constexpr int kMostEntries = SD_MOST_TOP;   // of a row: one per work-item of a workgroup
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
    // An entry as it is stored, for kernels that have other loads under way behind these: a conversion beside the load would wait for it.
    struct Raw { int low, high; uint32_t value; };
    __device__ __forceinline__ Raw raw(int64_t at) const {
        const int* c = static_cast<const int*>(classes);
        Raw e{c[wide ? 2 * at : at], c[wide ? 2 * at + 1 : at], 0};
        if (dtype == SD_FLOAT32) e.value = static_cast<const uint32_t*>(values)[at];
        else e.value = static_cast<const uint16_t*>(values)[at];
        return e;
    }
    __device__ __forceinline__ int64_t cls(const Raw& e) const { return wide ? (int64_t)((uint64_t)(uint32_t)e.high << 32 | (uint32_t)e.low) : (int64_t)e.low; }
    __device__ __forceinline__ float value(const Raw& e) const {
        if (dtype == SD_FLOAT32) return __uint_as_float(e.value);
        return dtype == SD_BFLOAT16 ? Elem<bf16>::get(bf16{(uint16_t)e.value}) : Elem<fp16>::get(fp16{(uint16_t)e.value});
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

struct Slopes {
    const float2* stats;
    const float* entries;
    const float *scale, *scale2;    // one number each that all is multiplied by (scale2 may be null)
    void* grad;                     // rows one behind the other
    bool unless_one;                // nothing is done where *scale2 is 1
    __device__ __forceinline__ float by() const { return scale2 ? *scale * *scale2 : *scale; }
};

struct Others { float top; double sum; };     // of the classes in no entry: sum of exp((z - top) / T)

// ---- the outcomes of a row -------------------------------------------------------------------------------------------------
// An entry: its class (negative: none), the teacher's logit and the student's.  `said`: 1 for an entry, 2 for one that is above -inf; a row counts, and is read, that
// has an entry and an entry or a rest above -inf.
struct Entry { int64_t cls; float t, z; };
__device__ __forceinline__ int said(int64_t cls, float t) { return cls < 0 ? 0 : t != -INFINITY ? 3 : 1; }

// over the entries: of the teacher's weights w = exp((t - most_t) / T), of the student's exp((z - base) / T), each class once, and of w times the difference of the two
// exponents
struct Sums { double w, p, a; };
__device__ __forceinline__ double add_entry(Sums& s, const Entry& e, float most_t, float base, bool first, const Temper& t) {
    const double at = ((double)e.t - (double)most_t) * t.inverse, az = ((double)e.z - (double)base) * t.inverse, w = exp(at), p = exp(az);
    s.w += w;
    if (w != 0.0) s.a += w * (at - az);
    if (first) s.p += p;
    return p;
}

// What a row comes to.  The entries' sums are relative to most_t and to their own largest logit (where none is above -inf, to 0); the rest, which may lie far above the
// entries, to the larger of the two, and the student's outcomes to base, the largest of its logits: with p = exp((entries - base) / T), o = exp((top - base) / T),
//   W = sum_w exp(-up) + w_r,  P = sum_p p + S o,  D = (exp(-up) (sum_a - (up + log p) sum_w) + w_r (left - up - log(S o))) / W - log W + log P.
// The four lanes of a quad hold the same row: one call of a 64-bit function, some 50 instructions, is for up to four numbers of it.
template <int LANE> __device__ __forceinline__ double of_quad(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t low = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)bits, LANE * 0x55, 0xf, 0xf, false);
    const uint32_t high = (uint32_t)__builtin_amdgcn_mov_dpp((int)(uint32_t)(bits >> 32), LANE * 0x55, 0xf, 0xf, false);
    return __builtin_bit_cast(double, (uint64_t)high << 32 | low);
}
template <class F> __device__ __forceinline__ void four_of(double& x, double& y, double& z, double& w, F&& f) {
    const int lane = threadIdx.x & 3;
    const double v = f(lane == 0 ? x : lane == 1 ? y : lane == 2 ? z : w);
    x = of_quad<0>(v); y = of_quad<1>(v); z = of_quad<2>(v); w = of_quad<3>(v);
}

struct Rest { double left, up, log_p, top, scale, w, p, o; };      // of the teacher's others; (top - base) / T; exp(-up), w_r, p and o
__device__ __forceinline__ Rest rest_of(double rest, float most_t, float entries, float top, const Temper& t) {
    const double left = rest - (double)most_t * t.inverse, up = left > 0.0 ? left : 0.0, high = (double)finite(top);
    const double base = entries == -INFINITY ? high : fmax((double)entries, high);
    const double log_p = entries == -INFINITY ? 0.0 : ((double)entries - base) * t.inverse, log_o = (high - base) * t.inverse;
    Rest e{left, up, log_p, log_o, -up, left - up, log_p, log_o};
    four_of(e.scale, e.w, e.p, e.o, [](double v) { return exp(v); });
    return e;
}
struct Row { double over_w, per_w, per_p; float factor; };      // 1 / W, the same for sum_w, p / P; factor = (p_r - q_r) / S
__device__ __forceinline__ Row ratios_of(const Sums& s, const Rest& rest, const Others& o, bool bad) {
    double w = s.w * rest.scale + rest.w, p = s.p * rest.p + (o.sum > 0.0 ? o.sum * rest.o : 0.0), others = o.sum, one = 1.0;
    four_of(w, p, others, one, [](double v) { return 1.0 / v; });
    if (bad) p = __builtin_nan("");
    return Row{w, rest.scale * w, rest.p * p, o.sum > 0.0 || bad ? (float)(rest.o * p - rest.w * w * others) : 0.f};
}
__device__ __forceinline__ double divergence_of(const Sums& s, const Rest& rest, const Others& o, const Row& row, bool bad) {
    double log_s = o.sum, w = s.w * rest.scale + rest.w, p = s.p * rest.p + (o.sum > 0.0 ? o.sum * rest.o : 0.0), one = 1.0;
    four_of(log_s, w, p, one, [](double v) { return log(v); });
    log_s = o.sum > 0.0 ? log_s + rest.top : -INFINITY;
    double a = rest.scale != 0.0 ? rest.scale * (s.a - (rest.up + rest.log_p) * s.w) : 0.0;
    if (rest.w != 0.0) a += rest.w * (rest.left - rest.up - log_s);
    return bad ? __builtin_nan("") : a * row.over_w - w + p;
}
__device__ __forceinline__ double teacher_share(const Row& r, float v, float most_t, const Temper& t) { return exp(((double)v - (double)most_t) * t.inverse) * r.per_w; }
__device__ __forceinline__ double student_share(const Row& r, float z, float base, const Temper& t) { return exp(((double)z - (double)base) * t.inverse) * r.per_p; }

// d D / d (z / T) of the class of an entry; q: of its entry alone, unless `repeats`: a class may stand in several
__device__ __forceinline__ float entry_slope(const Lists& l, int64_t r, const Entry& e, const Row& row, float most_t, float base, bool repeats, const Temper& t) {
    double q = 0.0;
    if (repeats) {
        for (int i = 0; i < l.k; i++)
            if (l.cls(r * l.k + i) == e.cls) q += teacher_share(row, l.value(r * l.k + i), most_t, t);
    } else q = teacher_share(row, e.t, most_t, t);
    return (float)(student_share(row, e.z, base, t) - q);
}
// whether no entry before j has its class
__device__ __forceinline__ bool first_of(const Lists& l, int64_t r, int j, int64_t cls) {
    for (int i = 0; i < j; i++)
        if (l.cls(r * l.k + i) == cls) return false;
    return true;
}

struct First { double share, weight; };     // of a lane's first entry, the student's and the teacher's, where no class repeats: there seldom is a second one

// The outcomes of row r by a group of 2^shift lanes of a wavefront, all of which call it, with what they give for the row.  `skip`: the row does not count.
template <class T> __device__ __forceinline__ void outcomes_of(const LogitRows& a, const Lists& l, const Temper& t, const Outcome& e, int64_t r, const Others& o, bool skip, bool repeats,
                                                              int lane, int shift, float2& stats, float& most_t, float& base, Row& row, First& first) {
    const int lanes = 1 << shift;
    const T* z = row_start<T>(a, r);
    stats = make_float2(0.f, 0.f);
    row = Row{0.0, 0.0, 0.0, 0.f};
    first = First{0.0, 0.0};
    double divergence = 0.0;
    most_t = base = 0.f;
    if (!skip) {
        float bad = 0.f;
        most_t = base = -INFINITY;
        for (int j = lane; j < l.k; j += lanes) {
            const int64_t c = l.cls(r * l.k + j);
            if (c < 0) continue;
            const float v = l.value(r * l.k + j), u = c < a.classes ? Elem<T>::get(z[c]) : __builtin_nanf("");
            most_t = fmaxf(most_t, v);
            base = fmaxf(base, u);
            if (v != v || u != u) bad = 1.f;
        }
        const double rest = l.rest ? (double)l.rest[r] : -INFINITY;
        if (rest != rest || o.sum != o.sum) bad = 1.f;
        most_t = group_max(most_t, shift); base = group_max(base, shift); bad = group_max(bad, shift);
        const float entries = base;
        if (most_t == -INFINITY) most_t = 0.f;
        if (base == -INFINITY) base = 0.f;
        Sums s{0.0, 0.0, 0.0};
        for (int j = lane; j < l.k; j += lanes) {
            const int64_t c = l.cls(r * l.k + j);
            if (c < 0 || c >= a.classes) continue;
            const double share = add_entry(s, Entry{c, l.value(r * l.k + j), Elem<T>::get(z[c])}, most_t, base, !repeats || first_of(l, r, j, c), t);
            if (j == lane) first = First{share, s.w};
        }
        s.w = group_total(s.w, shift); s.p = group_total(s.p, shift); s.a = group_total(s.a, shift);
        const Rest left = rest_of(rest, most_t, entries, o.top, t);
        row = ratios_of(s, left, o, bad != 0.f);
        divergence = divergence_of(s, left, o, row, bad != 0.f);
        stats = make_float2(finite(o.top), row.factor);
    }
    if (lane == 0) {
        e.divergences[r] = (float)divergence;
        e.kept[r] = skip ? 0.f : 1.f;
        if (e.stats) e.stats[r] = stats;
    }
}

// The entries of row r, once its outcomes are known: f gets each one's class (inside the row) and slope; the slopes are kept for a later gradient.
template <class T> __device__ __forceinline__ void each_slope(const LogitRows& a, const Lists& l, const Temper& t, const Outcome& e, int64_t r, bool skip, bool repeats, int lane, int shift,
                                                                     float most_t, float base, const Row& row, const First& first) {
    const T* z = row_start<T>(a, r);
    for (int j = lane; j < l.k; j += 1 << shift) {
        const int64_t c = skip ? -1 : l.cls(r * l.k + j);
        const bool inside = c >= 0 && c < a.classes;
        float slope = 0.f;
        if (inside) slope = j == lane && !repeats ? (float)(first.share * row.per_p - first.weight * row.per_w)
                                                  : entry_slope(l, r, Entry{c, l.value(r * l.k + j), Elem<T>::get(z[c])}, row, most_t, base, repeats, t);
        e.entries[r * l.k + j] = slope;
    }
}

// whether row r counts, by a group of lanes that all call it
__device__ __forceinline__ bool counts(const Lists& l, int64_t r, int lane, int shift) {
    float entry = 0.f, live = l.rest && l.rest[r] != -INFINITY ? 1.f : 0.f;
    for (int j = lane; j < l.k; j += 1 << shift) {
        const int64_t c = l.cls(r * l.k + j);
        const int what = c < 0 ? 0 : said(c, l.value(r * l.k + j));
        if (what) entry = 1.f;
        if (what & 2) live = 1.f;
    }
    return group_max(entry, shift) != 0.f && group_max(live, shift) != 0.f;
}

// (of the lanes of a wavefront, which go through these in step)
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// N values become those of a row's gradient
template <class T, int N> __device__ __forceinline__ void gradient_values(float (&f)[N], float top, float w, const Temper& t) {
    #pragma unroll
    for (int i = 0; i < N; i++) f[i] = exp_stored<T>(f[i] - top, t) * w;
}

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

// -inf in the place of those values of a vector whose bit is set
template <class T> __device__ __forceinline__ u32x4 without(u32x4 v, uint32_t bits) {
    const u32x4 none = Elem<T>::splat(Elem<T>::put(-INFINITY));
    #pragma unroll
    for (int w = 0; w < 4; w++) {
        if constexpr (sizeof(T) == 4) v[w] = bits >> w & 1 ? none[w] : v[w];
        else {
            v[w] = bits >> (2 * w) & 1 ? (v[w] & 0xffff0000u) | (none[w] & 0xffffu) : v[w];
            v[w] = bits >> (2 * w + 1) & 1 ? (v[w] & 0xffffu) | (none[w] & 0xffff0000u) : v[w];
        }
    }
    return v;
}

// ---- short rows ------------------------------------------------------------------------------------------------------------
// Lanes that hold a row mark the entries' classes for each other; a value of the row that is marked becomes -inf.
template <class T, int NV> __device__ __forceinline__ bool take_out(HeldRow<T, NV>& row, const Lists& l, int64_t r, uint32_t (&marks)[256][2]) {
    constexpr int V = Elem<T>::kVec;
    const int first = (int)threadIdx.x - row.lane;
    uint32_t* own = marks[threadIdx.x];
    own[0] = own[1] = 0u;
    wave_fence();
    float twice = 0.f;
    const auto mark = [&](int i, int e) {
        const int bit = (i >> row.shift) * V + e;
        const uint32_t one = 1u << (bit & 31);
        return atomicOr(&marks[first + (i & ((1 << row.shift) - 1))][bit >> 5], one) & one;
    };
    for (int j = row.lane; j < l.k; j += 1 << row.shift) {
        const int64_t c64 = l.cls(r * l.k + j);
        if (c64 < 0 || c64 >= row.n) continue;
        const int c = (int)c64, i = c / V, start = row.n >= V ? row.column(i) : 0;
        if (mark(i, c - start)) twice = 1.f;
        // (the last vector has some of the values of the one before it)
        if (row.n >= V && i != row.vecs - 1 && c >= row.n - V) mark(row.vecs - 1, c - (row.n - V));
    }
    wave_fence();
    const uint32_t low = own[0], high = own[1];
    if (low | high) {
        #pragma unroll
        for (int k = 0; k < NV; k++) {
            const uint32_t bits = (k * V < 32 ? low >> (k * V & 31) : high >> (k * V & 31)) & ((1u << V) - 1u);
            if (bits) row.v[k] = without<T>(row.v[k], bits);
        }
    }
    return group_max(twice, row.shift) != 0.f;
}

template <class T, int NV> __device__ __forceinline__ Others others_of(const HeldRow<T, NV>& row, const Temper& t) {
    constexpr int V = Elem<T>::kVec;
    float top = -INFINITY;
    #pragma unroll
    for (int k = 0; k < NV; k++)
        if (row.index(k) < row.vecs) {
            float f[V];
            Elem<T>::unpack(row.v[k], f);
            #pragma unroll
            for (int i = 0; i < V; i++) top = fmaxf(top, f[i]);
        }
    top = group_max(top, row.shift);
    const float b = finite(top);
    double s = 0.0;
    #pragma unroll
    for (int k = 0; k < NV; k++)
        if (row.index(k) < row.vecs) {
            const int past = row.n >= V ? row.index(k) * V - row.column(row.index(k)) : 0;      // values that the vector before has, too
            float f[V];
            Elem<T>::unpack(row.v[k], f);
            #pragma unroll
            for (int i = 0; i < V; i++) f[i] = exp_at(f[i] - b, t);
            if (past > 0) {
                #pragma unroll
                for (int i = 0; i < V; i++) f[i] = i < past ? 0.f : f[i];
            }
            s += (double)tree(f);
        }
    return Others{top, group_total(s, row.shift)};
}

// the row's part of a gradient, the entries' classes left to be stored
template <class T, int NV> __device__ __forceinline__ void store_gradient(const HeldRow<T, NV>& row, T* q, float2 stats, float by, const Temper& t) {
    constexpr int V = Elem<T>::kVec;
    #pragma unroll
    for (int k = 0; k < NV; k++)
        if (row.index(k) < row.vecs) {
            const int c = row.n >= V ? row.column(row.index(k)) : 0;
            float f[V];
            if (stats.y == 0.f) {
                #pragma unroll
                for (int i = 0; i < V; i++) f[i] = 0.f;
            } else {
                Elem<T>::unpack(row.v[k], f);
                gradient_values<T>(f, stats.x, stats.y * by, t);
            }
            if (row.n >= V) {
                store16(q + c, Elem<T>::pack(f));
            } else {
                #pragma unroll
                for (int i = 0; i < V; i++)
                    if (i < row.n) q[i] = Elem<T>::put(f[i]);
            }
        }
}

// Short rows, one by each group of lanes.  Bound by a row's 64-bit functions: 65536 x 1000 bf16 65 us (2.0 TB/s).
template <class T, int NV> __global__ void __launch_bounds__(256) distill_short_kernel(LogitRows a, Lists l, Temper t, Outcome e, int shift, int64_t row0) {
    __shared__ uint32_t marks[256][2];
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    HeldRow<T, NV> row;
    row.n = (int)a.classes; row.shift = shift;
    row.lane = threadIdx.x & ((1 << shift) - 1);
    row.vecs = (row.n + Elem<T>::kVec - 1) / Elem<T>::kVec;
    const int64_t r = row0 + (int64_t)blockIdx.x * (256 >> shift) + (threadIdx.x >> shift);
    if (r >= a.rows) return;
    const bool skip = !counts(l, r, row.lane, shift);
    Others o{-INFINITY, 0.0};
    bool repeats = false;
    if (!skip) {
        row.load(row_start<T>(a, r));
        repeats = take_out(row, l, r, marks);
        o = others_of(row, t);
    }
    float2 stats;
    float most_t, base;
    Row end;
    First first;
    outcomes_of<T>(a, l, t, e, r, o, skip, repeats, row.lane, shift, stats, most_t, base, end, first);
    if (e.entries) each_slope<T>(a, l, t, e, r, skip, repeats, row.lane, shift, most_t, base, end, first);
}

// Their gradient, bound by its bytes: 65536 x 1000 bf16 57 us (4.6 TB/s).
template <class T, int NV> __global__ void __launch_bounds__(256) distill_short_gradient_kernel(LogitRows a, Lists l, Temper t, Slopes g, int shift) {
    if (g.unless_one && *g.scale2 == 1.f) return;
    const int per = 256 >> shift;
    HeldRow<T, NV> row;
    row.n = (int)a.classes; row.shift = shift;
    row.lane = threadIdx.x & ((1 << shift) - 1);
    row.vecs = (row.n + Elem<T>::kVec - 1) / Elem<T>::kVec;
    const float by = g.by();
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += (int64_t)gridDim.x * per) {
        const float2 stats = g.stats[r];
        if (stats.y != 0.f) row.load(row_start<T>(a, r));
        T* q = static_cast<T*>(g.grad) + r * a.classes;
        store_gradient(row, q, stats, by, t);
        wave_fence();
        for (int j = row.lane; j < l.k; j += 1 << shift) {
            const int64_t c = l.cls(r * l.k + j);
            if (c >= 0 && c < a.classes) q[c] = Elem<T>::put(g.entries[r * l.k + j] * by);
        }
    }
}

// ---- long rows ---------------------------------------------------------------------------------------------------------------
// Marks of the entries' classes among the vectors that a workgroup holds, by the work-item that holds each: NV vectors, the k-th vector item + k THREADS.
template <class T, int NV, int THREADS> struct Marks {
    static constexpr int V = Elem<T>::kVec, kWords = (NV * V + 31) / 32;
    uint32_t words[THREADS][kWords];
    int repeats;
    __device__ __forceinline__ void clear() {
        #pragma unroll
        for (int w = 0; w < kWords; w++) words[threadIdx.x][w] = 0u;
        if (threadIdx.x == 0) repeats = 0;
    }
    __device__ __forceinline__ void mark(int at) {      // at: the class behind those before the vectors
        const int vec = at / V, bit = vec / THREADS * V + at % V;
        const uint32_t one = 1u << (bit & 31);
        if (atomicOr(&words[vec % THREADS][bit >> 5], one) & one) repeats = 1;
    }
    __device__ __forceinline__ uint32_t bits(int k) const { return words[threadIdx.x][k * V / 32] >> (k * V & 31) & ((1u << V) - 1u); }
};

// the vector `item` behind a pointer that is the same for all lanes: an offset of 32 bits is added by the load or store itself
template <class T> __device__ __forceinline__ T* behind(T* p, int item) { return (T*)((const char*)p + (uint32_t)item * 16u); }

// The workgroup holds a row in its registers, at most 16 vectors per work-item, and an entry per work-item.  FUSED: the logits are read once and the gradient leaves
// with the row, and these are read past the caches.
// A row per workgroup and no loop over them: the constants of the 64-bit functions would be kept in registers that the row needs.  What the entries give is summed
// while the row is on its way; when it is there a wavefront's part, one barrier and a few 64-bit functions of one wavefront stand between its sums and its gradient.
// 4096 x 131072 bf16 431 us (4.7 TB/s): a compute unit has one such row at a time, and what it waits for between loads and stores, and its vector instructions, hide in part only.
template <class T, int NV, int THREADS, bool FUSED> __global__ void __launch_bounds__(THREADS, 4) distill_held_kernel(LogitRows a, Lists l, Temper t, Outcome e, Slopes g, int64_t row0) {
    constexpr int V = Elem<T>::kVec, WAVES = THREADS / 64, kChunk = NV < 32 / V ? NV : 32 / V;
    constexpr int kShift = WAVES == 4 ? 2 : WAVES == 8 ? 3 : 4;      // (the wavefronts' results in the lanes of each group of so many)
    static_assert(kMostEntries <= 256 && WAVES >= 4, "the first four wavefronts have the entries");
    __shared__ Marks<T, NV + 1, THREADS> marks;       // (one more: the values behind the last whole vector)
    __shared__ float most[4][2];
    __shared__ double sums[4][3];
    __shared__ Others others[WAVES];
    __shared__ double weights[kMostEntries];        // the teacher's, relative to the largest, and what
    __shared__ int theirs_of[kMostEntries];         // class each is for
    __shared__ Row end;
    __shared__ float end_top;
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    const int n = (int)a.classes, full = n / V, rest_at = full * V + (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63;
    const T lowest = Elem<T>::put(-INFINITY);
    const float by = FUSED ? *g.scale : 0.f;
    const int64_t r = a.rows - 1 - (row0 + blockIdx.x);     // (the producer's last rows may be in the caches)
    T* q = static_cast<T*>(g.grad) + r * a.classes;
    const bool own = (int)threadIdx.x < l.k;
    bool skip;
    // a work-item's entry: its class (-1: none, n: one that is not in the row) and the two logits
    int cls = -1;
    float value = -INFINITY, z = -INFINITY;
    const auto decode = [&](const Lists::Raw& mine) {
        if (own) {
            const int64_t c = l.cls(mine);
            cls = c < 0 ? -1 : c < n ? (int)c : n;
            value = l.value(mine);
        }
    };
    if (FUSED) skip = e.kept[r] == 0.f;
    const Lists::Raw entry = l.raw(r * l.k + (own ? (int)threadIdx.x : 0));
    if (!FUSED) {
        decode(entry);
        const int what = said(cls, value);
        const bool any = __syncthreads_or(what & 1), live = __syncthreads_or(what & 2);
        skip = !any || !(live || (l.rest && l.rest[r] != -INFINITY));
    }
    if (skip) {     // (the whole workgroup's)
        if (own && e.entries) e.entries[r * l.k + threadIdx.x] = 0.f;
        if (threadIdx.x == 0) {
            e.divergences[r] = 0.f;
            e.kept[r] = 0.f;
            if (e.stats) e.stats[r] = make_float2(0.f, 0.f);
        }
        if (FUSED) clear_row(q, n, THREADS);
        return;
    }
    const T* p = row_start<T>(a, r);
    // the entries' logits are asked for before the row: loads arrive in their order
    T theirs_z = lowest;
    if (64 * wave < l.k) {
        if (FUSED) decode(entry);
        theirs_z = p[cls >= 0 && cls < n ? cls : 0];
    }
    u32x4 v[NV];
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int i = (int)threadIdx.x + k * THREADS;
        const T* from = behind(p, i < full ? i : full - 1);     // (under no condition: behind one no load can be waited for by itself)
        v[k] = FUSED ? stream16(from) : load16(from);
    }
    T last = p[rest_at < n ? rest_at : n - 1];
    const double rest = l.rest ? (double)l.rest[r] : -INFINITY;
    const bool inside = cls >= 0 && cls < n;
    marks.clear();
    __syncthreads();
    // (the values behind the last whole vector are held by the first work-items, one each, as the first value of a vector of their own)
    if (inside) marks.mark(cls < full * V ? cls : (NV * THREADS + (cls - full * V)) * V);
    if (own) theirs_of[threadIdx.x] = inside ? cls : -1;
    if (wave < 4) {
        if (inside) z = Elem<T>::get(theirs_z);
        const float m0 = group_max(inside ? value : -INFINITY, 6), m1 = group_max(z, 6);
        if (lane == 0) { most[wave][0] = m0; most[wave][1] = m1; }
    }
    __syncthreads();
    const bool repeats = marks.repeats != 0;
    float most_t = 0.f, entries = 0.f;
    double share = 0.0;
    if (wave < 4) {
        most_t = fmaxf(fmaxf(most[0][0], most[1][0]), fmaxf(most[2][0], most[3][0]));
        entries = fmaxf(fmaxf(most[0][1], most[1][1]), fmaxf(most[2][1], most[3][1]));
        if (most_t == -INFINITY) most_t = 0.f;
        Sums s{0.0, 0.0, 0.0};
        if (64 * wave < l.k) {
            if (inside) {
                bool first = true;
                if (repeats)
                    for (int i = 0; i < (int)threadIdx.x; i++) first = first && theirs_of[i] != cls;
                share = add_entry(s, Entry{cls, value, z}, most_t, entries == -INFINITY ? 0.f : entries, first, t);
                weights[threadIdx.x] = s.w;
            }
            if (rest != rest || (cls >= 0 && (!inside || value != value || z != z))) s.p = __builtin_nan("");      // (something is wrong with the row)
            s.w = wave_total(s.w); s.p = wave_total(s.p); s.a = wave_total(s.a);
        }
        if (lane == 0) { sums[wave][0] = s.w; sums[wave][1] = s.p; sums[wave][2] = s.a; }
    }
    float top = -INFINITY;
    double sum = 0.0;
    #pragma unroll
    for (int c = 0; c < NV; c += kChunk) {
        float f[kChunk * V];
        #pragma unroll
        for (int k = c; k < c + kChunk; k++) {
            const uint32_t listed = marks.bits(k);
            if ((k + 1) * THREADS > full) {
                asm volatile("");       // (a branch of the whole workgroup's)
                if ((int)threadIdx.x + k * THREADS >= full) v[k] = Elem<T>::splat(lowest);
            }
            if (listed) v[k] = without<T>(v[k], listed);
            Elem<T>::unpack(v[k], reinterpret_cast<float (&)[V]>(f[(k - c) * V]));
        }
        take(f, top, sum, t);
        asm volatile("" : "+v"(top), "+v"(sum));     // (here, while the next vectors are on their way, and not behind them all)
    }
    if (rest_at >= n || (marks.bits(NV) & 1u)) last = lowest;
    float f1[1] = {Elem<T>::get(last)};
    take(f1, top, sum, t);
    {
        const float m = group_max(top, 6);
        sum = wave_total(sum * (double)exp_at(finite(top) - finite(m), t));
        if (lane == 0) others[wave] = Others{m, sum};
    }
    __syncthreads();
    Others o{-INFINITY, 0.0};
    Sums s{0.0, 0.0, 0.0};
    Rest left;
    bool odd = false;
    if (wave == 0) {        // (the others wait: with four wavefronts to a unit that each did this it would take four times as long)
        const Others part = others[lane & (WAVES - 1)];
        o.top = group_max(part.top, kShift);
        o.sum = group_total(part.sum * (double)exp_at(finite(part.top) - finite(o.top), t), kShift);
        s = Sums{group_total(sums[lane & 3][0], 2), group_total(sums[lane & 3][1], 2), group_total(sums[lane & 3][2], 2)};
        odd = o.sum != o.sum || s.p != s.p;
        left = rest_of(rest, most_t, entries, o.top, t);
        const Row row = ratios_of(s, left, o, odd);
        if (lane == 0) { end = row; end_top = finite(o.top); }
    }
    __syncthreads();
    const Row row = end;
    const float high = end_top;
    if (FUSED) {
        if (row.factor == 0.f) clear_row(q, n, THREADS);
        else {
            // what was derived from the vectors is derived again: kept, it would be twice their registers
            int item = threadIdx.x;
            asm("" : "+v"(item));
            #pragma unroll
            for (int k = 0; k < NV; k++) asm("" : "+v"(v[k]));
            const float w = row.factor * by;
            #pragma unroll
            for (int k = 0; k < NV; k++) {
                const int i = item + k * THREADS;
                float f[V];
                Elem<T>::unpack(v[k], f);
                gradient_values<T>(f, high, w, t);
                if (i < full) put_stream16(behind(q, i), Elem<T>::pack(f));
            }
            if (rest_at < n) {
                float f[1] = {Elem<T>::get(last)};
                gradient_values<T>(f, high, w, t);
                q[rest_at] = Elem<T>::put(f[0]);
            }
        }
    }
    float slope = 0.f;
    if (inside) {
        double weight = weights[threadIdx.x];
        if (repeats) {
            weight = 0.0;
            for (int i = 0; i < l.k; i++) weight += theirs_of[i] == cls ? weights[i] : 0.0;
        }
        slope = (float)(share * row.per_p - weight * row.per_w);
    }
    if (own && e.entries) e.entries[r * l.k + threadIdx.x] = slope;
    if (wave == 0) {
        const double divergence = divergence_of(s, left, o, row, odd);
        if (lane == 0) {
            e.divergences[r] = (float)divergence;
            e.kept[r] = 1.f;
            if (e.stats) e.stats[r] = make_float2(high, row.factor);
        }
    }
    if (FUSED) {
        __syncthreads();        // (the entries' values stand where the others' stood)
        if (inside) q[cls] = Elem<T>::put(slope * by);
    }
}

// Rows that no workgroup can hold: parts of them, whose others distill_join_kernel joins.  16 x 200001 bf16
// 12 us, the join 6, the gradient 6: launches and chains of loads.
constexpr int kPartVectors = 8;
template <class T> __global__ void __launch_bounds__(256) distill_part_kernel(LogitRows a, Lists l, Temper t, Outcome e, int splits, int64_t part, Others* parts, int* twice) {
    constexpr int V = Elem<T>::kVec, kSpan = 256 * kPartVectors * V;
    __shared__ Marks<T, kPartVectors, 256> marks;
    __shared__ Others waves[4];
    if (e.ticket && blockIdx.x == 0 && threadIdx.x == 0) *e.ticket = 0u;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = b / splits, s = b - r * splits, from = s * part, until = a.classes - from < part ? a.classes : from + part;
        const T* p = row_start<T>(a, r);
        int64_t cls = -1;
        float value = -INFINITY;
        if ((int)threadIdx.x < l.k) { cls = l.cls(r * l.k + threadIdx.x); value = l.value(r * l.k + threadIdx.x); }
        const int what = said(cls, value);
        const bool entry = __syncthreads_or(what & 1), live = __syncthreads_or(what & 2);
        float top = -INFINITY;
        double sum = 0.0;
        bool repeats = false;
        if (entry && (live || (l.rest && l.rest[r] != -INFINITY))) {
            for (int64_t c0 = from; c0 < until; c0 += kSpan) {
                const int64_t n = until - c0;
                u32x4 v[kPartVectors];
                #pragma unroll
                for (int k = 0; k < kPartVectors; k++) {
                    const int c = (k * 256 + (int)threadIdx.x) * V;
                    v[k] = Elem<T>::splat(Elem<T>::put(-INFINITY));
                    if (c + V <= n) v[k] = load16(p + c0 + c);
                    else if (c < n) {
                        float f[V];
                        #pragma unroll
                        for (int i = 0; i < V; i++) f[i] = c + i < n ? Elem<T>::get(p[c0 + c + i]) : -INFINITY;
                        v[k] = Elem<T>::pack(f);
                    }
                }
                marks.clear();
                __syncthreads();
                if (cls >= c0 && cls < until && cls < c0 + kSpan) marks.mark((int)(cls - c0));
                __syncthreads();
                repeats |= marks.repeats != 0;
                #pragma unroll
                for (int k = 0; k < kPartVectors; k += 2) {
                    float f[2 * V];
                    Elem<T>::unpack(without<T>(v[k], marks.bits(k)), reinterpret_cast<float (&)[V]>(f[0]));
                    Elem<T>::unpack(without<T>(v[k + 1], marks.bits(k + 1)), reinterpret_cast<float (&)[V]>(f[V]));
                    take(f, top, sum, t);
                }
                __syncthreads();
            }
        }
        const float m = group_max(top, 6);
        sum = wave_total(sum * (double)exp_at(finite(top) - finite(m), t));
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = Others{m, sum};
        __syncthreads();
        if (threadIdx.x == 0) {
            Others o{-INFINITY, 0.0};
            for (int w = 0; w < 4; w++) o.top = fmaxf(o.top, waves[w].top);
            for (int w = 0; w < 4; w++) o.sum += waves[w].sum * (double)exp_at(finite(waves[w].top) - finite(o.top), t);
            parts[b] = o;
            twice[b] = repeats;
        }
        __syncthreads();
    }
}

// a wavefront per row
template <class T> __global__ void __launch_bounds__(256) distill_join_kernel(LogitRows a, Lists l, Temper t, Outcome e, int splits, const Others* parts, const int* twice) {
    const int lane = threadIdx.x & 63;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < a.rows; r += (int64_t)gridDim.x * 4) {
        const bool skip = !counts(l, r, lane, 6);
        float top = -INFINITY, repeats = 0.f;
        for (int k = lane; k < splits; k += 64) {
            top = fmaxf(top, parts[r * splits + k].top);
            if (twice[r * splits + k]) repeats = 1.f;
        }
        top = group_max(top, 6);
        double sum = 0.0;
        for (int k = lane; k < splits; k += 64) sum += parts[r * splits + k].sum * (double)exp_at(finite(parts[r * splits + k].top) - finite(top), t);
        const Others o{top, wave_total(sum)};
        const bool twice_there = group_max(repeats, 6) != 0.f;
        float2 stats;
        float most_t, base;
        Row end;
        First first;
        outcomes_of<T>(a, l, t, e, r, o, skip, twice_there, lane, 6, stats, most_t, base, end, first);
        if (e.entries) each_slope<T>(a, l, t, e, r, skip, twice_there, lane, 6, most_t, base, end, first);
    }
}

// A workgroup writes `part` columns of a row's gradient, then those of its entries that lie there.
template <class T> __global__ void __launch_bounds__(256) distill_long_gradient_kernel(LogitRows a, Lists l, Temper t, Slopes g, int splits, int64_t part) {
    constexpr int V = Elem<T>::kVec, kUnroll = 4;
    if (g.unless_one && *g.scale2 == 1.f) return;
    const float by = g.by();
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = b / splits, c0 = (b - r * splits) * part, c1 = a.classes - c0 < part ? a.classes : c0 + part, full = c1 / V;
        const float2 stats = g.stats[r];
        const float w = stats.y * by;
        const T* src = row_start<T>(a, r);
        T* q = static_cast<T*>(g.grad) + r * a.classes;
        const bool own = (int)threadIdx.x < l.k;
        const int64_t cls = own ? l.cls(r * l.k + threadIdx.x) : -1;
        const float slope = own ? g.entries[r * l.k + threadIdx.x] * by : 0.f;
        for (int64_t i = c0 / V + threadIdx.x; i < full; i += kUnroll * 256) {
            u32x4 v[kUnroll];
            #pragma unroll
            for (int k = 0; k < kUnroll; k++)
                if (stats.y != 0.f && i + k * 256 < full) v[k] = load16(src + (i + k * 256) * V);
            #pragma unroll
            for (int k = 0; k < kUnroll; k++) {
                if (i + k * 256 >= full) continue;
                float f[V];
                if (stats.y == 0.f) {
                    #pragma unroll
                    for (int m = 0; m < V; m++) f[m] = 0.f;
                } else {
                    Elem<T>::unpack(v[k], f);
                    gradient_values<T>(f, stats.x, w, t);
                }
                put_stream16(q + (i + k * 256) * V, Elem<T>::pack(f));
            }
        }
        for (int64_t j = full * V + threadIdx.x; j < c1; j += 256) q[j] = Elem<T>::put(stats.y == 0.f ? 0.f : exp_stored<T>(Elem<T>::get(src[j]) - stats.x, t) * w);
        __syncthreads();        // (the entries' values stand where these stood)
        if (cls >= c0 && cls < c1) q[cls] = Elem<T>::put(slope);
    }
}

// ---- the loss --------------------------------------------------------------------------------------------------------------------
// Which rows count, before they are read: a wavefront per row; the workgroups' numbers of them to `counted`.
__global__ void __launch_bounds__(256) distill_rows_that_count_kernel(Lists l, int64_t rows, float* kept, int* counted) {
    __shared__ int waves[4];
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4) {
        const bool here = counts(l, r, lane, 6);
        if (lane == 0) kept[r] = here ? 1.f : 0.f;
        n += here;
    }
    if (lane == 0) waves[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) counted[blockIdx.x] = waves[0] + waves[1] + waves[2] + waves[3];
}
// scale = factor / their number
__global__ void __launch_bounds__(256) distill_scale_kernel(const int* counted, int blocks, double factor, float* scale) {
    __shared__ int waves[4];
    int n = 0;
    for (int i = threadIdx.x; i < blocks; i += 256) n += counted[i];
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = n;
    __syncthreads();
    if (threadIdx.x == 0) {
        n = waves[0] + waves[1] + waves[2] + waves[3];
        *scale = (float)(factor / (n > 1 ? n : 1));
    }
}

// loss = weight T^2 mean of the divergences over the rows that count (0 where there are none), scale = weight T / their number (or null: it is there)
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

// ---- host ------------------------------------------------------------------------------------------------------------------------
namespace {

constexpr int kMeanBlocks = 128, kCountBlocks = 256;

int check_lists(const sd_top_lists* in, const char* who, Lists* l) {
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

// scratch: the ticket, sums of workgroups (the counts' place before), a mark for each row that counts, parts of long rows
constexpr int64_t kDistillSums = 4 + 4 * kMeanBlocks;
static_assert(4 * kMeanBlocks >= kCountBlocks, "counts of workgroups stand where their sums will");
int64_t kept_floats(int64_t rows) { return (rows + 3) / 4 * 4; }

struct Cut { int splits; int64_t part; };
Cut cut_of(const LogitRows& a, int vec) {
    int splits = row_splits(a.rows, a.classes, vec);
    const int64_t part = part_of(a.classes, splits, vec);
    return {(int)((a.classes + part - 1) / part), part};
}

// Lanes for a short row: whole quads (see four_of), and of many rows more of them in a wavefront, for each of which a row's 64-bit functions cost
// as much: 8192 x 1000 fp32, k = 16, 22.0 us with 64 lanes for a row, 17.4 with 32.  The border at half and at four times as many, k = 3 and 16:
// 4000 x 2000 bf16 14.6 and 16.3 us (2^17 and 2^18), 16384 x 200 fp32 13.4 and 14.7, 65536 x 200 bf16 30 and 29 (2^18 and 2^20); of lists longer than a row's lanes each lane
// has several entries, one behind the other: k = 64, 65536 x 200 fp32 110 and 58.
constexpr int64_t kFewLanes = 1 << 18;
Group short_group(const LogitRows& a, int vec) {
    Group g = group_of(a.rows, a.classes, vec);
    if (g.shift < 0) return g;
    while (g.shift < 2) { g.shift++; g.vectors = g.vectors > 1 ? g.vectors / 2 : 1; }
    while (g.vectors < kHeld && g.shift > 2 && a.rows << g.shift > kFewLanes) { g.shift--; g.vectors *= 2; }
    return g;
}

// Whether a row is read in parts, being more than a workgroup can hold.  Where it can, few rows are no reason: 16 x 65536 bf16 21.5 us with the gradient, held 18.7.
bool in_parts(const LogitRows& a, int vec) { return (a.classes + vec - 1) / vec > 16 * 512; }

int64_t distill_floats(const LogitRows& a, int dtype) {
    const int vec = vec_of(dtype);
    return kDistillSums + kept_floats(a.rows) + (in_parts(a, vec) ? ((int64_t)(sizeof(Others) + sizeof(int)) / 4 * a.rows * cut_of(a, vec).splits + 3) / 4 * 4 : 0);
}

// Whether the gradient leaves with the rows: it then costs one reading of the logits less and two launches more.  A workgroup must be able to hold a row, and there
// must be rows for all compute units.  Loss and gradient of 4500 x 4096 bf16 (35 MiB) 43.7 us with it and 39.9 without, 800 x 30001 (46 MiB) 42.0 and 44.4, 8192 x 4096
// 63.7 and 68.7, 4096 x 131072 479 and 665; of short rows, whose 64-bit functions the gradient would wait for, 65536 x 1000 fp32 232 and 207.
bool fuses(const LogitRows& a, int dtype) {
    const int vec = vec_of(dtype);
    return a.rows * a.classes * (16 / vec) >= (40ll << 20) && short_group(a, vec).shift < 0 && a.rows >= 512 && a.classes <= kHeldLong * vec;
}

}  // namespace

}  // namespace sd

using namespace sd;

extern "C" int64_t sd_distill_scratch(const sd_logit_rows* rows, int64_t k) {
    LogitRows a;
    if (check_logits(rows, "distill_scratch", &a) != SD_OK) return -1;
    if (k < 1 || k > kMostEntries) { set_error("distill_scratch: k=%lld entries for each row: 1..%d are possible", (long long)k, kMostEntries); return -1; }
    return distill_floats(a, rows->dtype);
}

extern "C" int sd_distill_fuses(const sd_logit_rows* rows) {
    LogitRows a;
    return check_logits(rows, "distill_fuses", &a) == SD_OK && fuses(a, rows->dtype) ? 1 : 0;
}

extern "C" int sd_distill_loss(const sd_logit_rows* rows, const sd_top_lists* lists, double temperature, double weight, float* stats, float* entries, float* scale, void* grad,
                               float* loss, float* divergences, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    Lists l;
    Temper t;
    if (int rc = check_logits(rows, "distill_loss", &a)) return rc;
    if (int rc = check_lists(lists, "distill_loss", &l)) return rc;
    if (int rc = check_temper(temperature, weight, "distill_loss", &t)) return rc;
    SD_REQUIRE(loss && divergences && scratch, "distill_loss: null argument");
    SD_REQUIRE(!stats == !entries && !stats == !scale, "distill_loss: the gradient needs stats, entries and scale");
    SD_REQUIRE(!grad || stats, "distill_loss: a gradient that leaves with the rows needs stats, entries and scale, too");
    SD_REQUIRE(!grad || fuses(a, rows->dtype), "distill_loss: the gradient of these rows does not leave with them (sd_distill_fuses)");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (reinterpret_cast<uintptr_t>(scratch) & 15) == 0 &&
               (reinterpret_cast<uintptr_t>(grad) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0, "distill_loss: stats must be aligned to 8 bytes, scratch to 16, the gradient to its type");
    hipStream_t s = static_cast<hipStream_t>(stream);
    float* kept = scratch + kDistillSums;
    const Outcome e{reinterpret_cast<float2*>(stats), entries, divergences, kept, reinterpret_cast<uint32_t*>(scratch)};
    const Slopes g{nullptr, nullptr, scale, nullptr, grad, false};
    const double scale_factor = weight * temperature;
    if (grad) {
        int* counted = reinterpret_cast<int*>(scratch + 4);
        const int64_t want = (a.rows + 3) / 4;
        const int blocks = (int)(want < kCountBlocks ? want : kCountBlocks);
        hipLaunchKernelGGL(distill_rows_that_count_kernel, dim3(blocks), dim3(256), 0, s, l, a.rows, kept, counted);
        hipLaunchKernelGGL(distill_scale_kernel, dim3(1), dim3(256), 0, s, counted, blocks, scale_factor, scale);
        if (int rc = check_launch("distill_rows_that_count_kernel or distill_scale_kernel")) return rc;
    }
    const int vec = vec_of(rows->dtype);
    const Group group = short_group(a, vec);
    const char* kernel = group.shift >= 0 ? "distill_short_kernel" : grad || !in_parts(a, vec) ? "distill_held_kernel" : "distill_part_kernel or distill_join_kernel";
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        if (group.shift >= 0) {
            const int per = 256 >> group.shift;
            with_vectors(group.vectors, [&](auto nv) {
                in_slices((a.rows + per - 1) / per, [&](int64_t from, unsigned blocks) {
                    hipLaunchKernelGGL((distill_short_kernel<T, nv.value>), dim3(blocks), dim3(256), 0, s, a, l, t, e, group.shift, from * per);
                });
            });
            return;
        }
        if (grad || !in_parts(a, vec)) {
            const int64_t vecs = (a.classes + vec - 1) / vec;
            const auto held = [&](auto fused) {
                in_slices(a.rows, [&](int64_t from, unsigned blocks) {
                    const dim3 grid(blocks);
                    if (vecs <= 4 * 256) hipLaunchKernelGGL((distill_held_kernel<T, 4, 256, fused.value>), grid, dim3(256), 0, s, a, l, t, e, g, from);
                    else if (vecs <= 8 * 256) hipLaunchKernelGGL((distill_held_kernel<T, 8, 256, fused.value>), grid, dim3(256), 0, s, a, l, t, e, g, from);
                    else if (vecs <= 16 * 256) hipLaunchKernelGGL((distill_held_kernel<T, 16, 256, fused.value>), grid, dim3(256), 0, s, a, l, t, e, g, from);
                    else if (vecs <= 16 * 512) hipLaunchKernelGGL((distill_held_kernel<T, 16, 512, fused.value>), grid, dim3(512), 0, s, a, l, t, e, g, from);
                    else if constexpr (fused.value) hipLaunchKernelGGL((distill_held_kernel<T, 16, 1024, true>), grid, dim3(1024), 0, s, a, l, t, e, g, from);
                });
            };
            if (grad) held(std::true_type());
            else held(std::false_type());
            return;
        }
        const Cut cut = cut_of(a, vec);
        Others* parts = reinterpret_cast<Others*>(kept + kept_floats(a.rows));
        int* twice = reinterpret_cast<int*>(parts + a.rows * cut.splits);
        hipLaunchKernelGGL(distill_part_kernel<T>, dim3(blocks_for(a.rows * cut.splits)), dim3(256), 0, s, a, l, t, e, cut.splits, cut.part, parts, twice);
        hipLaunchKernelGGL(distill_join_kernel<T>, dim3(blocks_for((a.rows + 3) / 4)), dim3(256), 0, s, a, l, t, e, cut.splits, parts, twice);
    });
    if (int rc = check_launch(kernel)) return rc;
    const int64_t want = (a.rows + 16383) / 16384;
    const Mean m{divergences, kept, a.rows, weight * temperature * temperature, scale_factor, loss, grad ? nullptr : scale, reinterpret_cast<double*>(scratch + 4), e.ticket};
    hipLaunchKernelGGL(distill_mean_kernel, dim3((unsigned)(want < kMeanBlocks ? want : kMeanBlocks)), dim3(1024), 0, s, m);
    return check_launch("distill_mean_kernel");
}

extern "C" int sd_distill_gradient(const sd_logit_rows* rows, const sd_top_lists* lists, double temperature, const float* stats, const float* entries, const float* scale,
                                   const float* scale2, int unless_one, void* grad, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    Lists l;
    Temper t;
    if (int rc = check_logits(rows, "distill_gradient", &a)) return rc;
    if (int rc = check_lists(lists, "distill_gradient", &l)) return rc;
    if (int rc = check_temper(temperature, 1.0, "distill_gradient", &t)) return rc;
    SD_REQUIRE(stats && entries && scale && grad, "distill_gradient: null argument");
    SD_REQUIRE(!unless_one || scale2, "distill_gradient: unless_one needs scale2");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(stats) & 7) == 0 && (reinterpret_cast<uintptr_t>(grad) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0,
               "distill_gradient: stats must be aligned to 8 bytes, the gradient to its type");
    const Slopes g{reinterpret_cast<const float2*>(stats), entries, scale, scale2, grad, unless_one != 0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const int vec = vec_of(rows->dtype);
    const Group group = short_group(a, vec);
    // a launch that mostly finds nothing to do has no more workgroups than run at once: each takes time to come and go
    const auto blocks = [&](int64_t n) { return dim3(unless_one && n > 8 * num_cus() ? (unsigned)(8 * num_cus()) : blocks_for(n)); };
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        if (group.shift >= 0) {
            const int per = 256 >> group.shift;
            with_vectors(group.vectors, [&](auto nv) {
                hipLaunchKernelGGL((distill_short_gradient_kernel<T, nv.value>), blocks((a.rows + per - 1) / per), dim3(256), 0, s, a, l, t, g, group.shift);
            });
            return;
        }
        const int64_t part = 256 * vec * 4;
        const int splits = (int)((a.classes + part - 1) / part);
        hipLaunchKernelGGL(distill_long_gradient_kernel<T>, blocks(a.rows * splits), dim3(256), 0, s, a, l, t, g, splits, part);
    });
    return check_launch(group.shift >= 0 ? "distill_short_gradient_kernel" : "distill_long_gradient_kernel");
}
