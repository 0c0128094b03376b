// The k largest logits of each row in order (of equal ones the lower class first), their classes, and the log-sum of the others at a temperature:
//   rest = log sum over the classes that are not among the k of exp(z[v] / T)   (-inf where there are none).
// Values are compared by whole numbers in their order (order_of): NaN above all, -0 as 0.  With the class behind it, upside down, every logit
// has a number of its own, so the k largest are the same in every call.
//
// A row is read once.  A bound that at least k of its logits reach comes from the work-items' own maxima over its first vectors: the least of the
// wavefronts' (k / wavefronts)-th largest ones.  What reaches the bound is put on a list in LDS, about 1.3 k of the first vectors' logits and with
// each further part of the row as many again; of what does not, the exponentials are summed (relative to the largest of them).  A list that gets long is cut
// to the k largest numbers, the last of which becomes the bound.  At the end the list is sorted by counting.  Few rows are read in parts, whose
// lists a second kernel joins.  Bound by the bytes of the logits where there are many, else by the steps of a row, which other rows' loads hide.
// Logits of -inf are never listed: where there are not k others the first classes that are -inf follow, which are among the row's first k.
#include <climits>
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kMostTop = SD_MOST_TOP;
constexpr int64_t kMostClasses = 1ll << 30;

__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
constexpr uint32_t kLowestOrder = 0x00800000u;      // of -FLT_MAX; that of -inf is one less

typedef unsigned long long Number;      // order << 32 | ~class; 0: none
__device__ __forceinline__ Number number_of(float v, int cls) { return (Number)order_of(v) << 32 | (uint32_t)~cls; }
__device__ __forceinline__ float number_value(Number x) { return value_of((uint32_t)(x >> 32)); }
__device__ __forceinline__ int number_class(Number x) { return (int)~(uint32_t)x; }

struct Top {
    int k;
    double inverse;         // 1 / temperature
    float high, low;        // log2(e) / temperature in two positive parts (see exp_of)
    void* values;
    int* classes;
    float* rest;
};
__device__ __forceinline__ float exp_at(float v, const Top& t) { return __builtin_amdgcn_exp2f(fmaf(v, t.high, v * t.low)); }

struct Others { float top; double sum; };       // sum of exp((v - top) / T)
// two of them as one; `top` may be infinite
__device__ __forceinline__ void join(Others& o, float top, double sum, const Top& t) {
    if (top > o.top) {
        o.sum *= (double)exp_at(o.top - top, t);
        o.top = top;
    }
    o.sum += sum * (top == o.top ? 1.0 : (double)exp_at(top - o.top, t));
}

// The parts of a row: the k largest numbers in order (0 where there are fewer) and the others of each; the sum is NaN in a part that has a NaN.
struct Parts { Number* numbers; Others* others; };

template <int THREADS> struct Shared {
    static constexpr int kCap = THREADS == 64 ? 512 : 2048;     // numbers of the list
    static constexpr int kLong = kCap / 2;                      // from here on it is cut; what an exact choice adds has room behind it
    static constexpr int kShort = kCap / 8;                     // and at the end from here on: sorting takes the square of the numbers
    static constexpr int kWaves = THREADS / 64;
    static constexpr int kOwn = kCap / THREADS;
    Number list[kCap];
    Others others[kWaves];
    uint32_t bounds[kWaves];
    int counts[2][kWaves];
    int count, bad, nan;
    uint32_t left_top;
    unsigned long long left_sum;
};
static_assert(Shared<256>::kShort >= kMostTop && Shared<256>::kShort <= 256 && Shared<64>::kShort <= 64, "a work-item per number at the end");

// The list of a row or part, kept by all work-items of a workgroup together: they all call every member but `push` and `leave`, which come between barriers.
template <int THREADS> struct Keeper {
    using S = Shared<THREADS>;
    S& s;
    const Top& t;
    float bound = -FLT_MAX;     // what reaches it is listed
    Others others{-INFINITY, 0.0};     // this work-item's
    int lane, wave, turn = 0;

    __device__ __forceinline__ Keeper(S& shared, const Top& top) : s(shared), t(top), lane(threadIdx.x & 63), wave(threadIdx.x >> 6) {
        if (threadIdx.x == 0) { s.count = 0; s.nan = 0; s.bad = 0; s.left_top = 0u; s.left_sum = 0ull; }
    }
    __device__ __forceinline__ void push(Number x) {
        const int at = atomicAdd(&s.count, 1);
        if (at < S::kCap) s.list[at] = x;
    }
    __device__ __forceinline__ void leave(float v) {
        if (v == v && v != -INFINITY) join(others, v, 1.0, t);
    }
    // The same for numbers of the list, whose places vary from call to call: their shares of the largest of them are added as whole numbers of 2^-40, in whatever
    // order.  (The first of `take(visit)`'s two passes comes after a barrier.)
    template <class Take> __device__ __forceinline__ void leave_listed(Take&& take) {
        uint32_t most = 0u;
        take([&](Number x) { const uint32_t order = (uint32_t)(x >> 32); most = order > most ? order : most; });
        if (most != 0u) atomicMax(&s.left_top, most);
        __syncthreads();
        const float top = value_of(s.left_top);
        unsigned long long share = 0;
        take([&](Number x) { const float v = number_value(x); share += (unsigned long long)((v == top ? 1.f : exp_at(v - top, t)) * 0x1p40f); });
        if (share != 0ull) atomicAdd(&s.left_sum, share);
        __syncthreads();
        if (threadIdx.x == 0 && s.left_sum != 0ull) {
            if (top == top) join(others, top, (double)s.left_sum * 0x1p-40, t);
            s.left_top = 0u;
            s.left_sum = 0ull;
        }
    }
    // how many of a work-item's numbers there are over all of them
    __device__ __forceinline__ int total(int mine) {
        uint32_t u = (uint32_t)mine;
        const auto add = [](uint32_t a, uint32_t b) { return a + b; };
        u = lanes_step<0>(u, add); u = lanes_step<1>(u, add); u = lanes_step<2>(u, add);
        u = lanes_step<3>(u, add); u = lanes_step<4>(u, add); u = lanes_step<5>(u, add);
        if (S::kWaves == 1) return (int)u;
        int* counts = s.counts[turn++ & 1];     // (the other one may still be read)
        if (lane == 0) counts[wave] = (int)u;
        __syncthreads();
        int sum = 0;
        #pragma unroll
        for (int w = 0; w < S::kWaves; w++) sum += counts[w];
        return sum;
    }
    // What follows has higher classes than the k numbers listed at `order` and above: it is listed above that, or from it on if `also`.
    __device__ __forceinline__ void raise(uint32_t order, bool also) {
        if (order < kLowestOrder) return;
        const float from = order >= 0xff800000u ? INFINITY : value_of(also ? order : order + 1u);
        bound = fmaxf(bound, from);
    }
    // The list of n > k numbers becomes the k largest of them.
    __device__ __forceinline__ void cut(int n) {
        Number own[S::kOwn];
        #pragma unroll
        for (int i = 0; i < S::kOwn; i++) {
            const int at = threadIdx.x + i * THREADS;
            own[i] = at < n ? s.list[at] : 0ull;
        }
        Number least = 0;       // the largest prefix found that k numbers reach
        for (int bit = 63; bit >= 0; bit--) {
            const Number next = least | 1ull << bit;
            int c = 0;
            #pragma unroll
            for (int i = 0; i < S::kOwn; i++) c += own[i] >= next;
            c = total(c);
            if (c >= t.k) least = next;
            if (c == t.k) break;
        }
        __syncthreads();
        if (threadIdx.x == 0) s.count = 0;
        __syncthreads();
        #pragma unroll
        for (int i = 0; i < S::kOwn; i++) {
            if (own[i] >= least && own[i] != 0ull) push(own[i]);
        }
        leave_listed([&](auto&& visit) {
            #pragma unroll
            for (int i = 0; i < S::kOwn; i++)
                if (own[i] < least && own[i] != 0ull) visit(own[i]);
        });
        raise((uint32_t)(least >> 32), (uint32_t)least == 0u);
        __syncthreads();
    }
    // The end of a row or part that has n numbers listed, at most one for each work-item: what `put` gets are the k largest of them with their places.
    template <class Put> __device__ __forceinline__ void sort(int n, Put&& put) {
        const Number mine = (int)threadIdx.x < n ? s.list[threadIdx.x] : 0ull;
        int place = 0;
        for (int j = 0; j < n; j++) place += s.list[j] > mine;
        if (mine != 0ull && place < t.k) put(place, mine);
        if (n > t.k) leave_listed([&](auto&& visit) { if (mine != 0ull && place >= t.k) visit(mine); });
    }
    // all work-items' others, to the first one
    __device__ __forceinline__ Others all_others() {
        const float m = group_max(others.top, 6);
        Others o{m, group_total(others.top == m ? others.sum : others.sum * (double)exp_at(others.top - m, t), 6)};
        if (S::kWaves > 1) {
            if (lane == 0) s.others[wave] = o;
            __syncthreads();
            if (threadIdx.x == 0)
                for (int w = 1; w < S::kWaves; w++) join(o, s.others[w].top, s.others[w].sum, t);
        }
        if (s.nan) o.sum = __builtin_nan("");
        return o;
    }
    // The same for a whole row: its results.
    template <class T> __device__ __forceinline__ void finish(int n, const T* row, int64_t r) {
        T* values = static_cast<T*>(t.values) + r * t.k;
        int* classes = t.classes + r * t.k;
        const auto put = [&](int place, int cls) { values[place] = row[cls]; classes[place] = cls; };
        sort(n, [&](int place, Number x) { put(place, number_class(x)); });
        if (n < t.k) {      // the first classes that are -inf
            const bool none = (int)threadIdx.x < t.k && Elem<T>::get(row[threadIdx.x]) == -INFINITY;
            const uint64_t lanes = __ballot(none);
            if (lane == 0) s.counts[0][wave] = __popcll(lanes);
            __syncthreads();
            int place = n + __popcll(lanes & ((1ull << lane) - 1ull));
            for (int w = 0; w < wave; w++) place += s.counts[0][w];
            if (none && place < t.k) put(place, threadIdx.x);
        }
        const Others o = all_others();
        if (threadIdx.x == 0) t.rest[r] = o.sum == 0.0 ? -INFINITY : (float)(log(o.sum) + (double)o.top * t.inverse);
    }
};

// Where vector c of the n classes from p on is read: one that would pass the end is that which ends with it, and holds -inf in the place of what the vector before
// it has, too (rows have more than 64 classes, of which a part may hold fewer than a vector).
template <int V> __device__ __forceinline__ int column_of(int c, int n) { return c + V <= n ? c : n - V; }
template <class T> __device__ __forceinline__ u32x4 without_first(u32x4 v, int count) {
    const u32x4 none = Elem<T>::splat(Elem<T>::put(-INFINITY));
    #pragma unroll
    for (int w = 0; w < 4; w++) {
        if constexpr (sizeof(T) == 4) v[w] = w < count ? none[w] : v[w];
        else v[w] = 2 * w + 1 < count ? none[w] : 2 * w < count ? (v[w] & 0xffff0000u) | (none[w] & 0xffffu) : v[w];
    }
    return v;
}

// NV vectors of a row for each work-item, the k-th being vector threadIdx.x + k THREADS of those from c0 on; -inf behind the end
template <class T, int THREADS, int NV> __device__ __forceinline__ void load_vectors(u32x4 (&v)[NV], const T* p, int c0, int n) {
    constexpr int V = Elem<T>::kVec;
    if (c0 + THREADS * NV * V <= n) {
        #pragma unroll
        for (int k = 0; k < NV; k++) v[k] = load16(p + c0 + ((int)threadIdx.x + k * THREADS) * V);
        return;
    }
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = c0 + ((int)threadIdx.x + k * THREADS) * V;
        v[k] = Elem<T>::splat(Elem<T>::put(-INFINITY));
        if (c < n) v[k] = load16(p + column_of<V>(c, n));
    }
    #pragma unroll
    for (int k = 0; k < NV; k++) {
        const int c = c0 + ((int)threadIdx.x + k * THREADS) * V;
        if (c < n && c + V > n) v[k] = without_first<T>(v[k], c + V - n);
    }
}

template <int V> __device__ __forceinline__ float largest(const float (&f)[V]) {
    float m = f[0];
    #pragma unroll
    for (int i = 1; i < V; i++) m = fmaxf(m, f[i]);
    return m;
}

// one of these vectors and where it begins
template <class T> __device__ __forceinline__ int load_one(float (&f)[Elem<T>::kVec], const T* p, int c, int n) {
    constexpr int V = Elem<T>::kVec;
    const int at = column_of<V>(c, n);
    if (c >= n) {
        #pragma unroll
        for (int i = 0; i < V; i++) f[i] = -INFINITY;
    } else Elem<T>::unpack(without_first<T>(load16(p + at), c - at), f);
    return at;
}

// The exact choice of the k first numbers of THREADS * nv vectors, where more of them reach the bound than the list has room for, and where a logit is NaN:
// the k-th largest order bit by bit.  The vectors are read again for each bit: it is rare, and held in registers they would crowd out the rest.
template <class T, int THREADS> __device__ __forceinline__ void choose_exactly(Keeper<THREADS>& keep, const T* p, int c0, int n, int class0, int have, int nv) {
    constexpr int V = Elem<T>::kVec;
    const int k_most = keep.t.k;
    uint32_t kth = 0;
    #pragma unroll 1
    for (int bit = 31; bit >= 0; bit--) {
        const uint32_t next = kth | 1u << bit;
        int count = 0;
        #pragma unroll 1
        for (int k = 0; k < nv; k++) {
            float f[V];
            load_one(f, p, c0 + ((int)threadIdx.x + k * THREADS) * V, n);
            #pragma unroll
            for (int i = 0; i < V; i++) count += order_of(f[i]) >= next;
        }
        if (keep.total(count) >= k_most) kth = next;
    }
    const bool enough = kth >= kLowestOrder;        // else all above -inf are chosen
    if (!enough) kth = kLowestOrder - 1u;
    __syncthreads();
    if (threadIdx.x == 0) keep.s.count = have;
    __syncthreads();
    bool nan = false;
    #pragma unroll 1
    for (int k = 0; k < nv; k++) {
        float f[V];
        const int c = load_one(f, p, c0 + ((int)threadIdx.x + k * THREADS) * V, n);
        #pragma unroll 1
        for (int i = 0; i < V; i++) {
            float v = f[0];
            #pragma unroll
            for (int m = 1; m < V; m++) v = i == m ? f[m] : v;
            const uint32_t order = order_of(v);
            nan |= v != v;
            if (order > kth) keep.push(number_of(v, class0 + c + i));
            else if (!enough || order != kth) keep.leave(v);
        }
    }
    if (nan) keep.s.nan = 1;
    __syncthreads();
    if (enough) {       // equal ones in the order of their classes
        int at = keep.s.count;
        const int end = have + k_most;
        __syncthreads();
        #pragma unroll 1
        for (int k = 0; k < nv; k++) {
            float f[V];
            const int c = load_one(f, p, c0 + ((int)threadIdx.x + k * THREADS) * V, n);
            uint32_t equal = 0;
            #pragma unroll
            for (int i = 0; i < V; i++) equal |= order_of(f[i]) == kth ? 1u << i : 0u;
            const int mine = __popc(equal);
            int before = mine;      // of the lanes up to this one
            #pragma unroll
            for (int s = 1; s < 64; s <<= 1) {
                const int other = __shfl_up(before, s);
                if (keep.lane >= s) before += other;
            }
            int* counts = keep.s.counts[k & 1];
            if (keep.lane == 63) counts[keep.wave] = before;
            __syncthreads();
            int place = at + before - mine;
            #pragma unroll
            for (int w = 0; w < Shared<THREADS>::kWaves; w++) {
                if (w < keep.wave) place += counts[w];
                at += counts[w];
            }
            const float value = value_of(kth);
            for (; equal != 0u; equal &= equal - 1u, place++) {
                if (place < end) keep.s.list[place] = (Number)kth << 32 | (uint32_t)~(class0 + c + __ffs(equal) - 1);
                else keep.leave(value);
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) keep.s.count = end;
        keep.raise(kth, false);
    }
    __syncthreads();
}

// A workgroup per row, or per one of `splits` parts of `part` classes of a row.
template <class T, int THREADS, int NV> __global__ void __launch_bounds__(THREADS, NV > 4 ? 6 : 8) top_rows_kernel(LogitRows a, Top t, int splits, int part, Parts out) {
    constexpr int V = Elem<T>::kVec, kSpan = THREADS * NV * V;
    using S = Shared<THREADS>;
    __shared__ S s;
    for (int64_t b = blockIdx.x; b < a.rows * splits; b += gridDim.x) {
        const int64_t r = splits == 1 ? b : b / splits;
        const int q = (int)(b - r * splits), class0 = q * part, n = a.classes - class0 < part ? (int)a.classes - class0 : part;
        const T* row = row_start<T>(a, r);
        const T* p = row + class0;
        Keeper<THREADS> keep(s, t);
        int have = 0;
        for (int c0 = 0, step = 1; c0 < n; c0 += kSpan, step++) {
            u32x4 v[NV];
            load_vectors<T, THREADS, NV>(v, p, c0, n);
            if (c0 == 0) {
                float m = -INFINITY;
                #pragma unroll
                for (int k = 0; k < NV; k++) {
                    float f[V];
                    Elem<T>::unpack(v[k], f);
                    m = fmaxf(m, largest(f));
                }
                // the largest number of 16 bits that at least k / wavefronts of the lanes' maxima reach
                const int want = (t.k + S::kWaves - 1) / S::kWaves;
                const uint32_t order = order_of(m);
                uint32_t least = 0;
                if (want <= 64) {
                    #pragma unroll
                    for (int bit = 31; bit >= 16; bit--) {
                        const uint32_t next = least | 1u << bit;
                        if (__popcll(__ballot(order >= next)) >= want) least = next;
                    }
                }
                if (S::kWaves > 1) {
                    if (keep.lane == 0) s.bounds[keep.wave] = least;
                    __syncthreads();
                    #pragma unroll
                    for (int w = 0; w < S::kWaves; w++) least = s.bounds[w] < least ? s.bounds[w] : least;
                }
                keep.raise(least, true);
                // what was derived from the vectors is derived again: kept, it would be twice their registers
                #pragma unroll
                for (int k = 0; k < NV; k++) asm("" : "+v"(v[k]));
            }
            Others mine = keep.others;
            #pragma unroll
            for (int k = 0; k < NV; k++) {
                asm volatile("" : "+v"(v[k]), "+v"(mine.sum));      // (one vector after the other: all of them unpacked would not fit)
                float f[V];
                Elem<T>::unpack(v[k], f);
                float m = largest(f);
                if (m >= keep.bound) {
                    const int c = class0 + column_of<V>(c0 + ((int)threadIdx.x + k * THREADS) * V, n);
                    #pragma unroll
                    for (int i = 0; i < V; i++)
                        if (f[i] >= keep.bound) {
                            keep.push(number_of(f[i], c + i));
                            f[i] = -INFINITY;
                        }
                    m = largest(f);
                }
                if (m > mine.top) {
                    mine.sum *= (double)exp_at(mine.top - m, t);
                    mine.top = m;
                }
                const float base = finite(mine.top);
                #pragma unroll
                for (int i = 0; i < V; i++) f[i] = exp_at(f[i] - base, t);
                mine.sum += (double)tree(f);
            }
            if (mine.sum != mine.sum) s.bad = step;
            __syncthreads();
            const int listed = s.count, bad = s.bad;
            __syncthreads();
            if (listed > S::kCap || bad == step) {
                choose_exactly<T, THREADS>(keep, p, c0, n, class0, have, NV);
                have = s.count;
                __syncthreads();
            } else {
                keep.others = mine;
                have = listed;
            }
            if (have > (c0 + kSpan < n ? S::kLong : S::kShort) && have > t.k) {
                keep.cut(have);
                have = t.k;
            }
        }
        if (splits == 1) keep.template finish<T>(have, row, r);
        else {
            Number* numbers = out.numbers + (r * splits + q) * t.k;
            keep.sort(have, [&](int place, Number x) { numbers[place] = x; });
            for (int i = have + threadIdx.x; i < t.k; i += THREADS) numbers[i] = 0ull;
            const Others o = keep.all_others();
            if (threadIdx.x == 0) out.others[r * splits + q] = o;
        }
        __syncthreads();
    }
}

// A workgroup per row joins its parts' lists: of k / splits numbers of each list at least the least is a bound.
template <class T> __global__ void __launch_bounds__(256) top_join_kernel(LogitRows a, Top t, int splits, Parts in) {
    using S = Shared<256>;
    __shared__ S s;
    __shared__ Number leasts[4];
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        Keeper<256> keep(s, t);
        const Number* numbers = in.numbers + r * splits * t.k;
        const int total = splits * t.k, nth = (t.k + splits - 1) / splits - 1;
        Number least = ~0ull;
        __syncthreads();
        for (int q = threadIdx.x; q < splits; q += 256) {
            const Number x = numbers[q * t.k + nth];
            least = x < least ? x : least;
            const Others o = in.others[r * splits + q];
            if (o.sum != o.sum) s.bad = 1;
            else if (o.sum != 0.0) join(keep.others, o.top, o.sum, t);
        }
        for (int step = 32; step > 0; step >>= 1) {
            const Number x = __shfl_xor(least, step);
            least = x < least ? x : least;
        }
        if (keep.lane == 0) leasts[keep.wave] = least;
        __syncthreads();
        #pragma unroll
        for (int w = 0; w < 4; w++) least = leasts[w] < least ? leasts[w] : least;
        if (threadIdx.x == 0) s.nan = s.bad;
        int have = 0;
        for (int i0 = 0; i0 < total; i0 += 1024) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const int at = i0 + i * 256 + threadIdx.x;
                const Number x = at < total ? numbers[at] : 0ull;
                if (x == 0ull) continue;
                if (x >= least) keep.push(x);
                else keep.leave(number_value(x));
            }
            __syncthreads();
            have = s.count;
            __syncthreads();
            if (have > (i0 + 1024 < total ? S::kLong : S::kShort) && have > t.k) {
                keep.cut(have);
                have = t.k;
            }
        }
        keep.template finish<T>(have, row_start<T>(a, r), r);
        __syncthreads();
    }
}

// Rows of at most 64 classes: 2^shift lanes of a wavefront per row, one class each, whose place is the number of classes before it.
template <class T> __global__ void __launch_bounds__(256) top_short_kernel(LogitRows a, Top t, int shift) {
    const int lane = threadIdx.x & ((1 << shift) - 1), lead = (threadIdx.x & 63) - lane, n = (int)a.classes;
    const int64_t per = 256 >> shift;
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += gridDim.x * per) {
        const T* p = row_start<T>(a, r);
        const T raw = p[lane < n ? lane : 0];
        const float v = lane < n ? Elem<T>::get(raw) : -INFINITY;
        const uint32_t mine = lane < n ? order_of(v) : 0u;
        int place = 0;
        for (int j = 0; j < n; j++) {
            const uint32_t other = (uint32_t)__shfl((int)mine, lead + j);
            place += other > mine || (other == mine && j < lane);
        }
        const bool chosen = lane < n && place < t.k;
        if (chosen) {
            static_cast<T*>(t.values)[r * t.k + place] = raw;
            t.classes[r * t.k + place] = lane;
        }
        const float other = chosen ? -INFINITY : v, top = group_max(other, shift);
        const double sum = group_total(other == -INFINITY ? 0.0 : other == top ? 1.0 : (double)exp_at(other - top, t), shift);
        const float nan = group_max(v != v ? 1.f : 0.f, shift);
        if (lane == 0) t.rest[r] = nan != 0.f ? __builtin_nanf("") : sum == 0.0 ? -INFINITY : (float)(log(sum) + (double)top * t.inverse);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
namespace {

// How rows are read: 0 short ones by lanes, 64 by a wavefront each, 256 by workgroups, in `splits` parts.
struct Plan { int threads, vectors, splits; int64_t part; };
Plan plan_of(const LogitRows& a, int64_t k, int vec) {
    if (a.classes <= 64) return {0, 1, 1, a.classes};
    if (k <= 64 && a.classes <= 64 * 4 * vec) return {64, 4, 1, a.classes};
    const int64_t want = (2048 + a.rows - 1) / a.rows, span = 256 * vec;
    int vectors = 8;
    while (vectors > 2 && a.classes < want * span * vectors) vectors /= 2;
    int64_t splits = (a.classes + span * vectors - 1) / (span * vectors);
    if (splits > want) splits = want;
    if (splits > 256) splits = 256;
    if (splits == 1) return {256, vectors, 1, a.classes};
    const int64_t part = ((a.classes + splits - 1) / splits + span - 1) / span * span;
    return {256, vectors, (int)((a.classes + part - 1) / part), part};
}

int64_t part_floats(const LogitRows& a, int64_t k, const Plan& plan) {
    if (plan.splits == 1) return 0;
    return a.rows * plan.splits * (2 * k + (int64_t)(sizeof(Others) / sizeof(float)));
}

}  // namespace

}  // namespace sd

using namespace sd;

extern "C" int64_t sd_top_scratch(const sd_logit_rows* rows, int64_t k) {
    LogitRows a;
    if (check_logits(rows, "top_scratch", &a) != SD_OK) return -1;
    if (k < 1 || k > kMostTop || k > a.classes || a.classes >= kMostClasses) { set_error("top_scratch: k=%lld of %lld classes: 1..%d of fewer than 2^30 are possible", (long long)k, (long long)a.classes, kMostTop); return -1; }
    return (part_floats(a, k, plan_of(a, k, vec_of(rows->dtype))) + 3) / 4 * 4;
}

extern "C" int sd_top_logits(const sd_logit_rows* rows, int64_t k, double temperature, void* values, int* classes, float* rest, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    if (int rc = check_logits(rows, "top_logits", &a)) return rc;
    SD_REQUIRE(k >= 1 && k <= kMostTop && k <= a.classes && a.classes < kMostClasses, "top_logits: k=%lld of %lld classes: 1..%d of fewer than 2^30 are possible", (long long)k, (long long)a.classes, kMostTop);
    SD_REQUIRE(temperature >= 1e-4 && temperature <= 1e4, "top_logits: temperature=%g outside 1e-4..1e4", temperature);
    SD_REQUIRE(values && classes && rest, "top_logits: null argument");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(values) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0 && ((reinterpret_cast<uintptr_t>(classes) | reinterpret_cast<uintptr_t>(rest)) & 3) == 0 &&
               (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "top_logits: results are not aligned to their types, or scratch to 16 bytes");
    const Plan plan = plan_of(a, k, vec_of(rows->dtype));
    SD_REQUIRE(scratch || plan.splits == 1, "top_logits: null scratch");
    const double by = 1.4426950408889634074 / temperature;
    float high = (float)by;
    if ((double)high >= by) high = nextafterf(high, 0.f);
    const Top t{(int)k, 1.0 / temperature, high, (float)(by - (double)high), values, classes, rest};
    const int64_t lists = a.rows * plan.splits;
    Parts parts{};
    if (plan.splits > 1) parts = Parts{reinterpret_cast<Number*>(scratch), reinterpret_cast<Others*>(scratch + 2 * lists * k)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    with_dtype(rows->dtype, [&](auto* p) {
        using T = std::remove_pointer_t<decltype(p)>;
        if (plan.threads == 0) {
            int shift = 0;
            while ((1 << shift) < a.classes) shift++;
            const int64_t per = 256 >> shift, blocks = (a.rows + per - 1) / per;
            hipLaunchKernelGGL(top_short_kernel<T>, dim3(blocks_for(blocks)), dim3(256), 0, s, a, t, shift);
            return;
        }
        const dim3 grid(blocks_for(lists));
        if (plan.threads == 64) hipLaunchKernelGGL((top_rows_kernel<T, 64, 4>), grid, dim3(64), 0, s, a, t, 1, (int)plan.part, parts);
        else if (plan.vectors == 2) hipLaunchKernelGGL((top_rows_kernel<T, 256, 2>), grid, dim3(256), 0, s, a, t, plan.splits, (int)plan.part, parts);
        else if (plan.vectors == 4) hipLaunchKernelGGL((top_rows_kernel<T, 256, 4>), grid, dim3(256), 0, s, a, t, plan.splits, (int)plan.part, parts);
        else hipLaunchKernelGGL((top_rows_kernel<T, 256, 8>), grid, dim3(256), 0, s, a, t, plan.splits, (int)plan.part, parts);
        if (plan.splits > 1) hipLaunchKernelGGL(top_join_kernel<T>, dim3(blocks_for(a.rows)), dim3(256), 0, s, a, t, plan.splits, parts);
    });
    return check_launch("top_rows_kernel");
}
