// The k largest logits of each row in order (of equal ones the lower class first), their classes, and the log-sum of the others at a temperature:
//   rest = log sum over the classes that are not among the k of exp(z[v] / T)   (-inf where there are none).
// Values are compared by whole numbers in their order (order_of): NaN above all, -0 as 0.  With the class behind it, upside down, every logit
// has a number of its own, so the k largest are the same in every call.
//
// A row is read once, in vectors of 16 bytes, whose largest logits decide: the k largest logits of a row lie in the k vectors that are first by their largest
// logit and place, since any other logit has those k before it.  Vectors that reach a bound which k of them are known to reach are put on a list in LDS; of the
// others the exponentials are summed.  The first bound comes from the work-items' own maxima over their first vectors: the least of the wavefronts'
// (k / wavefronts)-th largest ones, reached by about 1.3 k vectors; a list that gets long is cut to k vectors, the last of which is the new bound (what is
// cut is read again and summed).  At the end the listed vectors' logits are chosen from in the same way and sorted by counting.  Few rows are read in
// parts, whose results a second kernel joins.  Logits of -inf are never listed: where there are not k others the first classes that are -inf follow,
// which are among the row's first k.
// Bound by the instructions of a logit, of which the exponential is half (it takes the time of four), and by the bytes of the logits.
#include <type_traits>
#include "label_rows.h"

namespace sd {

constexpr int kMostTop = SD_MOST_TOP;
constexpr int64_t kMostClasses = 1ll << 30;
constexpr int kTopVectors = 4;          // 16-byte vectors of a row for each work-item at a time

__device__ __forceinline__ uint32_t order_of(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0xffffffffu : b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t order) {
    return __uint_as_float(order & 0x80000000u ? order ^ 0x80000000u : ~order);
}
constexpr uint32_t kLowestOrder = 0x00800000u;      // of -FLT_MAX; that of -inf is one less
constexpr uint32_t kInfiniteOrder = 0xff800000u;
constexpr uint32_t kZeroOrder = 0x80000000u, kNanOrder = 0xffffffffu;
// of several values (two zeros, all NaN): which of them it was stands in the row
__device__ __forceinline__ bool shared_order(uint32_t order) { return order == kZeroOrder || order == kNanOrder; }

typedef unsigned long long Number;      // order << 32 | ~class; 0: none
__device__ __forceinline__ Number number_of(uint32_t order, int cls) { return (Number)order << 32 | (uint32_t)~cls; }
__device__ __forceinline__ uint32_t number_order(Number x) { return (uint32_t)(x >> 32); }
__device__ __forceinline__ int number_class(Number x) { return (int)~(uint32_t)x; }

struct Top {
    int k;
    float by;               // log2(e) / temperature
    double inverse;         // 1 / temperature
    void* values;
    int* classes;
    float* rest;
};

// Sums of exp(v / T) are kept as multiples of exp(top / T), top being the largest v in them: differences to it, by log2(e) / T rounded to fp32, are all that an exponential
// sees, and top / T, in 64 bits, comes to the logarithm of the sum at the end.  Where many values are taken relative to one number m, m log2(e) / T is the sum of two fp32
// numbers, of which a fused multiply-add takes the first; beyond 2^28, where the second would be more than 2^4, differences are formed in 64 bits.
constexpr float kNear = 0x1p28f;
struct Others { float top; double sum; };       // (top: -inf where there are none, never +inf)
__device__ __forceinline__ double in_powers(float top, float of, const Top& t) { return top == of ? 1.0 : (double)__builtin_amdgcn_exp2f((float)(((double)top - (double)of) * (double)t.by)); }
__device__ __forceinline__ void join(Others& o, float top, double sum, const Top& t) {
    if (sum == 0.0) return;
    if (top > o.top) {
        if (o.sum != 0.0) o.sum *= in_powers(o.top, top, t);
        o.top = top;
    }
    o.sum += sum * in_powers(top, o.top, t);
}

template <int V> __device__ __forceinline__ float largest(const float (&f)[V]) {
    float m = f[0];
    #pragma unroll
    for (int i = 1; i < V; i++) m = fmaxf(m, f[i]);
    return m;
}

// The parts of a row: the k largest numbers in order (0 where there are fewer) and the others of each.  The sum is NaN in a part that has a NaN.
struct Parts { Number* numbers; Others* others; };

template <int THREADS> struct Shared {
    static constexpr int kWaves = THREADS / 64;
    static constexpr int kRoom = 512;               // numbers of a wavefront's part of the list
    static constexpr int kMost = THREADS < 320 ? THREADS : 320;    // numbers that a cut may leave: at most one for each work-item
    Number list[kWaves][kRoom];
    Number first[THREADS];                          // those of a list that is no longer than that, one behind the other
    Others others[kWaves];
    uint64_t words[2][kWaves];                      // (or as many of 32 bits)
    Number kth;                                     // the k-th number of a row or part
    int again;
};

// The list of a row or part, kept by all work-items of a workgroup together: they all call every member but `leave`; `push` is a wavefront's.  A wavefront has a
// part of the list to itself, in the order in which it found the numbers, so that nothing waits for it and every call sees the same list.
template <int THREADS> struct Keeper {
    using S = Shared<THREADS>;
    S& s;
    const Top& t;
    float bound = -FLT_MAX;         // what reaches it is listed
    Others others{-INFINITY, 0.0};  // this work-item's
    int mine = 0;                   // numbers of this wavefront
    int all = 0, longest = 0;       // of all and of the longest part, as of the last `settle`
    bool nan = false, infinite = false;     // a NaN is there; +inf is among the others
    int lane, wave, turn = 0;

    __device__ __forceinline__ Keeper(S& shared, const Top& top) : s(shared), t(top), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) {}

    __device__ __forceinline__ void leave(float v) {
        if (v == INFINITY) infinite = true;
        else if (v > -INFINITY) join(others, v, 1.0, t);
    }
    // logits that are all among the others
    template <int V> __device__ __forceinline__ void leave_all(float (&f)[V]) {
        float m = largest(f);
        if (m == INFINITY) {
            infinite = true;
            #pragma unroll
            for (int i = 0; i < V; i++) f[i] = f[i] == INFINITY ? -INFINITY : f[i];
            m = largest(f);
        }
        if (m == -INFINITY) return;
        const float power = m * t.by;
        if (fabsf(power) <= kNear) {
            const float low = fmaf(m, t.by, -power);
            #pragma unroll
            for (int i = 0; i < V; i++) f[i] = __builtin_amdgcn_exp2f(fmaf(f[i], t.by, -power) - low);
        } else {
            #pragma unroll
            for (int i = 0; i < V; i++) f[i] = __builtin_amdgcn_exp2f((float)(((double)f[i] - (double)m) * (double)t.by));
        }
        join(others, m, (double)tree(f), t);
    }
    static __device__ __forceinline__ int before(uint64_t lanes) {     // of them, below this one
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0u));
    }
    // the numbers of those lanes of the wavefront that have one here
    __device__ __forceinline__ void push(uint64_t lanes, bool has, Number x) {
        if (has) s.list[wave][mine + before(lanes)] = x;
        mine += __popcll(lanes);
    }
    // a word of each wavefront, of which `op` makes one
    template <class Word, class Op> __device__ __forceinline__ Word share(Word word, Op&& op) {
        if (S::kWaves == 1) { __syncthreads(); return word; }
        Word* words = reinterpret_cast<Word*>(s.words[turn++ & 1]);      // (the other ones may still be read)
        if (lane == 0) words[wave] = word;
        __syncthreads();
        Word r = words[0];
        #pragma unroll
        for (int w = 1; w < S::kWaves; w++) r = op(r, words[w]);
        return r;
    }
    template <class Op> static __device__ __forceinline__ uint32_t lanes_make(uint32_t u, Op&& op) {
        u = lanes_step<0>(u, op); u = lanes_step<1>(u, op); u = lanes_step<2>(u, op);
        u = lanes_step<3>(u, op); u = lanes_step<4>(u, op);
        return __builtin_amdgcn_readfirstlane(lanes_step<5>(u, op));
    }
    template <class Op> __device__ __forceinline__ uint32_t share_lanes(uint32_t u, Op&& op) { return share(lanes_make(u, op), op); }
    static __device__ __forceinline__ uint32_t least_of(uint32_t a, uint32_t b) { return a < b ? a : b; }
    // the lists' lengths
    __device__ __forceinline__ void settle() {
        const uint32_t r = share((uint32_t)mine << 16 | (uint32_t)mine, [](uint32_t a, uint32_t b) {
            return (a >> 16 > b >> 16 ? a >> 16 : b >> 16) << 16 | ((a & 0xffffu) + (b & 0xffffu));
        });
        all = (int)(r & 0xffffu);
        longest = (int)(r >> 16);
    }
    // What follows has higher classes than the k numbers or more listed at `order` and above: it is listed above that, or from it on if `also`.
    __device__ __forceinline__ void raise(uint32_t order, bool also) {
        if (order < kLowestOrder) return;
        const float from = order >= kInfiniteOrder ? INFINITY : value_of(also ? order : order + 1u);
        bound = fmaxf(bound, from);
    }
    // The list of more than `most` numbers becomes at least k and at most `most` of the largest of them; `out` gets the others.  OWN: the wavefront's alone.
    template <bool OWN, class Out> __device__ __forceinline__ void cut(int most, Out&& out) {
        constexpr int kOwn = 4;         // numbers that a lane has in registers meanwhile
        const auto shared = [&](auto word, auto&& op) { return OWN ? word : share(word, op); };
        const Number* own = s.list[wave];
        Number held[kOwn];
        uint32_t every = ~0u, some = 0u;
        const auto look = [&](Number x) {
            every &= number_order(x);
            some |= number_order(x);
        };
        #pragma unroll
        for (int h = 0; h < kOwn; h++) {
            held[h] = lane + 64 * h < mine ? own[lane + 64 * h] : 0ull;
            if (lane + 64 * h < mine) look(held[h]);
        }
        #pragma unroll 1
        for (int i = lane + 64 * kOwn; i < mine; i += 64) look(own[i]);
        const auto both = [](uint32_t a, uint32_t b) { return a & b; };
        const auto either = [](uint32_t a, uint32_t b) { return a | b; };
        every = shared(lanes_make(every, both), both);
        some = shared(lanes_make(some, either), either);
        // The bits in which the orders differ are all that is looked for, two at a time: three counts, of at most kRoom numbers in each wavefront, and one barrier.
        const uint32_t differ = every ^ some;
        const int high = differ == 0u ? 0 : 32 - __clz(differ);
        Number least = (Number)(high == 32 ? 0u : every >> high << high) << 32;     // the largest prefix found that k numbers reach
        static_assert(S::kWaves * S::kRoom < 1 << 16, "a count of all wavefronts' numbers has 16 bits");
        #pragma unroll 1
        for (int bit = 30 + high + (high & 1); bit >= 0; bit -= 2) {     // (of an odd number of bits the first one is one that all share, or none has)
            const Number low = least | 1ull << bit, next = least | 2ull << bit, top = next | low;
            uint64_t c = 0;
            const auto count = [&](Number x) {
                c += (uint64_t)__popcll(__ballot(x >= low)) | (uint64_t)__popcll(__ballot(x >= next)) << 16 | (uint64_t)__popcll(__ballot(x >= top)) << 32;
            };
            #pragma unroll
            for (int h = 0; h < kOwn; h++) count(held[h]);
            #pragma unroll 1
            for (int i = 64 * kOwn; i < mine; i += 64) count(lane + i < mine ? own[lane + i] : 0ull);
            c = shared(c, [](uint64_t a, uint64_t b) { return a + b; });
            const int low_and_next = __builtin_amdgcn_readfirstlane((int)(uint32_t)c), reach[3] = {low_and_next & 0xffff, low_and_next >> 16 & 0xffff, __builtin_amdgcn_readfirstlane((int)(c >> 32))};
            int reached;
            if (reach[2] >= t.k) { least = top; reached = reach[2]; }
            else if (reach[1] >= t.k) { least = next; reached = reach[1]; }
            else if (reach[0] >= t.k) { least = low; reached = reach[0]; }
            else continue;
            if (reached <= most) break;
        }
        const int had = mine;
        mine = 0;
        #pragma unroll 1
        for (int i = 0; i < had; i += 64) {     // (what stays is stored no later than where it stood)
            const Number x = lane + i < had ? own[lane + i] : 0ull;
            const bool stays = x >= least && x != 0ull;
            push(__ballot(stays), stays, x);
            if (!stays && x != 0ull) out(x);
        }
        raise(number_order(least), (uint32_t)least == 0u);
        if (!OWN) settle();
    }
    // the list, at most THREADS long, in `first`
    __device__ __forceinline__ void gather() {
        int at = lane;
        if (S::kWaves > 1) {
            uint32_t* words = reinterpret_cast<uint32_t*>(s.words[turn++ & 1]);
            if (lane == 0) words[wave] = (uint32_t)mine;
            __syncthreads();
            for (int w = 0; w < wave; w++) at += (int)words[w];
        }
        for (int i = lane; i < mine; i += 64, at += 64) s.first[at] = s.list[wave][i];
        __syncthreads();
    }
    // The end of a row or part: what `put` gets are the k largest numbers with their places, of a list of logits that is at most THREADS long.
    template <class Put> __device__ __forceinline__ void sort(Put&& put) {
        gather();
        if (64 * wave >= all) return;
        const Number own = (int)threadIdx.x < all ? s.first[threadIdx.x] : 0ull;
        int place = 0;
        #pragma unroll 4
        for (int j = 0; j < all; j++) place += s.first[j] > own;
        if (own != 0ull) {
            if (place < t.k) put(place, own);
            else leave(value_of(number_order(own)));
            if (place == t.k - 1) s.kth = own;
        }
    }
    // all work-items' others, to the first one; NaN where the row or part has a NaN
    __device__ __forceinline__ Others all_others() {
        const float m = group_max(others.top, 6);
        Others o{m, group_total(others.sum == 0.0 ? 0.0 : others.sum * in_powers(others.top, m, t), 6)};
        if (lane == 0) s.others[wave] = o;
        const uint32_t odd = share((__ballot(nan) ? 1u : 0u) | (__ballot(infinite) ? 2u : 0u), [](uint32_t x, uint32_t y) { return x | y; });
        if (S::kWaves > 1) {
            constexpr int kShift = S::kWaves == 2 ? 1 : S::kWaves == 4 ? 2 : 3;
            const Others theirs = s.others[lane & (S::kWaves - 1)];
            o.top = group_max(theirs.top, kShift);
            o.sum = group_total(theirs.sum == 0.0 ? 0.0 : theirs.sum * in_powers(theirs.top, o.top, t), kShift);
        }
        if (odd & 2) o = Others{FLT_MAX, INFINITY};
        if (odd & 1) o.sum = __builtin_nan("");
        return o;
    }
    // The same for a whole row: what it chooses.
    template <class T> __device__ __forceinline__ void finish(const T* row, int64_t r) {
        T* values = static_cast<T*>(t.values) + r * t.k;
        int* classes = t.classes + r * t.k;
        const auto put = [&](int place, T v, int cls) { values[place] = v; classes[place] = cls; };
        sort([&](int place, Number x) {
            const uint32_t order = number_order(x);
            const int cls = number_class(x);
            put(place, shared_order(order) ? row[cls] : Elem<T>::put(value_of(order)), cls);
        });
        if (all < t.k) {      // the first classes that are -inf
            const bool none = (int)threadIdx.x < t.k && Elem<T>::get(row[threadIdx.x]) == -INFINITY;
            const uint64_t lanes = __ballot(none);
            int place = all + before(lanes);
            if (S::kWaves > 1) {
                uint32_t* words = reinterpret_cast<uint32_t*>(s.words[turn++ & 1]);
                if (lane == 0) words[wave] = (uint32_t)__popcll(lanes);
                __syncthreads();
                for (int w = 0; w < wave; w++) place += (int)words[w];
            }
            if (none && place < t.k) put(place, Elem<T>::put(-INFINITY), threadIdx.x);
        }
    }
    __device__ __forceinline__ void store_rest(const Others& o, int64_t r) const {
        t.rest[r] = o.sum == 0.0 ? -INFINITY : (float)(log(o.sum) + (double)o.top * t.inverse);
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
// the vector that was read at column `at` (a multiple of V but for the last)
template <class T> __device__ __forceinline__ void read_again(float (&f)[Elem<T>::kVec], const T* p, int at) {
    constexpr int V = Elem<T>::kVec;
    Elem<T>::unpack(without_first<T>(load16(p + at), (V - (at & (V - 1))) & (V - 1)), f);
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

// Shares of the others below this, relative to the bound, are formed again: of terms below 2^-126 nothing is left, 2^30 of them are 2^-36 of it.
constexpr double kLeastShare = 0x1p-60;

// A workgroup per row, or per one of `splits` parts of `part` classes of a row.  What is not listed lies below the wavefront's bound, to which the exponentials are relative;
// where they come out too small, or the bound too large, for fp32, the others are gone through again at the end.
// 4096 x 131072 bf16, k = 64, 217 us (4.9 TB/s; reading alone 163 to 185); 1 x 131072, k = 50, in 16 parts 12 us and the join 7, of which each waits for its own steps.
template <class T, int THREADS> __global__ void __launch_bounds__(THREADS, 8) top_rows_kernel(LogitRows a, Top t, int splits, int part, Parts out, int64_t first) {
    constexpr int V = Elem<T>::kVec, NV = kTopVectors, kSpan = THREADS * NV * V;
    using S = Shared<THREADS>;
    static_assert(64 * NV + kMostTop <= S::kRoom, "a wavefront's part of the list has room for all vectors behind the k that a cut of its own leaves");
    static_assert(64 * V <= S::kRoom, "and for the logits of a vector for each work-item");
    __shared__ S s;
    const int64_t b = first + blockIdx.x;
    const int64_t r = splits == 1 ? b : b / splits;
    const int q = (int)(b - r * splits), class0 = q * part, n = a.classes - class0 < part ? (int)a.classes - class0 : part;
    const T* row = row_start<T>(a, r);
    const T* p = row + class0;
    Keeper<THREADS> keep(s, t);
    // a vector that is cut: its logits are among the others
    const auto leave_vector = [&](Number x) {
        float f[V];
        read_again(f, p, number_class(x));
        keep.leave_all(f);
    };
    double sum = 0.0;                       // of 2^(v by - power)
    float base = -FLT_MAX, power = 0.f;     // (nothing but -inf is summed as long as this is the bound)
    bool again = false;
    const int most = t.k + t.k / 4 < S::kMost ? t.k + t.k / 4 : S::kMost;      // vectors that a cut leaves
    const auto rebase = [&]() {
        if (keep.bound == base) return;
        const float before = power;
        base = keep.bound;
        power = base * t.by;
        if (!(fabsf(power) <= kNear)) { power = 0.f; again = true; }
        if (sum != 0.0) sum *= (double)__builtin_amdgcn_exp2f((float)((double)before - (double)power));
    };
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
            keep.raise(keep.share(least, Keeper<THREADS>::least_of), true);
            rebase();
            // what was derived from the vectors is derived again: kept, it would be twice their registers
            #pragma unroll
            for (int k = 0; k < NV; k++) asm("" : "+v"(v[k]));
        }
        #pragma unroll
        for (int k = 0; k < NV; k += 2) {
            asm volatile("" : "+v"(v[k]), "+v"(v[k + 1]), "+v"(sum));      // (two vectors after two: all of them unpacked would not fit)
            float f[2][V], m[2];
            bool listed[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                Elem<T>::unpack(v[k + h], f[h]);
                m[h] = largest(f[h]);
                listed[h] = m[h] >= keep.bound;
            }
            const auto column = [&](int h) { return column_of<V>(c0 + ((int)threadIdx.x + (k + h) * THREADS) * V, n); };
            const int had = keep.mine;
            const uint64_t lanes[2] = {__ballot(listed[0]), __ballot(listed[1])};
            if (lanes[0] | lanes[1]) {
                #pragma unroll
                for (int h = 0; h < 2; h++)
                    if (lanes[h]) keep.push(lanes[h], listed[h], number_of(order_of(m[h]), column(h)));
            }
            float part[2];
            #pragma unroll
            for (int h = 0; h < 2; h++) {
                #pragma unroll
                for (int i = 0; i < V; i++) f[h][i] = __builtin_amdgcn_exp2f(fmaf(f[h][i], t.by, -power));
                part[h] = tree(f[h]);
            }
            if (__ballot(part[0] + part[1] != part[0] + part[1])) {     // a NaN is above all: the vector's number is to say so, and has to be on the list
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    const bool nan = part[h] != part[h], more = nan && !listed[h];
                    const Number x = number_of(0xffffffffu, column(h));
                    if (nan && listed[h]) s.list[keep.wave][had + (h ? __popcll(lanes[0]) : 0) + keep.before(lanes[h])] = x;
                    keep.push(__ballot(more), more, x);
                    keep.nan |= nan;
                    part[h] = nan ? 0.f : part[h];
                }
            }
            sum += (double)((listed[0] ? 0.f : part[0]) + (listed[1] ? 0.f : part[1]));
        }
        // The wavefronts go on by themselves; they meet, and cut the list together, behind the first, second, fourth, .. and last of their steps.
        const bool last = c0 + kSpan >= n;
        if (last || (step & (step - 1)) == 0) {
            keep.settle();
            if (keep.all > most) { keep.template cut<false>(most, leave_vector); rebase(); }
        }
        if (!last && keep.mine > S::kRoom - 64 * NV) { keep.template cut<true>(S::kRoom - 64 * NV, leave_vector); rebase(); }
    }
    // The logits of the listed vectors.  Each of these has one that reaches the least of their largest ones.
    keep.gather();
    const Number x = (int)threadIdx.x < keep.all ? s.first[threadIdx.x] : 0ull;
    const uint32_t least = keep.share_lanes(x != 0ull ? number_order(x) : ~0u, Keeper<THREADS>::least_of);
    keep.bound = -FLT_MAX;
    if (keep.all >= t.k) keep.raise(least, true);
    keep.mine = 0;
    if (__ballot(x != 0ull)) {
        float f[V];
        const int at = x != 0ull ? number_class(x) : 0;
        if (x != 0ull) read_again(f, p, at);
        #pragma unroll
        for (int i = 0; i < V; i++) {
            const bool listed = x != 0ull && !(f[i] < keep.bound);      // (a NaN, too)
            const uint64_t lanes = __ballot(listed);
            if (lanes) keep.push(lanes, listed, number_of(order_of(f[i]), class0 + at + i));
            f[i] = listed ? -INFINITY : f[i];
        }
        if (x != 0ull) keep.leave_all(f);
    }
    keep.settle();
    if (keep.all > THREADS) keep.template cut<false>(S::kMost, [&](Number y) { keep.leave(value_of(number_order(y))); });
    if (splits == 1) keep.template finish<T>(row, r);
    else {
        Number* numbers = out.numbers + (r * splits + q) * t.k;
        keep.sort([&](int place, Number y) { numbers[place] = y; });
        for (int i = keep.all + threadIdx.x; i < t.k; i += THREADS) numbers[i] = 0ull;
    }
    // (where fewer than k logits are above -inf there are no others)
    if (!again && sum != 0.0) join(keep.others, base, sum * (double)__builtin_amdgcn_exp2f(-fmaf(base, t.by, -power)), t);
    Others o = keep.all_others();
    const uint32_t bases = keep.share(order_of(again ? INFINITY : base), [](uint32_t x, uint32_t y) { return x > y ? x : y; });
    if (threadIdx.x == 0) {
        const float highest = value_of(bases);
        s.again = keep.all >= t.k && o.sum == o.sum && highest > -FLT_MAX && (highest == INFINITY || !(o.sum * in_powers(o.top, highest, t) >= kLeastShare));
    }
    __syncthreads();
    if (s.again) {
        const Number kth = s.kth;
        keep.others = Others{-INFINITY, 0.0};
        #pragma unroll 1
        for (int c = (int)threadIdx.x * V; c < n; c += THREADS * V) {
            float f[V];
            const int at = column_of<V>(c, n);
            Elem<T>::unpack(without_first<T>(load16(p + at), c - at), f);
            #pragma unroll
            for (int i = 0; i < V; i++)
                if (number_of(order_of(f[i]), class0 + at + i) < kth) keep.leave(f[i]);
        }
        o = keep.all_others();
    }
    if (threadIdx.x == 0) {
        if (splits == 1) keep.store_rest(o, r);
        else out.others[r * splits + q] = o;
    }
}

// A workgroup per row joins its parts' lists: of k / splits numbers of each list at least the least is a bound.
constexpr int kJoin = 512;
template <class T> __global__ void __launch_bounds__(kJoin) top_join_kernel(LogitRows a, Top t, int splits, Parts in, int64_t first) {
    using S = Shared<kJoin>;
    constexpr int kTurn = (S::kRoom - kMostTop) / 64;      // numbers of a work-item before the lists' lengths are looked at
    __shared__ S s;
    const int64_t r = first + blockIdx.x;
    Keeper<kJoin> keep(s, t);
    const Number* numbers = in.numbers + r * splits * t.k;
    const int total = splits * t.k, nth = (t.k + splits - 1) / splits - 1, most = t.k + t.k / 4;
    uint32_t least = ~0u;       // (by their orders: lists with nothing there have 0)
    for (int q = threadIdx.x; q < splits; q += kJoin) {
        least = Keeper<kJoin>::least_of(least, number_order(numbers[q * t.k + nth]));
        const Others o = in.others[r * splits + q];
        if (o.sum != o.sum) keep.nan = true;
        else if (o.sum == INFINITY) keep.infinite = true;
        else join(keep.others, o.top, o.sum, t);
    }
    keep.raise(keep.share_lanes(least, Keeper<kJoin>::least_of), true);
    for (int i0 = 0; i0 < total; i0 += kTurn * kJoin) {
        const uint32_t from = order_of(keep.bound);     // (a NaN is above every bound)
        #pragma unroll
        for (int i = 0; i < kTurn; i++) {
            const int at = i0 + i * kJoin + threadIdx.x;
            const Number x = at < total ? numbers[at] : 0ull;
            const bool listed = x != 0ull && number_order(x) >= from;
            const uint64_t lanes = __ballot(listed);
            if (lanes) keep.push(lanes, listed, x);
            if (x != 0ull && !listed) keep.leave(value_of(number_order(x)));
        }
        keep.settle();
        if (keep.all > kJoin || keep.longest > kMostTop) {
            const auto leave = [&](Number y) { keep.leave(value_of(number_order(y))); };
            if (keep.all > most) keep.template cut<false>(most, leave);
            if (i0 + kTurn * kJoin < total && keep.mine > kMostTop) keep.template cut<true>(kMostTop, leave);
        }
    }
    keep.template finish<T>(row_start<T>(a, r), r);
    const Others o = keep.all_others();
    if (threadIdx.x == 0) keep.store_rest(o, r);
}

__device__ __forceinline__ uint32_t group_most(uint32_t u, int shift) {
    const auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    if (shift > 0) u = lanes_step<0>(u, larger);
    if (shift > 1) u = lanes_step<1>(u, larger);
    if (shift > 2) u = lanes_step<2>(u, larger);
    if (shift > 3) u = lanes_step<3>(u, larger);
    if (shift > 4) u = lanes_step<4>(u, larger);
    if (shift > 5) u = lanes_step<5>(u, larger);
    return u;
}

// Rows of at most 64 classes: 2^shift lanes of a wavefront per row, one class each.  Its place is the number of classes before it, or the turn in which it is the first of
// the largest ones that are left, where the turns, each of which takes as long as four comparisons with a class, are few: 65536 x 50 bf16, k = 5, 58 and 35 us.
template <class T> __global__ void __launch_bounds__(256) top_short_kernel(LogitRows a, Top t, int shift) {
    const int lane = threadIdx.x & ((1 << shift) - 1), lead = (threadIdx.x & 63) - lane, n = (int)a.classes;
    const uint64_t whole = shift == 6 ? ~0ull : (1ull << (1 << shift)) - 1ull;
    const int64_t per = 256 >> shift;
    for (int64_t r = (int64_t)blockIdx.x * per + (threadIdx.x >> shift); r < a.rows; r += gridDim.x * per) {
        const T* p = row_start<T>(a, r);
        const T raw = p[lane < n ? lane : 0];
        const float v = lane < n ? Elem<T>::get(raw) : -INFINITY;
        const uint32_t mine = lane < n ? order_of(v) : 0u;
        int place = t.k;
        if (4 * t.k <= n) {
            uint32_t left = mine;
            for (int turn = 0; turn < t.k; turn++) {
                const uint32_t most = group_most(left, shift);
                if (lane == __ffsll((long long)(__ballot(left == most) >> lead & whole)) - 1) { place = turn; left = 0u; }
            }
        } else {
            place = 0;
            for (int j = 0; j < n; j++) {
                const uint32_t other = (uint32_t)__shfl((int)mine, lead + j);
                place += other > mine || (other == mine && j < lane);
            }
        }
        const bool chosen = lane < n && place < t.k;
        if (chosen) {
            static_cast<T*>(t.values)[r * t.k + place] = raw;
            t.classes[r * t.k + place] = lane;
        }
        // (exponentials and the logarithm in 32 bits: there are 63 numbers at most, 1 among them, and in 64 they took longer than all the rest)
        const float other = chosen ? -INFINITY : v, top = group_max(other, shift);
        const float sum = (float)group_total(other == -INFINITY ? 0.0 : other == top ? 1.0 : top == INFINITY ? 0.0 : (double)__builtin_amdgcn_exp2f((other - top) * t.by), shift);
        const float nan = group_max(v != v ? 1.f : 0.f, shift);
        if (lane == 0)
            t.rest[r] = nan != 0.f ? __builtin_nanf("") : sum == 0.f ? -INFINITY : top == INFINITY ? INFINITY : (float)((double)logf(sum) + (double)top * t.inverse);
    }
}

// ---- host ------------------------------------------------------------------------------------------------------------------------
namespace {

// How rows are read: by `threads` work-items each (0: short ones, by lanes; 30000 x 10 fp32 8.6 us, by a wavefront each 35), in `splits` parts.
// A list is cut to 1.25 k, which is no more than the work-items, so that a prefix of the numbers does for it (k = 256 with 256 of them 4096 x 131072 bf16 660 us, with
// 512 316).  Above that as many as the card runs at once, since what is left over costs as much time as all the others: 300 x 50001 fp16, k = 200, in 7 parts 70 us, in
// 5 53 (whole 38, see below); 20000 x 9001 fp32, k = 20, by 256 work-items 232 us, by 128 168 (but 4096 x 131072 bf16, which is twice the card by 256, 206 and 218).
struct Plan { int threads, splits; int64_t part; };
Plan plan_of(const LogitRows& a, int64_t k, int vec) {
    if (a.classes <= 64) return {0, 1, a.classes};
    const int64_t most = k + k / 4, card = 1 << 19;
    int threads = 64;
    while (threads < most) threads *= 2;
    if (a.classes <= (int64_t)threads * kTopVectors * vec) return {threads, 1, a.classes};
    // A workgroup that is done with a row in two turns needs no parts and no join, nor in four where every compute unit has one: bf16, k = 5 / 50 / 200, 64 x 12000 24 / 15.5 / 19 us,
    // in parts 24 / 19.5 / 28.5; 64 x 30000 28 / 21 / 23 and 24 / 20 / 31; 300 x 50001 43 / 35 / 39 and 39 / 37 / 52; 512 x 65536 47 / 36 / 40 and 49 / 42 / 59; where it would take
    // four turns and there are fewer rows 16 x 50001 32 / 28 / 31 and 24 / 25 / 33; 200 x 50001 35 / 29 / 32 and 32 / 32 / 46.
    if (a.rows * 512 <= card && a.classes <= 512 * kTopVectors * vec * (a.rows >= 256 ? 4 : 2)) return {512, 1, a.classes};
    if (threads < 128) threads = 128;
    while (threads < 256 && a.rows * threads * 2 <= card) threads *= 2;
    const int64_t fit = card / (a.rows * threads), want = fit > 1 ? fit : 1, span = threads * vec;
    int64_t splits = (a.classes + span * kTopVectors - 1) / (span * kTopVectors);
    if (splits > want) splits = want;
    if (splits > 256) splits = 256;
    if (splits == 1) return {threads, 1, a.classes};
    const int64_t part = ((a.classes + splits - 1) / splits + span - 1) / span * span;
    return {threads, (int)((a.classes + part - 1) / part), part};
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
    if (k < 1 || k > kMostTop || k > a.classes || a.classes >= kMostClasses) {
        set_error("top_scratch: k=%lld of %lld classes: 1..%d of fewer than 2^30 are possible", (long long)k, (long long)a.classes, kMostTop);
        return -1;
    }
    return (part_floats(a, k, plan_of(a, k, vec_of(rows->dtype))) + 3) / 4 * 4;
}

extern "C" int sd_top_logits(const sd_logit_rows* rows, int64_t k, double temperature, void* values, int* classes, float* rest, float* scratch, sd_stream_t stream) {
    sd::CallGuard call_guard;
    LogitRows a;
    if (int rc = check_logits(rows, "top_logits", &a)) return rc;
    SD_REQUIRE(k >= 1 && k <= kMostTop && k <= a.classes && a.classes < kMostClasses, "top_logits: k=%lld of %lld classes: 1..%d of fewer than 2^30 are possible",
               (long long)k, (long long)a.classes, kMostTop);
    SD_REQUIRE(temperature >= 1e-4 && temperature <= 1e4, "top_logits: temperature=%g outside 1e-4..1e4", temperature);
    SD_REQUIRE(values && classes && rest, "top_logits: null argument");
    SD_REQUIRE((reinterpret_cast<uintptr_t>(values) & (rows->dtype == SD_FLOAT32 ? 3 : 1)) == 0 && ((reinterpret_cast<uintptr_t>(classes) | reinterpret_cast<uintptr_t>(rest)) & 3) == 0 &&
               (reinterpret_cast<uintptr_t>(scratch) & 15) == 0, "top_logits: results are not aligned to their types, or scratch to 16 bytes");
    const Plan plan = plan_of(a, k, vec_of(rows->dtype));
    SD_REQUIRE(scratch || plan.splits == 1, "top_logits: null scratch");
    const Top t{(int)k, (float)(1.4426950408889634074 / temperature), 1.0 / temperature, values, classes, rest};
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
        const auto launch = [&](auto threads) {
            in_slices(lists, [&](int64_t from, unsigned blocks) {
                hipLaunchKernelGGL((top_rows_kernel<T, threads.value>), dim3(blocks), dim3(threads.value), 0, s, a, t, plan.splits, (int)plan.part, parts, from);
            });
        };
        switch (plan.threads) {
            case 64: launch(std::integral_constant<int, 64>()); break;
            case 128: launch(std::integral_constant<int, 128>()); break;
            case 256: launch(std::integral_constant<int, 256>()); break;
            default: launch(std::integral_constant<int, 512>());
        }
        if (plan.splits > 1) {
            in_slices(a.rows, [&](int64_t from, unsigned blocks) { hipLaunchKernelGGL(top_join_kernel<T>, dim3(blocks), dim3(kJoin), 0, s, a, t, plan.splits, parts, from); });
        }
    });
    return check_launch(plan.threads == 0 ? "top_short_kernel" : plan.splits == 1 ? "top_rows_kernel" : "top_rows_kernel or top_join_kernel");
}
