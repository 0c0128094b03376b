// Logits as they stand when a class is chosen: per row and class v, with n = how often v stands in the row's history,
//   y = z;  where n > 0  y = (z > 0 ? z / repetition : z * repetition) - frequency n - presence;  y += bias[v];  -inf where v is not allowed,
// in 32 bits and in this order, rounded once.  The gradient is 0 where v is not allowed, g / repetition or g * repetition where n > 0, else g.
// Bound by the bytes of the logits in and out.  The counts of a workgroup's columns stand in its LDS, for which it reads the whole history of
// its rows: no scratch, nothing to sort, and any number of repeated classes.
#include <type_traits>
#include "label_rows.h"

namespace sd {

// What a workgroup counts in (16 KiB): 8192 columns by 16 bits, or 4096 by 32 where a history has more places than 16 bits count.  Against 32 bits for 8192 columns:
// 4096 x 65536 bf16 with 1024 places and a bit mask 237 -> 229 us, its gradient 315 -> 282.
constexpr int kCountWords = 4096;
enum { kPlain, kBiased, kGradient };
enum { kNone, kShort, kLong };          // histories: none, of fewer than 2^16 places, of more
enum { kAll = 0, kFlags = SD_ALLOWED_FLAGS, kBits = SD_ALLOWED_BITS };

struct Shape {
    const void *history, *lengths;
    int64_t length, history_outer, history_inner;
    int wide_history, wide_lengths;             // int64 instead of int32
    const float *repetition_rows, *presence_rows, *frequency_rows;
    float repetition, inverse, presence, frequency;
    const float* bias;
    int64_t bias_outer, bias_inner;
    const void* allowed;
    int64_t allowed_outer, allowed_inner;
    const void* grad;                           // backward: what flows into the result, rows one behind the other
    void* out;
    int64_t part;                               // columns of a workgroup, a multiple of 8
    int parts, group;                           // parts of a row, or (with one part) rows of a workgroup
    uint32_t first;                             // of the launch's workgroups (see in_slices)
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

// What classes of the history pay: a positive logit times `inverse`, another one times `repetition`.  A quotient is a product with the reciprocal in fp32, off by up to 1.5 units
// of fp32 instead of half of one: with a division, whose instructions each logit of a vector pays in which one counts, 4096 x 65536 bf16 with 1024 places and a bit mask
// takes 220 us instead of 209.  Both numbers have to be normal ones; a row's repetition that is none makes what it applies to NaN.
constexpr float kLeastRepetition = 0x1p-126f, kMostRepetition = 0x1p126f;
struct Penalties { float repetition, inverse, presence, frequency; };
__device__ __forceinline__ Penalties penalties_of(const Shape& s, int64_t r) {
    Penalties p{s.repetition, s.inverse, s.presence, s.frequency};
    if (s.repetition_rows) {
        const float given = s.repetition_rows[r];
        p.repetition = given >= kLeastRepetition && given <= kMostRepetition ? given : __builtin_nanf("");
        p.inverse = 1.f / p.repetition;
    }
    if (s.presence_rows) p.presence = s.presence_rows[r];
    if (s.frequency_rows) p.frequency = s.frequency_rows[r];
    return p;
}
__device__ __forceinline__ float penalised(float z, uint32_t n, const Penalties& p) {
    return n ? z * (z > 0.f ? p.inverse : p.repetition) - p.frequency * (float)n - p.presence : z;
}
__device__ __forceinline__ float penalised_slope(float g, float z, uint32_t n, const Penalties& p) { return n ? g * (z > 0.f ? p.inverse : p.repetition) : g; }

// the count of column `at`
template <int HISTORY> __device__ __forceinline__ void count_one(uint32_t* counts, uint32_t at) {
    if constexpr (HISTORY == kLong) atomicAdd(&counts[at], 1u);
    else atomicAdd(&counts[at >> 1], 1u << (16 * (at & 1)));
}
template <int HISTORY> __device__ __forceinline__ uint32_t count_of(const uint32_t* counts, int at) {
    if constexpr (HISTORY == kLong) return counts[at];
    else return counts[at >> 1] >> (16 * (at & 1)) & 0xffffu;
}

// 16 bytes of a row's history, 4 places of 32 bits or 2 of 64
struct Places { u32x4 v; };
template <bool WIDE> __device__ __forceinline__ Places load_places(const void* past, int64_t pack) {
    if constexpr (WIDE) {
        struct __attribute__((packed, aligned(8))) Pack { u32x4 v; };
        return Places{static_cast<const Pack*>(past)[pack].v};
    } else return Places{load16(static_cast<const float*>(past) + 4 * pack)};
}
// adds those of the places from `first` on that are below n to the counts of columns [c0, c0 + columns)
template <bool WIDE, int HISTORY> __device__ __forceinline__ void count_places(uint32_t* counts, const Places& p, int64_t first, int64_t n, uint32_t c0, uint32_t columns) {
    #pragma unroll
    for (int i = 0; i < (WIDE ? 2 : 4); i++) {
        const uint32_t at = (WIDE ? p.v[2 * i] : p.v[i]) - c0;
        if (first + i < n && at < columns && (!WIDE || p.v[2 * i + 1] == 0u)) count_one<HISTORY>(counts, at);
    }
}
constexpr int64_t kGroupPlaces = 1 << 12;       // of the histories of rows that a workgroup shapes together

// the first places of a history, which are on their way before it is known how many of them count
constexpr int kAhead = 2;
template <bool WIDE> __device__ __forceinline__ void load_ahead(Places (&p)[kAhead], const void* past, int64_t length) {
    constexpr int kPer = WIDE ? 2 : 4;
    #pragma unroll
    for (int k = 0; k < kAhead; k++) {
        const int64_t pack = (int)threadIdx.x + k * 256;
        if ((pack + 1) * kPer <= length) p[k] = load_places<WIDE>(past, pack);
    }
}
template <bool WIDE, int HISTORY> __device__ __forceinline__ void count_history(uint32_t* counts, const Places (&ahead)[kAhead], const void* past, int64_t length, int64_t n,
                                                                  uint32_t c0, uint32_t columns) {
    constexpr int kPer = WIDE ? 2 : 4;
    constexpr int64_t from = kAhead * 256;
    #pragma unroll
    for (int k = 0; k < kAhead; k++) {
        const int64_t pack = (int)threadIdx.x + k * 256;
        if ((pack + 1) * kPer <= length) count_places<WIDE, HISTORY>(counts, ahead[k], pack * kPer, n, c0, columns);
    }
    const int64_t packs = n / kPer;
    #pragma unroll 2
    for (int64_t pack = from + threadIdx.x; pack < packs; pack += 256) count_places<WIDE, HISTORY>(counts, load_places<WIDE>(past, pack), pack * kPer, n, c0, columns);
    // the places behind the last whole 16 bytes, unless they were among those
    int64_t j = packs * kPer + threadIdx.x;
    if (packs < from && (packs + 1) * kPer <= length) return;
    if (j < n) {
        const uint32_t* word = static_cast<const uint32_t*>(past) + (WIDE ? 2 * j : j);
        const uint32_t at = word[0] - c0;
        if (at < columns && (!WIDE || word[1] == 0u)) count_one<HISTORY>(counts, at);
    }
}

// 4096 x 65536 bf16 with 1024 places and a bit mask 211 us (5.1 TB/s), its gradient 254 (4.2: a cache line for each counted logit).
// A workgroup shapes `part` columns of a row, or `group` whole rows.  A work-item's vectors are on their way together, the first of them while the
// history is counted.
template <class T, int ALLOWED, int HISTORY, int KIND> __global__ void __launch_bounds__(256, HISTORY == kNone ? 8 : 6) shape_kernel(LogitRows a, Shape s) {
    constexpr bool GRAD = KIND == kGradient, BIAS = KIND == kBiased;
    // (16-byte vectors of a work-item that are on their way together; each of them takes two or three with a bias, and four of those the registers of half the wavefronts:
    // 256 x 50001 fp16 with a bias and a history of 4000 places for each row 28.1 us, with two 25.0, but 2000 x 32000 bf16 with 500 places 102 and 105)
    constexpr int kShapeVectors = BIAS ? 2 : 4;
    constexpr int V = Elem<T>::kVec, kAny = ALLOWED == kAll ? kBits : ALLOWED, kPer = HISTORY == kLong ? 1 : 2;     // (kPer: columns of a word of counts)
    __shared__ __align__(16) uint32_t counts[HISTORY ? kCountWords : 4];
    const uint32_t block = s.first + blockIdx.x;
    const int64_t r0 = (int64_t)(block / s.parts) * s.group, c0 = (int64_t)(block % s.parts) * s.part;
    const int rows = (int)(a.rows - r0 < s.group ? a.rows - r0 : s.group);
    const int columns = (int)(a.classes - c0 < s.part ? a.classes - c0 : s.part), width = (columns + 7) & ~7, vecs = columns / V, items = rows * vecs;
    const auto place = [&](int64_t r, int64_t outer, int64_t inner) {
        const uint32_t o = (uint32_t)r / a.inner, i = (uint32_t)r - o * a.inner;
        return o * outer + i * inner;
    };
    const auto allowed_row = [&](int64_t r) { return static_cast<const uint8_t*>(s.allowed) + (ALLOWED == kBits ? 4 : 1) * place(r, s.allowed_outer, s.allowed_inner); };
    const auto split = [&](int item, int per, int& i) { i = rows == 1 ? 0 : item / per; return item - i * per; };
    u32x4 v[kShapeVectors], b[BIAS ? kShapeVectors : 1][V / 4];
    uint32_t bits[kShapeVectors];
    const auto load = [&](int first) {
        #pragma unroll
        for (int k = 0; k < kShapeVectors; k++) {
            const int item = first + k * 256 + (int)threadIdx.x;
            if (item >= items) continue;
            int i;
            const int c = split(item, vecs, i) * V;
            const int64_t r = r0 + i;
            v[k] = load16(GRAD ? static_cast<const T*>(s.grad) + r * a.classes + c0 + c : row_start<T>(a, r) + c0 + c);
            if constexpr (BIAS) {
                const float* bias = s.bias + place(r, s.bias_outer, s.bias_inner) + c0 + c;
                #pragma unroll
                for (int m = 0; m < V / 4; m++) b[k][m] = load16(bias + 4 * m);
            }
            if (ALLOWED != kAll) bits[k] = allowed_bits<V, kAny>(allowed_row(r), (int)c0 + c);
        }
    };
    // (loads arrive in their order: the history's first)
    Places ahead[kAhead];
    const void* past = nullptr;
    if (HISTORY != kNone && rows == 1) {
        past = static_cast<const uint8_t*>(s.history) + place(r0, s.history_outer, s.history_inner) * (s.wide_history ? 8 : 4);
        if (s.wide_history) load_ahead<true>(ahead, past, s.length);
        else load_ahead<false>(ahead, past, s.length);
    }
    load(0);
    if (HISTORY) {
        for (int i = threadIdx.x; i < rows * width / (4 * kPer); i += 256) reinterpret_cast<u32x4*>(counts)[i] = u32x4{0u, 0u, 0u, 0u};
        __syncthreads();
        const auto counted = [&](int64_t r) {       // places of a row's history that count
            if (!s.lengths) return s.length;
            const int64_t given = s.wide_lengths ? static_cast<const int64_t*>(s.lengths)[r] : static_cast<const int*>(s.lengths)[r];
            return given < 0 ? 0 : given < s.length ? given : s.length;
        };
        if (rows == 1) {
            const int64_t n = counted(r0);
            if (s.wide_history) count_history<true, HISTORY>(counts, ahead, past, s.length, n, (uint32_t)c0, (uint32_t)columns);
            else count_history<false, HISTORY>(counts, ahead, past, s.length, n, (uint32_t)c0, (uint32_t)columns);
        } else {        // all rows' places one behind the other: in a turn for each row there would be little to do
            const auto count_rows = [&](auto wide) {
                constexpr bool WIDE = decltype(wide)::value;
                constexpr uint32_t kPlaces = WIDE ? 2 : 4;
                const uint32_t length = (uint32_t)s.length, packs = (length + kPlaces - 1) / kPlaces;
                #pragma unroll 2
                for (uint32_t j = threadIdx.x; j < rows * packs; j += 256) {
                    const uint32_t i = j / packs, pack = j - i * packs;
                    const int64_t r = r0 + i, n = counted(r);
                    const uint32_t* words = static_cast<const uint32_t*>(s.history) + place(r, s.history_outer, s.history_inner) * (WIDE ? 2 : 1);
                    Places p;
                    if ((pack + 1) * kPlaces <= length) p = load_places<WIDE>(words, pack);
                    else {
                        #pragma unroll
                        for (int m = 0; m < 4; m++) p.v[m] = (pack * 4 + m) < length * (WIDE ? 2 : 1) ? words[pack * 4 + m] : ~0u;
                    }
                    count_places<WIDE, HISTORY>(counts + i * width / kPer, p, pack * kPlaces, n, 0, (uint32_t)columns);
                }
            };
            if (s.wide_history) count_rows(std::true_type());
            else count_rows(std::false_type());
        }
        __syncthreads();
    }
    Penalties paid{};
    if (HISTORY && rows == 1) paid = penalties_of(s, r0);
    for (int first = 0; first < items; first += kShapeVectors * 256) {
        if (first > 0) load(first);
        uint32_t seen = 0;          // bit k: a class of vector k is in the history
        u32x4 z[GRAD && HISTORY ? kShapeVectors : 1];
        if (HISTORY) {
            #pragma unroll
            for (int k = 0; k < kShapeVectors; k++) {
                const int item = first + k * 256 + (int)threadIdx.x;
                if (item >= items) continue;
                int i;
                const int c = split(item, vecs, i) * V;
                uint32_t any = 0;
                #pragma unroll
                for (int m = 0; m < V / kPer; m++) any |= counts[(i * width + c) / kPer + m];
                if (any) {
                    seen |= 1u << k;
                    if constexpr (GRAD && HISTORY) z[k] = load16(row_start<T>(a, r0 + i) + c0 + c);
                }
            }
        }
        #pragma unroll
        for (int k = 0; k < kShapeVectors; k++) {
            const int item = first + k * 256 + (int)threadIdx.x;
            if (item >= items) continue;
            int i;
            const int c = split(item, vecs, i) * V;
            const int64_t r = r0 + i;
            float f[V];
            Elem<T>::unpack(v[k], f);
            if (HISTORY && seen >> k & 1) {
                if (rows > 1) paid = penalties_of(s, r);
                float zf[V];
                if constexpr (GRAD && HISTORY) Elem<T>::unpack(z[k], zf);
                #pragma unroll
                for (int m = 0; m < V; m++) {
                    const uint32_t n = count_of<HISTORY>(counts, i * width + c + m);
                    f[m] = GRAD ? penalised_slope(f[m], zf[m], n, paid) : penalised(f[m], n, paid);
                }
            }
            if constexpr (BIAS) {
                #pragma unroll
                for (int m = 0; m < V; m++) f[m] += __uint_as_float(b[k][m / 4][m % 4]);
            }
            if (ALLOWED != kAll) {
                #pragma unroll
                for (int m = 0; m < V; m++) f[m] = bits[k] >> m & 1 ? f[m] : GRAD ? 0.f : -INFINITY;
            }
            T* to = static_cast<T*>(s.out) + r * a.classes + c0 + c;
            store16(to, Elem<T>::pack(f));
        }
    }
    // the values behind the last whole vector of each row
    const int rest = columns - vecs * V;
    for (int item = threadIdx.x; item < rows * rest; item += 256) {
        int i;
        const int c = vecs * V + split(item, rest, i);
        const int64_t r = r0 + i;
        const T* z = row_start<T>(a, r) + c0 + c;
        float f = Elem<T>::get(GRAD ? static_cast<const T*>(s.grad)[r * a.classes + c0 + c] : *z);
        if (HISTORY) {
            const uint32_t n = count_of<HISTORY>(counts, i * width + c);
            if (rows > 1) paid = penalties_of(s, r);
            if (!GRAD) f = penalised(f, n, paid);
            else if (n) f = penalised_slope(f, Elem<T>::get(*z), n, paid);
        }
        if (BIAS) f += s.bias[place(r, s.bias_outer, s.bias_inner) + c0 + c];
        if (ALLOWED != kAll && !allowed_one<kAny>(allowed_row(r), (int)c0 + c)) f = GRAD ? 0.f : -INFINITY;
        static_cast<T*>(s.out)[r * a.classes + c0 + c] = Elem<T>::put(f);
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
    SD_REQUIRE(c->repetition_rows || (c->repetition >= kLeastRepetition && c->repetition <= kMostRepetition), "%s: repetition=%g outside 2^-126..2^126", who, c->repetition);
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
        s.repetition = (float)c->repetition; s.inverse = (float)(1.0 / c->repetition); s.presence = (float)c->presence; s.frequency = (float)c->frequency;
    }
    s.bias = c->bias; s.bias_outer = c->bias_outer; s.bias_inner = c->bias_inner;
    s.allowed = c->allowed; s.allowed_outer = c->allowed_outer; s.allowed_inner = c->allowed_inner;
    s.grad = grad; s.out = out;
    const int64_t width = (a.classes + 7) / 8 * 8, most = s.length >= 1 << 16 ? kCountWords : 2 * kCountWords;
    if (width <= most) {
        // Short rows are shaped together, as many as leave 1024 workgroups: 100000 x 10 fp32 with 4 places each 6.9 us, in a workgroup each 136.  But a long history is
        // read faster where a workgroup has one row: 8192 x 2000 bf16 with 2000 places 43 us, in groups of 2 47, of 4 52.5.
        const int64_t places = s.length > 0 ? kGroupPlaces / s.length : most, fit = most / width, want = (a.rows + 1023) / 1024;
        const int64_t group = want < fit ? want : fit;
        s.group = (int)(group < places ? group : places > 1 ? places : 1);
        s.parts = 1;
        s.part = width;
    } else {
        const int64_t want = (a.classes * a.rows / 1024 + 2047) / 2048 * 2048;
        s.group = 1;
        s.part = want < 2048 ? 2048 : want < most ? want : most;
        s.parts = (int)((a.classes + s.part - 1) / s.part);
    }
    const int64_t blocks = (a.rows + s.group - 1) / s.group * s.parts;
    SD_REQUIRE(blocks < (1ll << 31), "%s: %lld rows of %lld classes are too many for one call", who, (long long)a.rows, (long long)a.classes);
    with_dtype(in->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto launch = [&](auto allowed, auto with_history) {
            in_slices(blocks, [&](int64_t from, unsigned n) {
                s.first = (uint32_t)from;
                if (grad) hipLaunchKernelGGL((shape_kernel<T, allowed.value, with_history.value, kGradient>), dim3(n), dim3(256), 0, stream, a, s);
                else if (s.bias) hipLaunchKernelGGL((shape_kernel<T, allowed.value, with_history.value, kBiased>), dim3(n), dim3(256), 0, stream, a, s);
                else hipLaunchKernelGGL((shape_kernel<T, allowed.value, with_history.value, kPlain>), dim3(n), dim3(256), 0, stream, a, s);
            });
        };
        const auto with = [&](auto allowed) {
            if (!history) launch(allowed, std::integral_constant<int, kNone>());
            else if (s.length < 1 << 16) launch(allowed, std::integral_constant<int, kShort>());
            else launch(allowed, std::integral_constant<int, kLong>());
        };
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
