// The next token of every row from its logits and a random number (tvk_sample).
//
// With s = x / T a token weighs exp(s - max s); what the filters leave is a prefix
// of the tokens in the order of their logits, equal ones in that of their indexes:
// those above a border value and the first few that equal it. So nothing is
// sorted. A histogram over the logits' distance from the largest, of counts or of
// weights, says which bin the border of a filter falls into; the bin's own values,
// a few, are compared with each other in LDS, or spread over a histogram of their
// own until they are few or all equal. The token is then the first in the
// vocabulary's order at which the sum of kept weights passes the random number's
// share of their total: sums over stretches of the row say in which it lies.
//
// Weights are integers: 2^44 exp(s - max s) from float64, rounded. Their sums are
// exact in 64 bits whatever the order (2^44 times at most 2^19 tokens), so that the
// atomics of a histogram and the split of a row over threads and workgroups leave
// no trace in the result, and the borders fall where the formulas in 64 bits put
// them: float32 weights would put one in 10^4 draws from a flat distribution
// elsewhere.
//
// The row stays in the registers of 1024 threads, 32 K values in 16 bits or 16 K in
// 32, and is read again, stretch by stretch, for every pass past that. Most of a small call is latency, and much of
// that the code's own: a line of 64 bytes that no cache holds takes as long as a
// load. So passes are loops over a thread's words, not unrolled, helpers are called,
// not inlined, and nothing is read in a chain that can be read at once. Few rows are
// cut among workgroups, in four launches: the largest, the histogram, what lies in
// and above the border's bin, the token.
//
// Measured: 1 x 50001 of bfloat16 with top_k and top_p 22 us (launches of 3.7, 4.9, 7.5
// and 6.7), 64 x 128000 with top_p at temperatures from 0.5 to 1.5 61 us (4.9, 16, 24
// and 17), 200 x 32003 of float32 with every filter 47 us (rows that are read again for
// every pass); in a replayed graph, whose start is 5 of them, the largest logit alone
// 18 us of 1 x 50001 and 21 of 64 x 128000, without filters 23 and 30. The weights of a
// row, some 210 cycles for 64 of them, and their atomics in LDS bound the larger; a
// series without the table of fractions was slower (18.9 us for 16.5 in the histogram's
// launch), and neither comparisons with a bin's ends in place of its number nor sums
// over runs of one place before the atomics changed the third.
#include "norm_rows.h"

#include <cfloat>

using namespace tvk;

namespace {

typedef unsigned long long u64;

constexpr int SA_THREADS = 1024, SA_WAVES = SA_THREADS / 64;
constexpr int SA_BINS = 2 * SA_THREADS;
constexpr int SA_CHUNKS = 4;       // of 16 bytes, that a thread holds
constexpr int SA_LIST = 256;       // values of a bin that are compared with each other
constexpr int SA_FEW = 512;        // tokens that are
constexpr int SA_SOME = 128;       // more of them than this are first spread over bins
constexpr int SA_KEPT = 8192;      // tokens that are weighed from a list
constexpr int SA_PIECES = 32;      // of a row, at most
constexpr int64_t SA_MOST_COLS = 1 << 19;

// Where a row that is cut among workgroups goes on.
enum { SA_FIRST, SA_ALL, SA_TOKENS, SA_SUMS, SA_WHOLE };
struct RowState {
    int mode, bin;
    u64 above, need;
};

struct SampleArgs {
    const void* x;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* random;
    int64_t* token;
    float* logprob;
    int64_t rows, stride, row0;   // row0: of a launch
    int cols;
    // of rows cut into pieces
    int pieces, piece;     // chunks of a piece
    RowState* state;       // [rows]
    u64* bins;             // [rows][pieces][SA_BINS]
    u64* places;           // [rows][SA_BINS]
    float* tops;           // [rows][pieces]
    unsigned* listed;      // [rows][pieces]
    float* list_v;         // [rows][pieces][SA_FEW]
    int* list_at;
};

constexpr int SA_STEPS = 64;   // of a power of two in a table

// 2^(44 + j / 64), from the exponential's series.
struct StepTable {
    double v[SA_STEPS];
    constexpr StepTable() : v{} {
        for (int j = 0; j < SA_STEPS; ++j) {
            double term = 0x1p44, sum = 0x1p44;
            for (int n = 1; n < 24; ++n) sum += term *= 0.693147180559945309 * j / SA_STEPS / n;
            v[j] = sum;
        }
    }
};
__constant__ StepTable kSteps = StepTable();

// A row's weights: exp((x - top) / T) = 2^(n / 64) 2^r, n whole and |r| <= 1 / 128.
struct Heat {
    float top;             // the largest logit
    double c;              // 64 log2(e) / T
    const double* table;   // 2^(44 + j / 64), in LDS

    // 2^44 times the weight, within 2^-44 of it; next to nothing below 2^-60. Beside an infinite logit the others weigh nothing.
    __device__ __forceinline__ double large_weight(float x) const {
        if (top == INFINITY) return x == top ? 0x1p44 : 0.0;
        const double y = fmax(((double)x - (double)top) * c, -60.0 * SA_STEPS);
        const double shifted = y + 0x1.8p52;   // n in its low bits
        const int n = (int)(uint32_t)__builtin_bit_cast(u64, shifted);
        const double f = y - (shifted - 0x1.8p52), ln = 0.0108304246962491454;   // ln 2 / 64; f ln at most 0.0054 in magnitude
        // its exponential: (f ln)^5 / 120 is left, 4e-14
        const double p = fma(fma(fma(fma(f, ln * ln * ln * ln / 24, ln * ln * ln / 6), f, ln * ln / 2), f, ln), f, 1.0);
        return __builtin_bit_cast(double, __builtin_bit_cast(u64, table[n & (SA_STEPS - 1)] * p) + ((u64)(uint32_t)(n >> 6) << 52));
    }
    __device__ static u64 whole(double w) {   // rounded: the low bits of a sum whose last place is 1
        return __builtin_bit_cast(u64, w + 0x1p52) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ u64 whole_weight(float x) const { return whole(large_weight(x)); }
};

// Chunks [first, end) of 16 bytes of a row, thread t those at first + t + 1024 j, C of them in registers.
template <int DT, int C = SA_CHUNKS>
struct RowIn {
    typedef typename elem<DT>::T T;
    typedef uint32_t W __attribute__((ext_vector_type(4 * C)));
    static constexpr int VEC = 16 / (int)sizeof(T), HELD = C * SA_THREADS;   // chunks that are held
    static constexpr int N = 2, STEP = DT == TVK_F32 ? 2 : 1;                // values handled together, their words
    const T* row;
    int cols, first, end, at, words;   // at: the first of the held; words of a thread
    const int* places = nullptr;       // of a list
    W w;

    __device__ __forceinline__ RowIn(const SampleArgs& p, int64_t r, int first, int last)
        : row(static_cast<const T*>(p.x) + r * p.stride), cols(p.cols), first(first), end(min(last, (p.cols + VEC - 1) / VEC)) {
        load(first);
    }
    __device__ __forceinline__ void load(int from) {
        at = from;
        words = min(C, (end - from + SA_THREADS - 1) / SA_THREADS) * 4;
        const int whole = min(end, cols / VEC), mine = from + (int)threadIdx.x;   // past `whole` lies at most a piece of a chunk
        const T* p = row + (int64_t)mine * VEC;
        Words<16> c[C];
#pragma unroll
        for (int j = 0; j < C; ++j) {
            c[j] = {};
            if (mine + j * SA_THREADS < whole) c[j] = load_words<16, sizeof(T)>(p + j * SA_THREADS * VEC);
        }
#pragma unroll
        for (int j = 0; j < 4 * C; ++j) w[j] = c[j / 4].w[j % 4];
        if (from + words / 4 * SA_THREADS <= whole) return;
        constexpr uint32_t LOWEST = DT == TVK_F32 ? 0xff800000u : DT == TVK_F16 ? 0xfc00fc00u : 0xff80ff80u;   // -inf
#pragma unroll 1
        for (int k = words - 4; k < words; ++k) {   // of a thread's last chunk
            uint32_t v = w[k];
            const int i = mine + k / 4 * SA_THREADS;
            if (i >= whole) {
                v = LOWEST;
                const int e = i * VEC + k % 4 * (VEC / 4);   // the word's first value
                if (i < end && e < cols) {
                    if constexpr (DT == TVK_F32) v = __builtin_bit_cast(uint32_t, row[e]);
                    else {
                        v = (LOWEST & 0xffff0000u) | __builtin_bit_cast(uint16_t, row[e]);
                        if (e + 1 < cols) v = (v & 0xffffu) | (uint32_t)__builtin_bit_cast(uint16_t, row[e + 1]) << 16;
                    }
                }
            }
            w[k] = v;
        }
    }
    // From here on the n tokens of a list instead (at most as many as are held), whose places are in LDS.
    __device__ __forceinline__ void take(const float* v, const int* v_places, int n) {
        static_assert(SA_KEPT <= 4 * C / STEP * N * SA_THREADS, "a list is held");
        first = at = 0;
        end = 1;
        words = (n + N * SA_THREADS - 1) / (N * SA_THREADS) * STEP;
        places = v_places;
        auto value = [&](int i) { return elem<DT>::from_f32(i < n ? v[i] : -INFINITY); };
#pragma unroll 1
        for (int k = 0; k < words; k += STEP) {
            const int i = threadIdx.x + k / STEP * N * SA_THREADS;
            if constexpr (DT == TVK_F32) {
                w[k] = __builtin_bit_cast(uint32_t, value(i));
                w[k + 1] = __builtin_bit_cast(uint32_t, value(i + SA_THREADS));
            } else {
                w[k] = __builtin_bit_cast(uint16_t, value(i)) | (uint32_t)__builtin_bit_cast(uint16_t, value(i + SA_THREADS)) << 16;
            }
        }
    }
    // f(indexes, two values) over the chunks; NaN as -inf. A chunk's last call is where (the second index + 1) % VEC is 0.
    template <class F>
    __device__ __forceinline__ void each(F&& f) {
#pragma unroll 1
        for (int from = first; from < end; from += HELD) {
            if (at != from) load(from);
#pragma unroll 1
            for (int k = 0; k < words; k += STEP) {
                const Words<8> two{{w[k], w[k + STEP - 1]}};
                const float v[N] = {fmaxf(word_at<DT>(two, 0), -INFINITY), fmaxf(word_at<DT>(two, 1), -INFINITY)};
                const int e = (from + (int)threadIdx.x + k / 4 * SA_THREADS) * VEC + k % 4 * (VEC / 4);
                int i[N] = {e, e + 1};
                if (places) {
                    i[0] = places[threadIdx.x + k / STEP * N * SA_THREADS];
                    i[1] = places[threadIdx.x + (k / STEP * N + 1) * SA_THREADS];
                }
                f(i, v);
            }
        }
    }
    __device__ float value(int i) const {
        const float v = elem<DT>::to_f32(row[i]);
        return v == v ? v : -INFINITY;
    }
};

struct AddOp { template <class V> __device__ static V of(V a, V b) { return a + b; } };
struct LeastOp { template <class V> __device__ static V of(V a, V b) { return a < b ? a : b; } };
struct MostOp { template <class V> __device__ static V of(V a, V b) { return a > b ? a : b; } };

// A value from another lane, by CTRL; lanes without a source, or outside ROWS (bits of groups of 16), get `none`.
template <int CTRL, int ROWS = 0xf, class V>
__device__ __forceinline__ V from_lane(V v, V none) {
    if constexpr (sizeof(V) == 8) {
        const u64 u = __builtin_bit_cast(u64, v), n = __builtin_bit_cast(u64, none);
        const uint32_t lo = __builtin_amdgcn_update_dpp((int)n, (int)u, CTRL, ROWS, 0xf, false);
        const uint32_t hi = __builtin_amdgcn_update_dpp((int)(n >> 32), (int)(u >> 32), CTRL, ROWS, 0xf, false);
        return __builtin_bit_cast(V, (u64)hi << 32 | lo);
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none), __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
    }
}

// Over 16 lanes, in each of them.
template <class Op, class V>
__device__ __forceinline__ V lanes16(V v) {
    v = Op::of(v, from_lane<0xB1>(v, v));    // lane ^ 1
    v = Op::of(v, from_lane<0x4E>(v, v));    // lane ^ 2
    v = Op::of(v, from_lane<0x141>(v, v));   // mirrored in 8
    return Op::of(v, from_lane<0x140>(v, v));   // mirrored in 16
}

// What is the same in every lane, in a scalar register: vector registers are what the kernels run out of.
template <class V>
__device__ __forceinline__ V of_all(V v) {
    if constexpr (sizeof(V) == 8) {
        const u64 u = __builtin_bit_cast(u64, v);
        return __builtin_bit_cast(V, (u64)(uint32_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 |
                                         (uint32_t)__builtin_amdgcn_readfirstlane((int)u));
    } else {
        return __builtin_bit_cast(V, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
    }
}

// Over the workgroup, the same bits in every thread: waves first, then the waves' results.
template <class Op, class V>
__device__ __forceinline__ V all_threads(V v) {
    __shared__ V part[SA_WAVES * 4];
    v = lanes16<Op>(v);
    __syncthreads();
    if (threadIdx.x % 16 == 0) part[threadIdx.x / 16] = v;
    __syncthreads();
    v = part[threadIdx.x % 16];
#pragma unroll
    for (int i = 1; i < 4; ++i) v = Op::of(v, part[threadIdx.x % 16 + 16 * i]);
    return lanes16<Op>(v);
}

// Sum of the lanes up to this one.
template <class V>
__device__ __forceinline__ V lanes_up_to(V v) {
    v += from_lane<0x111>(v, (V)0);         // from the lane before, and 2, 4, 8 before, in groups of 16
    v += from_lane<0x112>(v, (V)0);
    v += from_lane<0x114>(v, (V)0);
    v += from_lane<0x118>(v, (V)0);
    v += from_lane<0x142, 0xa>(v, (V)0);    // the first group's last to the second, the third's to the fourth
    v += from_lane<0x143, 0xc>(v, (V)0);    // the first half's last to the second half
    return v;
}

// Sums by bin: of weights, or counts in the same words.
union Bins {
    u64 w[SA_BINS];
    unsigned n[2 * SA_BINS];
};

struct Shared {
    Bins all, part;
    float list[SA_KEPT];
    int list_at[SA_KEPT], kept_at[SA_KEPT];
    double table[SA_STEPS];
    u64 list_w[SA_FEW], before[SA_FEW];
    unsigned rank[SA_FEW];
    u64 sums[SA_WAVES];
    unsigned counts[SA_PIECES];
    // what one thread finds for all
    u64 found_w, found_own;
    unsigned found_n, found_count, listed;
    int found, last;
    float border;
};

// For each of the n <= SA_FEW entries of s.list (list_at, list_w) the weight, s.before, and the number, s.rank, of those that
// `front(v, at, other v, other at)` puts in front of it. Waves share the comparisons out: 64 entries each with a part of all.
template <class F>
__device__ __forceinline__ void compare_all(int n, Shared& s, F&& front) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
    if (threadIdx.x < SA_FEW) s.before[threadIdx.x] = 0, s.rank[threadIdx.x] = 0;
    __syncthreads();
    const int groups = (n + 63) / 64, parts = SA_WAVES / groups;   // (no groups: nothing to do)
    const int each = (n + parts - 1) / parts, i = wave % groups * 64 + lane, first = wave / groups * each;
    if (i < n && wave / groups < parts) {
        const float v = s.list[i];
        const int at = s.list_at[i];
        u64 before = 0;
        unsigned rank = 0;
#pragma unroll 4
        for (int k = first; k < min(first + each, n); ++k) {
            const bool f = front(v, at, s.list[k], s.list_at[k]);
            rank += f;
            before += f ? s.list_w[k] : 0;
        }
        if (rank) {
            atomicAdd(&s.rank[i], rank);
            atomicAdd(&s.before[i], before);
        }
    }
    __syncthreads();
}
__device__ __forceinline__ bool in_front(float v, int at, float o, int o_at) { return o > v || (o == v && o_at < at); }

// Values between lo and hi in bins of equal width, the largest first. Rounding moves no value past another, so what is in a
// bin is settled by the same expression wherever it is asked; and float64 tells any two values apart, so that lo and hi share
// no bin where the scale is that of their distance. float32 is enough, and faster, where only the first range is asked for.
template <class F>
struct Range {
    float lo, hi;
    F scale;
    __device__ __forceinline__ bool has(float x) const { return x >= lo && x <= hi; }
    __device__ __forceinline__ int bin(float x) const {
        const F b = ((F)hi - (F)x) * scale;
        return (int)(b < (F)(SA_BINS - 1) ? b : (F)(SA_BINS - 1));   // infinities and NaN: the last
    }
    // the bin within a bin
    __device__ __forceinline__ int part(float x, int bin) const {
        const double b = ((double)((F)hi - (F)x) * (double)scale - bin) * SA_BINS;
        return b > 0.0 ? (int)fmin(b, (double)(SA_BINS - 1)) : 0;
    }
};

// Weights from 1 to 2^-40, the rest in the last bin.
template <class F>
__device__ inline Range<F> first_range(float top, float heat) {
    return {top == INFINITY ? top : -FLT_MAX, top, (F)(SA_BINS / (28.0 * heat))};
}

// The values that a filter keeps: above t, and the first `ties` of the `equal` that equal it.
struct Border {
    float t;
    unsigned ties, equal;
};

// A row's filters.
struct Filters {
    float heat, top_p, least, random;
    int top_k;
    bool by_k, by_p;
    __device__ Filters(const SampleArgs& p, int64_t row) {
        heat = p.temperature ? p.temperature[row] : 1.0f;
        top_p = p.top_p ? p.top_p[row] : 1.0f;
        least = p.min_p ? p.min_p[row] : 0.0f;
        top_k = p.top_k ? p.top_k[row] : 0;
        random = p.random[row];
        by_k = top_k > 0 && top_k < p.cols;
        by_p = top_p < 1.0f;
    }
    __device__ bool first_only(float top) const { return top == -INFINITY || !(heat > 0.0f) || top_k == 1 || top_p <= 0.0f; }
    __device__ Heat weights(float top, const Shared& s) const { return {top, SA_STEPS * 1.4426950408889634 / heat, s.table}; }
    // the weight that reaches top_p's share
    __device__ u64 share(u64 total) const { return min(total, max((u64)1, (u64)ceil((double)top_p * (double)total))); }
    // what the sum of weights up to the token is to pass
    __device__ u64 goal(u64 total) const {
        const double share = random > 0.0f ? (double)random * (double)total : 0.0;
        return min(share < (double)total ? (u64)share : total - 1, total - 1);
    }
    // 2^44 v's weight, zero where min_p drops it
    __device__ __forceinline__ u64 weigh(const Heat& h, float v) const {
        const double w = h.large_weight(v);
        return least > 0.0f && w < fmin((double)least, 1.0) * 0x1p44 ? (u64)0 : Heat::whole(w);
    }
};

__device__ inline void make_table(Shared& s) {
    if (threadIdx.x < SA_STEPS) s.table[threadIdx.x] = kSteps.v[threadIdx.x];
    __syncthreads();
}

__device__ __forceinline__ void clear(Bins& b) {
    __syncthreads();
    b.w[threadIdx.x] = b.w[threadIdx.x + SA_THREADS] = 0;
    __syncthreads();
}

__device__ __forceinline__ u64 sum_of(const Bins& b, Shared& s) {
    return all_threads<AddOp>(b.w[threadIdx.x] + b.w[threadIdx.x + SA_THREADS]);
}

template <int DT, int C, class F>
__device__ __forceinline__ void fill_bins(RowIn<DT, C>& x, const Heat& h, const Range<F>& r, bool counts, Bins& b) {
    constexpr int N = RowIn<DT>::N;
    clear(b);
    if (counts)
        x.each([&](const int (&)[N], const float (&v)[N]) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (r.has(v[k])) atomicAdd(&b.n[r.bin(v[k])], 1u);
        });
    else
        x.each([&](const int (&)[N], const float (&v)[N]) {
            u64 w[N];
            int bin[N];
#pragma unroll
            for (int k = 0; k < N; ++k) {
                w[k] = h.whole_weight(v[k]);
                bin[k] = r.bin(v[k]);
            }
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (r.has(v[k]) && w[k]) atomicAdd(&b.w[bin[k]], w[k]);
        });
    __syncthreads();
}

// The first bin with which the count, or the weight, reaches `need`: s.found (-1: none), s.found_w before it, s.found_own in it.
__device__ __forceinline__ void find_bin(bool part, bool counts, u64 need, Shared& s) {
    const Bins& b = part ? s.part : s.all;
    const int i = 2 * threadIdx.x, wave = threadIdx.x / 64;
    const u64 v0 = counts ? b.n[i] : b.w[i], v1 = counts ? b.n[i + 1] : b.w[i + 1];
    u64 v = lanes_up_to(v0 + v1);
    __syncthreads();
    if (threadIdx.x == 0) s.found = -1;
    if (threadIdx.x % 64 == 63) s.sums[wave] = v;
    __syncthreads();
    const int other = threadIdx.x % SA_WAVES;
    v += lanes16<AddOp>(other < wave ? s.sums[other] : (u64)0) - (v0 + v1);
    const bool first = v < need && v + v0 >= need, second = v + v0 < need && v + v0 + v1 >= need;
    if (first || second) {
        s.found = first ? i : i + 1;
        s.found_w = first ? v : v + v0;
        s.found_own = first ? v0 : v1;
    }
    __syncthreads();
}

// The border among the values of one bin: those before it count, or weigh, `above`.
struct InBin {
    bool done;
    Border b;
    float lo, hi;
};

template <int DT, int C>
__device__ __forceinline__ InBin border_in_bin(RowIn<DT, C>& x, const Heat& h, const Range<double>& r, int bin, bool counts, u64 need, u64 above,
                                               Shared& s) {
    constexpr int N = RowIn<DT>::N;
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    float lo = INFINITY, hi = -INFINITY;
    x.each([&](const int (&)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) {
            if (!r.has(v[k]) || r.bin(v[k]) != bin) continue;
            lo = fminf(lo, v[k]);
            hi = fmaxf(hi, v[k]);
            const unsigned i = atomicAdd(&s.listed, 1u);
            if (i < SA_LIST) s.list[i] = v[k];
        }
    });
    lo = all_threads<LeastOp>(lo);
    hi = all_threads<MostOp>(hi);
    const unsigned count = s.listed;
    if (lo == hi) {
        const u64 left = need - above, w = h.whole_weight(lo);
        return {true, {lo, counts ? (unsigned)left : (unsigned)((left + w - 1) / w), count}, lo, hi};
    }
    if (count > SA_LIST) return {false, {-INFINITY, 0, 0}, lo, hi};
    const bool there = threadIdx.x < count;
    const float own = there ? s.list[threadIdx.x] : 0.0f;
    const u64 each = there ? counts ? 1 : h.whole_weight(own) : 0;
    if (there) s.list_w[threadIdx.x] = each, s.list_at[threadIdx.x] = (int)threadIdx.x;
    compare_all((int)count, s, [](float v, int, float o, int) { return o > v; });
    const u64 before = there ? above + s.before[threadIdx.x] : 0;
    const unsigned larger = there ? s.rank[threadIdx.x] : 0;
    compare_all((int)count, s, [](float v, int, float o, int) { return o >= v; });
    const unsigned equal = there ? s.rank[threadIdx.x] - larger : 0;
    if (there && before < need && need <= before + equal * each) {   // all that equal the border write the same
        s.border = own;
        s.found_n = (unsigned)((need - before + each - 1) / each);
        s.found_count = equal;
    }
    __syncthreads();
    return {true, {s.border, s.found_n, s.found_count}, lo, hi};
}

// Places in the vocabulary's order in bins of 2^SHIFT: a wave's chunks of one step.
template <int DT>
struct Places {
    static constexpr int SHIFT = DT == TVK_F32 ? 8 : 9, MASK = (1 << SHIFT) - 1;
    static_assert(1 << SHIFT == 64 * RowIn<DT>::VEC && SA_MOST_COLS >> SHIFT <= SA_BINS, "a wave's chunks; bins for all");
};

// The index of the last of the first b.ties tokens that equal the border.
template <int DT, int C>
__device__ __forceinline__ int last_tie(RowIn<DT, C>& x, const Border& b, Shared& s) {
    typedef Places<DT> At;
    constexpr int N = RowIn<DT>::N;
    if (b.ties == b.equal) return 0x7fffffff;
    clear(s.part);
    x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (v[k] == b.t) atomicAdd(&s.part.n[i[k] >> At::SHIFT], 1u);
    });
    __syncthreads();
    find_bin(true, true, b.ties, s);
    const int bin = s.found, i = (bin << At::SHIFT) + (int)threadIdx.x;
    const u64 need = b.ties - s.found_w;
    clear(s.part);
    if (threadIdx.x <= At::MASK && i >= 0 && i < x.cols) s.part.n[threadIdx.x] = x.value(i) == b.t;
    __syncthreads();
    find_bin(true, true, need, s);
    return (bin << At::SHIFT) + s.found;
}

// What the filters leave.
struct Keep {
    float t;
    int last;   // the index of the last tie
    __device__ __forceinline__ bool has(int i, float v) const { return v > t || (v == t && i <= last); }
};

// The tokens that `has` names, with their places: s.listed of them, at most MOST kept.
template <int MOST, int DT, int C, class F>
__device__ __forceinline__ void list_tokens(RowIn<DT, C>& x, float* v_out, int* at_out, Shared& s, F&& has) {
    constexpr int N = RowIn<DT>::N;
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (has(i[k], v[k])) {
                const unsigned o = atomicAdd(&s.listed, 1u);
                if (o < MOST) {
                    v_out[o] = v[k];
                    at_out[o] = i[k];
                }
            }
    });
    __syncthreads();
}

// The same, none kept where they are more, in two passes: `count` (which may do more) first, so that a wave asks for its
// share of the list once and not for each word. Many tokens of a piece are faster listed so, 64 x 128000 with flat
// distributions 60 us and 66; rows that one workgroup takes, with what they do besides, are not: 256 x 128000 148 and 134.
template <int MOST, int DT, int C, class G, class F>
__device__ __forceinline__ void list_counted(RowIn<DT, C>& x, float* v_out, int* at_out, Shared& s, G&& count, F&& has) {
    constexpr int N = RowIn<DT>::N;
    __syncthreads();
    if (threadIdx.x == 0) s.listed = 0;
    __syncthreads();
    unsigned n = 0;
    x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) n += count(i[k], v[k]);
    });
    const unsigned up_to = lanes_up_to(n);
    unsigned o = 0;
    if (threadIdx.x % 64 == 63) o = atomicAdd(&s.listed, up_to);
    o = (unsigned)__builtin_amdgcn_readlane((int)o, 63) + up_to - n;
    __syncthreads();
    if (s.listed <= MOST && __any(n))
        x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (has(i[k], v[k])) {
                    v_out[o] = v[k];
                    at_out[o++] = i[k];
                }
        });
    __syncthreads();
}

// The weights of the tokens that `has` keeps, in the places' bins: a wave's step is a bin, and nobody else's.
template <int DT, int C, class F>
__device__ __forceinline__ void add_all_places(RowIn<DT, C>& x, const Heat& h, const Filters& f, u64* places, F&& has) {
    constexpr int N = RowIn<DT>::N, VEC = RowIn<DT>::VEC;
    u64 sum = 0;   // of a chunk, then of a wave's
    x.each([&](const int (&i)[N], const float (&v)[N]) {
        bool keep[N], any = false;
#pragma unroll
        for (int k = 0; k < N; ++k) any |= keep[k] = has(i[k], v[k]);
        if (any) {
            u64 w[N];
#pragma unroll
            for (int k = 0; k < N; ++k) w[k] = f.weigh(h, v[k]);
#pragma unroll
            for (int k = 0; k < N; ++k) sum += keep[k] ? w[k] : 0;
        }
        if (i[0] % VEC == VEC - N) {   // (the same for all) the chunk's end
            sum = lanes_up_to(sum);
            if (threadIdx.x % 64 == 63 && i[0] / VEC - 63 < x.end) places[i[0] >> Places<DT>::SHIFT] = sum;
            sum = 0;
        }
    });
}

// The same where some may be left out: those that are kept were listed (s.list), where the list holds them, and are weighed
// by as many threads. s.part is used.
template <int DT, int C, class F>
__device__ __forceinline__ void add_listed_places(RowIn<DT, C>& x, const Heat& h, const Filters& f, u64* places, Shared& s, F&& has) {
    const unsigned n = s.listed;
    if (n > SA_KEPT) return add_all_places(x, h, f, places, has);   // (not of a list)
    clear(s.part);
    for (unsigned t = threadIdx.x; t < n; t += SA_THREADS) {
        const u64 w = f.weigh(h, s.list[t]);
        if (w) atomicAdd(&s.part.w[s.list_at[t] >> Places<DT>::SHIFT], w);
    }
    __syncthreads();
    constexpr int PER = 64;   // chunks of a place
    const int from = x.places ? 0 : x.first / PER, to = x.places ? SA_BINS : (x.end + PER - 1) / PER;
    for (int i = from + (int)threadIdx.x; i < to; i += SA_THREADS) places[i] = s.part.w[i];
}

template <int DT, int C, class F>
__device__ __forceinline__ void add_places(RowIn<DT, C>& x, const Heat& h, const Filters& f, u64* places, Shared& s, F&& has) {
    list_tokens<SA_KEPT>(x, s.list, s.list_at, s, has);
    add_listed_places(x, h, f, places, s, has);
}

__device__ inline void put(const SampleArgs& p, int64_t row, int token, float v, const Heat& h, const Filters& f, u64 total) {
    p.token[row] = token;
    if (!p.logprob) return;
    const double d = v == h.top ? 0.0 : ((double)v - (double)h.top) / f.heat;
    // log of the total in float32, and one step of Newton's method: e is within 2^-20 of 1
    const double sum = (double)total * 0x1p-44;
    const float log32 = __builtin_amdgcn_logf((float)sum) * 0.693147181f;
    const double e = sum * (Heat{0.0f, SA_STEPS * 1.4426950408889634, h.table}.large_weight(-log32) * 0x1p-44) - 1.0;
    p.logprob[row] = (float)(d - (log32 + (e - 0.5 * e * e)));
}

// The token, from the places' sums of weights (s.all): the first at which they pass the random number's share.
template <int DT>
__device__ __forceinline__ void draw(const SampleArgs& p, int64_t row, const typename elem<DT>::T* x, const Heat& h, const Filters& f,
                                     const Keep& k, Shared& s) {
    typedef Places<DT> At;
    const u64 total = sum_of(s.all, s), goal = f.goal(total);
    find_bin(false, false, goal + 1, s);
    const int bin = s.found, i = (bin << At::SHIFT) + (int)threadIdx.x;
    const u64 need = goal + 1 - s.found_w;
    clear(s.part);
    float v = -INFINITY;
    if (threadIdx.x <= At::MASK && i >= 0 && i < p.cols) {
        v = elem<DT>::to_f32(x[i]);
        if (k.has(i, v)) s.part.w[threadIdx.x] = f.weigh(h, v);   // (NaN is not kept)
    }
    __syncthreads();
    find_bin(true, false, need, s);
    if ((int)threadIdx.x == s.found) put(p, row, i, v, h, f, total);
}

__device__ inline void put_first(const SampleArgs& p, int64_t row, float top, unsigned at) {
    if (threadIdx.x != 0) return;
    p.token[row] = top == -INFINITY ? -1 : (int64_t)at;
    if (p.logprob) p.logprob[row] = top == -INFINITY ? NAN : 0.0f;
}

// The first place of the largest among a thread's values.
template <int DT, int C>
__device__ __forceinline__ unsigned first_of(RowIn<DT, C>& x, float top) {
    constexpr int N = RowIn<DT>::N;
    unsigned at = 0x7fffffff;
    x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) at = min(at, v[k] == top ? (unsigned)i[k] : at);
    });
    return at;
}

// All that is left, of n <= SA_FEW tokens (s.list, s.list_at) that hold what the filters can keep: compared with each other, a
// thread each.
__device__ __forceinline__ void finish_few(const SampleArgs& p, int64_t row, int n, const Heat& h, const Filters& f, Shared& s) {
    const int t = threadIdx.x;
    const bool there = t < n;
    const float v = there ? s.list[t] : -INFINITY;
    const int at = there ? s.list_at[t] : 0;
    const u64 w = there ? h.whole_weight(v) : 0;
    if (there) s.list_w[t] = w;
    compare_all(n, s, in_front);
    const u64 above = there ? s.before[t] : 0;   // of the tokens in front of this one
    const int rank = there ? (int)s.rank[t] : 0;
    bool keep = there && (!f.by_k || rank < f.top_k);
    if (f.by_p) {
        const u64 need = f.share(all_threads<AddOp>(keep ? w : (u64)0));
        keep = keep && above < need;
    }
    const u64 own = keep ? f.weigh(h, v) : 0;
    const u64 total = all_threads<AddOp>(own), goal = f.goal(total);
    if (there) s.list_w[t] = own;
    compare_all(n, s, [](float, int at, float, int o) { return o < at; });
    const u64 before = there ? s.before[t] : 0;
    if (before <= goal && goal < before + own) put(p, row, at, v, h, f, total);
}

// A row by one workgroup, with its largest logit known.
template <int DT, int C>
__device__ __forceinline__ void whole_row(const SampleArgs& p, int64_t row, RowIn<DT, C>& x, float top, const Filters& f, Shared& s) {
    if (f.first_only(top)) {
        put_first(p, row, top, all_threads<LeastOp>(first_of(x, top)));
        return;
    }
    const Heat h = f.weights(top, s);
    Border b{-INFINITY, 0, 0};
    const Range<double> whole = first_range<double>(top, f.heat);
#pragma unroll 1
    for (int filter = 0; filter < 2; ++filter) {
        const bool counts = filter == 0;   // top_k needs no weights; top_p's are of what that leaves
        if (!(counts ? f.by_k : f.by_p)) continue;
        if (!counts && f.by_k && b.t != -INFINITY) {   // from here on the tokens that top_k leaves, where a list holds them
            list_tokens<SA_KEPT>(x, s.list, s.kept_at, s, [&](int, float v) { return v >= b.t; });
            if (s.listed <= SA_KEPT) x.take(s.list, s.kept_at, (int)s.listed);
            __syncthreads();
        }
        Range<double> r = whole;
        r.lo = fmaxf(r.lo, b.t);
        u64 need = 0, above = 0;
#pragma unroll 1
        for (bool first = true;; first = false) {
            fill_bins(x, h, r, counts, s.all);
            if (first) {
                u64 total = sum_of(s.all, s);   // (of weights)
                if (b.equal > b.ties) total -= (b.equal - b.ties) * h.whole_weight(b.t);
                need = counts ? (u64)f.top_k : f.share(total);
            }
            find_bin(false, counts, need - above, s);
            const int bin = s.found;
            if (bin < 0) break;   // fewer tokens than top_k (other sums are exact: they reach what is asked of them)
            above += s.found_w;
            if (first && counts && above + s.found_own <= SA_FEW) {
                list_tokens<SA_FEW>(x, s.list, s.list_at, s, [&](int, float v) { return r.has(v) && r.bin(v) <= bin; });
                return finish_few(p, row, (int)s.listed, h, f, s);
            }
            const InBin in = border_in_bin(x, h, r, bin, counts, need, above, s);
            b = in.b;
            if (in.done) break;
            // a bin's values are fewer than its range's or lie closer, until they are equal
            r = {in.lo, in.hi, SA_BINS / ((double)in.hi - (double)in.lo)};
        }
    }
    const Keep k{b.t, last_tie(x, b, s)};
    clear(s.all);
    auto has = [&](int i, float v) { return k.has(i, v); };
    if (f.by_k || f.by_p) {
        add_places(x, h, f, s.all.w, s, has);
    } else {
        add_all_places(x, h, f, s.all.w, has);
    }
    __syncthreads();
    draw<DT>(p, row, x.row, h, f, k, s);
}

template <int DT, int C>
__device__ __forceinline__ float largest(RowIn<DT, C>& x, Shared& s) {
    constexpr int N = RowIn<DT>::N;
    float top = -INFINITY;
    x.each([&](const int (&)[N], const float (&v)[N]) {
#pragma unroll
        for (int k = 0; k < N; ++k) top = fmaxf(top, v[k]);
    });
    return all_threads<MostOp>(top);
}

// (No loop over rows: what it would keep from one to the next does not fit the registers, and scratch memory costs a launch
// 7 us.)
template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_rows_kernel(SampleArgs p) {
    __shared__ Shared s;
    make_table(s);
    const int64_t row = p.row0 + blockIdx.x;
    RowIn<DT> x(p, row, 0, 0x7fffffff);
    whole_row(p, row, x, largest(x, s), Filters(p, row), s);
}

// ---------------------------------------------------------------------------
// rows cut among workgroups
// ---------------------------------------------------------------------------

template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_top_kernel(SampleArgs p) {
    __shared__ Shared s;
    const int64_t row = blockIdx.x / (unsigned)p.pieces;
    const int piece = blockIdx.x % (unsigned)p.pieces;
    RowIn<DT> x(p, row, piece * p.piece, (piece + 1) * p.piece);
    const float top = largest(x, s);
    if (threadIdx.x == 0) p.tops[blockIdx.x] = top;
}

__device__ __forceinline__ float top_of(const SampleArgs& p, int64_t row) {
    const int lane = threadIdx.x % 64;
    return of_all(lanes64_all<MaxOp>(lane < p.pieces ? p.tops[row * p.pieces + lane] : -INFINITY));
}

// A piece's histogram; or where no border is wanted what the token is found from.
template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_bins_kernel(SampleArgs p) {
    __shared__ Shared s;
    make_table(s);
    const int64_t row = blockIdx.x / (unsigned)p.pieces;
    const int piece = blockIdx.x % (unsigned)p.pieces;
    RowIn<DT> x(p, row, piece * p.piece, (piece + 1) * p.piece);
    const float top = top_of(p, row);
    const Filters f(p, row);
    if (f.first_only(top)) {
        const unsigned at = all_threads<LeastOp>(first_of(x, top));
        if (threadIdx.x == 0) p.listed[blockIdx.x] = at;
        return;
    }
    const Heat h = f.weights(top, s);
    if (!f.by_k && !f.by_p) {
        add_all_places(x, h, f, p.places + row * SA_BINS, [](int, float) { return true; });
        return;
    }
    fill_bins(x, h, first_range<float>(top, f.heat), f.by_k, s.all);
    u64* out = p.bins + (int64_t)blockIdx.x * SA_BINS;
    out[threadIdx.x] = s.all.w[threadIdx.x];
    if (!f.by_k) out[threadIdx.x + SA_THREADS] = s.all.w[threadIdx.x + SA_THREADS];   // (counts are in the first half)
}

// The border's bin, from all pieces' histograms, and what of a piece lies in it and above.
template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_border_kernel(SampleArgs p) {
    __shared__ Shared s;
    make_table(s);
    const int64_t row = blockIdx.x / (unsigned)p.pieces;
    const int piece = blockIdx.x % (unsigned)p.pieces;
    RowIn<DT> x(p, row, piece * p.piece, (piece + 1) * p.piece);
    const float top = top_of(p, row);
    const Filters f(p, row);
    auto state = [&](int mode, int bin, u64 above, u64 need) {
        if (piece == 0 && threadIdx.x == 0) p.state[row] = {mode, bin, above, need};
    };
    if (f.first_only(top)) return state(SA_FIRST, 0, 0, 0);
    if (!f.by_k && !f.by_p) return state(SA_ALL, 0, 0, 0);
    const Heat h = f.weights(top, s);
    const u64* in = p.bins + row * p.pieces * SA_BINS + threadIdx.x;
    auto sum = [&](const u64* first) {
        u64 v = 0;   // counts are two to a word, and do not carry: there are at most 2^19
#pragma unroll 1
        for (int i = 0; i < p.pieces; i += 8) {
            u64 w[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) w[k] = first[(int64_t)min(i + k, p.pieces - 1) * SA_BINS];
#pragma unroll
            for (int k = 0; k < 8; ++k) v += i + k < p.pieces ? w[k] : 0;
        }
        return v;
    };
    s.all.w[threadIdx.x] = sum(in);
    s.all.w[threadIdx.x + SA_THREADS] = f.by_k ? 0 : sum(in + SA_THREADS);
    __syncthreads();
    const u64 need = f.by_k ? (u64)f.top_k : f.share(sum_of(s.all, s));
    find_bin(false, f.by_k, need, s);
    const int bin = s.found;
    const u64 above = s.found_w, own = s.found_own;
    u64* places = p.places + row * SA_BINS;
    if (bin < 0) {   // fewer tokens than top_k
        if (f.by_p) return state(SA_WHOLE, 0, 0, 0);
        add_all_places(x, h, f, places, [](int, float) { return true; });
        return state(SA_ALL, 0, 0, 0);
    }
    const Range<float> r = first_range<float>(top, f.heat);
    const bool few = f.by_k && above + own <= SA_FEW;
    if (f.by_k && f.by_p && !few) return state(SA_WHOLE, 0, 0, 0);
    // the bin's tokens, or all down to it, are listed; those above it weighed
    const int64_t list = (int64_t)blockIdx.x * SA_FEW;
    if (threadIdx.x == 0) s.found_n = 0;
    constexpr int N = RowIn<DT>::N;
    auto above_it = [&](int i, float v) {
        const int o = r.has(v) ? r.bin(v) : SA_BINS;
        if (o == bin || (few && o < bin)) {
            const unsigned at = atomicAdd(&s.found_n, 1u);
            if (at < SA_FEW) {
                p.list_v[list + at] = v;
                p.list_at[list + at] = i;
            }
        }
        return o < bin;
    };
    if (few) {
        __syncthreads();
        x.each([&](const int (&i)[N], const float (&v)[N]) {
#pragma unroll
            for (int k = 0; k < N; ++k) above_it(i[k], v[k]);
        });
        __syncthreads();
    } else {
        auto has = [&](int, float v) { return r.has(v) && r.bin(v) < bin; };
        list_counted<SA_KEPT>(x, s.list, s.list_at, s, above_it, has);
        add_listed_places(x, h, f, places, s, has);
    }
    if (threadIdx.x == 0) p.listed[blockIdx.x] = s.found_n;
    state(few ? SA_TOKENS : SA_SUMS, bin, above, need);
}

template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_token_kernel(SampleArgs p) {
    __shared__ Shared s;
    make_table(s);
    const int64_t row = blockIdx.x;
    const float top = top_of(p, row);
    const Filters f(p, row);
    const RowState st = p.state[row];
    const int lane = threadIdx.x % 64;
    const unsigned listed = lane < p.pieces ? p.listed[row * p.pieces + lane] : st.mode == SA_FIRST ? 0x7fffffffu : 0u;
    if (st.mode == SA_FIRST) return put_first(p, row, top, all_threads<LeastOp>(listed));
    const Heat h = f.weights(top, s);
    const typename elem<DT>::T* x = static_cast<const typename elem<DT>::T*>(p.x) + row * p.stride;
    int n = 0, base = 0;   // entries, and where they lie in s.list
    bool whole = st.mode == SA_WHOLE;
    if (st.mode == SA_TOKENS || st.mode == SA_SUMS) {   // the pieces' lists, one behind the other: a thread an entry
        const unsigned up_to = lanes_up_to(listed);
        n = (int)__builtin_amdgcn_readlane((int)up_to, 63);   // (at most 2^19)
        if (threadIdx.x < SA_PIECES) s.counts[threadIdx.x] = up_to;
        __syncthreads();
        whole = n > (st.mode == SA_TOKENS ? SA_FEW : SA_KEPT / 2) || (lane < p.pieces && listed > SA_FEW);
        whole = __any(whole);
        base = st.mode == SA_SUMS && n > SA_SOME ? SA_KEPT / 2 : 0;
        if (!whole)
            for (int t = threadIdx.x; t < n; t += SA_THREADS) {
                int i = 0;   // the first piece whose entries reach past this one
                for (int half = SA_PIECES / 2; half > 0; half /= 2)
                    if (s.counts[i + half - 1] <= t) i += half;
                const int64_t from = (row * p.pieces + i) * SA_FEW + t - (i ? s.counts[i - 1] : 0);
                s.list[base + t] = p.list_v[from];
                s.list_at[base + t] = p.list_at[from];
            }
        __syncthreads();
    }
    clear(s.all);
    const int places = (p.cols >> Places<DT>::SHIFT) + 1;
    if (st.mode == SA_ALL || st.mode == SA_SUMS)
        for (int i = threadIdx.x; i < places && i < SA_BINS; i += SA_THREADS)
            if (i << Places<DT>::SHIFT < p.cols) s.all.w[i] = p.places[row * SA_BINS + i];
    u64 before_list = st.above;
    if (base && !whole) {   // of many, those are weighed that lie above the border's bin within the bin
        const Range<float> r = first_range<float>(top, f.heat);
        clear(s.part);
        for (int t = threadIdx.x; t < n; t += SA_THREADS)
            atomicAdd(&s.part.w[r.part(s.list[base + t], st.bin)], f.by_k ? (u64)1 : h.whole_weight(s.list[base + t]));
        __syncthreads();
        find_bin(true, false, st.need - st.above, s);
        const int part = s.found;
        before_list += s.found_w;
        if (threadIdx.x == 0) s.listed = 0;
        __syncthreads();
        for (int t = threadIdx.x; t < n; t += SA_THREADS) {
            const float v = s.list[base + t];
            const int at = s.list_at[base + t], bin = r.part(v, st.bin);
            if (bin < part) {
                const u64 w = f.weigh(h, v);
                if (w) atomicAdd(&s.all.w[at >> Places<DT>::SHIFT], w);
            } else if (bin == part) {
                const unsigned o = atomicAdd(&s.listed, 1u);
                if (o < SA_FEW) s.list[o] = v, s.list_at[o] = at;
            }
        }
        __syncthreads();
        n = (int)s.listed;
        whole = n > SA_FEW;
        __syncthreads();
    }
    if (whole) {   // too many of them: from the start
        RowIn<DT, SA_CHUNKS / 2> all(p, row, 0, 0x7fffffff);   // (the others' registers are in use here)
        return whole_row(p, row, all, top, f, s);
    }
    if (st.mode == SA_TOKENS) return finish_few(p, row, n, h, f, s);
    Keep k{-INFINITY, 0x7fffffff};
    if (st.mode == SA_SUMS) {   // the bin's tokens, compared with each other
        const int t = threadIdx.x;
        const bool there = t < n;
        const float v = there ? s.list[t] : 0.0f;
        const int at = there ? s.list_at[t] : 0;
        const u64 each = there ? f.by_k ? 1 : h.whole_weight(v) : 0;
        if (there) s.list_w[t] = each;
        compare_all(n, s, in_front);
        const u64 before = there ? before_list + s.before[t] : 0;
        if (there && before < st.need) {
            const u64 w = f.weigh(h, v);
            if (w) atomicAdd(&s.all.w[at >> Places<DT>::SHIFT], w);
            if (before + each >= st.need) {   // the last of them
                s.border = v;
                s.last = at;
            }
        }
        __syncthreads();
        k = {s.border, s.last};
    }
    __syncthreads();
    draw<DT>(p, row, x, h, f, k, s);
}

template <int DT>
tvk_status launch(SampleArgs p, hipStream_t s) {
    // A workgroup a CU is wanted, for pieces of 512 chunks or more, and the three launches more that they take: one row of
    // bfloat16, top_k 50 and top_p 0.9, in pieces and not, 16000 values 21.6 and 14.6 us, 32000 22.3 and 19.4, 128000 24 and 51;
    // top_p alone 27.6 and 25.8, 27.7 and 38.7, 39 and 121.
    const int chunks = (p.cols + RowIn<DT>::VEC - 1) / RowIn<DT>::VEC;
    const int64_t pieces = chunks <= 2048 ? 1 : std::min<int64_t>({SA_PIECES, 256 / p.rows, chunks / 512});
    const dim3 block(SA_THREADS);
    if (pieces < 2) {
        constexpr int64_t MOST = 1 << 21;   // rows of a launch: 2^32 threads are too many
        for (p.row0 = 0; p.row0 < p.rows; p.row0 += MOST)
            hipLaunchKernelGGL((sample_rows_kernel<DT>), dim3((unsigned)std::min(p.rows - p.row0, MOST)), block, 0, s, p);
        return TVK_OK;
    }
    p.piece = (int)((chunks + pieces - 1) / pieces + 63) / 64 * 64;   // whole places
    p.pieces = (chunks + p.piece - 1) / p.piece;
    const int64_t all = p.rows * p.pieces;
    Scratch scratch;
    char* at = static_cast<char*>(scratch.get((size_t)(all * (SA_BINS * 8 + SA_FEW * 8 + 8) + p.rows * (SA_BINS * 8 + (int64_t)sizeof(RowState))), s));
    if (!at) return fail(TVK_ERR_OOM, "tvk_sample: workspace allocation failed");
    auto take = [&](auto*& to, int64_t n) {
        to = reinterpret_cast<std::remove_reference_t<decltype(to)>>(at);
        at += n * sizeof(*to);
    };
    take(p.bins, all * SA_BINS);
    take(p.places, p.rows * SA_BINS);
    take(p.state, p.rows);
    take(p.list_v, all * SA_FEW);
    take(p.list_at, all * SA_FEW);
    take(p.tops, all);
    take(p.listed, all);
    hipLaunchKernelGGL((sample_top_kernel<DT>), dim3((unsigned)all), block, 0, s, p);
    hipLaunchKernelGGL((sample_bins_kernel<DT>), dim3((unsigned)all), block, 0, s, p);
    hipLaunchKernelGGL((sample_border_kernel<DT>), dim3((unsigned)all), block, 0, s, p);
    hipLaunchKernelGGL((sample_token_kernel<DT>), dim3((unsigned)p.rows), block, 0, s, p);
    return TVK_OK;
}

}  // namespace

extern "C" tvk_status tvk_sample(const tvk_sample_desc* d) {
    auto bad = [](tvk_status st, const char* m) { return fail(st, std::string("tvk_sample: ") + m); };
    if (!d) return bad(TVK_ERR_INVALID, "desc is NULL");
    if (!norm_dtype(d->dtype)) return bad(TVK_ERR_UNSUPPORTED, "dtype must be float32, float16 or bfloat16");
    if (d->rows < 0 || d->cols < 0) return bad(TVK_ERR_INVALID, "negative size");
    if (d->rows > 0x7fffffff) return bad(TVK_ERR_UNSUPPORTED, "rows up to 2^31 - 1 only");
    if (d->cols > SA_MOST_COLS) return bad(TVK_ERR_UNSUPPORTED, "up to 2^19 columns only");
    if (d->rows == 0) return TVK_OK;
    if ((d->cols > 0 && !d->logits) || !d->random || !d->token) return bad(TVK_ERR_INVALID, "NULL tensor");
    if (d->logits_stride < 0) return bad(TVK_ERR_INVALID, "negative strides");
    SampleArgs p{};
    p.x = d->logits;
    p.temperature = d->temperature;
    p.top_k = d->top_k;
    p.top_p = d->top_p;
    p.min_p = d->min_p;
    p.random = d->random;
    p.token = d->token;
    p.logprob = d->logprob;
    p.rows = d->rows;
    p.stride = d->logits_stride;
    p.cols = (int)d->cols;
    const hipStream_t s = resolve_stream(d->stream);
    const tvk_status st = d->dtype == TVK_F32 ? launch<TVK_F32>(p, s) : d->dtype == TVK_F16 ? launch<TVK_F16>(p, s) : launch<TVK_BF16>(p, s);
    if (st != TVK_OK) return st;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return bad(TVK_ERR_DEVICE, (std::string("launch failed: ") + hipGetErrorString(e)).c_str());
    return TVK_OK;
}
