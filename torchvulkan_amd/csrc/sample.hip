// The next token of every row from its logits and a random number (tvk_sample).
//
// With s = x / T a token weighs exp(s - max s); what the filters leave is a prefix
// of the tokens in the order of their logits, equal ones in that of their indexes:
// those above a border value and the first few that equal it. So nothing is
// sorted. A histogram over the logits' distance from the largest, counts and sums
// of weights, says which bin the border of a filter falls into; the bin's own
// values, a few, are compared with each other in LDS, or spread over a histogram
// of their own until they are few or all equal. The token is then the first in the
// vocabulary's order at which the sum of kept weights passes the random number's
// share of their total, found by halving ranges 16 ways.
//
// Weights are integers: 2^44 exp(s - max s) from float64, rounded. Their sums are
// exact in 64 bits whatever the order (2^44 times at most 2^19 tokens), so that the
// atomics of a histogram and the split of a row over threads leave no trace in the
// result, and the borders fall where the formulas in 64 bits put them: float32
// weights would put one in 10^4 draws from a flat distribution elsewhere.
#include "norm_rows.h"

using namespace tvk;

namespace {

typedef unsigned long long u64;

constexpr int SA_THREADS = 1024, SA_WAVES = SA_THREADS / 64;
constexpr int SA_BINS = 2 * SA_THREADS;
constexpr int SA_LIST = 256;       // values of a bin that are compared with each other
constexpr int64_t SA_MOST_COLS = 1 << 19;

struct SampleArgs {
    const void* x;
    const float* temperature;
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    const float* random;
    int64_t* token;
    float* logprob;
    int64_t rows, stride;
    int cols;
};

// A row's weights.
struct Heat {
    float top;   // the largest logit
    double c;    // log2(e) / T
    // exp((x - top) / T), within 2^-46 of itself; below 2^-50 zero
    __device__ double weight(float x) const {
        if (x == top) return 1.0;   // infinities too
        const double t = ((double)x - (double)top) * c;
        if (!(t > -50.0)) return 0.0;
        const double n = rint(t), f = (t - n) * 0.693147180559945309;
        // the exponential's series up to f^11 / 11!: |f| <= 0.3466, so what follows is below 7e-15
        double p = 1.0 / 39916800;
        p = fma(p, f, 1.0 / 3628800);
        p = fma(p, f, 1.0 / 362880);
        p = fma(p, f, 1.0 / 40320);
        p = fma(p, f, 1.0 / 5040);
        p = fma(p, f, 1.0 / 720);
        p = fma(p, f, 1.0 / 120);
        p = fma(p, f, 1.0 / 24);
        p = fma(p, f, 1.0 / 6);
        p = fma(p, f, 0.5);
        p = fma(p, f, 1.0);
        p = fma(p, f, 1.0);
        return ldexp(p, (int)n);
    }
    __device__ static u64 whole(double w) {   // 2^44 w rounded: the low bits of a sum whose last place is 1
        return __builtin_bit_cast(u64, fma(w, 0x1p44, 0x1p52)) & ((1ull << 52) - 1);
    }
    __device__ u64 whole_weight(float x) const { return whole(weight(x)); }
};

// A row in chunks of 16 bytes; -inf past its end and for NaN, and zeros of one sign.
template <int DT>
struct Logits {
    typedef typename elem<DT>::T T;
    static constexpr int VEC = 16 / (int)sizeof(T);
    const T* row;
    int cols, chunks;
    __device__ static float cleaned(float v) { return v == v ? v + 0.0f : -INFINITY; }
    __device__ void load(int c, float (&v)[VEC]) const {
        if ((c + 1) * VEC <= cols) {
            const Words<16> w = load_words<16, sizeof(T)>(row + c * VEC);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = cleaned(word_at<DT>(w, k));
        } else {
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = c * VEC + k < cols ? cleaned(elem<DT>::to_f32(row[c * VEC + k])) : -INFINITY;
        }
    }
    // f(chunk, values) over the row
    template <class F>
    __device__ void each(F&& f) const {
        for (int c = threadIdx.x; c < chunks; c += SA_THREADS) {
            float v[VEC];
            load(c, v);
            f(c, v);
        }
    }
};

// A sum or a maximum over the workgroup, the same bits in every thread.
template <class V, class F>
__device__ V all_threads(V v, V* part, F&& f) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = f(v, __shfl_xor(v, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
    for (int w = 1; w < SA_WAVES; ++w) v = f(v, part[w]);
    return v;
}

// Sum of the lanes before this one.
template <class V>
__device__ V lanes_before(V v) {
    const V own = v;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const V o = __shfl_up(v, m);
        if ((int)(threadIdx.x % 64) >= m) v += o;
    }
    return v - own;
}

struct Bins {
    u64 w[SA_BINS];
    unsigned n[SA_BINS];
};

struct Shared {
    Bins all, part;        // of the whole row, of a bin
    float list[SA_LIST];
    u64 list_w[SA_LIST];
    u64 sums[SA_WAVES];
    unsigned counts[SA_WAVES];
    float values[SA_WAVES];
    // what one thread finds for all
    u64 found_w;
    unsigned found_n, found_count, listed;
    int found;
    float border;
    int64_t token;
};

// Values between lo and hi in bins of equal width, the largest first.
struct Range {
    float lo, hi;
    double scale;
    __device__ bool has(float x) const { return x >= lo && x <= hi; }
    __device__ int bin(float x) const { return (int)fmin(((double)hi - (double)x) * scale, (double)(SA_BINS - 1)); }
};

// The values that a filter keeps: above t, and the first `ties` that equal it. w: weight of those above.
struct Border {
    float t;
    unsigned ties;
    u64 w;
};

template <int DT>
__device__ void fill_bins(const Logits<DT>& x, const Heat& h, const Range& r, Bins& b) {
    for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) b.w[i] = 0, b.n[i] = 0;
    __syncthreads();
    x.each([&](int, const float (&v)[Logits<DT>::VEC]) {
#pragma unroll
        for (int k = 0; k < Logits<DT>::VEC; ++k)
            if (r.has(v[k])) {
                const int i = r.bin(v[k]);
                atomicAdd(&b.n[i], 1u);
                const u64 w = h.whole_weight(v[k]);
                if (w) atomicAdd(&b.w[i], w);
            }
    });
    __syncthreads();
}

// The first bin with which the count, or the weight, reaches `need`: s.found, and what is before it.
__device__ inline void find_bin(const Bins& b, bool by_count, u64 need, Shared& s) {
    const int i = 2 * threadIdx.x, wave = threadIdx.x / 64;
    const u64 w0 = b.w[i], w1 = b.w[i + 1];
    const unsigned n0 = b.n[i], n1 = b.n[i + 1];
    u64 w = lanes_before(w0 + w1);
    unsigned n = lanes_before(n0 + n1);
    __syncthreads();
    if (threadIdx.x == 0) s.found = -1;
    if (threadIdx.x % 64 == 63) s.sums[wave] = w + w0 + w1, s.counts[wave] = n + n0 + n1;
    __syncthreads();
    for (int k = 0; k < wave; ++k) w += s.sums[k], n += s.counts[k];
    auto reaches = [&](u64 w, unsigned n) { return by_count ? n >= need : w >= need; };
    const bool first = !reaches(w, n) && reaches(w + w0, n + n0), second = !reaches(w + w0, n + n0) && reaches(w + w0 + w1, n + n0 + n1);
    if (first || second) {
        s.found = first ? i : i + 1;
        s.found_w = first ? w : w + w0;
        s.found_n = first ? n : n + n0;
        s.found_count = first ? n0 : n1;
    }
    __syncthreads();
}

// Where the first `need` tokens end, or those that weigh `need` together.
template <int DT>
__device__ Border find_border(const Logits<DT>& x, const Heat& h, Range r, bool by_count, u64 need, Shared& s) {
    u64 above_w = 0;
    unsigned above_n = 0;
    const Bins* bins = &s.all;
    for (;;) {   // a bin's values are fewer than its range's or lie closer, until they are equal
        find_bin(*bins, by_count, need - (by_count ? above_n : above_w), s);
        const int bin = s.found;
        if (bin < 0) return {-INFINITY, 0, above_w};   // (sums are exact: they reach what is asked of them)
        above_w += s.found_w;
        above_n += s.found_n;
        const unsigned count = s.found_count;
        __syncthreads();
        if (threadIdx.x == 0) s.listed = 0;
        __syncthreads();
        float lo = INFINITY, hi = -INFINITY;
        x.each([&](int, const float (&v)[Logits<DT>::VEC]) {
#pragma unroll
            for (int k = 0; k < Logits<DT>::VEC; ++k)
                if (r.has(v[k]) && r.bin(v[k]) == bin) {
                    lo = fminf(lo, v[k]);
                    hi = fmaxf(hi, v[k]);
                    if (count <= SA_LIST) {
                        const unsigned i = atomicAdd(&s.listed, 1u);
                        s.list[i] = v[k];
                        s.list_w[i] = h.whole_weight(v[k]);
                    }
                }
        });
        lo = all_threads(lo, s.values, [](float a, float b) { return fminf(a, b); });
        hi = all_threads(hi, s.values, [](float a, float b) { return fmaxf(a, b); });
        if (lo == hi) {
            const u64 left = need - (by_count ? above_n : above_w), w = h.whole_weight(lo);
            return {lo, by_count ? (unsigned)left : (unsigned)((left + w - 1) / w), above_w};
        }
        if (count <= SA_LIST) {
            if (threadIdx.x < count) {
                const float own = s.list[threadIdx.x];
                u64 w = above_w;
                unsigned n = above_n, equal = 0;
                for (unsigned i = 0; i < count; ++i) {
                    const float o = s.list[i];
                    if (o > own) w += s.list_w[i], ++n;
                    equal += o == own;
                }
                const u64 each = s.list_w[threadIdx.x], before = by_count ? n : w;
                if (before < need && need <= before + (by_count ? equal : equal * each)) {   // all that equal the border write the same
                    s.border = own;
                    s.found_n = by_count ? (unsigned)(need - before) : (unsigned)((need - before + each - 1) / each);
                    s.found_w = w;
                }
            }
            __syncthreads();
            return {s.border, s.found_n, s.found_w};
        }
        r = {lo, hi, SA_BINS / ((double)hi - (double)lo)};
        fill_bins(x, h, r, s.part);
        bins = &s.part;
    }
}

template <int DT>
__device__ void sample_row(const SampleArgs& p, int64_t row, Shared& s) {
    constexpr int VEC = Logits<DT>::VEC;
    const Logits<DT> x{static_cast<const typename elem<DT>::T*>(p.x) + row * p.stride, p.cols, (p.cols + VEC - 1) / VEC};
    float top = -INFINITY, low = INFINITY;
    int at = 0x7fffffff;
    unsigned count = 0;   // of tokens that weigh anything
    x.each([&](int c, const float (&v)[VEC]) {
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if (v[k] > top) top = v[k], at = c * VEC + k;
            if (v[k] != -INFINITY) low = fminf(low, v[k]), ++count;
        }
    });
    const float own = top;
    top = all_threads(top, s.values, [](float a, float b) { return fmaxf(a, b); });
    at = (int)all_threads(own == top ? (unsigned)at : 0x7fffffffu, s.counts, [](unsigned a, unsigned b) { return a < b ? a : b; });
    const float heat = p.temperature ? p.temperature[row] : 1.0f, random = p.random[row];
    const float top_p = p.top_p ? p.top_p[row] : 1.0f, least = p.min_p ? p.min_p[row] : 0.0f;
    const int top_k = p.top_k ? p.top_k[row] : 0;
    if (top == -INFINITY || !(heat > 0.0f) || top_k == 1 || top_p <= 0.0f) {   // nothing, or the largest
        if (threadIdx.x == 0) {
            p.token[row] = top == -INFINITY ? -1 : at;
            if (p.logprob) p.logprob[row] = top == -INFINITY ? NAN : 0.0f;
        }
        return;
    }
    low = all_threads(low, s.values, [](float a, float b) { return fminf(a, b); });
    count = all_threads(count, s.counts, [](unsigned a, unsigned b) { return a + b; });
    const Heat h{top, 1.4426950408889634 / heat};
    if (top == INFINITY) low = top;   // beside an infinite logit the others weigh nothing
    const bool by_k = top_k > 0 && (unsigned)top_k < count, by_p = top_p < 1.0f;
    Border b{-INFINITY, 0, 0};
    if (by_k || by_p) {
        if (low == top) {   // all equal
            unsigned n = 0;
            x.each([&](int, const float (&v)[VEC]) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) n += v[k] == top;
            });
            n = all_threads(n, s.counts, [](unsigned a, unsigned b) { return a + b; });
            if (by_k) n = min(n, (unsigned)top_k);
            b = {top, by_p ? max(1u, (unsigned)ceil((double)top_p * n)) : n, 0};
        } else {
            const double span = fmin((double)top - (double)low, 28.0 * heat);   // weights from 1 to 2^-40; the rest in the last bin
            const Range r{low, top, SA_BINS / span};
            fill_bins(x, h, r, s.all);
            u64 total = 0;
            if (by_k) {
                b = find_border(x, h, r, true, (u64)top_k, s);
                total = b.w + b.ties * h.whole_weight(b.t);
            } else {
                u64 w = 0;
                for (int i = threadIdx.x; i < SA_BINS; i += SA_THREADS) w += s.all.w[i];
                total = all_threads(w, s.sums, [](u64 a, u64 b) { return a + b; });
            }
            if (by_p) {
                const u64 need = min(total, max((u64)1, (u64)ceil((double)top_p * (double)total)));
                b = find_border(x, h, r, false, need, s);
            }
        }
    }
    // Kept: v > b.t, the first b.ties that equal it, and of those what weighs `least` of the largest.
    const bool by_least = least > 0.0f;
    const double floor_w = fmin((double)least, 1.0);
    auto weigh = [&](float v) {
        const double w = h.weight(v);
        return by_least && w < floor_w ? (u64)0 : Heat::whole(w);
    };
    const u64 tie_w = b.ties ? weigh(b.t) : 0;
    // chunks [first, end) hold the token; before them lie `ties` equal to the border and the weight `base`
    int first = 0, end = x.chunks;
    unsigned ties = 0;
    u64 base = 0, goal = 0, total = 0;
    for (bool whole_row = true; whole_row || end - first > 64; whole_row = false) {
        const int each = ((end - first + SA_WAVES - 1) / SA_WAVES + 63) / 64 * 64, wave = threadIdx.x / 64;
        u64 w = 0;
        unsigned n = 0;
        for (int c = first + wave * each + threadIdx.x % 64; c < min(first + (wave + 1) * each, end); c += 64) {
            float v[VEC];
            x.load(c, v);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if (v[k] > b.t) w += weigh(v[k]);
                n += v[k] == b.t;
            }
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) w += __shfl_xor(w, m), n += __shfl_xor(n, m);
        __syncthreads();
        if (threadIdx.x % 64 == 0) s.sums[wave] = w, s.counts[wave] = n;
        __syncthreads();
        auto kept_ties = [&](unsigned before, unsigned n) { return min(before + n, max(b.ties, before)) - before; };
        if (whole_row) {
            unsigned t = 0;
            for (int k = 0; k < SA_WAVES; ++k) total += s.sums[k] + kept_ties(t, s.counts[k]) * tie_w, t += s.counts[k];
            const double share = random > 0.0f ? (double)random * (double)total : 0.0;
            goal = share < (double)total ? (u64)share : total - 1;
            goal = min(goal, total - 1);
        }
        for (int k = 0;; ++k) {   // the first wave whose chunks pass the goal
            const u64 sum = s.sums[k] + kept_ties(ties, s.counts[k]) * tie_w;
            if (base + sum > goal || k == SA_WAVES - 1) {
                first = min(first + k * each, end);
                end = min(first + each, end);
                break;
            }
            base += sum;
            ties += s.counts[k];
        }
    }
    if (threadIdx.x < 64) {
        float v[VEC];
        const int c = first + threadIdx.x;
        if (c < end) x.load(c, v);
        else
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[k] = -INFINITY;
        unsigned n = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) n += b.ties && v[k] == b.t;
        ties += lanes_before(n);
        u64 w[VEC], sum = 0;
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            w[k] = v[k] > b.t ? weigh(v[k]) : v[k] == b.t && b.ties && ties++ < b.ties ? tie_w : 0;
            sum += w[k];
        }
        base += lanes_before(sum);
        if (base <= goal && base + sum > goal) {   // one lane's
            int k = 0;
#pragma unroll
            for (int i = 0; i < VEC; ++i)
                if (base <= goal) base += w[i], k = i;
            p.token[row] = c * VEC + k;
            if (p.logprob) {
                float picked = v[0];
#pragma unroll
                for (int i = 1; i < VEC; ++i) picked = k == i ? v[i] : picked;
                const double d = picked == top ? 0.0 : ((double)picked - (double)top) / heat;
                p.logprob[row] = (float)(d - log((double)total * 0x1p-44));
            }
        }
    }
}

template <int DT>
__global__ __launch_bounds__(SA_THREADS) void sample_kernel(SampleArgs p) {
    __shared__ Shared s;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        sample_row<DT>(p, row, s);
        __syncthreads();
    }
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
    const SampleArgs p{d->logits, d->temperature, d->top_k, d->top_p, d->min_p, d->random, d->token, d->logprob,
                       d->rows, d->logits_stride, (int)d->cols};
    const hipStream_t s = resolve_stream(d->stream);
    const dim3 grid((unsigned)std::min<int64_t>(d->rows, 1 << 20)), block(SA_THREADS);
    if (d->dtype == TVK_F32) hipLaunchKernelGGL((sample_kernel<TVK_F32>), grid, block, 0, s, p);
    else if (d->dtype == TVK_F16) hipLaunchKernelGGL((sample_kernel<TVK_F16>), grid, block, 0, s, p);
    else hipLaunchKernelGGL((sample_kernel<TVK_BF16>), grid, block, 0, s, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return bad(TVK_ERR_DEVICE, (std::string("launch failed: ") + hipGetErrorString(e)).c_str());
    return TVK_OK;
}
