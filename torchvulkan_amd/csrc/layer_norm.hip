// Layer norm (tvk_layer_norm_fwd, tvk_layer_norm_bwd).
//
// Both directions read and write each value once and are bound by that. A row is
// in registers (norm_rows.h) while two reductions run over it: its sum, then the
// squares of its distances d from the mean m that the sum gives. The second takes
// sum(d) too, which would be zero if m were exact: with e = sum(d) / cols the
// centred values are d - e and the variance sum(d^2) / cols - e^2, so that a row
// far from zero loses nothing to its mean's rounding. A row about zero has e = 0
// (see Left). Backward, the same two
// reductions carry sum(g), g = dy w, and sum(g d), and
//   dx = inv (g - mean(g) - n mean(g n)) + dh,   n = (d - e) inv;
// a workgroup takes rows in turn and keeps the sums of dweight (dy n) and dbias
// (dy) in registers; a second launch adds the workgroups' up in a fixed order.
// 8-bit output has a scale for each 128 columns: 16 or 32 neighbouring lanes,
// whose largest value is one reduction among them.
//
// Measured, where a copy reaches 5.2 TB/s: 16384 x 4096 of bfloat16 with a residual
// to 8 bits 91 us (472 MB, 5.2 TB/s); backward of 16384 x 2048 62 us, 5 of them the
// second launch (268 MB); 5 x 1024 3.3 us, a launch; backward of 1000 x 777 of float32
// 10 us, two launches. A row of 512 chunks by 512 threads with one chunk each was slower,
// 101 us and 92, and so was one kept packed between the sums, which fits five
// workgroups a CU for four, 97 us.
#include "f8_blocks.h"
#include "norm_rows.h"

using namespace tvk;

namespace {

struct LayerArgs {
    const void* x;
    const void* r;
    const void* w;
    const void* b;
    void* out;
    void* h;
    float* scale;
    int64_t sx, sr, so, sh;   // row strides, elements
    int64_t ss[2];            // scale: row, block
    int64_t rows, cols;
    float eps, rcols;
    int w32, out8;
};

struct LayerBwdArgs {
    const void* dy;
    const void* h;
    const void* dh;
    const void* w;
    void* dx;
    void* dw;      // of a single workgroup, which needs no partials; or NULL
    void* db;
    float* stats;  // [rows][3]: m, e and 1 / sqrt(variance + eps), of long rows
    int64_t sdy, sh, sdh, sdx;
    int64_t rows, cols;
    float eps, rcols;
    int w32, want;   // gradients wanted: 1 dweight, 2 dbias
};

// Sums over a row's TPR threads, the same bits in each; `turn` as in row_all.
template <int TPR, int N>
__device__ __forceinline__ void row_sums(float (&v)[N], int turn) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = TPR == 16 ? lanes16_all<SumOp>(v[i]) : lanes64_all<SumOp>(v[i]);
    if constexpr (TPR > 64) {
        __shared__ float part[2][1024 / 64][N];
        const int wave = threadIdx.x / 64, w0 = threadIdx.x / TPR * (TPR / 64);
        if (threadIdx.x % 64 == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) part[turn][wave][i] = v[i];
        __syncthreads();
        constexpr int AT_ONCE = TPR > 512 && N > 2 ? 3 : TPR / 64;   // (three sums of 16 waves take too many registers)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            v[i] = part[turn][w0][i];
#pragma unroll AT_ONCE
            for (int w = 1; w < TPR / 64; ++w) v[i] += part[turn][w0 + w][i];
        }
    }
}

// The largest of LANES (16 or 32) neighbouring lanes, in each of them.
template <int LANES>
__device__ __forceinline__ float lanes_top(float v) {
    v = lanes16_all<MaxOp>(v);
    if constexpr (LANES == 32) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        v = fmaxf(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    }
    return v;
}

// What is left of a row's mean m, e = sum(d) / cols, and the squares about m + e, from sum(d) and sum(d^2).
//
// m is off by a few 2^-24 |m|, by additions most of which are of like size. e is off by what rounding did to the d: in a
// binade all d are off by the same part of their last place, where the values are of fewer bits, which comes to 2^-26 of the
// deviation on the whole. The values near the mean, whose d is exact to the last place of their own, would all be moved by that.
// So e is zero for a mean below an eighth of the deviation, where either is off by about the same: of 16384 x 4096
// bfloat16 values about zero, in 8 bits, 77 came out on the other side of a rounding than in 64 bits; 145 with e (three draws).
struct Left {
    float e, squares;
    __device__ __forceinline__ Left(float mean, float sum, float sq, float cols_inverse) {
        const bool small = 64.0f * mean * mean < sq * cols_inverse;   // (not of NaN)
        e = small ? 0.0f : sum * cols_inverse;
        squares = small ? sq : fmaxf(sq - sum * e, 0.0f);
    }
};

// 1 / sqrt(ss * rcols + eps): the instruction's, a step of 2^-23 or so off, once by Newton's method.
__device__ __forceinline__ float inv_std(float ss, float rcols, float eps) {
    const float x = fmaf(ss, rcols, eps), r = inv_rms(ss, rcols, eps);
    return x > 1e-30f && x < 1e30f ? fmaf(0.5f * r, fmaf(-x * r, r, 1.0f), r) : r;
}

template <int DT, bool OUT8, int NC, int TPR>
__global__ __launch_bounds__(row_threads(TPR)) void layer_norm_kernel(LayerArgs p) {
    typedef Row<DT, NC, TPR> R;
    typedef typename R::T T;
    constexpr int VEC = R::VEC, SUBS = row_threads(TPR) / TPR;
    constexpr int LANES = F8_BLOCK / VEC < TPR ? F8_BLOCK / VEC : TPR;   // that share a block
    const int t = threadIdx.x % TPR, chunks = (int)p.cols / VEC, tail = (int)p.cols % VEC;
    // 8 bits: the values past the last whole chunk are held beside their block's chunks, block `tb`
    const int tb = VEC * chunks / F8_BLOCK, tc = tb * (F8_BLOCK / VEC);
    const int tt = OUT8 ? (t - tc % TPR + TPR) % TPR : t;
    const bool has_last = tt < tail;
    Weights<DT, NC, TPR> w, b;
    w.load(p.w, p.w32, t, chunks, tail, tt, 1.0f);
    b.load(p.b, p.w32, t, chunks, tail, tt, 0.0f);
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * SUBS; first < p.rows; first += (int64_t)gridDim.x * SUBS) {
        const int64_t row = first + row_of_thread<TPR>();
        if (TPR < RN_THREADS && row >= p.rows) break;   // (rows of whole workgroups are always there)
        R h, r;
        h.load(static_cast<const T*>(p.x) + row * p.sx, t, chunks, tail, tt);
        if (p.r) {
            r.load(static_cast<const T*>(p.r) + row * p.sr, t, chunks, tail, tt);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                float s[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = h.at(i, k) + r.at(i, k);
                h.c[i] = pack<DT, VEC>(s);
            }
            h.last = elem<DT>::to_f32(elem<DT>::from_f32(h.last + r.last));
        }
        float v[NC][VEC], sum[1] = {has_last ? h.last : 0.0f};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float part = 0.0f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) part += v[i][k] = h.at(i, k);   // chunks past the row are zeros
            sum[0] += part;
        }
        row_sums<TPR>(sum, turn);
        const float mean = sum[0] * p.rcols;
        float last = has_last ? h.last - mean : 0.0f, dev[2] = {last * last, last};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const bool in = t + TPR * i < chunks;
            float sq = 0.0f, part = 0.0f;
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[i][k] -= mean;
                sq = fmaf(v[i][k], v[i][k], sq);
                part += v[i][k];
            }
            dev[0] += in ? sq : 0.0f;
            dev[1] += in ? part : 0.0f;
        }
        row_sums<TPR>(dev, turn ^ 1);
        const Left left(mean, dev[1], dev[0], p.rcols);
        const float e = left.e, inv = inv_std(left.squares, p.rcols, p.eps);
        if (p.h) {
            T* o = static_cast<T*>(p.h) + row * p.sh;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (t + TPR * i < chunks) store_words<16, sizeof(T)>(o + (uint32_t)(VEC * (t + TPR * i)), h.c[i]);
            if (has_last) o[VEC * chunks + tt] = elem<DT>::from_f32(h.last);
        }
        const float shift = -e * inv;
        last = fmaf(fmaf(last, inv, shift), w.r.last, b.r.last);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], g[VEC];
            w.chunk(i, t, chunks, f);
            b.chunk(i, t, chunks, g);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i][k] = fmaf(fmaf(v[i][k], inv, shift), f[k], g[k]);
        }
        if constexpr (OUT8) {
            uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.so;
            float* scale = p.scale + row * p.ss[0];
            const float last_top = has_last ? fabsf(last) : 0.0f;
            float tops[NC];
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                tops[i] = 0.0f;
                if (t + TPR * i < chunks)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) tops[i] = fmaxf(tops[i], fabsf(v[i][k]));
                if (tc / TPR == i) tops[i] = fmaxf(tops[i], last_top);
            }
            if constexpr (TPR * VEC < F8_BLOCK && NC == 2) tops[0] = tops[1] = fmaxf(tops[0], tops[1]);   // the row is one block
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                const F8Scale s(lanes_top<LANES>(tops[i]));
                const int c = t + TPR * i;
                if (c < chunks) {
                    Words<VEC> q;
#pragma unroll
                    for (int k = 0; k < VEC; k += 4) q.w[k / 4] = s.divide4(v[i][k], v[i][k + 1], v[i][k + 2], v[i][k + 3]);
                    store_words<VEC, 1>(o + (uint32_t)(VEC * c), q);
                }
                const bool ours = tc / TPR == i;
                if (ours && has_last) o[VEC * chunks + tt] = s.divide1(last);
                // the block's first chunk, or its first value past the chunks
                if (VEC * c % F8_BLOCK == 0 && c < chunks) scale[VEC * c / F8_BLOCK * p.ss[1]] = s.s;
                if (ours && tc >= chunks && has_last && tt == 0) scale[tb * p.ss[1]] = s.s;
            }
            if (tc / TPR >= NC) {   // registers full of chunks, and the values past them a block of their own
                const F8Scale s(lanes_top<LANES>(last_top));
                if (has_last) o[VEC * chunks + tt] = s.divide1(last);
                if (has_last && tt == 0) scale[tb * p.ss[1]] = s.s;
            }
        } else {
            T* o = static_cast<T*>(p.out) + row * p.so;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (t + TPR * i < chunks) store_words<16, sizeof(T)>(o + (uint32_t)(VEC * (t + TPR * i)), pack<DT, VEC>(v[i]));
            if (has_last) o[VEC * chunks + tt] = elem<DT>::from_f32(last);
        }
    }
}

// part: [2][gridDim.x][cols], the workgroups' sums of dy * n and of dy over their rows; NULL: not wanted.
template <int DT, int NC, int TPR, int THREADS>
__global__ __launch_bounds__(THREADS) void layer_norm_bwd_kernel(LayerBwdArgs p, float* part) {
    typedef Row<DT, NC, TPR> R;
    typedef typename R::T T;
    constexpr int VEC = R::VEC, SUBS = THREADS / TPR;
    const int t = threadIdx.x % TPR, sub = row_of_thread<TPR>(), chunks = (int)p.cols / VEC, tail = (int)p.cols % VEC;
    Weights<DT, NC, TPR> w;
    w.load(p.w, p.w32, t, chunks, tail);
    // The longest rows leave no registers for the sums of dweight and dbias, nor for the next row: each thread has its sums in
    // LDS (4096 x 16384 of bfloat16 182 us, in registers with spills 380, and 640 with the next row too).
    constexpr bool LONG = NC * TPR >= 2048;
    __shared__ f32x4 acc_lds[LONG ? 2 : 1][LONG ? NC * VEC / 4 : 1][LONG ? TPR : 1];
    float acc[2][NC][VEC], acc_last[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            if constexpr (LONG) acc_lds[0][(i * VEC + k) / 4][t] = acc_lds[1][(i * VEC + k) / 4][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            else acc[0][i][k] = acc[1][i][k] = 0.0f;
        }
    int64_t row = (int64_t)blockIdx.x * SUBS + sub;
    const int64_t step = (int64_t)gridDim.x * SUBS;
    R dy, h, dh;   // of the next row, on their way while one is computed
    auto load = [&]() {
        dy.load(static_cast<const T*>(p.dy) + row * p.sdy, t, chunks, tail);
        h.load(static_cast<const T*>(p.h) + row * p.sh, t, chunks, tail);
        if (p.dh) dh.load(static_cast<const T*>(p.dh) + row * p.sdh, t, chunks, tail);
    };
    if (!LONG && row < p.rows) load();
    // a workgroup's rows keep step: their sums meet at barriers
    for (int64_t first = (int64_t)blockIdx.x * SUBS; first < p.rows; first += step) {
        if (LONG && row < p.rows) load();
        R gy = dy, x = h, add = dh;
        const bool live = row < p.rows;
        T* dx = static_cast<T*>(p.dx) + row * p.sdx;
        row += step;
        if (!LONG && row < p.rows) load();
        const bool has_last = t < tail;
        float one[2] = {has_last ? x.last : 0.0f, has_last ? gy.last * w.r.last : 0.0f};   // sums of h and of g
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], px = 0.0f, pg = 0.0f;
            w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                px += x.at(i, k);
                pg = fmaf(gy.at(i, k), f[k], pg);
            }
            one[0] += px;
            one[1] += pg;
        }
        row_sums<TPR>(one, 0);
        if constexpr (NC > 1) {   // (one chunk's floats have room)
            gy.packed();
            x.packed();
            w.r.packed();
        }
        const float mean = one[0] * p.rcols;
        const float d_last = has_last ? x.last - mean : 0.0f;
        float two[3] = {d_last * d_last, d_last, gy.last * w.r.last * d_last};   // of d^2, d and g d
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const bool in = t + TPR * i < chunks;
            float f[VEC], sq = 0.0f, pd = 0.0f, pg = 0.0f;
            w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float d = x.at(i, k) - mean;
                sq = fmaf(d, d, sq);
                pd += d;
                pg = fmaf(gy.at(i, k) * f[k], d, pg);
            }
            two[0] += in ? sq : 0.0f;
            two[1] += in ? pd : 0.0f;
            two[2] += in ? pg : 0.0f;
        }
        row_sums<TPR>(two, 1);
        if (!live) continue;
        add.packed();
        if constexpr (NC > 1) {
            gy.packed();
            x.packed();
            w.r.packed();
        }
        const Left left(mean, two[1], two[0], p.rcols);
        const float e = left.e, inv = inv_std(left.squares, p.rcols, p.eps);
        const float gmean = one[1] * p.rcols;
        const float nmean = (two[2] - e * one[1]) * inv * p.rcols;   // of g * n
        auto centred = [&](float v) { return (v - mean) - e; };
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], o[VEC];
            f32x4 grads[2];   // of four columns, LONG
            w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float n = centred(x.at(i, k)) * inv, d = gy.at(i, k);
                if constexpr (LONG)
                    if (k % 4 == 0) grads[0] = acc_lds[0][(i * VEC + k) / 4][t], grads[1] = acc_lds[1][(i * VEC + k) / 4][t];
                if constexpr (LONG) {
                    grads[0][k % 4] = fmaf(d, n, grads[0][k % 4]);
                    grads[1][k % 4] += d;
                    if (k % 4 == 3) acc_lds[0][(i * VEC + k) / 4][t] = grads[0], acc_lds[1][(i * VEC + k) / 4][t] = grads[1];
                } else {
                    acc[0][i][k] = fmaf(d, n, acc[0][i][k]);
                    acc[1][i][k] += d;
                }
                o[k] = inv * (fmaf(d, f[k], -gmean) - n * nmean);
                if (p.dh) o[k] += add.at(i, k);
            }
            if (t + TPR * i < chunks) store_words<16, sizeof(T)>(dx + (uint32_t)(VEC * (t + TPR * i)), pack<DT, VEC>(o));
        }
        if (has_last) {
            const float n = centred(x.last) * inv;
            acc_last[0] = fmaf(gy.last, n, acc_last[0]);
            acc_last[1] += gy.last;
            float o = inv * (fmaf(gy.last, w.r.last, -gmean) - n * nmean);
            if (p.dh) o += add.last;
            dx[VEC * chunks + t] = elem<DT>::from_f32(o);
        }
    }
    if (!part && !p.dw && !p.db) return;
    if constexpr (LONG) {   // a workgroup a row at a time: every thread stores its own sums
        for (int what = 0; what < 2; ++what) {
            if (!(p.want >> what & 1)) continue;
            float* out = part + ((int64_t)what * gridDim.x + blockIdx.x) * p.cols;
            void* grad = what ? p.db : p.dw;
            auto store = [&](int c, float v) {
                if (part) out[c] = v;
                else if (p.w32) static_cast<float*>(grad)[c] = v;
                else put<DT>(grad, c, v);
            };
            for (int q = 0; q < NC * VEC / 4; ++q) {
                const int i = q / (VEC / 4), c = VEC * (t + TPR * i) + 4 * (q % (VEC / 4));
                if (t + TPR * i < chunks)
#pragma unroll
                    for (int k = 0; k < 4; ++k) store(c + k, acc_lds[what][q][t][k]);
            }
            if (t < tail) store(VEC * chunks + t, acc_last[what]);
        }
        return;
    }
    __shared__ __attribute__((aligned(16))) float sum[LONG ? 1 : SUBS][LONG ? 1 : VEC * (NC * TPR + 1)];
#pragma unroll
    for (int what = 0; what < 2; ++what) {
        if (!(p.want >> what & 1)) continue;
        float* out = part + ((int64_t)what * gridDim.x + blockIdx.x) * p.cols;
        void* grad = what ? p.db : p.dw;
        auto put_chunks = [&](float* to) {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (t + TPR * i < chunks)
#pragma unroll
                    for (int k = 0; k < VEC; k += 4) {
                        const float four[4] = {acc[what][i][k], acc[what][i][k + 1], acc[what][i][k + 2], acc[what][i][k + 3]};
                        store_words<16, 4>(to + (uint32_t)(VEC * (t + TPR * i) + k), pack<TVK_F32, 4>(four));
                    }
            if (t < tail) to[VEC * chunks + t] = acc_last[what];
        };
        if (SUBS == 1 && part) {
            put_chunks(out);
            continue;
        }
        __syncthreads();
        put_chunks(sum[sub]);
        __syncthreads();
        for (int c = threadIdx.x; c < (int)p.cols; c += THREADS) {
            float v = sum[0][c];
#pragma unroll
            for (int i = 1; i < SUBS; ++i) v += sum[i][c];
            if (part) out[c] = v;
            else if (p.w32) static_cast<float*>(grad)[c] = v;
            else put<DT>(grad, c, v);
        }
    }
}

// ---------------------------------------------------------------------------
// rows past what registers hold: read again for every pass
// ---------------------------------------------------------------------------

// What the values that `value` gives are normalised with, the same bits in every thread.
struct Stats {
    float m, e, inv;
    __device__ float centred(float v) const { return (v - m) - e; }
};

template <class F>
__device__ inline Stats long_stats(int64_t cols, float eps, F&& value) {
    float s = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += RN_THREADS) s += value(c);
    const float m = block_all<SumOp>(s) / (float)cols;
    float sq = 0.0f, d = 0.0f;
    for (int64_t c = threadIdx.x; c < cols; c += RN_THREADS) {
        const float v = value(c) - m;
        sq += v * v;
        d += v;
    }
    d = block_all<SumOp>(d);
    sq = block_all<SumOp>(sq);
    const Left left(m, d, sq, 1.0f / (float)cols);
    return {m, left.e, 1.0f / sqrtf(left.squares / (float)cols + eps)};
}

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void layer_norm_any_kernel(LayerArgs p) {
    typedef typename elem<DT>::T T;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.sx;
        const T* r = p.r ? static_cast<const T*>(p.r) + row * p.sr : nullptr;
        T* h = p.h ? static_cast<T*>(p.h) + row * p.sh : nullptr;
        auto sum = [&](int64_t c) {
            float v = at<DT>(x, c);
            if (r) v = elem<DT>::to_f32(elem<DT>::from_f32(v + at<DT>(r, c)));
            return v;
        };
        if (h)   // may lie over x or residual: from here on h is read, by the threads that wrote it until a barrier
            for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) put<DT>(h, c, sum(c));
        auto value = [&](int64_t c) { return h ? at<DT>(h, c) : sum(c); };
        const Stats st = long_stats(p.cols, p.eps, value);
        auto norm = [&](int64_t c) {
            return fmaf(st.centred(value(c)) * st.inv, weight_at<DT>(p.w, p.w32, c), p.b ? weight_at<DT>(p.b, p.w32, c) : 0.0f);
        };
        if (p.out8) {
            uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.so;
            const int lane = threadIdx.x % 64;
            for (int64_t blk = threadIdx.x / 64; blk * F8_BLOCK < p.cols; blk += RN_THREADS / 64) {
                const int64_t c0 = blk * F8_BLOCK + lane, c1 = c0 + 64;
                const float a = c0 < p.cols ? norm(c0) : 0.0f, b = c1 < p.cols ? norm(c1) : 0.0f;
                const F8Scale s(lanes64_all<MaxOp>(fmaxf(fabsf(a), fabsf(b))));
                if (c0 < p.cols) o[c0] = s.divide1(a);
                if (c1 < p.cols) o[c1] = s.divide1(b);
                if (lane == 0) p.scale[row * p.ss[0] + blk * p.ss[1]] = s.s;
            }
        } else {
            T* o = static_cast<T*>(p.out) + row * p.so;
            for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) put<DT>(o, c, norm(c));
        }
    }
}

// Every row's statistics, for the sums over rows. dx comes after those: it may lie over dy or h.
template <int DT>
__global__ __launch_bounds__(RN_THREADS) void layer_norm_stats_kernel(LayerBwdArgs p) {
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const void* h = static_cast<const typename elem<DT>::T*>(p.h) + row * p.sh;
        const Stats st = long_stats(p.cols, p.eps, [&](int64_t c) { return at<DT>(h, c); });
        if (threadIdx.x == 0) {
            p.stats[3 * row] = st.m;
            p.stats[3 * row + 1] = st.e;
            p.stats[3 * row + 2] = st.inv;
        }
    }
}

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void layer_norm_bwd_any_kernel(LayerBwdArgs p) {
    typedef typename elem<DT>::T T;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.sdy;
        const T* h = static_cast<const T*>(p.h) + row * p.sh;
        const T* dh = p.dh ? static_cast<const T*>(p.dh) + row * p.sdh : nullptr;
        const Stats st = long_stats(p.cols, p.eps, [&](int64_t c) { return at<DT>(h, c); });
        float g = 0.0f, gn = 0.0f;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            const float v = at<DT>(dy, c) * weight_at<DT>(p.w, p.w32, c);
            g += v;
            gn += v * (st.centred(at<DT>(h, c)) * st.inv);
        }
        g = block_all<SumOp>(g) / (float)p.cols;
        gn = block_all<SumOp>(gn) / (float)p.cols;
        T* dx = static_cast<T*>(p.dx) + row * p.sdx;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            float v = st.inv * (at<DT>(dy, c) * weight_at<DT>(p.w, p.w32, c) - g - st.centred(at<DT>(h, c)) * st.inv * gn);
            if (dh) v += at<DT>(dh, c);
            put<DT>(dx, c, v);
        }
    }
}

// The sums over rows: a workgroup takes 64 columns and every gridDim.y-th group of 4 rows; partials [2][gridDim.y][cols].
template <int DT>
__global__ __launch_bounds__(RN_THREADS) void layer_norm_sums_kernel(LayerBwdArgs p, float* part, int64_t first) {
    __shared__ float sum[2][4][64];
    typedef typename elem<DT>::T T;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = first + (int64_t)blockIdx.x * 64 + lane;
    float dw = 0.0f, db = 0.0f;
    if (c < p.cols)
        for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < p.rows; row += (int64_t)gridDim.y * 4) {
            const float dy = at<DT>(static_cast<const T*>(p.dy) + row * p.sdy, c);
            const float h = at<DT>(static_cast<const T*>(p.h) + row * p.sh, c);
            const Stats st{p.stats[3 * row], p.stats[3 * row + 1], p.stats[3 * row + 2]};
            dw += dy * (st.centred(h) * st.inv);
            db += dy;
        }
    sum[0][wave][lane] = dw;
    sum[1][wave][lane] = db;
    __syncthreads();
    if (wave < 2 && c < p.cols)
        part[((int64_t)wave * gridDim.y + blockIdx.y) * p.cols + c] =
            sum[wave][0][lane] + sum[wave][1][lane] + sum[wave][2][lane] + sum[wave][3][lane];
}

template <int DT>
void forward(const LayerArgs& p, hipStream_t s) {
    const bool done = row_shape(p.rows, 1024, p.cols * (int64_t)dtype_size(DT) / 16, [&](auto nc, auto tpr) {
        constexpr int NC = decltype(nc)::value, TPR = decltype(tpr)::value, SUBS = row_threads(TPR) / TPR;
        const dim3 grid((unsigned)std::min<int64_t>((p.rows + SUBS - 1) / SUBS, 1 << 20)), block(row_threads(TPR));
        if (p.out8) hipLaunchKernelGGL((layer_norm_kernel<DT, true, NC, TPR>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((layer_norm_kernel<DT, false, NC, TPR>), grid, block, 0, s, p);
    });
    if (!done) hipLaunchKernelGGL((layer_norm_any_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
}

template <int DT>
tvk_status backward(LayerBwdArgs p, void* dw, void* db, hipStream_t s) {
    Scratch scratch;
    float* part = nullptr;
    int64_t parts = 0;
    p.want = (dw ? 1 : 0) | (db ? 2 : 0);
    auto partials = [&](int64_t n, int64_t more) {   // n partials of both sums and `more` floats before them
        parts = n;
        if (!p.want) return true;
        part = static_cast<float*>(scratch.get((size_t)(more + parts * 2 * p.cols) * 4 + 4, s));
        return part != nullptr;
    };
    bool have = true, single = false;
    const bool done = row_shape(p.rows, 256, p.cols * (int64_t)dtype_size(DT) / 16, [&](auto nc, auto tpr) {
        // one chunk a thread where two leave no registers for a second workgroup a CU: bfloat16 8192 x 4096 65 us, with two
        // 80, 4096 x 8192 79 and 103
        constexpr bool TWICE = decltype(nc)::value == 2 && (decltype(tpr)::value == 256 || decltype(tpr)::value == 512);
        constexpr int NC = TWICE ? 1 : decltype(nc)::value, TPR = decltype(tpr)::value * (TWICE ? 2 : 1);
        constexpr int THREADS = bwd_threads(TPR), SUBS = THREADS / TPR;
        const int64_t groups = std::min<int64_t>((p.rows + SUBS - 1) / SUBS, RN_BWD_THREADS / THREADS);
        single = groups == 1;
        if (single) p.dw = dw, p.db = db;
        else have = partials(groups, 0);
        if (have && p.rows > 0)
            hipLaunchKernelGGL((layer_norm_bwd_kernel<DT, NC, TPR, THREADS>), dim3((unsigned)groups), dim3(THREADS), 0, s, p, part);
    });
    if (!done) {   // a workgroup a row, dx last: it may lie over dy or h
        have = partials(std::max<int64_t>(1, std::min<int64_t>(64, p.rows / 64)), 3 * p.rows);
        if (have && p.want) {
            p.stats = part;
            part += 3 * p.rows;
            if (p.rows > 0) hipLaunchKernelGGL((layer_norm_stats_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
            over_columns<64>(p.cols, [&](int64_t first, unsigned groups) {
                hipLaunchKernelGGL((layer_norm_sums_kernel<DT>), dim3(groups, (unsigned)parts), dim3(RN_THREADS), 0, s, p, part, first);
            });
        }
        if (have && p.rows > 0) hipLaunchKernelGGL((layer_norm_bwd_any_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
    }
    if (!have) return fail(TVK_ERR_OOM, "tvk_layer_norm_bwd: workspace allocation failed");
    if (p.want && !single) norm_fold<DT>(part, parts, p.cols, dw, db, p.w32, s);
    return TVK_OK;
}

}  // namespace

extern "C" tvk_status tvk_layer_norm_fwd(const tvk_layer_norm_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_layer_norm_fwd: desc is NULL");
    const tvk_status st = check_norm("tvk_layer_norm_fwd", d->dtype, d->weight_dtype, d->rows, d->cols, d->eps);
    if (st != TVK_OK) return st;
    const bool out8 = d->out_dtype == TVK_F8E4M3FN;
    if (!out8 && d->out_dtype != d->dtype)
        return fail(TVK_ERR_UNSUPPORTED, "tvk_layer_norm_fwd: the output's dtype must be the input's or float8_e4m3fn");
    if (d->rows == 0 || d->cols == 0) return TVK_OK;
    if (!d->x || !d->out || (out8 && !d->scale)) return fail(TVK_ERR_INVALID, "tvk_layer_norm_fwd: NULL tensor");
    if (d->x_stride < 0 || (d->residual && d->residual_stride < 0) || !rows_apart(d->out_stride, d->rows, d->cols) ||
        (d->residual_out && !rows_apart(d->residual_out_stride, d->rows, d->cols)))
        return fail(TVK_ERR_INVALID, "tvk_layer_norm_fwd: negative strides, or output rows that overlap");
    if (out8 && !apart2(d->scale_stride, d->rows, (d->cols + F8_BLOCK - 1) / F8_BLOCK))
        return fail(TVK_ERR_INVALID, "tvk_layer_norm_fwd: scales that overlap");
    LayerArgs p{};
    p.x = d->x;
    p.r = d->residual;
    p.w = d->weight;
    p.b = d->bias;
    p.out = d->out;
    p.h = d->residual_out;
    p.scale = d->scale;
    p.sx = d->x_stride;
    p.sr = d->residual_stride;
    p.so = d->out_stride;
    p.sh = d->residual_out_stride;
    p.ss[0] = d->scale_stride[0];
    p.ss[1] = d->scale_stride[1];
    p.rows = d->rows;
    p.cols = d->cols;
    p.eps = (float)d->eps;
    p.rcols = 1.0f / (float)d->cols;
    p.w32 = d->weight_dtype == TVK_F32;
    p.out8 = out8;
    const hipStream_t s = resolve_stream(d->stream);
    if (d->dtype == TVK_F32) forward<TVK_F32>(p, s);
    else if (d->dtype == TVK_F16) forward<TVK_F16>(p, s);
    else forward<TVK_BF16>(p, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_layer_norm_fwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}

extern "C" tvk_status tvk_layer_norm_bwd(const tvk_layer_norm_bwd_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_layer_norm_bwd: desc is NULL");
    tvk_status st = check_norm("tvk_layer_norm_bwd", d->dtype, d->weight_dtype, d->rows, d->cols, d->eps);
    if (st != TVK_OK) return st;
    if (d->cols == 0 || (d->rows == 0 && !d->dweight && !d->dbias)) return TVK_OK;
    if (d->rows > 0) {
        if (!d->dy || !d->h || !d->dx) return fail(TVK_ERR_INVALID, "tvk_layer_norm_bwd: NULL tensor");
        if (d->dy_stride < 0 || d->h_stride < 0 || (d->dh && d->dh_stride < 0) || !rows_apart(d->dx_stride, d->rows, d->cols))
            return fail(TVK_ERR_INVALID, "tvk_layer_norm_bwd: negative strides, or output rows that overlap");
    }
    LayerBwdArgs p{};
    p.dy = d->dy;
    p.h = d->h;
    p.dh = d->dh;
    p.w = d->weight;
    p.dx = d->dx;
    p.sdy = d->dy_stride;
    p.sh = d->h_stride;
    p.sdh = d->dh_stride;
    p.sdx = d->dx_stride;
    p.rows = d->rows;
    p.cols = d->cols;
    p.eps = (float)d->eps;
    p.rcols = 1.0f / (float)d->cols;
    p.w32 = d->weight_dtype == TVK_F32;
    const hipStream_t s = resolve_stream(d->stream);
    if (d->dtype == TVK_F32) st = backward<TVK_F32>(p, d->dweight, d->dbias, s);
    else if (d->dtype == TVK_F16) st = backward<TVK_F16>(p, d->dweight, d->dbias, s);
    else st = backward<TVK_BF16>(p, d->dweight, d->dbias, s);
    if (st != TVK_OK) return st;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_layer_norm_bwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}
