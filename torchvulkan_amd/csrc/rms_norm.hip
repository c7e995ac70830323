// Root-mean-square norm (tvk_rms_norm_fwd, tvk_rms_norm_bwd).
//
// Both directions read and write each value once and are bound by that. A row
// is held in the registers of TPR threads (part of a wave, a wave, or a workgroup
// of 256 to 1024), one or two chunks of 16 bytes each, while its sums are taken: one
// pass forward, for the 8-bit output too (max|h w| and the sum of squares come
// from the same pass, and scale both), one pass backward for both sums and dx.
// Backward, a workgroup takes rows in turn and keeps dweight's sums over them in
// registers; those are added up by a second launch in a fixed order, or stored as they
// are where one workgroup takes all rows. Rows start at any multiple of a value (16-byte
// accesses need no more); the values past a row's last whole chunk go one to a thread.
// Rows of more than 2048 chunks are read again for every pass.
//
// Measured (a 2 GiB copy moves 4.9 TB/s): residual, norm and 8 bits of 16384 x 4096 in
// bfloat16 81 us, 5.8 TB/s; its gradients at 16384 x 2048 56 us, 4.8 TB/s, 5 of them
// the second launch; 7 x 4096 3.9 us and gradients of 1000 x 777 8.1 us, the launches.
#include "words.h"

#include <algorithm>

using namespace tvk;

namespace {

constexpr int RN_THREADS = 256;
constexpr float kF8Max = 448.0f;

struct NormArgs {
    const void* x;
    const void* r;
    const void* w;
    void* out;
    void* h;
    float* scale;
    int64_t sx, sr, so, sh;   // row strides, elements
    int64_t rows, cols;
    float eps, rcols;
    int w32, out8;
};

struct NormBwdArgs {
    const void* dy;
    const void* h;
    const void* dh;
    const void* w;
    void* dx;
    void* dw;      // of a single workgroup, which needs no partials; or NULL
    float* inv;    // [rows], or NULL
    int64_t sdy, sh, sdh, sdx;
    int64_t rows, cols;
    float eps, rcols;
    int w32;
};

template <int DT>
__device__ inline float at(const void* p, int64_t i) {
    return elem<DT>::to_f32(static_cast<const typename elem<DT>::T*>(p)[i]);
}
template <int DT>
__device__ inline void put(void* p, int64_t i, float v) {
    static_cast<typename elem<DT>::T*>(p)[i] = elem<DT>::from_f32(v);
}
template <int DT>
__device__ inline float weight_at(const void* w, int w32, int64_t i) {
    return !w ? 1.0f : w32 ? static_cast<const float*>(w)[i] : at<DT>(w, i);
}

struct SumOp { __device__ static float of(float a, float b) { return a + b; } };
struct MaxOp { __device__ static float of(float a, float b) { return fmaxf(a, b); } };

// Every thread gets the workgroup's result, combined in one fixed order.
template <class Op>
__device__ inline float block_all(float v) {
    __shared__ float part[RN_THREADS / 64];
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v = Op::of(v, __shfl_xor(v, m));
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int w = 1; w < RN_THREADS / 64; ++w) v = Op::of(v, part[w]);
    return v;
}

// Workgroups that take rows in turn, 2^32 threads in a dimension of a grid being too many.
dim3 rows_grid(int64_t rows) { return dim3((unsigned)std::min<int64_t>(rows, 1 << 16)); }

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_any_kernel(NormArgs p) {
    typedef typename elem<DT>::T T;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.sx;
        const T* r = p.r ? static_cast<const T*>(p.r) + row * p.sr : nullptr;
        T* h = p.h ? static_cast<T*>(p.h) + row * p.sh : nullptr;
        auto value = [&](int64_t c) {
            float v = at<DT>(x, c);
            if (r) v = elem<DT>::to_f32(elem<DT>::from_f32(v + at<DT>(r, c)));
            return v;
        };
        float ss = 0.0f;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            const float v = value(c);
            ss += v * v;
            if (h) put<DT>(h, c, v);
        }
        const float inv = 1.0f / sqrtf(block_all<SumOp>(ss) / (float)p.cols + p.eps);
        // residual_out may lie over x or residual: from here on h is read back
        auto norm = [&](int64_t c) { return (h ? at<DT>(h, c) : value(c)) * inv * weight_at<DT>(p.w, p.w32, c); };
        if (p.out8) {
            float top = 0.0f;
            for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) top = fmaxf(top, fabsf(norm(c)));
            top = block_all<MaxOp>(top);
            const float s = top > 0.0f ? top / kF8Max : 1.0f;
            if (threadIdx.x == 0) p.scale[row] = s;
            uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.so;
            for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) o[c] = f32_to_f8(norm(c) / s, TVK_F8E4M3FN);
        } else {
            T* o = static_cast<T*>(p.out) + row * p.so;
            for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) put<DT>(o, c, norm(c));
        }
    }
}

// 1 / sqrt(mean(h^2) + eps) of every row, for dweight's sums. dx comes after those: it may lie over dy or h.
template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_inv_kernel(NormBwdArgs p) {
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const void* h = static_cast<const typename elem<DT>::T*>(p.h) + row * p.sh;
        float ss = 0.0f;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            const float v = at<DT>(h, c);
            ss += v * v;
        }
        ss = block_all<SumOp>(ss);
        if (threadIdx.x == 0) p.inv[row] = 1.0f / sqrtf(ss / (float)p.cols + p.eps);
    }
}

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_bwd_any_kernel(NormBwdArgs p) {
    typedef typename elem<DT>::T T;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* dy = static_cast<const T*>(p.dy) + row * p.sdy;
        const T* h = static_cast<const T*>(p.h) + row * p.sh;
        const T* dh = p.dh ? static_cast<const T*>(p.dh) + row * p.sdh : nullptr;
        float ss = 0.0f, gh = 0.0f;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            const float v = at<DT>(h, c);
            ss += v * v;
            gh += at<DT>(dy, c) * weight_at<DT>(p.w, p.w32, c) * v;
        }
        ss = block_all<SumOp>(ss);
        gh = block_all<SumOp>(gh);
        const float inv = 1.0f / sqrtf(ss / (float)p.cols + p.eps);
        const float mean = gh * inv / (float)p.cols;   // of g * n
        T* dx = static_cast<T*>(p.dx) + row * p.sdx;
        for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
            const float g = at<DT>(dy, c) * weight_at<DT>(p.w, p.w32, c);
            float v = inv * (g - at<DT>(h, c) * inv * mean);
            if (dh) v += at<DT>(dh, c);
            put<DT>(dx, c, v);
        }
    }
}

// dweight's sums: a workgroup takes 64 columns and every gridDim.y-th group of 4 rows; partials [gridDim.y][cols].
template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_dweight_kernel(NormBwdArgs p, float* part) {
    __shared__ float sum[4][64];
    typedef typename elem<DT>::T T;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < p.cols)
        for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < p.rows; row += (int64_t)gridDim.y * 4)
            s += at<DT>(static_cast<const T*>(p.dy) + row * p.sdy, c) * at<DT>(static_cast<const T*>(p.h) + row * p.sh, c) *
                 p.inv[row];
    sum[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.cols) part[blockIdx.y * p.cols + c] = sum[0][lane] + sum[1][lane] + sum[2][lane] + sum[3][lane];
}

// ---------------------------------------------------------------------------
// rows in registers
// ---------------------------------------------------------------------------

template <int CTRL>
__device__ __forceinline__ float moved(float v) {   // a lane's value from another lane of its 16
    const int i = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(i, i, CTRL, 0xf, 0xf, false));
}

// Over 16 lanes, then 64: every lane ends with the same bits. Moves between lanes are DPP and lane swaps, a fifth of the
// latency of the shuffles through LDS.
template <class Op>
__device__ __forceinline__ float lanes16_all(float v) {
    v = Op::of(v, moved<0xB1>(v));    // lane ^ 1
    v = Op::of(v, moved<0x4E>(v));    // lane ^ 2
    v = Op::of(v, moved<0x141>(v));   // mirrored in 8
    return Op::of(v, moved<0x140>(v));   // mirrored in 16
}
template <class Op>
__device__ __forceinline__ float lanes64_all(float v) {
    v = lanes16_all<Op>(v);
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = Op::of(__builtin_bit_cast(float, (uint32_t)a[0]), __builtin_bit_cast(float, (uint32_t)a[1]));
    u = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return Op::of(__builtin_bit_cast(float, (uint32_t)b[0]), __builtin_bit_cast(float, (uint32_t)b[1]));
}

// A row's two sums (or a sum and a maximum) over its TPR threads, the same bits in each: lanes, then the waves in order.
// `turn` alternates from row to row: with two sets of LDS words one barrier a row is enough.
template <int TPR, class OpA, class OpB>
__device__ __forceinline__ void row_all(float& a, float& b, int turn) {
    if constexpr (TPR == 16) {
        a = lanes16_all<OpA>(a);
        b = lanes16_all<OpB>(b);
    } else {
        a = lanes64_all<OpA>(a);
        b = lanes64_all<OpB>(b);
    }
    if constexpr (TPR > 64) {
        __shared__ float part[2][2][1024 / 64];
        const int wave = threadIdx.x / 64, w0 = threadIdx.x / TPR * (TPR / 64);
        if (threadIdx.x % 64 == 0) {
            part[turn][0][wave] = a;
            part[turn][1][wave] = b;
        }
        __syncthreads();
        a = part[turn][0][w0];
        b = part[turn][1][w0];
#pragma unroll
        for (int w = 1; w < TPR / 64; ++w) {
            a = OpA::of(a, part[turn][0][w0 + w]);
            b = OpB::of(b, part[turn][1][w0 + w]);
        }
    }
}

// A thread's row among its workgroup's: the wave's where a row takes whole waves, so that addresses are scalar.
template <int TPR>
__device__ __forceinline__ int row_of_thread() {
    return TPR < 64 ? threadIdx.x / TPR : __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
}

// 1 / sqrt(ss / cols + eps), rcols being 1 / cols: the reciprocal square root instruction is within a step of float32 where
// its argument is not near float32's ends.
__device__ __forceinline__ float inv_rms(float ss, float rcols, float eps) {
    const float x = fmaf(ss, rcols, eps);
    return x > 1e-30f && x < 1e30f ? __builtin_amdgcn_rsqf(x) : 1.0f / sqrtf(x);
}

constexpr int row_threads(int tpr) { return tpr < RN_THREADS ? RN_THREADS : tpr; }

// What a thread holds of a row: chunk i is the row's chunk t + TPR * i; then, in t < tail, one of the values past them.
template <int DT, int NC, int TPR>
struct Row {
    typedef typename elem<DT>::T T;
    static constexpr int VEC = 16 / (int)sizeof(T);
    Words<16> c[NC];
    float last = 0.0f;

    __device__ __forceinline__ void load(const void* row, int t, int chunks, int tail) {
        const T* p = static_cast<const T*>(row);
#pragma unroll
        for (int i = 0; i < NC; ++i) c[i] = t + TPR * i < chunks ? load_words<16, sizeof(T)>(p + (uint32_t)(VEC * (t + TPR * i))) : Words<16>{};
        if (t < tail) last = elem<DT>::to_f32(p[(uint32_t)(VEC * chunks + t)]);
    }
    __device__ __forceinline__ float at(int i, int k) const { return word_at<DT>(c[i], k); }
    // From here on the values are unpacked anew: kept unpacked across a row's sums they take twice the registers.
    __device__ __forceinline__ void packed() {
        if constexpr (DT != TVK_F32)
#pragma unroll
            for (int i = 0; i < NC; ++i) asm volatile("" : "+v"(c[i].w[0]), "+v"(c[i].w[1]), "+v"(c[i].w[2]), "+v"(c[i].w[3]));
    }
};

// A row's weights: the row's type in registers, or float32 ones beside a 16-bit row read as they are needed.
template <int DT, int NC, int TPR>
struct Weights {
    typedef Row<DT, NC, TPR> R;
    R r;
    const float* w32 = nullptr;

    __device__ __forceinline__ void load(const void* w, int is32, int t, int chunks, int tail) {
        if (!w || (is32 && DT != TVK_F32)) {
            float ones[R::VEC];
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) ones[k] = 1.0f;
#pragma unroll
            for (int i = 0; i < NC; ++i) r.c[i] = pack<DT, R::VEC>(ones);
            r.last = 1.0f;
            w32 = static_cast<const float*>(w);
            if (w32 && t < tail) r.last = w32[R::VEC * chunks + t];
        } else {
            r.load(w, t, chunks, tail);
        }
    }
    __device__ __forceinline__ void chunk(int i, int t, int chunks, float (&f)[R::VEC]) const {
        if (DT != TVK_F32 && w32) {
#pragma unroll
            for (int k = 0; k < R::VEC; k += 4) {
                const Words<16> v = t + TPR * i < chunks ? load_words<16, 4>(w32 + R::VEC * (t + TPR * i) + k) : Words<16>{};
#pragma unroll
                for (int j = 0; j < 4; ++j) f[k + j] = __builtin_bit_cast(float, v.w[j]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) f[k] = r.at(i, k);
        }
    }
};

template <int DT, bool OUT8, int NC, int TPR>
__global__ __launch_bounds__(row_threads(TPR)) void rms_norm_kernel(NormArgs p) {
    typedef Row<DT, NC, TPR> R;
    typedef typename R::T T;
    constexpr int VEC = R::VEC, SUBS = row_threads(TPR) / TPR;
    const int t = threadIdx.x % TPR, chunks = (int)p.cols / VEC, tail = (int)p.cols % VEC;
    Weights<DT, NC, TPR> w;
    w.load(p.w, p.w32, t, chunks, tail);
    int turn = 0;
    for (int64_t row = (int64_t)blockIdx.x * SUBS + row_of_thread<TPR>(); row < p.rows; row += (int64_t)gridDim.x * SUBS) {
        R h, r;
        h.load(static_cast<const T*>(p.x) + row * p.sx, t, chunks, tail);
        if (p.r) {
            r.load(static_cast<const T*>(p.r) + row * p.sr, t, chunks, tail);
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                float s[VEC];
#pragma unroll
                for (int k = 0; k < VEC; ++k) s[k] = h.at(i, k) + r.at(i, k);
                h.c[i] = pack<DT, VEC>(s);
            }
            h.last = elem<DT>::to_f32(elem<DT>::from_f32(h.last + r.last));
        }
        // v: the row's values, for the 8-bit output times the weights
        float ss = h.last * h.last, last = OUT8 ? h.last * w.r.last : h.last, top = fabsf(last), v[NC][VEC];
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], part = 0.0f;
            if (OUT8) w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                v[i][k] = h.at(i, k);
                part = fmaf(v[i][k], v[i][k], part);
                if (OUT8) {
                    v[i][k] *= f[k];
                    top = fmaxf(top, fabsf(v[i][k]));
                }
            }
            ss += part;
        }
        if (OUT8) row_all<TPR, SumOp, MaxOp>(ss, top, turn);
        else row_all<TPR, SumOp, SumOp>(ss, top, turn);
        turn ^= 1;
        const float inv = inv_rms(ss, p.rcols, p.eps);
        if (p.h) {
            T* o = static_cast<T*>(p.h) + row * p.sh;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (t + TPR * i < chunks) store_words<16, sizeof(T)>(o + (uint32_t)(VEC * (t + TPR * i)), h.c[i]);
            if (t < tail) o[VEC * chunks + t] = elem<DT>::from_f32(h.last);
        }
        if constexpr (OUT8) {
            // y = h w inv; its largest magnitude is max|h w| times inv, and y / scale = h w (inv / scale). An inv / scale
            // that leaves float32's range, for rows of values near its ends, is not taken as one factor.
            top *= inv;
            const float s = top > 0.0f ? top / kF8Max : 1.0f, f8 = inv * __builtin_amdgcn_rcpf(s);
            const bool plain = f8 < 1e30f && f8 > 1e-30f;
            const float a = plain ? f8 : inv, b = plain ? 1.0f : s;
            if (t == 0) p.scale[row] = s;
            uint8_t* o = static_cast<uint8_t*>(p.out) + row * p.so;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (t + TPR * i >= chunks) continue;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[i][k] *= a;
                if (!plain)
#pragma unroll
                    for (int k = 0; k < VEC; ++k) v[i][k] /= b;
                Words<VEC> e;
#pragma unroll
                for (int k = 0; k < VEC; k += 4) e.w[k / 4] = pack4_f8(v[i][k], v[i][k + 1], v[i][k + 2], v[i][k + 3]);
                store_words<VEC, 1>(o + (uint32_t)(VEC * (t + TPR * i)), e);
            }
            if (t < tail) o[VEC * chunks + t] = f32_to_f8(last * a / b, TVK_F8E4M3FN);
        } else {
            T* o = static_cast<T*>(p.out) + row * p.so;
#pragma unroll
            for (int i = 0; i < NC; ++i) {
                if (t + TPR * i >= chunks) continue;
                float f[VEC];
                w.chunk(i, t, chunks, f);
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[i][k] = v[i][k] * inv * f[k];
                store_words<16, sizeof(T)>(o + (uint32_t)(VEC * (t + TPR * i)), pack<DT, VEC>(v[i]));
            }
            if (t < tail) o[VEC * chunks + t] = elem<DT>::from_f32(last * inv * w.r.last);
        }
    }
}

// Backward, a workgroup keeps dweight's sums over all of its rows: as many workgroups as are resident together (16 waves a
// CU). Forward takes a row each: loading the next row's weights again costs less than waiting for it (bfloat16
// 16384 x 4096 to 8 bits: 82 us, 90 with 1024 workgroups that keep their weights).
constexpr int64_t RN_BWD_THREADS = 1024 * 256;

// Threads of a backward workgroup: two rows of 256 threads at a time halve the partials that are folded
// (bfloat16 16384 x 4096: 105.7 us, 110.7 with one row), four make the waves wait for each other.
constexpr int bwd_threads(int tpr) { return tpr < 512 ? 512 : tpr; }

// part: [gridDim.x][cols], the workgroups' sums of dy * n over their rows; NULL: not wanted.
template <int DT, int NC, int TPR, int THREADS>
__global__ __launch_bounds__(THREADS) void rms_norm_bwd_kernel(NormBwdArgs p, float* part) {
    typedef Row<DT, NC, TPR> R;
    typedef typename R::T T;
    constexpr int VEC = R::VEC, SUBS = THREADS / TPR;
    const int t = threadIdx.x % TPR, sub = row_of_thread<TPR>(), chunks = (int)p.cols / VEC, tail = (int)p.cols % VEC;
    Weights<DT, NC, TPR> w;
    w.load(p.w, p.w32, t, chunks, tail);
    float acc[NC][VEC], acc_last = 0.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) acc[i][k] = 0.0f;
    int64_t row = (int64_t)blockIdx.x * SUBS + sub;
    const int64_t step = (int64_t)gridDim.x * SUBS;
    int turn = 0;
    R dy, h, dh;   // of the next row, on their way while one is computed
    auto load = [&]() {
        dy.load(static_cast<const T*>(p.dy) + row * p.sdy, t, chunks, tail);
        h.load(static_cast<const T*>(p.h) + row * p.sh, t, chunks, tail);
        if (p.dh) dh.load(static_cast<const T*>(p.dh) + row * p.sdh, t, chunks, tail);
    };
    if (row < p.rows) load();
    // a workgroup's rows keep step: their sums meet at barriers
    for (int64_t first = (int64_t)blockIdx.x * SUBS; first < p.rows; first += step) {
        R g = dy, x = h, add = dh;
        const bool live = row < p.rows;
        T* dx = static_cast<T*>(p.dx) + row * p.sdx;
        row += step;
        if (row < p.rows) load();
        float ss = x.last * x.last, gh = g.last * w.r.last * x.last;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], ps = 0.0f, pg = 0.0f;
            w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float v = x.at(i, k);
                ps = fmaf(v, v, ps);
                pg = fmaf(g.at(i, k) * f[k], v, pg);
            }
            ss += ps;
            gh += pg;
        }
        row_all<TPR, SumOp, SumOp>(ss, gh, turn);
        turn ^= 1;
        if (!live) continue;
        g.packed();
        x.packed();
        add.packed();
        w.r.packed();
        const float inv = inv_rms(ss, p.rcols, p.eps);
        const float mean = gh * inv * p.rcols;   // of g * n
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            float f[VEC], o[VEC];
            w.chunk(i, t, chunks, f);
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                const float n = x.at(i, k) * inv, d = g.at(i, k);
                acc[i][k] = fmaf(d, n, acc[i][k]);
                o[k] = inv * (d * f[k] - n * mean);
                if (p.dh) o[k] += add.at(i, k);
            }
            if (t + TPR * i < chunks) store_words<16, sizeof(T)>(dx + (uint32_t)(VEC * (t + TPR * i)), pack<DT, VEC>(o));
        }
        if (t < tail) {
            const float n = x.last * inv;
            acc_last = fmaf(g.last, n, acc_last);
            float o = inv * (g.last * w.r.last - n * mean);
            if (p.dh) o += add.last;
            dx[VEC * chunks + t] = elem<DT>::from_f32(o);
        }
    }
    if (!part && !p.dw) return;
    float* out = part + (int64_t)blockIdx.x * p.cols;
    // chunks of floats, to a partial or LDS; a single workgroup's sums to dweight itself
    auto put_sum = [&](int c, float v) {
        if (!p.dw) out[c] = v;
        else if (p.w32) static_cast<float*>(p.dw)[c] = v;
        else put<DT>(p.dw, c, v);
    };
    auto put_chunks = [&](float* to) {
#pragma unroll
        for (int i = 0; i < NC; ++i)
            if (t + TPR * i < chunks)
#pragma unroll
                for (int k = 0; k < VEC; k += 4) {
                    const float four[4] = {acc[i][k], acc[i][k + 1], acc[i][k + 2], acc[i][k + 3]};
                    store_words<16, 4>(to + (uint32_t)(VEC * (t + TPR * i) + k), pack<TVK_F32, 4>(four));
                }
        if (t < tail) to[VEC * chunks + t] = acc_last;
    };
    if (SUBS == 1 && !p.dw) {
        put_chunks(out);
        return;
    }
    __shared__ __attribute__((aligned(16))) float sum[SUBS][VEC * (NC * TPR + 1)];
    put_chunks(sum[sub]);
    __syncthreads();
    for (int c = threadIdx.x; c < (int)p.cols; c += THREADS) {
        float v = sum[0][c];
#pragma unroll
        for (int i = 1; i < SUBS; ++i) v += sum[i][c];
        put_sum(c, v);
    }
}

// Adds the partials up: a workgroup FOLD_COLS columns, its threads every FOLD_ROWS-th partial, then those in order.
constexpr int FOLD_COLS = 16, FOLD_ROWS = 64;

template <int DT>
__global__ __launch_bounds__(FOLD_COLS * FOLD_ROWS) void rms_norm_fold_kernel(const float* part, int64_t parts, int64_t cols,
                                                                              void* dw, int w32) {
    __shared__ float sum[FOLD_ROWS][FOLD_COLS + 1];
    const int x = threadIdx.x % FOLD_COLS, y = threadIdx.x / FOLD_COLS;
    const int64_t c = (int64_t)blockIdx.x * FOLD_COLS + x;
    float s = 0.0f;
    if (c < cols) {
        for (int64_t i = y; i < parts; i += 8 * FOLD_ROWS) {   // eight loads on their way together
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = part[min(i + u * FOLD_ROWS, parts - 1) * cols + c];
#pragma unroll
            for (int u = 0; u < 8; ++u) s += i + u * FOLD_ROWS < parts ? v[u] : 0.0f;
        }
    }
    sum[y][x] = s;
#pragma unroll
    for (int m = FOLD_ROWS / 2; m > 0; m >>= 1) {
        __syncthreads();
        if (y < m) sum[y][x] += sum[y + m][x];
    }
    if (y != 0 || c >= cols) return;
    if (w32) static_cast<float*>(dw)[c] = sum[0][x];
    else put<DT>(dw, c, sum[0][x]);
}

// Calls f(NC, TPR) for rows of `chunks` whole chunks; false past what registers hold. At most two chunks a thread: more
// take the registers of the waves that hide the row's latency (bfloat16 16384 x 4096 to 8 bits: 82 us with two chunks in
// 256 threads, 197 with eight in a wave). A wave with two chunks beats four waves with half of one each where rows are many
// (float16 2000 x 1024: 4.5 us, 5.4), and loses where they are few; backward, where it halves the partials too, from fewer rows
// on (1000 x 777: 8.5 us, 9.1).
template <class F>
bool row_shape(int64_t rows, int64_t few, int64_t chunks, F&& f) {
#define TVK_ROW(nc, tpr) return f(std::integral_constant<int, nc>{}, std::integral_constant<int, tpr>{}), true
    if (chunks <= 16) TVK_ROW(1, 16);
    if (chunks <= 32) TVK_ROW(2, 16);
    if (chunks <= 64) TVK_ROW(1, 64);
    if (chunks <= 128 && rows > few) TVK_ROW(2, 64);
    if (chunks <= 256) TVK_ROW(1, 256);
    if (chunks <= 512) TVK_ROW(2, 256);
    if (chunks <= 1024) TVK_ROW(2, 512);
    if (chunks <= 2048) TVK_ROW(2, 1024);
#undef TVK_ROW
    return false;
}

template <int DT>
void forward(const NormArgs& p, hipStream_t s) {
    const bool done = row_shape(p.rows, 1024, p.cols * (int64_t)dtype_size(DT) / 16, [&](auto nc, auto tpr) {
        constexpr int NC = decltype(nc)::value, TPR = decltype(tpr)::value, SUBS = row_threads(TPR) / TPR;
        const dim3 grid((unsigned)std::min<int64_t>((p.rows + SUBS - 1) / SUBS, 1 << 20)), block(row_threads(TPR));
        if (p.out8) hipLaunchKernelGGL((rms_norm_kernel<DT, true, NC, TPR>), grid, block, 0, s, p);
        else hipLaunchKernelGGL((rms_norm_kernel<DT, false, NC, TPR>), grid, block, 0, s, p);
    });
    if (!done) hipLaunchKernelGGL((rms_norm_any_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
}

template <int DT>
tvk_status backward(NormBwdArgs p, void* dw, hipStream_t s) {
    Scratch scratch;
    float* part = nullptr;
    int64_t parts = 0;
    auto partials = [&](int64_t n, int64_t more) {   // n partials and `more` floats before them
        parts = n;
        if (!dw) return true;
        part = static_cast<float*>(scratch.get((size_t)(more + parts * p.cols) * 4 + 4, s));
        return part != nullptr;
    };
    bool have = true;
    const bool done = row_shape(p.rows, 256, p.cols * (int64_t)dtype_size(DT) / 16, [&](auto nc, auto tpr) {
        constexpr int NC = decltype(nc)::value, TPR = decltype(tpr)::value, THREADS = bwd_threads(TPR), SUBS = THREADS / TPR;
        const int64_t groups = std::min<int64_t>((p.rows + SUBS - 1) / SUBS, RN_BWD_THREADS / THREADS);
        if (dw && groups == 1) p.dw = dw;
        else have = partials(groups, 0);
        if (have && p.rows > 0)
            hipLaunchKernelGGL((rms_norm_bwd_kernel<DT, NC, TPR, THREADS>), dim3((unsigned)groups), dim3(THREADS), 0, s, p, part);
    });
    if (!done) {   // a workgroup a row, dx last: it may lie over dy or h
        have = partials(std::max<int64_t>(1, std::min<int64_t>(64, p.rows / 64)), p.rows);
        if (have && dw) {
            p.inv = part;
            part += p.rows;
            if (p.rows > 0) hipLaunchKernelGGL((rms_norm_inv_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
            hipLaunchKernelGGL((rms_norm_dweight_kernel<DT>), dim3((unsigned)((p.cols + 63) / 64), (unsigned)parts),
                               dim3(RN_THREADS), 0, s, p, part);
        }
        if (have && p.rows > 0) hipLaunchKernelGGL((rms_norm_bwd_any_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
    }
    if (!have) return fail(TVK_ERR_OOM, "tvk_rms_norm_bwd: workspace allocation failed");
    if (dw && !p.dw)
        hipLaunchKernelGGL((rms_norm_fold_kernel<DT>), dim3((unsigned)((p.cols + FOLD_COLS - 1) / FOLD_COLS)),
                           dim3(FOLD_COLS * FOLD_ROWS), 0, s, part, parts, p.cols, dw, p.w32);
    return TVK_OK;
}

bool norm_dtype(int32_t dt) { return dt == TVK_F32 || dt == TVK_F16 || dt == TVK_BF16; }

// What both directions ask of their sizes and types.
tvk_status check_norm(const char* who, int32_t dtype, int32_t weight_dtype, int64_t rows, int64_t cols, double eps) {
    auto bad = [&](tvk_status st, const char* m) { return fail(st, std::string(who) + ": " + m); };
    if (!norm_dtype(dtype)) return bad(TVK_ERR_UNSUPPORTED, "dtype must be float32, float16 or bfloat16");
    if (weight_dtype != dtype && weight_dtype != TVK_F32)
        return bad(TVK_ERR_UNSUPPORTED, "the weight's dtype must be the input's or float32");
    if (rows < 0 || cols < 0) return bad(TVK_ERR_INVALID, "negative size");
    if (!(eps >= 0.0)) return bad(TVK_ERR_INVALID, "eps must not be negative");
    if (rows > 0x7fffffff || cols > 0x7fffffff) return bad(TVK_ERR_UNSUPPORTED, "rows and columns up to 2^31 - 1 only");
    return TVK_OK;
}

// Rows that are written must not lie over each other.
bool rows_apart(int64_t stride, int64_t rows, int64_t cols) { return rows <= 1 || stride >= cols; }

}  // namespace

extern "C" tvk_status tvk_rms_norm_fwd(const tvk_rms_norm_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_rms_norm_fwd: desc is NULL");
    tvk_status st = check_norm("tvk_rms_norm_fwd", d->dtype, d->weight_dtype, d->rows, d->cols, d->eps);
    if (st != TVK_OK) return st;
    const bool out8 = d->out_dtype == TVK_F8E4M3FN;
    if (!out8 && d->out_dtype != d->dtype)
        return fail(TVK_ERR_UNSUPPORTED, "tvk_rms_norm_fwd: the output's dtype must be the input's or float8_e4m3fn");
    if (d->rows == 0 || (d->cols == 0 && !out8)) return TVK_OK;   // rows without values have a scale all the same
    if ((d->cols > 0 && (!d->x || !d->out)) || (out8 && !d->scale)) return fail(TVK_ERR_INVALID, "tvk_rms_norm_fwd: NULL tensor");
    if (d->x_stride < 0 || (d->residual && d->residual_stride < 0) || !rows_apart(d->out_stride, d->rows, d->cols) ||
        (d->residual_out && !rows_apart(d->residual_out_stride, d->rows, d->cols)))
        return fail(TVK_ERR_INVALID, "tvk_rms_norm_fwd: negative strides, or output rows that overlap");
    NormArgs p{};
    p.x = d->x;
    p.r = d->residual;
    p.w = d->weight;
    p.out = d->out;
    p.h = d->residual_out;
    p.scale = d->scale;
    p.sx = d->x_stride;
    p.sr = d->residual_stride;
    p.so = d->out_stride;
    p.sh = d->residual_out_stride;
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
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_rms_norm_fwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}

extern "C" tvk_status tvk_rms_norm_bwd(const tvk_rms_norm_bwd_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_rms_norm_bwd: desc is NULL");
    tvk_status st = check_norm("tvk_rms_norm_bwd", d->dtype, d->weight_dtype, d->rows, d->cols, d->eps);
    if (st != TVK_OK) return st;
    if (d->cols == 0 || (d->rows == 0 && !d->dweight)) return TVK_OK;
    if (d->rows > 0) {
        if (!d->dy || !d->h || !d->dx) return fail(TVK_ERR_INVALID, "tvk_rms_norm_bwd: NULL tensor");
        if (d->dy_stride < 0 || d->h_stride < 0 || (d->dh && d->dh_stride < 0) || !rows_apart(d->dx_stride, d->rows, d->cols))
            return fail(TVK_ERR_INVALID, "tvk_rms_norm_bwd: negative strides, or output rows that overlap");
    }
    NormBwdArgs p{};
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
    if (d->dtype == TVK_F32) st = backward<TVK_F32>(p, d->dweight, s);
    else if (d->dtype == TVK_F16) st = backward<TVK_F16>(p, d->dweight, s);
    else st = backward<TVK_BF16>(p, d->dweight, s);
    if (st != TVK_OK) return st;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_rms_norm_bwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}
