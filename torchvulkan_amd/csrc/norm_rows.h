// Rows of a norm in registers: what tvk_rms_norm_* (rms_norm.hip) and
// tvk_layer_norm_* (layer_norm.hip) share. A row is held by TPR threads (part of
// a wave, a wave, or a workgroup of 256 to 1024), one or two chunks of 16 bytes
// each, while its sums are taken; rows start at any multiple of a value (16-byte
// accesses need no more), and the values past a row's last whole chunk go one to
// a thread.
#pragma once

#include "words.h"

#include <algorithm>
#include <type_traits>

namespace tvk {
namespace {

constexpr int RN_THREADS = 256;
constexpr float kF8Max = 448.0f;

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

    __device__ __forceinline__ void load(const void* row, int t, int chunks, int tail) { load(row, t, chunks, tail, t); }
    // tt: t, or where the values past the last chunk are wanted in other threads, the place among them
    __device__ __forceinline__ void load(const void* row, int t, int chunks, int tail, int tt) {
        const T* p = static_cast<const T*>(row);
#pragma unroll
        for (int i = 0; i < NC; ++i) c[i] = t + TPR * i < chunks ? load_words<16, sizeof(T)>(p + (uint32_t)(VEC * (t + TPR * i))) : Words<16>{};
        if (tt < tail) last = elem<DT>::to_f32(p[(uint32_t)(VEC * chunks + tt)]);
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
        load(w, is32, t, chunks, tail, t, 1.0f);
    }
    // absent: the value of every weight where there are none
    __device__ __forceinline__ void load(const void* w, int is32, int t, int chunks, int tail, int tt, float absent) {
        if (!w || (is32 && DT != TVK_F32)) {
            float ones[R::VEC];
#pragma unroll
            for (int k = 0; k < R::VEC; ++k) ones[k] = absent;
#pragma unroll
            for (int i = 0; i < NC; ++i) r.c[i] = pack<DT, R::VEC>(ones);
            r.last = absent;
            w32 = static_cast<const float*>(w);
            if (w32 && tt < tail) r.last = w32[R::VEC * chunks + tt];
        } else {
            r.load(w, t, chunks, tail, tt);
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

// Backward, a workgroup keeps dweight's sums over all of its rows: as many workgroups as are resident together (16 waves a
// CU). Forward takes a row each: loading the next row's weights again costs less than waiting for it (bfloat16
// 16384 x 4096 to 8 bits: 82 us, 90 with 1024 workgroups that keep their weights).
constexpr int64_t RN_BWD_THREADS = 1024 * 256;

// Threads of a backward workgroup: two rows of 256 threads at a time halve the partials that are folded
// (bfloat16 16384 x 4096: 105.7 us, 110.7 with one row), four make the waves wait for each other.
constexpr int bwd_threads(int tpr) { return tpr < 512 ? 512 : tpr; }

// Adds the partials up: a workgroup FOLD_COLS columns, its threads every FOLD_ROWS-th partial, then those in order. A second
// row of workgroups does the same for the partials behind those, to db. first: of a launch's columns.
constexpr int FOLD_COLS = 16, FOLD_ROWS = 64;

// Calls launch(first column, workgroups) for all columns, WIDTH to a workgroup: 2^32 threads in a dimension of a grid are too many.
template <int WIDTH, class F>
void over_columns(int64_t cols, F&& launch) {
    constexpr int64_t MOST = 1 << 20;
    for (int64_t first = 0; first < cols; first += MOST * WIDTH)
        launch(first, (unsigned)std::min<int64_t>(MOST, (cols - first + WIDTH - 1) / WIDTH));
}

template <int DT>
__global__ __launch_bounds__(FOLD_COLS * FOLD_ROWS) void norm_fold_kernel(const float* part, int64_t parts, int64_t cols,
                                                                         int64_t first, void* dw, void* db, int w32) {
    part += blockIdx.y * parts * cols;
    void* out = blockIdx.y ? db : dw;
    if (!out) return;
    __shared__ float sum[FOLD_ROWS][FOLD_COLS + 1];
    const int x = threadIdx.x % FOLD_COLS, y = threadIdx.x / FOLD_COLS;
    const int64_t c = first + (int64_t)blockIdx.x * FOLD_COLS + x;
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
    if (w32) static_cast<float*>(out)[c] = sum[0][x];
    else put<DT>(out, c, sum[0][x]);
}

template <int DT>
void norm_fold(const float* part, int64_t parts, int64_t cols, void* dw, void* db, int w32, hipStream_t s) {
    over_columns<FOLD_COLS>(cols, [&](int64_t first, unsigned groups) {
        hipLaunchKernelGGL((norm_fold_kernel<DT>), dim3(groups, db ? 2 : 1), dim3(FOLD_COLS * FOLD_ROWS), 0, s, part, parts, cols, first, dw,
                           db, w32);
    });
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
}  // namespace tvk
