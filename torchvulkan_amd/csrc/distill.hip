// Distillation from a teacher's top logits (tvk_distill_fwd, tvk_distill_bwd).
//
// Forward, the logits are read once: every thread keeps the running maximum m of
// its values and the sum s of exp((x - m) / T), rescaled when a group of chunks
// brings a larger one; threads and, where a row is cut among workgroups, pieces
// are joined in a fixed order. What is left is a row's list of `top` entries: a
// softmax over the teacher's logits and the student's logits at their indexes.
// Backward reads the logits once more and writes p = exp((x - m) / T - log s) times
// the row's factor (m and log s apart: their sum in one float32 is off by half a step
// of its own size, and all p with it); the entries' places, q less, are written over that after a
// barrier, from logits read before it (dlogits may be logits). An index named
// twice would be two writes to one place, so forward gives the whole of an
// index's q to its first entry, found in a hash table in LDS.
//
// Measured: 4096 x 32000 of bfloat16 with 64 entries 62 to 79 us forward (262 MB) and
// 91 backward (524 MB, 5.8 TB/s: the rows that forward read last are still in the
// memory's cache, and come first; 115 us where none are); 33 x 50001 of float32 14 us,
// three launches. Forward is bound by memory past 16384 rows (5.4 TB/s) and by the
// rounds of five workgroups a CU before that; registers for more would not hold a
// row's loads (spilled, 180 us for 170 in both directions).
#include "norm_rows.h"

using namespace tvk;

namespace {

constexpr int DI_THREADS = 256;
constexpr int DI_MOST_TOP = 2048;   // the hash table takes 48 KB of LDS then
constexpr float kLog2e = 1.44269504088896f;

struct DistillArgs {
    const void* x;        // logits, or NULL
    const void* index;
    const void* teacher;
    float* loss;
    float* lse;
    float* softmax;       // [rows][2]: m and log s, or NULL
    float* target;
    const float* dloss;
    void* dx;
    float* part;          // [rows][pieces][2]: maximum and sum of a piece
    int64_t sx, si, st, sq, sd, sdx;
    int64_t rows, cols;
    int top, index64, teacher32, slots;   // slots: of the hash table, a power of two above top
    int64_t piece;                        // values of a row that a workgroup takes
    int pieces;
    float inv_t, t;
};

struct Soft {
    float m, s;   // maximum, sum of exp((x - m) / T)
};

static_assert(DI_THREADS == RN_THREADS, "block_all's threads");

__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }   // results below 2^-126 are zeros

// What values are taken from: their maximum, or where that is -inf any finite number, so that they weigh nothing.
__device__ inline float base_of(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ inline Soft join(Soft a, Soft b, float c) {
    const float m = fmaxf(a.m, b.m), f = base_of(m);
    return {m, a.s * exp2_of((a.m - f) * c) + b.s * exp2_of((b.m - f) * c)};
}

// Over a wave's lanes in their order, the same bits in each.
__device__ inline Soft join_lanes(Soft r, float c) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const Soft o{__shfl_xor(r.m, m), __shfl_xor(r.s, m)};
        r = threadIdx.x & m ? join(o, r, c) : join(r, o, c);
    }
    return r;
}

template <int VALUES>
__device__ inline void add_values(Soft& r, const float (&x)[VALUES], float c) {
    float m = r.m;
#pragma unroll
    for (int i = 0; i < VALUES; ++i) m = fmaxf(m, x[i]);
    const float f = base_of(m);
    float s = r.s * exp2_of((r.m - f) * c);
#pragma unroll
    for (int i = 0; i < VALUES; ++i) s += exp2_of((x[i] - f) * c);
    r = {m, s};
}

// Maximum and sum of values [begin, end) of a row over the workgroup, the same bits in every thread.
template <int DT>
__device__ Soft soft_piece(const typename elem<DT>::T* row, int64_t begin, int64_t end, float c) {
    constexpr int VEC = 16 / (int)sizeof(typename elem<DT>::T), GROUP = 4;   // chunks on their way together
    Soft r{-INFINITY, 0.0f};
    const int64_t chunks = (end - begin) / VEC;
    int64_t i = threadIdx.x;
    for (; i + (GROUP - 1) * DI_THREADS < chunks; i += GROUP * DI_THREADS) {
        Words<16> w[GROUP];
#pragma unroll
        for (int g = 0; g < GROUP; ++g) w[g] = load_words<16, sizeof(*row)>(row + begin + (i + g * DI_THREADS) * VEC);
        float x[GROUP * VEC];
#pragma unroll
        for (int g = 0; g < GROUP; ++g)
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[g * VEC + k] = word_at<DT>(w[g], k);
        add_values(r, x, c);
    }
    for (; i < chunks; i += DI_THREADS) {
        const Words<16> w = load_words<16, sizeof(*row)>(row + begin + i * VEC);
        float x[VEC];
#pragma unroll
        for (int k = 0; k < VEC; ++k) x[k] = word_at<DT>(w, k);
        add_values(r, x, c);
    }
    if (begin + chunks * VEC + threadIdx.x < end) {
        const float x[1] = {elem<DT>::to_f32(row[begin + chunks * VEC + threadIdx.x])};
        add_values(r, x, c);
    }
    r = join_lanes(r, c);
    __shared__ Soft part[DI_THREADS / 64];
    __syncthreads();
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = r;
    __syncthreads();
    r = part[0];
#pragma unroll
    for (int w = 1; w < DI_THREADS / 64; ++w) r = join(r, part[w], c);
    return r;
}

__device__ inline int64_t index_at(const DistillArgs& p, int64_t row, int j) {
    return p.index64 ? static_cast<const int64_t*>(p.index)[row * p.si + j] : static_cast<const int32_t*>(p.index)[row * p.si + j];
}

template <int DT>
__device__ inline float teacher_at(const DistillArgs& p, int64_t row, int j) {
    const int64_t i = row * p.st + j;
    return p.teacher32 ? static_cast<const float*>(p.teacher)[i] : elem<DT>::to_f32(static_cast<const typename elem<DT>::T*>(p.teacher)[i]);
}

// A thread's first entry, asked for before the row's logits and used after them.
struct Entry {
    int64_t at;
    float t;
};
template <int DT>
__device__ inline Entry first_entry(const DistillArgs& p, int64_t row) {
    const int j = threadIdx.x;
    if (j >= p.top) return {-1, 0.0f};
    return {index_at(p, row, j), teacher_at<DT>(p, row, j)};
}

// The row's loss, log sum of exponentials and the entries' shares, from the sum over its logits, by the workgroup's first N
// threads: all, or a wave, which has no barriers to wait at while the others make room for the next workgroup. Forward of 4096 x
// 32000 in bfloat16 with 64 entries 62 us, all threads 71; 8192 x 8000 58 and 75. More entries take all. LDS: table, slots x 3 words.
template <int DT, int N>
__device__ __forceinline__ void distill_row(const DistillArgs& p, int64_t row, const Entry& own, Soft soft, int* table) {
    typedef typename elem<DT>::T T;
    auto all = [](auto op, float v) {
        if constexpr (N == 64) {
            __threadfence_block();   // (LDS, as a barrier would)
            return lanes64_all<decltype(op)>(v);
        } else {
            return block_all<decltype(op)>(v);
        }
    };
    const float c = kLog2e * p.inv_t;
    const T* x = static_cast<const T*>(p.x) + row * p.sx;
    const float own_x = own.at >= 0 && own.at < p.cols ? elem<DT>::to_f32(x[own.at]) : 0.0f;
    int *key = table, *first = table + p.slots, *count = table + 2 * p.slots;
    __shared__ int twice;
    for (int i = threadIdx.x; i < p.slots; i += N) {
        key[i] = -1;
        first[i] = 0x7fffffff;
        count[i] = 0;
    }
    if (threadIdx.x == 0) twice = 0;
    auto named = [&](int j, int64_t& at) {
        at = j == (int)threadIdx.x ? own.at : index_at(p, row, j);
        return at >= 0 && at < p.cols;
    };
    auto logit = [&](int j) { return j == (int)threadIdx.x ? own.t : teacher_at<DT>(p, row, j); };
    float top = -INFINITY, bad = 0.0f;
    int64_t at;
    for (int j = threadIdx.x; j < p.top; j += N)
        if (named(j, at)) {
            const float v = logit(j);
            top = fmaxf(top, v);
            bad = v != v ? 1.0f : bad;
        }
    top = all(MaxOp(), top);   // (and every thread is past the table's first values)
    bad = all(MaxOp(), bad);
    if (top == -INFINITY && bad == 0.0f) {   // nothing to learn from: no loss, and a gradient of zeros whatever the logits are
        for (int j = threadIdx.x; j < p.top && p.target; j += N) p.target[row * p.sq + j] = 0.0f;
        if (threadIdx.x == 0) {
            p.loss[row] = 0.0f;
            if (p.lse) p.lse[row] = INFINITY;
            if (p.softmax) p.softmax[2 * row] = 0.0f, p.softmax[2 * row + 1] = INFINITY;
        }
        return;
    }
    auto slot_of = [&](int64_t at) { return (uint32_t)at * 2654435769u >> 8 & (uint32_t)(p.slots - 1); };   // multiplicative hash
    float sum = 0.0f;
    for (int j = threadIdx.x; j < p.top; j += N)
        if (named(j, at)) {
            sum += exp2_of((logit(j) - top) * c);
            for (uint32_t h = slot_of(at);; h = (h + 1) & (uint32_t)(p.slots - 1)) {   // fewer entries than slots
                const int old = atomicCAS(&key[h], -1, (int)at);
                if (old != -1 && old != (int)at) continue;
                atomicMin(&first[h], j);
                if (atomicAdd(&count[h], 1)) twice = 1;
                break;
            }
        }
    sum = all(SumOp(), sum);   // (and the table is filled)
    const float log_s = logf(soft.s), log_q = logf(sum);
    auto share = [&](int j) { return exp2_of((logit(j) - top) * c) / sum; };
    float loss = 0.0f;
    for (int j = threadIdx.x; j < p.top; j += N) {
        float q = 0.0f;
        if (named(j, at)) {
            q = share(j);
            if (q != 0.0f) {
                const float lq = (logit(j) - top) * p.inv_t - log_q;
                const float lp = ((j == (int)threadIdx.x ? own_x : elem<DT>::to_f32(x[at])) - soft.m) * p.inv_t - log_s;
                loss += q * (lq - lp);
            }
            if (twice && p.target) {
                uint32_t h = slot_of(at);
                while (key[h] != (int)at) h = (h + 1) & (uint32_t)(p.slots - 1);
                if (first[h] != j) q = 0.0f;
                else if (count[h] > 1)
                    for (int k = j + 1; k < p.top; ++k)
                        if (index_at(p, row, k) == at) q += share(k);
            }
        }
        if (p.target) p.target[row * p.sq + j] = q;
    }
    loss = all(SumOp(), loss);
    if (threadIdx.x == 0) {
        p.loss[row] = loss * p.t * p.t;
        if (p.lse) {
            const float lse = soft.m * p.inv_t + log_s;
            p.lse[row] = lse == INFINITY ? NAN : lse;   // +inf stands for a row without entries
        }
        if (p.softmax) p.softmax[2 * row] = soft.m, p.softmax[2 * row + 1] = log_s;   // (s is finite, or NaN)
    }
}

// A workgroup a row. N: threads for what follows the logits.
template <int DT, int N>
__global__ __launch_bounds__(DI_THREADS) void distill_rows_kernel(DistillArgs p) {
    extern __shared__ int table[];
    typedef typename elem<DT>::T T;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        if (row != blockIdx.x) __syncthreads();   // the table was the last row's
        const Entry own = first_entry<DT>(p, row);
        const Soft r = soft_piece<DT>(static_cast<const T*>(p.x) + row * p.sx, 0, p.cols, kLog2e * p.inv_t);
        if (threadIdx.x < N) distill_row<DT, N>(p, row, own, r, table);
    }
}

// Rows cut into pieces, a workgroup each; then a workgroup a row joins them.
template <int DT>
__global__ __launch_bounds__(DI_THREADS) void distill_pieces_kernel(DistillArgs p) {
    typedef typename elem<DT>::T T;
    const int64_t row = blockIdx.x / (unsigned)p.pieces, piece = blockIdx.x % (unsigned)p.pieces;
    const Soft r = soft_piece<DT>(static_cast<const T*>(p.x) + row * p.sx, piece * p.piece, min((piece + 1) * p.piece, p.cols),
                                  kLog2e * p.inv_t);
    if (threadIdx.x == 0) {
        p.part[2 * (int64_t)blockIdx.x] = r.m;
        p.part[2 * (int64_t)blockIdx.x + 1] = r.s;
    }
}

template <int DT, int N>
__global__ __launch_bounds__(N) void distill_join_kernel(DistillArgs p) {
    extern __shared__ int table[];
    const int64_t row = blockIdx.x;
    const float* part = p.part + 2 * row * p.pieces;
    const Entry own = first_entry<DT>(p, row);
    Soft r{-INFINITY, 0.0f};
    for (int i = threadIdx.x % 64; i < p.pieces; i += 64) r = join(r, Soft{part[2 * i], part[2 * i + 1]}, kLog2e * p.inv_t);
    distill_row<DT, N>(p, row, own, join_lanes(r, kLog2e * p.inv_t), table);
}

// LDS: top floats, the entries' gradients. APART: from m and log s, else from lse.
template <int DT, bool APART>
__global__ __launch_bounds__(DI_THREADS) void distill_bwd_kernel(DistillArgs p) {
    extern __shared__ float entry[];
    typedef typename elem<DT>::T T;
    constexpr int VEC = 16 / (int)sizeof(T), GROUP = 4;
    for (int64_t work = p.rows * p.pieces - 1 - blockIdx.x; work >= 0; work -= gridDim.x) {   // the rows that forward read last come first
        const int64_t row = work / p.pieces, begin = work % p.pieces * p.piece, end = min(begin + p.piece, p.cols);
        const T* x = static_cast<const T*>(p.x) + row * p.sx;
        T* o = static_cast<T*>(p.dx) + row * p.sdx;
        const float m = APART ? p.softmax[2 * row] : 0.0f, log_s = APART ? p.softmax[2 * row + 1] : p.lse[row];
        const bool none = log_s == INFINITY;
        const float f = p.dloss[row * p.sd] * p.t;
        auto grad = [&](float v, float q) {
            float g = f * (exp2_of(fmaf(APART ? v - m : v, p.inv_t, -log_s) * kLog2e) - q);
            asm("" : "+v"(g));   // a choice below, no branch for every value (33 x 50001 0.8 us)
            return none ? 0.0f : g;
        };
        for (int j = threadIdx.x; j < p.top; j += DI_THREADS) {
            const int64_t at = index_at(p, row, j);
            const float q = p.target[row * p.sq + j];
            if (q != 0.0f && at >= begin && at < end) entry[j] = grad(elem<DT>::to_f32(x[at]), q);
        }
        __syncthreads();   // dlogits may lie over logits
        const int64_t chunks = (end - begin) / VEC;
        auto store = [&](int64_t i, const Words<16>& w) {
            float g[VEC];
#pragma unroll
            for (int k = 0; k < VEC; ++k) g[k] = grad(word_at<DT>(w, k), 0.0f);
            store_words<16, sizeof(T)>(o + begin + i * VEC, pack<DT, VEC>(g));
        };
        int64_t i = threadIdx.x;
        for (; i + (GROUP - 1) * DI_THREADS < chunks; i += GROUP * DI_THREADS) {
            Words<16> w[GROUP];
#pragma unroll
            for (int g = 0; g < GROUP; ++g) w[g] = load_words<16, sizeof(T)>(x + begin + (i + g * DI_THREADS) * VEC);
#pragma unroll
            for (int g = 0; g < GROUP; ++g) store(i + g * DI_THREADS, w[g]);
        }
        for (; i < chunks; i += DI_THREADS) store(i, load_words<16, sizeof(T)>(x + begin + i * VEC));
        const int64_t last = begin + chunks * VEC + threadIdx.x;
        if (last < end) o[last] = elem<DT>::from_f32(grad(elem<DT>::to_f32(x[last]), 0.0f));
        __syncthreads();   // the entries' places come last
        for (int j = threadIdx.x; j < p.top; j += DI_THREADS) {
            const int64_t at = index_at(p, row, j);
            if (p.target[row * p.sq + j] != 0.0f && at >= begin && at < end) o[at] = elem<DT>::from_f32(entry[j]);
        }
        __syncthreads();
    }
}

constexpr int64_t kMostGroups = 1 << 20;

template <int DT, int N>
tvk_status forward(DistillArgs& p, hipStream_t s) {
    const size_t lds = (size_t)p.slots * 12;
    // Two workgroups a CU are wanted; rows that do not make them are cut, into pieces of 4 K values or more
    constexpr int64_t WANTED = 512, PIECE = 4096;
    const int64_t pieces = std::min((WANTED + p.rows - 1) / p.rows, p.cols / PIECE);
    if (pieces < 2) {
        hipLaunchKernelGGL((distill_rows_kernel<DT, N>), dim3((unsigned)std::min(p.rows, kMostGroups)), dim3(DI_THREADS), lds, s, p);
        return TVK_OK;
    }
    p.piece = ((p.cols + pieces - 1) / pieces + 7) / 8 * 8;
    p.pieces = (int)((p.cols + p.piece - 1) / p.piece);
    Scratch scratch;
    p.part = static_cast<float*>(scratch.get((size_t)(p.rows * p.pieces) * 8, s));
    if (!p.part) return fail(TVK_ERR_OOM, "tvk_distill_fwd: workspace allocation failed");
    hipLaunchKernelGGL((distill_pieces_kernel<DT>), dim3((unsigned)(p.rows * p.pieces)), dim3(DI_THREADS), 0, s, p);
    hipLaunchKernelGGL((distill_join_kernel<DT, N>), dim3((unsigned)p.rows), dim3(N), lds, s, p);
    return TVK_OK;
}

template <int DT>
tvk_status forward(DistillArgs& p, hipStream_t s) {
    return p.top <= 64 ? forward<DT, 64>(p, s) : forward<DT, DI_THREADS>(p, s);
}

template <int DT>
void backward(DistillArgs& p, hipStream_t s) {
    // pieces of 8 K values: enough workgroups for few rows, and few entries searched by each
    constexpr int64_t PIECE = 8192;
    p.piece = PIECE;
    p.pieces = (int)((p.cols + PIECE - 1) / PIECE);
    const int64_t groups = std::min(p.rows * p.pieces, kMostGroups);
    if (p.softmax) hipLaunchKernelGGL((distill_bwd_kernel<DT, true>), dim3((unsigned)groups), dim3(DI_THREADS), (size_t)p.top * 4, s, p);
    else hipLaunchKernelGGL((distill_bwd_kernel<DT, false>), dim3((unsigned)groups), dim3(DI_THREADS), (size_t)p.top * 4, s, p);
}

tvk_status check_distill(const char* who, int32_t dtype, int32_t index_dtype, int64_t rows, int64_t cols, int64_t top, double t) {
    auto bad = [&](tvk_status st, const char* m) { return fail(st, std::string(who) + ": " + m); };
    if (!norm_dtype(dtype)) return bad(TVK_ERR_UNSUPPORTED, "dtype must be float32, float16 or bfloat16");
    if (index_dtype != TVK_I32 && index_dtype != TVK_I64) return bad(TVK_ERR_UNSUPPORTED, "the indexes must be int32 or int64");
    if (rows < 0 || cols < 0 || top < 0) return bad(TVK_ERR_INVALID, "negative size");
    const float heat = (float)t;   // the kernels' factors are heat, heat * heat, 1 / heat and log2(e) / heat
    if (!(t > 0.0) || !(heat > 0.0f) || !(1.0f / heat > 0.0f) || !(heat * heat < INFINITY) || !(kLog2e * (1.0f / heat) < INFINITY))
        return bad(TVK_ERR_INVALID, "the temperature must be above zero and finite");
    if (rows > 0x7fffffff || cols > 0x7fffffff) return bad(TVK_ERR_UNSUPPORTED, "rows and columns up to 2^31 - 1 only");
    if (top > DI_MOST_TOP) return bad(TVK_ERR_UNSUPPORTED, "up to 2048 entries a row only");
    return TVK_OK;
}

}  // namespace

extern "C" tvk_status tvk_distill_fwd(const tvk_distill_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_distill_fwd: desc is NULL");
    tvk_status st = check_distill("tvk_distill_fwd", d->dtype, d->index_dtype, d->rows, d->cols, d->top, d->temperature);
    if (st != TVK_OK) return st;
    if (d->teacher_dtype != d->dtype && d->teacher_dtype != TVK_F32)
        return fail(TVK_ERR_UNSUPPORTED, "tvk_distill_fwd: the teacher's dtype must be the logits' or float32");
    if (d->rows == 0) return TVK_OK;
    if ((d->cols > 0 && !d->logits) || (d->top > 0 && (!d->index || !d->teacher)) || !d->loss)
        return fail(TVK_ERR_INVALID, "tvk_distill_fwd: NULL tensor");
    if (d->logits_stride < 0 || d->index_stride < 0 || d->teacher_stride < 0 || (d->target && !rows_apart(d->target_stride, d->rows, d->top)))
        return fail(TVK_ERR_INVALID, "tvk_distill_fwd: negative strides, or target rows that overlap");
    DistillArgs p{};
    p.x = d->logits;
    p.index = d->index;
    p.teacher = d->teacher;
    p.loss = d->loss;
    p.lse = d->lse;
    p.softmax = d->softmax;
    p.target = d->target;
    p.sx = d->logits_stride;
    p.si = d->index_stride;
    p.st = d->teacher_stride;
    p.sq = d->target_stride;
    p.rows = d->rows;
    p.cols = d->cols;
    p.top = (int)d->top;
    p.index64 = d->index_dtype == TVK_I64;
    p.teacher32 = d->teacher_dtype == TVK_F32;
    for (p.slots = 16; p.slots < 2 * p.top; p.slots *= 2) {}
    p.t = (float)d->temperature;
    p.inv_t = 1.0f / p.t;
    const hipStream_t s = resolve_stream(d->stream);
    if (d->dtype == TVK_F32) st = forward<TVK_F32>(p, s);
    else if (d->dtype == TVK_F16) st = forward<TVK_F16>(p, s);
    else st = forward<TVK_BF16>(p, s);
    if (st != TVK_OK) return st;
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_distill_fwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}

extern "C" tvk_status tvk_distill_bwd(const tvk_distill_bwd_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_distill_bwd: desc is NULL");
    const tvk_status st = check_distill("tvk_distill_bwd", d->dtype, d->index_dtype, d->rows, d->cols, d->top, d->temperature);
    if (st != TVK_OK) return st;
    if (d->rows == 0 || d->cols == 0) return TVK_OK;
    if (!d->logits || (d->top > 0 && (!d->index || !d->target)) || (!d->lse && !d->softmax) || !d->dloss || !d->dlogits)
        return fail(TVK_ERR_INVALID, "tvk_distill_bwd: NULL tensor");
    if (d->logits_stride < 0 || d->index_stride < 0 || d->target_stride < 0 || d->dloss_stride < 0 ||
        !rows_apart(d->dlogits_stride, d->rows, d->cols))
        return fail(TVK_ERR_INVALID, "tvk_distill_bwd: negative strides, or dlogits rows that overlap");
    DistillArgs p{};
    p.x = d->logits;
    p.index = d->index;
    p.target = const_cast<float*>(d->target);
    p.lse = const_cast<float*>(d->lse);
    p.softmax = const_cast<float*>(d->softmax);
    p.dloss = d->dloss;
    p.dx = d->dlogits;
    p.sx = d->logits_stride;
    p.si = d->index_stride;
    p.sq = d->target_stride;
    p.sd = d->dloss_stride;
    p.sdx = d->dlogits_stride;
    p.rows = d->rows;
    p.cols = d->cols;
    p.top = (int)d->top;
    p.index64 = d->index_dtype == TVK_I64;
    p.t = (float)d->temperature;
    p.inv_t = 1.0f / p.t;
    const hipStream_t s = resolve_stream(d->stream);
    if (d->dtype == TVK_F32) backward<TVK_F32>(p, s);
    else if (d->dtype == TVK_F16) backward<TVK_F16>(p, s);
    else backward<TVK_BF16>(p, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_distill_bwd: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}
