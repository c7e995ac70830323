// Values brought into 8-bit floats with a scale for each block of 128 columns of a
// row, or of 128 x 128 (tvk_quantize_f8); the former also as the first step of
// tvk_gemm_f8 with rows in 16 or 32 bits. A block's values are read once: in
// registers while their largest magnitude goes round the 16 lanes (or the
// workgroup) that hold them. Bound by memory: 8192 x 4096 of bfloat16 19.5 us
// (5.2 TB/s), 14336 x 4096 in blocks of 128 x 128 33.2 us (5.3 TB/s).
#include "gemm_f8.h"

using namespace tvk;

namespace {

constexpr int QF_THREADS = 256;
constexpr int64_t kMostGroups = 1 << 20;

struct QuantArgs {
    const void* x;
    uint8_t* out;
    float* scale;
    int64_t sx, so, ss[2];
    int64_t rows, cols, wide;   // wide: columns written, zeros past cols
};

// Eight values of a row from column c on, zeros past its end.
template <int DT>
__device__ inline void load8(const QuantArgs& p, int64_t row, int64_t c, float (&v)[8]) {
    typedef typename elem<DT>::T T;
    const T* x = static_cast<const T*>(p.x) + row * p.sx + c;
    if (c + 8 <= p.cols) {
        constexpr int BYTES = 8 * (int)sizeof(T), PART = BYTES < 16 ? BYTES : 16, PER = PART / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < 8; i += PER) {
            const Words<PART> w = load_words<PART, sizeof(T)>(x + i);
#pragma unroll
            for (int k = 0; k < PER; ++k) v[i + k] = word_at<DT>(w, k);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < p.cols ? elem<DT>::to_f32(x[k]) : 0.0f;
    }
}

__device__ inline float top8(const float (&v)[8]) {
    float top = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
    return top;
}

__device__ inline void store8(const QuantArgs& p, int64_t row, int64_t c, const float (&v)[8], const F8Scale& s) {
    uint8_t* o = p.out + row * p.so + c;
    Words<8> w;
    w.w[0] = s.pack4(v[0], v[1], v[2], v[3]);
    w.w[1] = s.pack4(v[4], v[5], v[6], v[7]);
    if (c + 8 <= p.wide) store_words<8, 1>(o, w);
    else
        for (int k = 0; k < 8 && c + k < p.wide; ++k) o[k] = (uint8_t)(w.w[k / 4] >> k % 4 * 8);
}

// Sixteen lanes a block of 128 columns of a row.
template <int DT>
__global__ __launch_bounds__(QF_THREADS) void quantize_rows_kernel(QuantArgs p, int64_t blocks, int64_t all) {
    for (int64_t b = (int64_t)blockIdx.x * (QF_THREADS / 16) + threadIdx.x / 16; b < all; b += (int64_t)gridDim.x * (QF_THREADS / 16)) {
        const int64_t row = b / blocks, blk = b - row * blocks, c = blk * F8_BLOCK + threadIdx.x % 16 * 8;
        float v[8];
        load8<DT>(p, row, c, v);
        float top = top8(v);
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
        const F8Scale s(top);
        store8(p, row, c, v, s);
        if (threadIdx.x % 16 == 0) p.scale[row * p.ss[0] + blk * p.ss[1]] = s.s;
    }
}

// A workgroup a block of 128 x 128, eight pieces of eight values a thread.
template <int DT>
__global__ __launch_bounds__(QF_THREADS) void quantize_blocks_kernel(QuantArgs p, int64_t blocks, int64_t all) {
    __shared__ float part[QF_THREADS / 64];
    for (int64_t b = blockIdx.x; b < all; b += gridDim.x) {
        const int64_t tall = b / blocks, blk = b - tall * blocks;
        const int64_t row0 = tall * F8_BLOCK + threadIdx.x / 16, c = blk * F8_BLOCK + threadIdx.x % 16 * 8;
        float v[8][8], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (row0 + 16 * i < p.rows) load8<DT>(p, row0 + 16 * i, c, v[i]);
            else
#pragma unroll
                for (int k = 0; k < 8; ++k) v[i][k] = 0.0f;
            top = fmaxf(top, top8(v[i]));
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
        __syncthreads();
        if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = top;
        __syncthreads();
        const F8Scale s(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (row0 + 16 * i < p.rows) store8(p, row0 + 16 * i, c, v[i], s);
        if (threadIdx.x == 0) p.scale[tall * p.ss[0] + blk * p.ss[1]] = s.s;
    }
}

template <int DT>
void launch(const QuantArgs& p, bool tall, hipStream_t s) {
    const int64_t blocks = (p.cols + F8_BLOCK - 1) / F8_BLOCK;
    const int64_t all = blocks * (tall ? (p.rows + F8_BLOCK - 1) / F8_BLOCK : p.rows);
    const int64_t groups = std::min(tall ? all : (all + QF_THREADS / 16 - 1) / (QF_THREADS / 16), kMostGroups);
    if (tall) hipLaunchKernelGGL((quantize_blocks_kernel<DT>), dim3((unsigned)groups), dim3(QF_THREADS), 0, s, p, blocks, all);
    else hipLaunchKernelGGL((quantize_rows_kernel<DT>), dim3((unsigned)groups), dim3(QF_THREADS), 0, s, p, blocks, all);
}

void launch(int dtype, const QuantArgs& p, bool tall, hipStream_t s) {
    if (dtype == TVK_F32) launch<TVK_F32>(p, tall, s);
    else if (dtype == TVK_F16) launch<TVK_F16>(p, tall, s);
    else launch<TVK_BF16>(p, tall, s);
}

// Rows of bytes copied to rows of whole blocks, zeros behind them.
__global__ __launch_bounds__(QF_THREADS) void pad_rows_kernel(const uint8_t* x, int64_t sx, uint8_t* out, int64_t rows, int64_t cols, int64_t wide) {
    const int64_t chunks = wide / 16, all = rows * chunks;
    for (int64_t i = (int64_t)blockIdx.x * QF_THREADS + threadIdx.x; i < all; i += (int64_t)gridDim.x * QF_THREADS) {
        const int64_t row = i / chunks, c = (i - row * chunks) * 16;
        const uint8_t* from = x + row * sx + c;
        Words<16> w{};
        if (c + 16 <= cols) w = load_words<16, 1>(from);
        else
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (c + k < cols) w.w[k / 4] |= (uint32_t)from[k] << k % 4 * 8;
        store_words<16, 16>(out + row * wide + c, w);
    }
}

}  // namespace

namespace tvk {

void f8_quantize_rows(int dtype, const void* x, int64_t x_stride, uint8_t* out, float* scale, int64_t rows, int64_t cols, hipStream_t s) {
    const int64_t wide = (cols + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK;
    launch(dtype, QuantArgs{x, out, scale, x_stride, wide, {1, rows}, rows, cols, wide}, false, s);
}

void f8_pad_rows(const uint8_t* x, int64_t x_stride, uint8_t* out, int64_t rows, int64_t cols, hipStream_t s) {
    const int64_t wide = (cols + F8_BLOCK - 1) / F8_BLOCK * F8_BLOCK, groups = (rows * (wide / 16) + QF_THREADS - 1) / QF_THREADS;
    hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)std::min(groups, kMostGroups)), dim3(QF_THREADS), 0, s, x, x_stride, out, rows, cols, wide);
}

}  // namespace tvk

extern "C" tvk_status tvk_quantize_f8(const tvk_quantize_f8_desc* d) {
    if (!d) return fail(TVK_ERR_INVALID, "tvk_quantize_f8: desc is NULL");
    if (!norm_dtype(d->dtype)) return fail(TVK_ERR_UNSUPPORTED, "tvk_quantize_f8: dtype must be float32, float16 or bfloat16");
    if (d->block_rows != 1 && d->block_rows != F8_BLOCK) return fail(TVK_ERR_UNSUPPORTED, "tvk_quantize_f8: blocks of 1 or 128 rows only");
    if (d->rows < 0 || d->cols < 0) return fail(TVK_ERR_INVALID, "tvk_quantize_f8: negative size");
    if (d->rows > 0x7fffffff || d->cols > 0x7fffffff)
        return fail(TVK_ERR_UNSUPPORTED, "tvk_quantize_f8: rows and columns up to 2^31 - 1 only");
    if (d->rows == 0 || d->cols == 0) return TVK_OK;
    if (!d->x || !d->out || !d->scale) return fail(TVK_ERR_INVALID, "tvk_quantize_f8: NULL tensor");
    const bool tall = d->block_rows != 1;
    if (d->x_stride < 0 || !rows_apart(d->out_stride, d->rows, d->cols) ||
        !apart2(d->scale_stride, tall ? (d->rows + F8_BLOCK - 1) / F8_BLOCK : d->rows, (d->cols + F8_BLOCK - 1) / F8_BLOCK))
        return fail(TVK_ERR_INVALID, "tvk_quantize_f8: negative strides, or outputs that overlap");
    const QuantArgs p{d->x, static_cast<uint8_t*>(d->out), d->scale, d->x_stride, d->out_stride, {d->scale_stride[0], d->scale_stride[1]},
                      d->rows, d->cols, d->cols};
    launch(d->dtype, p, tall, resolve_stream(d->stream));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_quantize_f8: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}
