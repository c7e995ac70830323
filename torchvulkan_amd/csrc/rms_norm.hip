// Root-mean-square norm (tvk_rms_norm_fwd, tvk_rms_norm_bwd): a workgroup a row.
#include "convert.h"

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
    float eps;
    int w32, out8;
};

struct NormBwdArgs {
    const void* dy;
    const void* h;
    const void* dh;
    const void* w;
    void* dx;
    float* inv;    // [rows], or NULL
    int64_t sdy, sh, sdh, sdx;
    int64_t rows, cols;
    float eps;
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

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_kernel(NormArgs p) {
    typedef typename elem<DT>::T T;
    const int64_t row = blockIdx.x;
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

// 1 / sqrt(mean(h^2) + eps) of every row, for dweight's sums. dx comes after those: it may lie over dy or h.
template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_inv_kernel(NormBwdArgs p) {
    const int64_t row = blockIdx.x;
    const void* h = static_cast<const typename elem<DT>::T*>(p.h) + row * p.sh;
    float ss = 0.0f;
    for (int64_t c = threadIdx.x; c < p.cols; c += RN_THREADS) {
        const float v = at<DT>(h, c);
        ss += v * v;
    }
    ss = block_all<SumOp>(ss);
    if (threadIdx.x == 0) p.inv[row] = 1.0f / sqrtf(ss / (float)p.cols + p.eps);
}

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_bwd_kernel(NormBwdArgs p) {
    typedef typename elem<DT>::T T;
    const int64_t row = blockIdx.x;
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

template <int DT>
__global__ __launch_bounds__(RN_THREADS) void rms_norm_fold_kernel(const float* part, int64_t parts, int64_t cols, void* dw,
                                                                   int w32) {
    const int64_t c = (int64_t)blockIdx.x * RN_THREADS + threadIdx.x;
    if (c >= cols) return;
    float s = 0.0f;
    for (int64_t i = 0; i < parts; ++i) s += part[i * cols + c];
    if (w32) static_cast<float*>(dw)[c] = s;
    else put<DT>(dw, c, s);
}

template <int DT>
void forward(const NormArgs& p, hipStream_t s) {
    hipLaunchKernelGGL((rms_norm_kernel<DT>), dim3((unsigned)p.rows), dim3(RN_THREADS), 0, s, p);
}

template <int DT>
tvk_status backward(NormBwdArgs p, void* dw, hipStream_t s) {
    Scratch scratch;
    float* part = nullptr;
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(64, p.rows / 64));
    if (dw) {
        p.inv = static_cast<float*>(scratch.get((size_t)(p.rows + parts * p.cols) * 4, s));
        if (!p.inv) return fail(TVK_ERR_OOM, "tvk_rms_norm_bwd: workspace allocation failed");
        part = p.inv + p.rows;
    }
    if (dw) {
        if (p.rows > 0) hipLaunchKernelGGL((rms_norm_inv_kernel<DT>), dim3((unsigned)p.rows), dim3(RN_THREADS), 0, s, p);
        hipLaunchKernelGGL((rms_norm_dweight_kernel<DT>), dim3((unsigned)((p.cols + 63) / 64), (unsigned)parts),
                           dim3(RN_THREADS), 0, s, p, part);
        hipLaunchKernelGGL((rms_norm_fold_kernel<DT>), dim3((unsigned)((p.cols + RN_THREADS - 1) / RN_THREADS)),
                           dim3(RN_THREADS), 0, s, part, parts, p.cols, dw, p.w32);
    }
    if (p.rows > 0) hipLaunchKernelGGL((rms_norm_bwd_kernel<DT>), dim3((unsigned)p.rows), dim3(RN_THREADS), 0, s, p);
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
    if (d->rows == 0 || d->cols == 0) return TVK_OK;
    if (!d->x || !d->out || (out8 && !d->scale)) return fail(TVK_ERR_INVALID, "tvk_rms_norm_fwd: NULL tensor");
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
