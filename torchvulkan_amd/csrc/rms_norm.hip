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
#include "f8_blocks.h"
#include "norm_rows.h"

using namespace tvk;

namespace {

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
            const float s = top > 0.0f ? fmaxf(top / kF8Max, F8_LEAST_SCALE) : 1.0f;
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
__global__ __launch_bounds__(RN_THREADS) void rms_norm_dweight_kernel(NormBwdArgs p, float* part, int64_t first) {
    __shared__ float sum[4][64];
    typedef typename elem<DT>::T T;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int64_t c = first + (int64_t)blockIdx.x * 64 + lane;
    float s = 0.0f;
    if (c < p.cols)
        for (int64_t row = (int64_t)blockIdx.y * 4 + wave; row < p.rows; row += (int64_t)gridDim.y * 4)
            s += at<DT>(static_cast<const T*>(p.dy) + row * p.sdy, c) * at<DT>(static_cast<const T*>(p.h) + row * p.sh, c) *
                 p.inv[row];
    sum[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && c < p.cols) part[blockIdx.y * p.cols + c] = sum[0][lane] + sum[1][lane] + sum[2][lane] + sum[3][lane];
}

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
            const float s = top > 0.0f ? fmaxf(top / kF8Max, F8_LEAST_SCALE) : 1.0f, f8 = inv * __builtin_amdgcn_rcpf(s);
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
            over_columns<64>(p.cols, [&](int64_t first, unsigned groups) {
                hipLaunchKernelGGL((rms_norm_dweight_kernel<DT>), dim3(groups, (unsigned)parts), dim3(RN_THREADS), 0, s, p, part, first);
            });
        }
        if (have && p.rows > 0) hipLaunchKernelGGL((rms_norm_bwd_any_kernel<DT>), rows_grid(p.rows), dim3(RN_THREADS), 0, s, p);
    }
    if (!have) return fail(TVK_ERR_OOM, "tvk_rms_norm_bwd: workspace allocation failed");
    if (dw && !p.dw) norm_fold<DT>(part, parts, p.cols, dw, nullptr, p.w32, s);
    return TVK_OK;
}

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
