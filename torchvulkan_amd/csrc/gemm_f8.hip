// Products of 8-bit floats with a scale for each block of 128 (tvk_gemm_f8):
//   out[m][n] = sum over blocks b of sa[m][b] sb[n / 128][b] sum over k in b of A[m][k] W[n][k]  (+ bias[n]).
// A matrix instruction takes 128 values of k, a block, into a sum of its own,
// which is added to the running one times the two scales: four multiply-adds a
// lane beside 32 cycles of the matrix unit.
//
// Up to 64 rows are bound by the bytes of W (this file): a workgroup takes 16 rows
// of W, its waves the blocks in turn, W and the rows of A straight from memory into
// the instruction's operands, several blocks on their way at once; the waves' sums
// meet in LDS. Up to 16 rows of A in 16 or 32 bits are brought into 8 bits on the
// way, by each workgroup for itself; more rows in a launch of their own. More than
// 64 rows run gemm_f8_ring.hip.
#include "gemm_f8.h"

using namespace tvk;

namespace {

constexpr int FR_WAVES = 8;
constexpr int NT4 = 12288, NT2 = 6144;   // columns

// 32 bytes of a row, of which `valid` are there (zeros behind them), at any alignment.
__device__ __forceinline__ i32x8 load32(const uint8_t* p, int valid) {
    union { Words<16> h[2]; i32x8 v; } u;
    u.v = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
    if (valid >= 32) {
        u.h[0] = load_words<16, 1>(p);
        u.h[1] = load_words<16, 1>(p + 16);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (i < valid) u.v[i / 4] |= (int)((uint32_t)p[i] << i % 4 * 8);
    }
    return u.v;
}

// The same of a row in DT, with the scale of the block that the lanes of one row share out.
template <int DT>
__device__ __forceinline__ i32x8 quantize32(const typename elem<DT>::T* p, int valid, float& scale) {
    typedef typename elem<DT>::T T;
    constexpr int VEC = 16 / (int)sizeof(T);
    float v[32];
    if (valid >= 32) {
#pragma unroll
        for (int i = 0; i < 32; i += VEC) {
            const Words<16> w = load_words<16, sizeof(T)>(p + i);
#pragma unroll
            for (int k = 0; k < VEC; ++k) v[i + k] = word_at<DT>(w, k);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = i < valid ? elem<DT>::to_f32(p[i]) : 0.0f;
    }
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[i]));
    top = fmaxf(top, __shfl_xor(top, 16));
    const F8Scale s(fmaxf(top, __shfl_xor(top, 32)));
    scale = s.s;
    i32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = (int)s.pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    return r;
}

// ADT: the type of A, TVK_F8E4M3FN with scales. MT, NT: blocks of 16 rows of A and of W; U: blocks of k on their way.
template <int ADT, int MT, int NT, int U, bool WIDE>
__global__ __launch_bounds__(64 * FR_WAVES) void gemm_f8_rows_kernel(GemmF8Args p) {
    constexpr bool IN8 = ADT == TVK_F8E4M3FN;
    static_assert(F8_BLOCK % (16 * NT) == 0, "one scale of W a workgroup and block");
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r = lane % 16, g = lane / 16, n0 = blockIdx.x * 16 * NT;
    const uint8_t* w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) w[i] = p.b + (int64_t)min(n0 + 16 * i + r, p.N - 1) * p.ldb + 32 * g;   // rows past N compute what is not stored
    const float* sb = p.sb + (int64_t)(n0 / F8_BLOCK) * p.sb_n;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int b0 = wave; b0 < p.blocks; b0 += FR_WAVES * U) {
        i32x8 fw[U][NT], fx[U][MT];
        float s[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + FR_WAVES * u;
            if (b >= p.blocks) continue;
#pragma unroll
            for (int i = 0; i < NT; ++i) fw[u][i] = load32(w[i] + (int64_t)b * F8_BLOCK, p.K - b * F8_BLOCK - 32 * g);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + FR_WAVES * u, valid = p.K - b * F8_BLOCK - 32 * g;
            if (b >= p.blocks) continue;
            const float scale = sb[(int64_t)b * p.sb_b];
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int m = min(16 * j + r, p.M - 1);   // rows past M compute what is not stored
                if constexpr (IN8) {
                    fx[u][j] = load32(static_cast<const uint8_t*>(p.a) + m * p.lda + (int64_t)b * F8_BLOCK + 32 * g, valid);
                    s[u][j] = p.sa[m * p.sa_m + b * p.sa_b] * scale;
                } else {
                    typedef typename elem<IN8 ? TVK_F32 : ADT>::T T;
                    fx[u][j] = quantize32<IN8 ? TVK_F32 : ADT>(static_cast<const T*>(p.a) + m * p.lda + (int64_t)b * F8_BLOCK + 32 * g,
                                                               valid, s[u][j]);
                    s[u][j] *= scale;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (b0 + FR_WAVES * u < p.blocks)
#pragma unroll
                for (int i = 0; i < NT; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        const f32x4 d = f8_mfma<WIDE>(fw[u][i], fx[u][j]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], s[u][j], acc[i][j][e]);
                    }
    }
    // [wave][m][n]: the waves' sums added in order
    __shared__ __attribute__((aligned(16))) float sum[FR_WAVES][MT * 16][NT * 16 + 4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(&sum[wave][16 * j + r][16 * i + 4 * g]) = acc[i][j];
    __syncthreads();
    for (int q = threadIdx.x; q < MT * 16 * NT * 16; q += 64 * FR_WAVES) {
        const int m = q / (NT * 16), c = q % (NT * 16);
        if (m >= p.M || n0 + c >= p.N) continue;
        float v = sum[0][m][c];
#pragma unroll
        for (int k = 1; k < FR_WAVES; ++k) v += sum[k][m][c];
        f8_put(p, m, n0 + c, v);
    }
}

template <int ADT, int MT, int NT, int U, bool WIDE>
void launch_rows(const GemmF8Args& p, hipStream_t s) {
    hipLaunchKernelGGL((gemm_f8_rows_kernel<ADT, MT, NT, U, WIDE>), dim3((unsigned)((p.N + 16 * NT - 1) / (16 * NT))), dim3(64 * FR_WAVES), 0, s, p);
}

template <int ADT, bool WIDE>
void few_rows(const GemmF8Args& p, hipStream_t s) {
    if (p.M <= 16) {
        if (p.N >= NT4) launch_rows<ADT, 1, 4, 2, WIDE>(p, s);
        else if (p.N >= NT2) launch_rows<ADT, 1, 2, 4, WIDE>(p, s);
        else launch_rows<ADT, 1, 1, 4, WIDE>(p, s);
    } else if constexpr (ADT == TVK_F8E4M3FN) {
        if (p.M <= 32) {
            if (p.N >= NT2) launch_rows<ADT, 2, 2, 2, WIDE>(p, s);
            else launch_rows<ADT, 2, 1, 2, WIDE>(p, s);
        } else {
            if (p.N >= NT2) launch_rows<ADT, 4, 2, 1, WIDE>(p, s);
            else launch_rows<ADT, 4, 1, 2, WIDE>(p, s);
        }
    }
}

template <int ADT>
void few_rows(const GemmF8Args& p, hipStream_t s) {
    if (p.out_dtype == TVK_F32) few_rows<ADT, true>(p, s);
    else few_rows<ADT, false>(p, s);
}

constexpr int64_t RING_MOST = 1 << 22;     // bytes from row to row, and
constexpr int64_t SCALES_MOST = 1 << 20;   // scales: a tile's offsets stay within 31 bits

// Rows that the tiled kernel's loads of 16 bytes meet.
bool ring_rows(const void* p, int64_t stride, int K) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride % 16 == 0 && stride <= RING_MOST && K % 16 == 0;
}

}  // namespace

extern "C" tvk_status tvk_gemm_f8(const tvk_gemm_f8_desc* d) {
    auto bad = [](tvk_status st, const char* m) { return fail(st, std::string("tvk_gemm_f8: ") + m); };
    if (!d) return bad(TVK_ERR_INVALID, "desc is NULL");
    const bool in8 = d->a_dtype == TVK_F8E4M3FN;
    if (!in8 && !norm_dtype(d->a_dtype)) return bad(TVK_ERR_UNSUPPORTED, "a's dtype must be float8_e4m3fn, float32, float16 or bfloat16");
    if (!norm_dtype(d->out_dtype)) return bad(TVK_ERR_UNSUPPORTED, "the output's dtype must be float32, float16 or bfloat16");
    if (d->bias_dtype != d->out_dtype && d->bias_dtype != TVK_F32)
        return bad(TVK_ERR_UNSUPPORTED, "the bias's dtype must be the output's or float32");
    if (d->M < 0 || d->N < 0 || d->K < 0) return bad(TVK_ERR_INVALID, "negative size");
    if (d->M > 0x7fffffff || d->N > 0x7fffffff || d->K > 0x7fff0000) return bad(TVK_ERR_UNSUPPORTED, "sizes below 2^31 only");
    if (d->M == 0 || d->N == 0) return TVK_OK;
    if ((d->K > 0 && (!d->a || !d->b || !d->b_scale || (in8 && !d->a_scale))) || !d->out) return bad(TVK_ERR_INVALID, "NULL tensor");
    if (d->a_stride < 0 || d->b_stride < 0 || d->a_scale_stride[0] < 0 || d->a_scale_stride[1] < 0 || d->b_scale_stride[0] < 0 ||
        d->b_scale_stride[1] < 0 || !rows_apart(d->out_stride, d->M, d->N))
        return bad(TVK_ERR_INVALID, "negative strides, or output rows that overlap");
    if (d->M > 64 && (d->a_scale_stride[0] > SCALES_MOST || d->b_scale_stride[0] > SCALES_MOST))
        return bad(TVK_ERR_UNSUPPORTED, "scales up to 2^20 from row to row only for more than 64 rows");
    if (d->M > 64 && d->K > RING_MOST) return bad(TVK_ERR_UNSUPPORTED, "K up to 2^22 only for more than 64 rows");
    if (((d->M + 127) / 128) * ((d->N + 127) / 128) > (1 << 22)) return bad(TVK_ERR_UNSUPPORTED, "more than 2^22 tiles of 128 x 128");
    GemmF8Args p{};
    p.a = d->a;
    p.b = static_cast<const uint8_t*>(d->b);
    p.sa = d->a_scale;
    p.sb = d->b_scale;
    p.bias = d->bias;
    p.out = d->out;
    p.lda = d->a_stride;
    p.ldb = d->b_stride;
    p.ldo = d->out_stride;
    p.sa_m = d->a_scale_stride[0];
    p.sa_b = d->a_scale_stride[1];
    p.sb_n = d->b_scale_stride[0];
    p.sb_b = d->b_scale_stride[1];
    p.M = (int)d->M;
    p.N = (int)d->N;
    p.K = (int)d->K;
    p.blocks = (p.K + F8_BLOCK - 1) / F8_BLOCK;
    p.out_dtype = d->out_dtype;
    p.bias32 = d->bias_dtype == TVK_F32;
    const hipStream_t s = resolve_stream(d->stream);
    const int64_t wide = (int64_t)p.blocks * F8_BLOCK;
    const bool ring = p.M > 64;
    // what has to be laid out first: rows of A in 16 or 32 bits, and for the tiled kernel rows that 16-byte loads do not meet
    const bool make_a = !in8 && p.M > 16, pad_a = ring && in8 && !ring_rows(d->a, d->a_stride, p.K);
    const bool pad_b = ring && !ring_rows(d->b, d->b_stride, p.K);
    const int splits = ring ? f8_ring_splits(p) : 1;
    Scratch scratch;
    if (splits > 1 || (p.K > 0 && (make_a || pad_a || pad_b))) {
        const int64_t bytes_a = make_a || pad_a ? p.M * wide : 0, bytes_b = pad_b ? p.N * wide : 0;
        const int64_t bytes_s = make_a ? ((int64_t)p.blocks * p.M * 4 + 15) / 16 * 16 : 0;
        p.part_n = (p.N + 3) / 4 * 4;
        const int64_t bytes_p = splits > 1 ? (int64_t)splits * p.M * p.part_n * 4 : 0;
        uint8_t* at = static_cast<uint8_t*>(scratch.get((size_t)(bytes_a + bytes_b + bytes_s + bytes_p) + 16, s));
        if (!at) return bad(TVK_ERR_OOM, "workspace allocation failed");
        if (splits > 1) p.part = reinterpret_cast<float*>(at + bytes_a + bytes_b + bytes_s);
        if (make_a) {
            float* scale = reinterpret_cast<float*>(at + bytes_a + bytes_b);
            f8_quantize_rows(d->a_dtype, d->a, d->a_stride, at, scale, p.M, p.K, s);
            p.sa = scale;
            p.sa_m = 1;
            p.sa_b = p.M;
        } else if (pad_a) {
            f8_pad_rows(static_cast<const uint8_t*>(d->a), d->a_stride, at, p.M, p.K, s);
        }
        if (bytes_a) p.a = at, p.lda = wide;
        if (pad_b) {
            f8_pad_rows(p.b, p.ldb, at + bytes_a, p.N, p.K, s);
            p.b = at + bytes_a;
            p.ldb = wide;
        }
    }
    if (ring && p.K % 16) p.K = (int)wide;   // both are copies then, with zeros up to there
    if (ring) f8_ring(p, splits, s);
    else if (in8 || make_a) few_rows<TVK_F8E4M3FN>(p, s);
    else if (d->a_dtype == TVK_F32) few_rows<TVK_F32>(p, s);
    else if (d->a_dtype == TVK_F16) few_rows<TVK_F16>(p, s);
    else few_rows<TVK_BF16>(p, s);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(TVK_ERR_DEVICE, std::string("tvk_gemm_f8: launch failed: ") + hipGetErrorString(e));
    return TVK_OK;
}
