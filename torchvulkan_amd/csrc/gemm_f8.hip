// Products of 8-bit floats with a scale for each block of 128 (tvk_gemm_f8):
//   out[m][n] = sum over blocks b of sa[m][b] sb[n / 128][b] sum over k in b of A[m][k] W[n][k]  (+ bias[n]).
// A matrix instruction takes 128 values of k, a block, into a sum of its own,
// which is added to the running one times the two scales: four multiply-adds a
// lane beside 32 cycles of the matrix unit.
//
// Up to 64 rows are bound by the bytes of W (this file): a workgroup takes 16 rows
// of W, or up to 64, its waves the blocks in turn, W and the rows of A straight from
// memory into the instruction's operands, several blocks on their way at once; the
// waves' sums meet in LDS. Up to 16 rows of A in 16 or 32 bits are brought into 8
// bits on the way, by each workgroup for itself; more rows in a launch of their
// own. More than 64 rows, and from 17 on those of long k, run gemm_f8_ring.hip.
//
// Measured, W from memory and, in brackets, from its cache: 1 x 14336 x 4096 13.5
// (12.4) us in 8 bits and 15.8 (11.4) from bfloat16 (11.3 for W's bytes at 5.2 TB/s, 3
// for a launch); 16 x 14336 x 4096 15.8 (13.3) and 17.2 (15.2); 1 x 8192 x 8192 13.9
// (12.9) and 17.2 (16.4); 64 x 14336 x 4096 22.3 (21.0) and 25.4 (24.0); 50 x 5000 x
// 4100, no row on 16 bytes, 16.5 (14.1), and 18.4 (17.2) from float16 with the launch
// that brings it into 8 bits.
// Loads on their way over the end of a loop's turn, with a next set of registers,
// were slower, 16.9 us for 15.1: a wave has four blocks of 4096 values in all.
#include "gemm_f8.h"

using namespace tvk;

namespace {

constexpr int FR_WAVES = 8;
// Past so many columns a workgroup takes 2 blocks of 16 rows of W, and 4, so that all workgroups make one round on the CUs, and
// the rows of A are read, and brought into 8 bits, less often. 16 rows from bfloat16 by 14336 x 4096, 1, 2 and 4 blocks: 34.1,
// 23.6 and 17.3 us; by 8192 x 4096 18.4, 12.1 and 15.3; by 4096 x 4096 10.3, 11.7 and 14.7. 50 rows by 5000 x 4100 21.6 and 14.8
// of 1 and 2.
constexpr int NT2 = 4096, NT4 = 8192;

// A lane's 32 values of a block of k, of A and of W alike, whose order does not matter to the sum: 16 of the first
// half and 16 of the second, so that the four lanes of a row load 64 bytes side by side.
__device__ __forceinline__ int half_at(int g, int half) { return 64 * half + 16 * g; }

// They of a row of bytes at any alignment, of a whole block.
__device__ __forceinline__ i32x8 load32(const uint8_t* block, int g) {
    union { Words<16> h[2]; i32x8 v; } u;
#pragma unroll
    for (int h = 0; h < 2; ++h) u.h[h] = load_words<16, 1>(block + half_at(g, h));
    return u.v;
}

// The same from `at` on in a row of K bytes, with zeros behind its end: the last 16 of the row, moved down, or where it
// has fewer, one after the other.
__device__ __forceinline__ i32x8 load_rest(const uint8_t* row, int at, int g, int K) {
    i32x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (K >= 16) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int k = at + half_at(g, h), from = min(k, K - 16), by = k - from;
            Words<16> w = load_words<16, 1>(row + from);
#pragma unroll
            for (int step = 2; step >= 1; step /= 2)   // words, then the bytes of one
#pragma unroll
                for (int i = 0; i < 4; ++i) w.w[i] = by & 4 * step ? (i + step < 4 ? w.w[i + step] : 0u) : w.w[i];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[4 * h + i] = by < 16 ? (int)__builtin_amdgcn_alignbyte(i < 3 ? w.w[i + 1] : 0u, w.w[i], (uint32_t)by % 4) : 0;
        }
    } else {
#pragma unroll 1
        for (int i = 0; i < 16; ++i) {
            const int k = half_at(g, 0) + i, byte = k < K ? row[k] : 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] |= i / 4 == q ? byte << i % 4 * 8 : 0;
        }
    }
    return v;
}

// How a wave has its rows of A: in 8 bits with scales; in wider types, 32 values a lane, each lane those of its
// operand; the same for up to 4 rows, 8 values a lane, handed round afterwards (a quarter of the arithmetic, which
// bounds few columns of a long k: 1 x 4096 x 14336 from bfloat16 15.8 us, each lane its own 24.4).
enum { X_F8, X_OWN, X_SHARED };

// What a lane loads of one block of A, and the operands that become of it.
template <int ADT, int FORM, int MT>
struct XBlock {
    typedef typename elem<FORM == X_F8 ? TVK_F32 : ADT>::T T;
    static constexpr int DT = FORM == X_F8 ? TVK_F32 : ADT, VALUES = FORM == X_OWN ? 32 : 8, VEC = 16 / (int)sizeof(T);
    i32x8 x[FORM == X_F8 ? MT : 1];
    float s[MT];
    Words<16> raw[VALUES / VEC];

    // Block b, all 128 values of it; rows past M compute what is not stored.
    __device__ __forceinline__ void load(const GemmF8Args& p, int lane, int b) {
        if constexpr (FORM == X_F8) {
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const int m = min(16 * j + lane % 16, p.M - 1);
                x[j] = load32(static_cast<const uint8_t*>(p.a) + m * p.lda + (int64_t)b * F8_BLOCK, lane / 16);
                s[j] = p.sa[m * p.sa_m + b * p.sa_b];
            }
        } else {
            const int m = min(FORM == X_OWN ? lane % 16 : lane / 16, p.M - 1);
            const T* block = static_cast<const T*>(p.a) + m * p.lda + (int64_t)b * F8_BLOCK;
#pragma unroll
            for (int i = 0; i < VALUES; i += VEC)
                raw[i / VEC] = load_words<16, sizeof(T)>(block + (FORM == X_OWN ? half_at(lane / 16, i / 16) + i % 16 : lane % 16 * 8 + i));
        }
    }

    // The same of a last block that is not whole.
    __device__ __forceinline__ void load_rest(const GemmF8Args& p, int lane, int b) {
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int m = min(16 * j + lane % 16, p.M - 1);
            if constexpr (FORM == X_F8) {
                x[j] = ::load_rest(static_cast<const uint8_t*>(p.a) + m * p.lda, b * F8_BLOCK, lane / 16, p.K);
                s[j] = p.sa[m * p.sa_m + b * p.sa_b];
            } else {
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const int k = b * F8_BLOCK + half_at(lane / 16, i / 16) + i % 16;
                    v[i] = elem<DT>::to_f32(static_cast<const T*>(p.a)[m * p.lda + min(k, p.K - 1)]);
                    v[i] = k < p.K ? v[i] : 0.0f;
                }
                quantize(v);
            }
        }
    }

    // 32 values a lane, with the scale of the block that the four lanes of one row share out.
    __device__ __forceinline__ void quantize(const float (&v)[32]) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[i]));
        top = fmaxf(top, __shfl_xor(top, 16));
        const F8Scale to(fmaxf(top, __shfl_xor(top, 32)));
        s[0] = to.s;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[0][i] = (int)to.pack4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }

    // Makes x and s of what load() brought.
    __device__ __forceinline__ void make(int lane) {
        if constexpr (FORM == X_OWN) {
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = word_at<DT>(raw[i / VEC], i % VEC);
            quantize(v);
        } else if constexpr (FORM == X_SHARED) {
            float v[8], top = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = word_at<DT>(raw[i / VEC], i % VEC), top = fmaxf(top, fabsf(v[i]));
#pragma unroll
            for (int i = 1; i < 16; i *= 2) top = fmaxf(top, __shfl_xor(top, i));
            const F8Scale to(top);
            const int lo = (int)to.pack4(v[0], v[1], v[2], v[3]), hi = (int)to.pack4(v[4], v[5], v[6], v[7]);
            const int from = lane % 4 * 16;   // lanes of the row that this lane's operand holds; its copies past 4 rows are not stored
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lane_of = from + (half_at(lane / 16, i / 2) + 8 * (i % 2)) / 8;
                x[0][2 * i] = __shfl(lo, lane_of);
                x[0][2 * i + 1] = __shfl(hi, lane_of);
            }
            s[0] = __shfl(to.s, from);
        }
    }
};

// ADT: the type of A. MT, NT: blocks of 16 rows of A and of W; U: blocks of k on their way.
template <int ADT, int FORM, int MT, int NT, int U, bool WIDE>
__global__ __launch_bounds__(64 * FR_WAVES, MT == 4 && NT == 1 ? 4 : 1) void gemm_f8_rows_kernel(GemmF8Args p) {
    static_assert(F8_BLOCK % (16 * NT) == 0, "one scale of W a workgroup and block");
    static_assert(FORM == X_F8 || MT == 1, "16 rows of A in wider types");
    const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const int r = lane % 16, g = lane / 16, n0 = p.first_n + blockIdx.x * 16 * NT;
    const uint8_t* w[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) w[i] = p.b + (int64_t)min(n0 + 16 * i + r, p.N - 1) * p.ldb;   // rows past N compute what is not stored
    const float* sb = p.sb + (int64_t)(n0 / F8_BLOCK) * p.sb_n;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    struct Block {
        i32x8 w[NT];
        XBlock<ADT, FORM, MT> x;
        float s;
    };
    auto add = [&](const Block& k) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) {
                const f32x4 d = f8_mfma<WIDE>(k.w[i], k.x.x[j]);
                const float scale = k.x.s[j] * k.s;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[e], scale, acc[i][j][e]);
            }
    };
    const int full = p.K / F8_BLOCK;
    for (int b0 = wave; b0 < full; b0 += FR_WAVES * U) {
        Block on[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = b0 + FR_WAVES * u;
            if (b >= full) continue;
#pragma unroll
            for (int i = 0; i < NT; ++i) on[u].w[i] = load32(w[i] + (int64_t)b * F8_BLOCK, g);
            on[u].x.load(p, lane, b);
            on[u].s = sb[(int64_t)b * p.sb_b];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (b0 + FR_WAVES * u >= full) continue;
            on[u].x.make(lane);
            add(on[u]);
        }
    }
    if (full < p.blocks && wave == full % FR_WAVES) {
        Block k;
#pragma unroll
        for (int i = 0; i < NT; ++i) k.w[i] = load_rest(w[i], full * F8_BLOCK, g, p.K);
        k.x.load_rest(p, lane, full);
        k.s = sb[(int64_t)full * p.sb_b];
        add(k);
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

template <int ADT, int FORM, int MT, int NT, int U, bool WIDE>
void launch_rows(GemmF8Args p, hipStream_t s) {
    // 2^32 threads in a dimension of a grid are too many; with a second dimension 50 x 5000 x 4100 took 0.7 us more
    constexpr int64_t MOST = 1 << 20;
    for (int64_t n = 0; n < p.N; n += MOST * 16 * NT) {
        p.first_n = (int)n;
        const int64_t groups = std::min<int64_t>(MOST, (p.N - n + 16 * NT - 1) / (16 * NT));
        hipLaunchKernelGGL((gemm_f8_rows_kernel<ADT, FORM, MT, NT, U, WIDE>), dim3((unsigned)groups), dim3(64 * FR_WAVES), 0, s, p);
    }
}

template <int ADT, int FORM, bool WIDE>
void rows_16(const GemmF8Args& p, hipStream_t s) {
    if (p.N > NT4) launch_rows<ADT, FORM, 1, 4, 2, WIDE>(p, s);
    else if (p.N > NT2) launch_rows<ADT, FORM, 1, 2, 4, WIDE>(p, s);
    else launch_rows<ADT, FORM, 1, 1, 4, WIDE>(p, s);
}

template <int ADT, bool WIDE>
void few_rows(const GemmF8Args& p, hipStream_t s) {
    constexpr bool IN8 = ADT == TVK_F8E4M3FN;
    if (p.M <= 4) {
        // from wider types 4 blocks of W a workgroup for as many columns as with more rows, where those make one round on the CUs.
        // 1 row of bfloat16, W from memory and, in brackets, from its cache: by 8192 x 4096 10.2 (8.0) us with one block and 11.5
        // (10.4) with four, by 8704 x 4096 12.4 (10.6) and 11.6 (10.5), by 14336 x 4096 15.6 (14.5) and 15.8 (11.4), by 14336 x
        // 14336 42.8 (37.3) and 37.7 (31.1), by 16384 x 4096 16.1 (14.7) and 17.5 (12.9), the most that it loses; two rounds, by
        // 20480 x 4096, 19.8 (18.1) and 25.7 (21.4).
        const int groups = (p.N + 63) / 64;
        if (!IN8 && p.N > NT4 && groups <= 256) launch_rows<ADT, IN8 ? X_F8 : X_SHARED, 1, IN8 ? 1 : 4, IN8 ? 4 : 2, WIDE>(p, s);
        else launch_rows<ADT, IN8 ? X_F8 : X_SHARED, 1, 1, 4, WIDE>(p, s);
    } else if (p.M <= 16) {
        rows_16<ADT, IN8 ? X_F8 : X_OWN, WIDE>(p, s);
    } else if constexpr (!IN8) {
        return;   // (8 bits by now)
    } else if (p.M <= 32) {
        if (p.N > NT4) launch_rows<ADT, X_F8, 2, 4, 1, WIDE>(p, s);
        else if (p.N > NT2) launch_rows<ADT, X_F8, 2, 2, 2, WIDE>(p, s);
        else launch_rows<ADT, X_F8, 2, 1, 2, WIDE>(p, s);
    } else {
        if (p.N > NT4) launch_rows<ADT, X_F8, 4, 4, 1, WIDE>(p, s);
        else if (p.N > NT2) launch_rows<ADT, X_F8, 4, 2, 1, WIDE>(p, s);
        else launch_rows<ADT, X_F8, 4, 1, 1, WIDE>(p, s);
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

// Where up to 64 rows run the tiled kernel too, rows that it can load as they lie: a workgroup of the other takes all of k for
// its rows of A, this splits k, and joins the sums in a launch of its own. Tiled against rows: 64 x 4096 x 4096 16.2 and 15.9 us,
// 64 x 4096 x 14336 23.8 and 46.1, 20 x 4096 x 14336 19.8 and 23.5, 48 x 8192 x 6144 20.4 and 22.1; 32 x 8192 x 6144 19.2 and
// 17.5, 20 x 14336 x 4096 20.7 and 16.2, 64 x 1024 x 1024 10.1 and 5.6.
bool tiles_pay(const GemmF8Args& p, const tvk_gemm_f8_desc* d) {
    return p.M > 16 && (int64_t)p.M * p.K >= 1 << 18 && p.K % 16 == 0 && p.K <= RING_MOST &&
           p.sa_m <= SCALES_MOST && p.sb_n <= SCALES_MOST && ring_rows(p.b, p.ldb, p.K) &&
           (d->a_dtype != TVK_F8E4M3FN || ring_rows(d->a, d->a_stride, p.K));
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
    if (((d->M + 127) / 128) * ((d->N + 127) / 128) >= (1 << 22)) return bad(TVK_ERR_UNSUPPORTED, "2^22 tiles of 128 x 128 or more");
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
    const bool ring = p.M > 64 || tiles_pay(p, d);
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
