// Products of 8-bit floats in blocks of 128 (tvk_gemm_f8): what its files share.
#pragma once

#include "f8_blocks.h"
#include "norm_rows.h"

namespace tvk {

typedef int i32x8 __attribute__((ext_vector_type(8)));

struct GemmF8Args {
    const void* a;          // [M][K], 8-bit or, in the kernel for few rows, a_dtype
    const uint8_t* b;       // [N][K]
    const float* sa;        // [M][ceil(K / 128)], at sa_m, sa_b
    const float* sb;        // [ceil(N / 128)][ceil(K / 128)], at sb_n, sb_b
    const void* bias;       // [N], or NULL
    void* out;
    int64_t lda, ldb, ldo, sa_m, sa_b, sb_n, sb_b;
    int M, N, K, blocks;    // blocks: ceil(K / 128)
    int tiles_m, tiles_n;
    int out_dtype, bias32;
    int first_n;            // of a launch of the few-row kernel
    // of the tiled kernel
    float* part;            // [splits][M][part_n], the sums of a split K, or NULL
    int part_n, split_blocks;
};

namespace {

// One 16 x 16 block of W X^T over 128 values of k: lane l holds 32 bytes of row l % 16 of each, the lanes of a row sharing a
// block out, and gets rows 4 (l / 16) .. + 3 (of W) of column l % 16 (a row of X).
//
// WIDE: in bfloat16, which holds an 8-bit value exactly, at half the rate. The 8-bit instructions align the products of
// eight neighbouring values of k to the largest of them and cut them off towards zero about 2^-13 below it: measured against
// sums in 64 bits, 1.5e-5 to 4e-5 of the result (root mean square over random operands of like and very unlike sizes). That is
// a tenth of what rounding to float16 leaves and nothing beside bfloat16's, but a float32 result would be left with 14 bits.
// Zeros in place of scales: the instruction without them.
template <bool WIDE>
__device__ __forceinline__ f32x4 f8_mfma(i32x8 w, i32x8 x) {
    f32x4 d{0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (!WIDE) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, d, 0, 0, 0, 0, 0, 0);
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    auto widen = [](int lo, int hi) {
        union { bf16x2 h[4]; bf16x8 v; } u;
        u.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, false);
        u.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)lo, 1.0f, true);
        u.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, false);
        u.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)hi, 1.0f, true);
        return u.v;
    };
#pragma unroll
    for (int i = 0; i < 8; i += 2)
        d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(w[i], w[i + 1]), widen(x[i], x[i + 1]), d, 0, 0, 0);
    return d;
}

template <int DT>
__device__ __forceinline__ float f8_bias(const GemmF8Args& p, int n) {
    return p.bias32 ? static_cast<const float*>(p.bias)[n] : at<DT>(p.bias, n);
}

// Stores one output from its float32 sum.
__device__ __forceinline__ void f8_put(const GemmF8Args& p, int64_t m, int n, float v) {
    const int64_t o = m * p.ldo + n;
    if (p.out_dtype == TVK_F32) {
        static_cast<float*>(p.out)[o] = p.bias ? v + f8_bias<TVK_F32>(p, n) : v;
    } else if (p.out_dtype == TVK_F16) {
        put<TVK_F16>(p.out, o, p.bias ? v + f8_bias<TVK_F16>(p, n) : v);
    } else {
        put<TVK_BF16>(p.out, o, p.bias ? v + f8_bias<TVK_BF16>(p, n) : v);
    }
}

}  // namespace

// Rows in 16 or 32 bits as 8-bit rows of whole blocks, zeros behind them; scale [ceil(cols / 128)][rows].
void f8_quantize_rows(int dtype, const void* x, int64_t x_stride, uint8_t* out, float* scale, int64_t rows, int64_t cols, hipStream_t s);
// 8-bit rows copied to rows of whole blocks, zeros behind them.
void f8_pad_rows(const uint8_t* x, int64_t x_stride, uint8_t* out, int64_t rows, int64_t cols, hipStream_t s);

// Queues the tiled kernel: 16-byte aligned 8-bit rows, K a multiple of 16. Of `splits` parts of K, which f8_ring_splits
// suggests, the sums go to p.part and are joined by a second launch.
int f8_ring_splits(const GemmF8Args& p);
void f8_ring(const GemmF8Args& p, int splits, hipStream_t s);

}  // namespace tvk
