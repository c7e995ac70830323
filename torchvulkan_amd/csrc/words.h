// Runs of a row's values as 32-bit words, at any alignment of a value: what the
// kernels that stream rows of any length and place load, compute on and store.
#pragma once

#include "convert.h"

namespace tvk {

template <int BYTES>
struct Words {
    uint32_t w[BYTES / 4];
};

// BYTES (a multiple of 4) at a multiple of ALIGN: one access, global memory takes any alignment.
template <int BYTES, int ALIGN>
__device__ __forceinline__ Words<BYTES> load_words(const void* p) {
    typedef uint32_t V __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN)));
    const V v = *static_cast<const V*>(p);
    Words<BYTES> r;
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) r.w[i] = v[i];
    return r;
}

template <int BYTES, int ALIGN>
__device__ __forceinline__ void store_words(void* p, const Words<BYTES>& r) {
    typedef uint32_t V __attribute__((ext_vector_type(BYTES / 4), aligned(ALIGN)));
    V v;
#pragma unroll
    for (int i = 0; i < BYTES / 4; ++i) v[i] = r.w[i];
    *static_cast<V*>(p) = v;
}

// Two floats rounded to nearest even into a packed pair (v_cvt_pk_f16_f32, v_cvt_pk_bf16_f32).
template <int DT>
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    if constexpr (DT == TVK_F16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, f16x2));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

// Value i of a run of DT (float32, float16, bfloat16).
template <int DT, int BYTES>
__device__ __forceinline__ float word_at(const Words<BYTES>& r, int i) {
    if constexpr (DT == TVK_F32) return __builtin_bit_cast(float, r.w[i]);
    else return elem<DT>::to_f32(__builtin_bit_cast(typename elem<DT>::T, (uint16_t)(i % 2 ? r.w[i / 2] >> 16 : r.w[i / 2])));
}

template <int DT, int VEC>
__device__ __forceinline__ Words<VEC * (DT == TVK_F32 ? 4 : 2)> pack(const float (&f)[VEC]) {
    Words<VEC * (DT == TVK_F32 ? 4 : 2)> r;
    if constexpr (DT == TVK_F32) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.w[i] = __builtin_bit_cast(uint32_t, f[i]);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; i += 2) r.w[i / 2] = pack_pair<DT>(f[i], f[i + 1]);
    }
    return r;
}

// Four floats within +-448 (or NaN) as e4m3fn, rounded to nearest even.
__device__ __forceinline__ uint32_t pack4_f8(float a, float b, float c, float d) {
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false), true);
}

}  // namespace tvk
