// 8-bit floats (e4m3fn) in blocks with a float32 scale each: how every kernel
// that makes them takes a block's scale and rounds its values, so that all that
// are given the same values give the same bits.
#pragma once

#include "words.h"

namespace tvk {

constexpr int F8_BLOCK = 128;   // columns of a block

// The least scale: 64 of the smallest float32's steps. A scale of fewer is off by so much of itself, or 0, that the block's
// largest value would be past 464, which is NaN. Values up to 448 times it are whole steps of 2^-6 over it.
constexpr float F8_LEAST_SCALE = 0x1p-143f;

// What a block's values are multiplied and divided by: the scale is the block's largest magnitude (NaN aside) over 448, the
// least one or more, and values go times its reciprocal. A scale whose reciprocal leaves float32's range is divided by.
struct F8Scale {
    float s, mul, div;
    __device__ explicit F8Scale(float top) {
        s = top > 0.0f ? fmaxf(top / 448.0f, F8_LEAST_SCALE) : 1.0f;
        const float r = 1.0f / s;
        const bool plain = r < 1e30f && r > 1e-30f;
        mul = plain ? r : 1.0f;
        div = plain ? 1.0f : s;
    }
    __device__ bool plain() const { return div == 1.0f; }
    // The largest of a block may come out above 448, by half a float32 step or, of a scale below float32's normal range, by as
    // much as that is off, 2^-7 of it at most: it rounds to 448.
    __device__ uint32_t pack4(float a, float b, float c, float d) const {
        a *= mul, b *= mul, c *= mul, d *= mul;
        if (!plain()) a /= div, b /= div, c /= div, d /= div;
        return pack4_f8(a, b, c, d);
    }
    // The same of quotients that are off by what a division's rounding leaves: where the values are a float32 result's own and
    // not a tensor's, each rounding on the way to 8 bits sends some to the other neighbour. (The remainder is exact.)
    __device__ uint32_t divide4(float a, float b, float c, float d) const {
        if (!plain()) return pack4(a, b, c, d);
        auto over = [&](float v) {
            const float q = v * mul;
            return fmaf(fmaf(-q, s, v), mul, q);
        };
        return pack4_f8(over(a), over(b), over(c), over(d));
    }
    __device__ uint8_t divide1(float a) const { return (uint8_t)divide4(a, 0.0f, 0.0f, 0.0f); }
};

// Whether no two places of a [rows, cols] array with these strides, in elements, are the same.
inline bool apart2(const int64_t* stride, int64_t rows, int64_t cols) {
    const int64_t a = stride[0], b = stride[1];
    if ((rows > 1 && a < 1) || (cols > 1 && b < 1)) return false;
    if (rows <= 1 || cols <= 1) return true;
    auto past = [](int64_t outer, int64_t inner, int64_t n) { return outer / inner >= n || (outer / inner == n - 1 && outer % inner); };
    return past(a, b, cols) || past(b, a, rows);
}

}  // namespace tvk
