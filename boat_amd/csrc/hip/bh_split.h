// bh_split.h - fp32 products on the bf16 matrix cores, without giving up fp32's precision (internal).
//
// A float has 24 significant bits, a bf16 has 8 and the same exponent range, so x = h + m + l with three bf16 exactly:
//   h = bf16(x), m = bf16(x - h), l = bf16(x - h - m)      (round to nearest; both differences are exact in fp32).
// Of the nine partial products of a*b the six largest are kept,
//   a*b ~ ah*bh + (ah*bm + am*bh) + (ah*bl + am*bm + al*bh),
// each exact in the matrix core's fp32 accumulator (8 x 8 bits).  What is dropped, am*bl + al*bm + al*bl, is below
// 2 * 2^-9 * 2^-18 + 2^-36 < 2^-25 of |a*b|: half of what rounding the product itself to fp32 may cost (2^-24).  So the sums
// are fp32 sums, and six v_mfma_f32_32x32x16_bf16 take 192 cycles of a SIMD for what takes v_mfma_f32_32x32x2_f32 512.
//
// Where the split does not hold it shows: an infinity leaves NaN in its remainders, and any sum it enters ends as NaN.  So does a
// finite value past the largest bf16 (3.3895e38; from 3.396e38 on the first part would be an infinity) unless the first part is
// kept to that bf16 (WIDE), which takes one instruction more a value; the remainder is then still exact.  What the kernels make of it: the dense
// product looks for sums that are not finite and makes those again in plain fp32 arithmetic from memory, so infinities and NaN
// come out as fp32 arithmetic gives them; attention splits its operands WIDE, and an infinity in them ends as NaN.  The parts of
// values below 2^-110 become subnormal; the matrix cores keep subnormals.
#pragma once

#include "bh_common.h"

namespace bh {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int kPlanes = 3;   // h, m, l

// two floats to their three packed bf16 pairs
template <bool WIDE = false>
__device__ __forceinline__ void split_pair(float x, float y, unsigned& h, unsigned& m, unsigned& l) {
    constexpr float kMost = 3.38953139e38f;      // the largest bf16
    const f32x2 first = WIDE ? (f32x2){__builtin_amdgcn_fmed3f(x, -kMost, kMost), __builtin_amdgcn_fmed3f(y, -kMost, kMost)} : (f32x2){x, y};
    h = __builtin_bit_cast(unsigned, __builtin_convertvector(first, bf16x2));
    const float rx = x - __uint_as_float(h << 16), ry = y - __uint_as_float(h & 0xffff0000u);
    m = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){rx, ry}, bf16x2));
    const float sx = rx - __uint_as_float(m << 16), sy = ry - __uint_as_float(m & 0xffff0000u);
    l = __builtin_bit_cast(unsigned, __builtin_convertvector((f32x2){sx, sy}, bf16x2));
}

// eight floats, consecutive in the contraction index, to a lane's fragment in each plane
template <bool WIDE = false>
__device__ __forceinline__ void split_eight(const float (&x)[8], u32x4 (&p)[kPlanes]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        unsigned h, m, l;
        split_pair<WIDE>(x[2 * i], x[2 * i + 1], h, m, l);
        p[0][i] = h; p[1][i] = m; p[2][i] = l;
    }
}

__device__ __forceinline__ f32x16 mfma_bf16(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// c += a . b over 16 of the contraction, smallest partial products first
__device__ __forceinline__ f32x16 mfma_split(const u32x4 (&a)[kPlanes], const u32x4 (&b)[kPlanes], f32x16 c) {
    c = mfma_bf16(a[1], b[1], c);
    c = mfma_bf16(a[0], b[2], c);
    c = mfma_bf16(a[2], b[0], c);
    c = mfma_bf16(a[0], b[1], c);
    c = mfma_bf16(a[1], b[0], c);
    c = mfma_bf16(a[0], b[0], c);
    return c;
}

// row of a lane's accumulator element i in a 32x32 product (its column is lane & 31)
__device__ __forceinline__ int acc_row(int i, int lane) { return 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3); }

}  // namespace bh
