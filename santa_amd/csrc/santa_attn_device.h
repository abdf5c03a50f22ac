// santa_attn_device.h -- gfx950 primitives shared by the exact attention
// kernels: matrix instructions on 16-bit fragments, the transposing LDS read,
// and the constants of their running maxima.
#pragma once

#include <type_traits>

#include "santa_device.h"

namespace santa {
namespace attn {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
struct Half8 {
  typedef __bf16 T __attribute__((ext_vector_type(8)));
};
template <>
struct Half8<false> {
  typedef _Float16 T __attribute__((ext_vector_type(8)));
};

// Eight 16-bit values travel as u32x4: the kernels' own code names no 16-bit
// vector type, which the host pass does not have.
template <bool BF16>
__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
  typedef typename Half8<BF16>::T H8;
  if constexpr (BF16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(H8, a), __builtin_bit_cast(H8, b), c, 0, 0, 0);
  }
}

// Eight floats rounded to nearest even into the 16-bit type.
template <bool BF16>
__device__ __forceinline__ u32x4 pack8(const float (&e)[8]) {
  typedef typename Half8<BF16>::T H8;
  H8 v;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = static_cast<std::remove_reference_t<decltype(v[0])>>(e[i]);
  return __builtin_bit_cast(u32x4, v);
}

// v of lane i ^ 32.
__device__ __forceinline__ float other_half(float v) {
  const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float((threadIdx.x & 32) ? s[0] : s[1]);
}

// This lane's column of two 4-row groups of a row-major 16-bit LDS tile, 8
// rows of ROW bytes apart, through the transposing read: in each 16-lane
// group, lane i passes the address of 4 elements of row i / 4 and receives
// the 4 rows' elements of column i.
template <int ROW>
__device__ __forceinline__ u32x4 read_tr8(const char* p) {
  typedef __attribute__((address_space(3))) s16x4* lds4;
  struct Two {
    s16x4 a, b;
  };
  const Two f = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p)),
                 __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 8 * ROW))};
  return __builtin_bit_cast(u32x4, f);
}

// Where running maxima start: below every finite score, so that scores of -inf
// (masked through K) weigh nothing as long as one key of the query is finite;
// relative to a maximum of -inf they would be NaN.
constexpr float kLowest = -3.402823466e38f;

// Above this a maximum in log2 units is subtracted from the scores before they
// are scaled: fma(score, scale, -round(max * scale)) is off by half an ulp of
// the product, up to a factor 2^(1/4) common to a query's probabilities here but
// an overflow from 2^31 on (scores from about 2e10).
constexpr float kHugeMax = 4194304.0f;

}  // namespace attn
}  // namespace santa
