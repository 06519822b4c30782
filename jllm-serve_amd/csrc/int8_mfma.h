// 8-bit integers on the matrix cores, and the epilogue of their products.
//
// v_mfma_i32_16x16x64_i8: D[16x16] += A[16x64] * B[64x16] in whole numbers. Lane l holds, of A, row l%16, k (l/16)*16 .. +16; of B,
// column l%16, k (l/16)*16 .. +16; of D, rows (l/16)*4 + i (i = 0..3), column l%16. In bytes that is the layout of the bf16 form of
// half the depth (mfma.h), and it takes as many clocks.
//
// The sums are exact (up to 131,071 inputs, where 128^2 K stays below 2^31), so an output does not depend on the tile, the cut of
// K or the order in which parts are added. It is (float(sum) * a_scale[m]) * w_scale[n], and from there on what the other
// products' epilogue makes of a sum (gemm_epilogue.h).
#pragma once
#include "common.h"
#include "gemm_epilogue.h"
#include "mfma.h"

typedef int intx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ intx4 mfma16_i8(u32x4 a, u32x4 b, intx4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
}

#define I8_MOST_K 131071

struct Int8Scales {
  const float *a, *w, *w2;  // per row of A, per row of W (and of the second weight)
};

// A wave's accumulators as tile_epilogue takes them: runs [.][j] of the first weight's outputs and, gated, [.][j + CN / 2] of the second's
template <bool GATED, int RM, int CN, int TBM, int TBN>
__device__ __forceinline__ void int8_epilogue(intx4 (&acc)[RM][CN], int lane, int wm, int wn, int m0, int n0, const Int8Scales& sc, const void* bias,
                                              int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int epilogue, GateSpec gs) {
  constexpr int NI = GATED ? CN / 2 : CN;
  const int row0 = m0 + wm * RM * 16 + lane % 16, col0 = n0 + wn * NI * 16 + lane / 16 * 4;
  float sa[RM], sw[CN][4];
#pragma unroll
  for (int i = 0; i < RM; ++i) sa[i] = sc.a[min(row0 + i * 16, M - 1)];
#pragma unroll
  for (int j = 0; j < CN; ++j)
#pragma unroll
    for (int c = 0; c < 4; ++c) sw[j][c] = (GATED && j >= NI ? sc.w2 : sc.w)[min(col0 + j % NI * 16 + c, N - 1)];
  floatx4 v[RM][CN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) v[i][j][c] = ((float)acc[i][j][c] * sa[i]) * sw[j][c];
  tile_epilogue<GATED, RM, CN, TBM, TBN>(v, lane, wm, wn, m0, n0, bias, bias_dtype, out, out_dtype, ldo, M, N, epilogue, gs, nullptr, 0, 1);
}
