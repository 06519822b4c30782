// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for many rows of 8-bit integers, in the large tiles of
// pingpong_tile.h (v_mfma_i32_16x16x64_i8).
//
// K may be cut over gridDim.z: the parts leave their whole-number sums, and a second kernel adds them and makes the outputs.
// Needs K % 16 == 0 and 16-byte aligned rows, K > 128; any M and N.
#include "int8_mfma.h"
#include "int8_parts.h"
#include "pingpong_tile.h"

struct PingpongInt8 {
  typedef signed char entry;
  typedef intx4 acc;
  static constexpr bool ANY_PIECES = true;
  static __device__ __forceinline__ const void* zeros() { return &int8_zeros; }
  static __device__ __forceinline__ acc multiply(u32x4 a, u32x4 b, acc c) { return mfma16_i8(a, b, c); }
};

template <bool GATED, int FM, int WGM>
__global__ __launch_bounds__(PP_WAVES * 64) void gemm_int8_large_kernel(Int8Args p) {
  int row, col;
  die_tile(blockIdx.x + blockIdx.y * gridDim.x, gridDim.y, gridDim.x, row, col);
  constexpr int TBM = WGM * FM * 32, TBN = PP_WAVES / WGM * 64;
  const int m0 = row * TBM, n0 = col * (GATED ? TBN / 2 : TBN);
  pingpong_tile<PingpongInt8, GATED, FM, WGM>(p.A, p.lda, p.W, p.W2, p.ldw, p.end.M, p.end.N, p.K, m0, n0, [&](auto& acc, int lane, int wm, int wn) {
    if (!GATED && gridDim.z > 1)
      int8_partial(acc, lane, wm, wn, m0, n0, p.partial + (size_t)blockIdx.z * p.end.M * p.end.N, p.end.M, p.end.N);
    else
      int8_epilogue<GATED, 2 * FM, 4>(acc, lane, wm, wn, m0, n0, p.end);
  });
}

template <int FM, int WGM>
static int launch_int8_large(const Int8Args& a, int parts, hipStream_t stream) {
  constexpr int TBM = WGM * FM * 32, TBN = PP_WAVES / WGM * 64;
  const int cols = a.W2 ? TBN / 2 : TBN;
  const dim3 grid((a.end.N + cols - 1) / cols, (a.end.M + TBM - 1) / TBM, parts);
  if (grid.y > 65535 || (unsigned long long)grid.x * grid.y > 0x7fffffffull) return 1;
  constexpr size_t smem = PingpongRing<FM, WGM>::BYTES;
  if (!(a.W2 ? int8_allow_lds<gemm_int8_large_kernel<true, FM, WGM>>((int)smem) : int8_allow_lds<gemm_int8_large_kernel<false, FM, WGM>>((int)smem)))
    JLLM_FAIL("gemm_int8_large: cannot reserve %zu bytes of LDS", smem);
  if (a.W2)
    gemm_int8_large_kernel<true, FM, WGM><<<grid, PP_WAVES * 64, smem, stream>>>(a);
  else
    gemm_int8_large_kernel<false, FM, WGM><<<grid, PP_WAVES * 64, smem, stream>>>(a);
  return 0;
}

// `tile`: rows * 1000 + columns of the output tile (gated: twice its outputs). `parts` > 1 cuts K into so many, in whole stages of 128 (not with
// the gated epilogue); `partial` then holds parts * M * N ints. Returns 0 when it ran, 1 when the shape is not one it takes, -1 on errors.
extern "C" int jllm_gemm_int8_large(const void* A, int lda, const float* a_scale, const void* W, int ldw, const float* w_scale, const void* W2, int ldw2,
                                    const float* w2_scale, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int K,
                                    int epilogue, float gate_limit, int tile, int parts, int* partial, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 128 || K > I8_MOST_K || (K & 15) || (lda & 15) || (ldw & 15) || (W2 && ldw2 != ldw)) return 1;
  if (((uintptr_t)A & 15) || ((uintptr_t)W & 15) || ((uintptr_t)W2 & 15)) return 1;
  JLLM_TAKE_GATE("gemm_int8_large", epilogue, gate_limit, gs);
  if (epilogue < 0 || epilogue > 2 || (epilogue == 2) != (W2 != nullptr)) JLLM_FAIL("gemm_int8_large: epilogue %d", epilogue);
  if (epilogue == 1 && out_dtype != JLLM_F32) JLLM_FAIL("gemm_int8_large: the accumulate epilogue adds into fp32");
  if (lda < 0 || ldw < 0 || ldo < N) JLLM_FAIL("gemm_int8_large: rows %d, %d and %d apart", lda, ldw, ldo);
  // a lane's place in an operand is a 32-bit byte offset from the operand's start
  if ((unsigned long long)M * (unsigned)lda >= (1ull << 32) || (unsigned long long)N * (unsigned)ldw >= (1ull << 32)) return 1;
  const int stages = (K + 127) / 128;
  if (parts < 1) parts = 1;
  if (parts > 1 && (W2 || !partial || ((uintptr_t)partial & 15))) JLLM_FAIL("gemm_int8_large: %d parts of K are not possible here", parts);
  if (parts > 65535 || (parts > 1 && stages <= (stages + parts - 1) / parts * (parts - 1))) return 1;  // a part without any
  const Int8Args a{(const signed char*)A, (const signed char*)W, (const signed char*)W2, partial, lda, ldw, K,
                   {{a_scale, w_scale, w2_scale}, bias, out, bias_dtype, out_dtype, ldo, M, N, epilogue, gs}};
  int rc;
  switch (tile) {
    case 256256: rc = launch_int8_large<4, 2>(a, parts, stream); break;
    case 192256: rc = launch_int8_large<3, 2>(a, parts, stream); break;
    case 128256: rc = launch_int8_large<2, 2>(a, parts, stream); break;
    case 256128: rc = launch_int8_large<2, 4>(a, parts, stream); break;
    default: JLLM_FAIL("gemm_int8_large: tiles of %d rows by %d columns are not built", tile / 1000, tile % 1000);
  }
  if (rc != 0) return rc;
  JLLM_CHECK_LAUNCH("gemm_int8_large");
  return parts > 1 ? int8_add_parts(partial, parts, a.end, false, stream) : 0;
}
