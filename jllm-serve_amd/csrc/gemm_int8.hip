// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for rows of 8-bit integers of any sizes, at any alignment and with
// any distance between rows: the general form of the product.
//
// A workgroup of four waves (2 x 2) owns 64 x 64 outputs (gated: 64 x 32, both weights'), a wave 2 x 2 accumulators of 16 x 16. K
// advances in stages of 128 through registers into two LDS buffers: 16 bytes a lane wherever the row begins (unaligned accesses are
// one load each), the last pieces of a row byte by byte, and zeros behind its end.
#include "int8_mfma.h"

#define G8_BK 128
#define G8_PITCH 144  // bytes of a row in LDS: 16 lanes that read one piece of 16 rows meet no bank twice in a turn

struct Gemm8Args {
  const signed char *A, *W, *W2;
  int lda, ldw, ldw2, K;
  Int8Epilogue end;
};

template <bool GATED>
__global__ __launch_bounds__(256) void gemm_int8_kernel(Gemm8Args p) {
  constexpr int TBM = 64, TBN = 64, COLS = GATED ? 32 : 64;
  const int M = p.end.M, N = p.end.N;
  __shared__ __align__(16) unsigned char lds[2][(TBM + TBN) * G8_PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, wm = wave >> 1, wn = wave & 1;
  const int m0 = blockIdx.y * TBM, n0 = blockIdx.x * COLS;
  // 128 rows of 8 pieces in a stage: thread t has piece t % 8 of rows t / 8, + 32, + 64 (the weights' first), + 96
  const int piece = tid & 7;
  const signed char* from[4];
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int r = (tid >> 3) + (c & 1) * 32;
    if (c < 2) {
      from[c] = p.A + (size_t)min(m0 + r, M - 1) * p.lda;
    } else {  // gated: of a wave's two blocks of 16 the first is gate rows, the second the up rows of the same outputs
      const bool second = GATED && (r & 16);
      const int n = GATED ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
      from[c] = (second ? p.W2 : p.W) + (size_t)min(n, N - 1) * (second ? p.ldw2 : p.ldw);
    }
  }
  u32x4 held[4];
  auto fetch = [&](int t) {
    const int k = t * G8_BK + piece * 16;
    if (k + 16 <= p.K) {
#pragma unroll
      for (int c = 0; c < 4; ++c) __builtin_memcpy(&held[c], from[c] + k, 16);
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (k + e < p.K) w[e >> 2] |= (uint32_t)(unsigned char)from[c][k + e] << (e & 3) * 8;
        held[c] = u32x4{w[0], w[1], w[2], w[3]};
      }
    }
  };
  auto put = [&](int buffer) {
#pragma unroll
    for (int c = 0; c < 4; ++c) *(u32x4*)(lds[buffer] + ((tid >> 3) + c * 32) * G8_PITCH + piece * 16) = held[c];
  };
  intx4 acc[2][2] = {};
  const int stages = (p.K + G8_BK - 1) / G8_BK;
  fetch(0);
  put(0);
  for (int t = 0; t < stages; ++t) {
    __syncthreads();
    if (t + 1 < stages) fetch(t + 1);
    const unsigned char* s = lds[t & 1] + (lane & 15) * G8_PITCH + (lane >> 4) * 16;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      u32x4 a[2], w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        a[i] = *(const u32x4*)(s + (wm * 32 + i * 16) * G8_PITCH + kk * 64);
        w[i] = *(const u32x4*)(s + (TBM + wn * 32 + i * 16) * G8_PITCH + kk * 64);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma16_i8(w[j], a[i], acc[i][j]);
    }
    if (t + 1 < stages) put((t + 1) & 1);
  }
  int8_epilogue<GATED, 2, 2>(acc, lane, wm, wn, m0, n0, p.end);
}

extern "C" int jllm_gemm_int8(const void* A, int lda, const float* a_scale, const void* W, int ldw, const float* w_scale, const void* W2, int ldw2,
                              const float* w2_scale, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int K,
                              int epilogue, float gate_limit, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > I8_MOST_K) JLLM_FAIL("gemm_int8: %d inputs (1 to %d: beyond, the sums could leave 32 bits)", K, I8_MOST_K);
  JLLM_TAKE_GATE("gemm_int8", epilogue, gate_limit, gs);
  if (epilogue < 0 || epilogue > 2 || (epilogue == 2) != (W2 != nullptr)) JLLM_FAIL("gemm_int8: epilogue %d", epilogue);
  if (epilogue == 1 && out_dtype != JLLM_F32) JLLM_FAIL("gemm_int8: the accumulate epilogue adds into fp32");
  if (lda < 0 || ldw < 0 || ldw2 < 0 || ldo < N) JLLM_FAIL("gemm_int8: rows %d, %d and %d apart", lda, ldw, ldo);
  const dim3 grid(W2 ? (N + 31) / 32 : (N + 63) / 64, (M + 63) / 64);
  if (grid.y > 65535) JLLM_FAIL("gemm_int8: %d rows are more than a grid takes", M);
  const Gemm8Args a{(const signed char*)A, (const signed char*)W, (const signed char*)W2, lda, ldw, ldw2, K,
                    {{a_scale, w_scale, w2_scale}, bias, out, bias_dtype, out_dtype, ldo, M, N, epilogue, gs}};
  if (W2)
    gemm_int8_kernel<true><<<grid, 256, 0, stream>>>(a);
  else
    gemm_int8_kernel<false><<<grid, 256, 0, stream>>>(a);
  JLLM_CHECK_LAUNCH("gemm_int8");
  return 0;
}
