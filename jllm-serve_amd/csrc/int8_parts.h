// Products of 8-bit integers whose K is cut over workgroups: the parts' whole-number sums in memory and the kernel that adds them.
#pragma once
#include "int8_mfma.h"

// what the tiled kernels take
struct Int8Args {
  const signed char *A, *W, *W2;
  int* partial;  // [part][weight][M][N]
  int lda, ldw, K;
  Int8Epilogue end;
};

// Which tile workgroup b of rows x cols takes: workgroups b, b + 8, b + 16 .. share a die, which gets a run of neighbouring tiles, in
// bands of eight columns, row by row inside a band, so that its L2 passes on fewer operands. us, bands of 2 / 4 / 8 / 16: 4,608 x 17,408 x 5,120
// gated in tiles of 256 x 256 639 / 632 / 624 / 629, 8,192 rows 1,115 / 1,094 / 1,085 / 1,104 (all before the outputs took less); at most sizes the
// same.
#define I8_BAND 8
__device__ __forceinline__ void int8_die_tile(int b, int rows, int cols, int& row, int& col) {
  const int tiles = rows * cols, each = tiles >> 3, more = tiles & 7, die = b & 7;
  const int i = die * each + min(die, more) + (b >> 3);
  const int band = i / (I8_BAND * rows), r = i - band * I8_BAND * rows, width = min(I8_BAND, cols - band * I8_BAND);
  row = r / width;
  col = band * I8_BAND + r - row * width;
}

// four neighbouring sums of row m from column n on, of which `there` exist
__device__ __forceinline__ void int8_part_store(int* __restrict__ part, int m, int n, int there, int N, intx4 v) {
  int* to = part + (size_t)m * N + n;
  if (there >= 4) {
    __builtin_memcpy(to, &v, 16);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c < there) to[c] = v[c];
  }
}

// A wave's sums (as `int8_epilogue` has them) as its part blockIdx.z of a cut K
template <bool GATED, int RM, int CN>
__device__ __forceinline__ void int8_partial(const intx4 (&acc)[RM][CN], int lane, int wm, int wn, int m0, int n0, int* partial, int M, int N) {
  constexpr int NI = GATED ? CN / 2 : CN;
  const size_t all = (size_t)M * N;
  int* part = partial + blockIdx.z * all * (GATED ? 2 : 1);
  const int row0 = m0 + wm * RM * 16 + lane % 16, col0 = n0 + wn * NI * 16 + lane / 16 * 4;
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) {
      const int n = col0 + j % NI * 16;
      if (row0 + i * 16 < M) int8_part_store(part + j / NI * all, row0 + i * 16, n, N - n, N, acc[i][j]);
    }
}

// The parts' sums ([part][weight][M][N]), V neighbouring outputs per thread (4, or 1 where N is no multiple of four): exact, so in any order.
// Bound by its bytes: three parts of 631 x 5,120 12 us (52 MB), four of 64 x 4,096 2.5 to 4.
template <int V, bool GATED>
__global__ __launch_bounds__(256) void int8_parts_kernel(const int* __restrict__ partial, int parts, Int8Epilogue p) {
  constexpr int MATS = GATED ? 2 : 1;
  const size_t all = (size_t)p.M * p.N, i = ((size_t)blockIdx.x * 256 + threadIdx.x) * V;
  if (i >= all) return;
  const int m = (int)(i / p.N), n = (int)(i - (size_t)m * p.N);
  floatx4 y{0.f, 0.f, 0.f, 0.f}, u = y, was = y;
  if (!GATED && p.epilogue == 1) {  // on its way together with the sums
    if (V == 4) was = int8_load4(p, m, n);
    else was[0] = ((const float*)p.out)[(size_t)m * p.ldo + n];
  }
  uint32_t bias[V];
  int8_load_bias(p, n, bias);
  int sum[MATS][V] = {};
#pragma unroll 4
  for (int z = 0; z < parts; ++z)
#pragma unroll
    for (int w = 0; w < MATS; ++w) {
      int s[V];
      __builtin_memcpy(s, (const int*)__builtin_assume_aligned(partial + ((size_t)z * MATS + w) * all + i, 4 * V), sizeof(s));
#pragma unroll
      for (int c = 0; c < V; ++c) sum[w][c] += s[c];
    }
  const Int8RowScale sa = int8_row_scale(p.scales.a[m]);
#pragma unroll
  for (int c = 0; c < V; ++c) {
    y[c] = int8_output(sum[0][c], sa, p.scales.w[n + c], int8_bias(p, bias[c]));
    if (GATED) u[c] = int8_output(sum[MATS - 1][c], sa, p.scales.w2[n + c], 0.f);
  }
  if (GATED) y = int8_gated4(y, u, p.gate, p.out_dtype);
  if (!GATED && p.epilogue == 1) y += was;
  int8_store4(p, m, n, V, y);
}

static inline int int8_add_parts(const int* partial, int parts, const Int8Epilogue& end, bool gated, hipStream_t stream) {
  const int v = end.N % 4 == 0 ? 4 : 1;
  const size_t groups = ((size_t)end.M * end.N / v + 255) / 256;
  if (groups > jllm_most_groups(256)) JLLM_FAIL("gemm_int8: %d x %d outputs are more than a grid takes", end.M, end.N);
  const unsigned n = (unsigned)groups;
  if (gated) {
    if (v == 4) int8_parts_kernel<4, true><<<n, 256, 0, stream>>>(partial, parts, end);
    else int8_parts_kernel<1, true><<<n, 256, 0, stream>>>(partial, parts, end);
  } else {
    if (v == 4) int8_parts_kernel<4, false><<<n, 256, 0, stream>>>(partial, parts, end);
    else int8_parts_kernel<1, false><<<n, 256, 0, stream>>>(partial, parts, end);
  }
  JLLM_CHECK_LAUNCH("gemm_int8: the sum of the parts");
  return 0;
}
