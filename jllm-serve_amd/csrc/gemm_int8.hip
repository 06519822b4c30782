// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for rows of 8-bit integers of any sizes, at any alignment and with
// any distance between rows: the general form of the product.
//
// A workgroup of four waves (2 x 2) owns 64 x 64 outputs (gated: 64 x 32, both weights'), a wave 2 x 2 accumulators of 16 x 16. K
// advances in stages of 128 through registers, four stages ahead, into two LDS buffers: 16 bytes a lane wherever the row begins (unaligned accesses are
// one load each); what would reach over a row's end is read up to it and moved down, with zeros behind. K may be cut over gridDim.z: the parts leave their
// whole-number sums, and a second kernel adds them and makes the outputs.
//
// Bound by the loads' latency where there are few workgroups and by LDS where there are many: a stage takes 0.42 us for each workgroup that a
// compute unit has. us inside a graph: 77 x 2,051 x 1,037 8.2 (with the scales and outputs one by one 9.7; besides, one stage ahead and
// the last bytes by branches 14.7), 64 x 4,096 x 12,288 23
// in four parts (the weight-streaming kernel 17), 2,048 x 4,096 x 4,096 114 (the large tiles 34: operands of many rows are laid out anew for them).
#include <type_traits>
#include "int8_mfma.h"
#include "int8_parts.h"

#define G8_BK 128
#define G8_AHEAD 4  // stages whose loads are on their way
#define G8_PITCH 144  // bytes of a row in LDS: 16 lanes that read one piece of 16 rows meet no bank twice in a turn

struct Gemm8Args {
  const signed char *A, *W, *W2;
  int* partial;  // [part][weight][M][N]
  int lda, ldw, ldw2, K, stages;  // stages of K per part
  Int8Epilogue end;
};

template <bool GATED, bool SHORT>
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
  u32x4 held[G8_AHEAD][4];  // stages on their way
  // A piece that reaches over the end of K is read up to it, from the row's last 16 bytes, and moved down where it goes to LDS
  auto fetch = [&](int t, u32x4 (&to)[4]) {
    const int k = t * G8_BK + piece * 16;
    if constexpr (SHORT) {  // rows of fewer than 16 bytes, byte by byte
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int e = 0; e < 15; ++e)
          if (k + e < p.K) w[e >> 2] |= (uint32_t)(unsigned char)from[c][k + e] << (e & 3) * 8;
        to[c] = u32x4{w[0], w[1], w[2], w[3]};
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) __builtin_memcpy(&to[c], from[c] + min(k, p.K - 16), 16);
    }
  };
  auto put = [&](int buffer, int t, const u32x4 (&of)[4]) {
    const bool whole = SHORT || (t + 1) * G8_BK <= p.K;  // the same in all lanes
    const int down = max(0, t * G8_BK + piece * 16 - (p.K - 16)) * 8;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      u32x4 v = of[c];
      if (!whole) {
        uint64_t lo = (uint64_t)v[1] << 32 | v[0], hi = (uint64_t)v[3] << 32 | v[2];
        if (down >= 64) lo = hi, hi = 0;
        const int s = down & 63;
        lo = down >= 128 ? 0 : s ? lo >> s | hi << (64 - s) : lo;
        hi = down >= 64 ? 0 : hi >> s;
        v = u32x4{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
      *(u32x4*)(lds[buffer] + ((tid >> 3) + c * 32) * G8_PITCH + piece * 16) = v;
    }
  };
  intx4 acc[2][2] = {};
  const int first = blockIdx.z * p.stages, stages = min((p.K + G8_BK - 1) / G8_BK - first, p.stages);
#pragma unroll
  for (int t = 0; t < G8_AHEAD; ++t) fetch(first + min(t, stages - 1), held[t]);
  // Stage t is multiplied from LDS while the next ones are on their way (behind the last it is asked for again: behind a branch the
  // compiler would wait for all); the buffer that it goes to was read in stage t - 2
  auto stage = [&](auto which, int t) {
    constexpr int H = decltype(which)::value, B = H % 2;  // t % G8_AHEAD
    put(B, first + t, held[H]);
    __syncthreads();
    fetch(first + min(t + G8_AHEAD, stages - 1), held[H]);
    const unsigned char* s = lds[B] + (lane & 15) * G8_PITCH + (lane >> 4) * 16;
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
  };
  int t = 0;
  for (; t + 4 <= stages; t += 4) {
    stage(std::integral_constant<int, 0>{}, t);
    stage(std::integral_constant<int, 1>{}, t + 1);
    stage(std::integral_constant<int, 2>{}, t + 2);
    stage(std::integral_constant<int, 3>{}, t + 3);
  }
  if (t < stages) stage(std::integral_constant<int, 0>{}, t);
  if (t + 1 < stages) stage(std::integral_constant<int, 1>{}, t + 1);
  if (t + 2 < stages) stage(std::integral_constant<int, 2>{}, t + 2);
  if (gridDim.z > 1) {
    int8_partial<GATED>(acc, lane, wm, wn, m0, n0, p.partial, M, N);
    return;
  }
  int8_epilogue<GATED, 2, 2>(acc, lane, wm, wn, m0, n0, p.end);
}

// `parts` > 1 cuts K, in whole stages of 128; `partial` then holds parts * (1 or, gated, 2) * M * N ints
extern "C" int jllm_gemm_int8(const void* A, int lda, const float* a_scale, const void* W, int ldw, const float* w_scale, const void* W2, int ldw2,
                              const float* w2_scale, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int K,
                              int epilogue, float gate_limit, int parts, int* partial, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > I8_MOST_K) JLLM_FAIL("gemm_int8: %d inputs (1 to %d: beyond, the sums could leave 32 bits)", K, I8_MOST_K);
  JLLM_TAKE_GATE("gemm_int8", epilogue, gate_limit, gs);
  if (epilogue < 0 || epilogue > 2 || (epilogue == 2) != (W2 != nullptr)) JLLM_FAIL("gemm_int8: epilogue %d", epilogue);
  if (epilogue == 1 && out_dtype != JLLM_F32) JLLM_FAIL("gemm_int8: the accumulate epilogue adds into fp32");
  if (lda < 0 || ldw < 0 || ldw2 < 0 || ldo < N) JLLM_FAIL("gemm_int8: rows %d, %d and %d apart", lda, ldw, ldo);
  const int stages = (K + G8_BK - 1) / G8_BK;
  parts = parts < 1 ? 1 : parts > stages ? stages : parts;
  const int each = (stages + parts - 1) / parts;
  parts = (stages + each - 1) / each;  // those that have any stage
  if (parts > 1 && (!partial || ((uintptr_t)partial & 15))) JLLM_FAIL("gemm_int8: %d parts of K need a buffer for their sums", parts);
  const dim3 grid((N - 1) / (W2 ? 32 : 64) + 1, (M - 1) / 64 + 1, parts);
  if (!jllm_grid_fits(grid, 256)) JLLM_FAIL("gemm_int8: %d x %d outputs are more than a grid takes", M, N);
  const Gemm8Args a{(const signed char*)A, (const signed char*)W, (const signed char*)W2, partial, lda, ldw, ldw2, K, each,
                    {{a_scale, w_scale, w2_scale}, bias, out, bias_dtype, out_dtype, ldo, M, N, epilogue, gs}};
  if (W2 && K < 16)
    gemm_int8_kernel<true, true><<<grid, 256, 0, stream>>>(a);
  else if (W2)
    gemm_int8_kernel<true, false><<<grid, 256, 0, stream>>>(a);
  else if (K < 16)
    gemm_int8_kernel<false, true><<<grid, 256, 0, stream>>>(a);
  else
    gemm_int8_kernel<false, false><<<grid, 256, 0, stream>>>(a);
  JLLM_CHECK_LAUNCH("gemm_int8");
  return parts > 1 ? int8_add_parts(partial, parts, a.end, W2 != nullptr, stream) : 0;
}

// Rows of 8-bit integers laid out for the fast kernels: row r at dst + r * ldd, zeros from `width` to ldd (a multiple of 16)
__global__ __launch_bounds__(256) void int8_lay_out_kernel(const signed char* __restrict__ src, int lds_, signed char* __restrict__ dst, int ldd, int rows, int width) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const unsigned pieces = (unsigned)ldd / 16;
  const size_t row = i / pieces;
  if (row >= (size_t)rows) return;
  const int at = (int)(i - row * pieces) * 16;
  const signed char* from = src + row * lds_ + at;
  uint32_t w[4] = {0, 0, 0, 0};
  if (at + 16 <= width) {
    __builtin_memcpy(w, from, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (at + e < width) w[e >> 2] |= (uint32_t)(unsigned char)from[e] << (e & 3) * 8;
  }
  *(u32x4*)(dst + row * ldd + at) = u32x4{w[0], w[1], w[2], w[3]};
}

extern "C" int jllm_int8_lay_out(const void* src, int ld, void* dst, int ldd, int rows, int width, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || ld < 0 || ldd < width || (ldd & 15) || ((uintptr_t)dst & 15)) JLLM_FAIL("int8_lay_out: rows of %d, %d and %d apart", width, ld, ldd);
  const unsigned pieces = (unsigned)ldd / 16, fit = jllm_most_groups(256) * 256u / pieces;
  const int most = fit > 0x7fffffffu ? 0x7fffffff : (int)fit;  // rows that one launch has threads for
  for (int first = 0; rows > 0; rows -= most, first += most) {
    const int n = min(rows, most);
    int8_lay_out_kernel<<<(unsigned)(((size_t)n * pieces + 255) / 256), 256, 0, stream>>>((const signed char*)src + (size_t)first * ld, ld,
                                                                                        (signed char*)dst + (size_t)first * ldd, ldd, n, width);
    JLLM_CHECK_LAUNCH("int8_lay_out");
    if (rows <= most) break;  // (first + most may not fit)
  }
  return 0;
}
