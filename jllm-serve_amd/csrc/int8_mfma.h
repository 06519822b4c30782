// 8-bit integers on the matrix cores, and the epilogue of their products.
//
// v_mfma_i32_16x16x64_i8: D[16x16] += A[16x64] * B[64x16] in whole numbers. Lane l holds, of A, row l%16, k (l/16)*16 .. +16; of B,
// column l%16, k (l/16)*16 .. +16; of D, rows (l/16)*4 + i (i = 0..3), column l%16. In bytes that is the layout of the bf16 form of
// half the depth (mfma.h), and it takes as many clocks.
//
// The sums are exact (up to 131,071 inputs, where 128^2 K stays below 2^31), so an output does not depend on the tile, the cut of
// K or the order in which parts are added. It is (float(sum) * a_scale[m]) * w_scale[n] without an overflow in between, and from there
// on what the other products make of a sum.
#pragma once
#include <atomic>
#include "common.h"
#include "mfma.h"

typedef int intx4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ intx4 mfma16_i8(u32x4 a, u32x4 b, intx4 c) {
  return __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, a), __builtin_bit_cast(intx4, b), c, 0, 0, 0);
}

#define I8_MOST_K 131071

// what loads of pieces behind the end of K fetch instead
__device__ const uint4 int8_zeros{0u, 0u, 0u, 0u};

struct Int8Scales {
  const float *a, *w, *w2;  // per row of A, per row of W (and of the second weight)
};

// What is done with a sum: the first weight's (with a bias and, gated, the second's), as the product's output
struct Int8Epilogue {
  Int8Scales scales;
  const void* bias;
  void* out;
  int bias_dtype, out_dtype, ldo, M, N, epilogue;
  GateSpec gate;
};

// The bias of C columns from n on (the last column's behind it) as it lies in memory: to make numbers of it would be to wait for it
template <int C>
__device__ __forceinline__ void int8_load_bias(const Int8Epilogue& p, int n, uint32_t (&raw)[C]) {
#pragma unroll
  for (int c = 0; c < C; ++c) raw[c] = 0;
  if (!p.bias) return;
  if (p.bias_dtype == JLLM_BF16) {
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = ((const uint16_t*)p.bias)[min(n + c, p.N - 1)];
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) raw[c] = ((const uint32_t*)p.bias)[min(n + c, p.N - 1)];
  }
}
__device__ __forceinline__ float int8_bias(const Int8Epilogue& p, uint32_t raw) { return __uint_as_float(p.bias_dtype == JLLM_BF16 ? raw << 16 : raw); }

// A row's scale as its sums are multiplied by it: from 2^96 on a sum's product with it may be beyond fp32 where the channel's scale brings the output
// back, so 2^32 of it waits until then (exact on both ways: sums are whole numbers, so nothing falls below fp32's normal numbers meanwhile)
#define I8_FAR 0x1p96f
struct Int8RowScale {
  float a, back;
};
__device__ __forceinline__ Int8RowScale int8_row_scale(float sa) { return fabsf(sa) >= I8_FAR ? Int8RowScale{sa * 0x1p-32f, 0x1p32f} : Int8RowScale{sa, 1.0f}; }

// A sum with its scales and bias. Every kernel rounds here alike (no product joined with an addition), so that a row's outputs have the same
// bits from all of them.
__device__ __forceinline__ float int8_output(int sum, Int8RowScale s, float sw, float b) {
#pragma clang fp contract(off)
  const float y = (((float)sum * s.a) * sw) * s.back;
  return y + b;
}

// 1 / (1 + exp(-slope x)), SLOPE in millionths, for outputs in fp32: the hardware's exp2 of the rounded exponent, times what the rounding left of it (by itself
// that is |slope x| halves of a step), so that the exponential and the reciprocal are off by one unit each. The bounds of x change no result (2^x is 0
// or infinite long before) and keep what is left a number. us, as for bf16 / so: 64 x 12,288 x 4,096 gated in fp32 23.6 / 24.2, 8,192 x 17,408 x 5,120 1,099 / 1,108.
template <int SLOPE>
__device__ __forceinline__ float int8_sigmoid(float x) {
#pragma clang fp contract(off)
  constexpr double RATE = SLOPE * 1e-6 * 1.4426950408889634074;
  constexpr float HI = (float)RATE, LO = (float)(RATE - (double)HI);
  x = fminf(fmaxf(x, -256.0f), 256.0f);
  const float t = x * HI, left = fmaf(x, LO, fmaf(x, HI, -t));
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-t) * fmaf(left, -0.6931471805599453f, 1.0f));
}

// The gate of two of them; FINE: of an output in fp32, where common.h's fast form would show. Rows without numbers have a scale of NaN, and clamps
// would lose it.
template <bool FINE>
__device__ __forceinline__ float int8_gated(float z, float u, GateSpec gs) {
#pragma clang fp contract(off)
  float y;
  if (!FINE) {
    y = gated<true>(z, u, gs);
  } else if (gs.fn == JLLM_GATE_SILU) {
    y = z * int8_sigmoid<1000000>(z) * u;
  } else if (gs.fn == JLLM_GATE_GELU_TANH) {  // 0.5 (1 + tanh x) = 1 / (1 + exp(-2x))
    y = z * int8_sigmoid<2000000>(0.7978845608028654f * (z + 0.044715f * z * z * z)) * u;
  } else {
    const float g = fminf(z, gs.limit), v = fminf(fmaxf(u, -gs.limit), gs.limit);
    y = g * int8_sigmoid<1702000>(g) * (v + 1.0f);
  }
  return gs.fn != JLLM_GATE_SWISH_CLAMPED || (z == z && u == u) ? y : z + u;
}
__device__ __forceinline__ floatx4 int8_gated4(floatx4 z, floatx4 u, GateSpec gs, int out_dtype) {
  floatx4 y;
  if (out_dtype == JLLM_BF16) {
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = int8_gated<false>(z[c], u[c], gs);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = int8_gated<true>(z[c], u[c], gs);
  }
  return y;
}

// What four neighbouring outputs of row m from column n on are added to
__device__ __forceinline__ floatx4 int8_load4(const Int8Epilogue& p, int m, int n) {
  floatx4 v;
  __builtin_memcpy(&v, (const float*)p.out + (size_t)m * p.ldo + n, 16);
  return v;
}

// Four neighbouring outputs of row m from column n on, of which `there` exist (what they are added to is in them). All four are one access
// wherever the row begins (the hardware takes it at any element).
__device__ __forceinline__ void int8_store4(const Int8Epilogue& p, int m, int n, int there, floatx4 v) {
  const size_t o = (size_t)m * p.ldo + n;
  if (there == 4) {
    if (p.out_dtype == JLLM_BF16) {
      const u32x2 w{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
      __builtin_memcpy((bf16_t*)p.out + o, &w, 8);
    } else {
      __builtin_memcpy((float*)p.out + o, &v, 16);
    }
    return;
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (c >= there) continue;
    if (p.out_dtype == JLLM_BF16)
      stf((bf16_t*)p.out, o + c, v[c]);
    else
      stf((float*)p.out, o + c, v[c]);
  }
}

// The four values of a vector per column from column n on, `whole`: all of them there. Any alignment of an entry.
__device__ __forceinline__ void int8_columns(const float* from, int n, int N, bool whole, float (&to)[4]) {
  if (whole) {
    __builtin_memcpy(to, from + n, 16);
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c) to[c] = from[min(n + c, N - 1)];
  }
}

// A wave's accumulators, CN runs of four columns for each of its RM blocks of 16 rows (gated: [.][j] and [.][j + CN / 2] are the two weights' of the
// same outputs), row block by row block, so that hardly more than the sums themselves is in registers. Where all of its columns are there
// (and no row's scale is far beyond others') it goes without a branch per output, and everything is requested before the first output is stored (behind a store the compiler moves no
// load forward, and each would wait for its own way); what the outputs are added to, one block of rows ahead.
template <bool GATED, int FN, bool FINE, int RM, int CN>
__device__ __forceinline__ void int8_outputs(const intx4 (&acc)[RM][CN], int lane, int wm, int wn, int m0, int n0, const Int8Epilogue& p) {
  constexpr int NI = GATED ? CN / 2 : CN;
  const int group = lane / 16, row0 = m0 + wm * RM * 16 + lane % 16, col0 = n0 + wn * NI * 16 + group * 4;
  const bool whole = n0 + (wn + 1) * NI * 16 <= p.N;  // the same in all lanes
  float sa[RM], sw[NI][4], su[NI][4], bv[NI][4];
#pragma unroll
  for (int i = 0; i < RM; ++i) sa[i] = p.scales.a[min(row0 + i * 16, p.M - 1)];
#pragma unroll
  for (int j = 0; j < NI; ++j) {
    int8_columns(p.scales.w, col0 + j * 16, p.N, whole, sw[j]);
    if (GATED) int8_columns(p.scales.w2, col0 + j * 16, p.N, whole, su[j]);
  }
  if (!p.bias) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) bv[j][c] = 0.f;
  } else if (p.bias_dtype == JLLM_BF16) {
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) bv[j][c] = ldf((const bf16_t*)p.bias, min(col0 + j * 16 + c, p.N - 1));
  } else {
#pragma unroll
    for (int j = 0; j < NI; ++j) int8_columns((const float*)p.bias, col0 + j * 16, p.N, whole, bv[j]);
  }
  auto scaled = [&](int i, int j, Int8RowScale s) {
    floatx4 v;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float z = int8_output(acc[i][j][c], s, sw[j][c], bv[j][c]);
      v[c] = GATED ? int8_gated<FINE>(z, int8_output(acc[i][GATED ? NI + j : 0][c], s, su[j][c], 0.f), GateSpec{FN, p.gate.limit}) : z;
    }
    return v;
  };
  auto outputs = [&](int i, int j) { return scaled(i, j, Int8RowScale{sa[i], 1.0f}); };
  float most = fabsf(sa[0]);  // of a row's scale in this wave
#pragma unroll
  for (int i = 1; i < RM; ++i) most = fmaxf(most, fabsf(sa[i]));
  if (!whole || __any(most >= I8_FAR)) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int m = row0 + i * 16;
      if (m >= p.M) continue;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int n = col0 + j * 16;
        if (n >= p.N) continue;
        floatx4 v = scaled(i, j, int8_row_scale(sa[i]));
        if (!GATED && p.epilogue == 1) {
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] += ((const float*)p.out)[(size_t)m * p.ldo + min(n + c, p.N - 1)];
        }
        int8_store4(p, m, n, min(4, p.N - n), v);
      }
    }
  } else if (!GATED && p.epilogue == 1) {
    float* out = (float*)p.out + col0;
    floatx4 was[2][NI];
    auto fetch = [&](int i) {
#pragma unroll
      for (int j = 0; j < NI; ++j) was[i & 1][j] = int8_load4(p, min(row0 + i * 16, p.M - 1), col0 + j * 16);
    };
    fetch(0);
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      if (i + 1 < RM) fetch(i + 1);
      if (row0 + i * 16 >= p.M) continue;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const floatx4 v = was[i & 1][j] + outputs(i, j);
        __builtin_memcpy(out + (size_t)(row0 + i * 16) * p.ldo + j * 16, &v, 16);
      }
    }
  } else if (GATED ? !FINE : p.out_dtype == JLLM_BF16) {
    bf16_t* out = (bf16_t*)p.out + col0;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      if (row0 + i * 16 >= p.M) continue;
      bf16_t* to = out + (size_t)(row0 + i * 16) * p.ldo;
      if constexpr (NI % 2 == 0) {  // two neighbouring runs exchange halves between lanes first, so that a lane stores eight columns
#pragma unroll
        for (int j = 0; j < NI; j += 2) {
          const floatx4 v = outputs(i, j), w = outputs(i, j + 1);
          const u32x2 lo = {pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])}, hi = {pack_bf16(w[0], w[1]), pack_bf16(w[2], w[3])};
          const auto a = __builtin_amdgcn_permlane16_swap(lo.x, hi.x, false, false);
          const auto b = __builtin_amdgcn_permlane16_swap(lo.y, hi.y, false, false);
          const u32x4 w4{a[0], b[0], a[1], b[1]};
          __builtin_memcpy(to + j * 16 - group * 4 + (group & 1) * 16 + (group >> 1) * 8, &w4, 16);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NI; ++j) {
          const floatx4 v = outputs(i, j);
          const u32x2 w{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
          __builtin_memcpy(to + j * 16, &w, 8);
        }
      }
    }
  } else {
    float* out = (float*)p.out + col0;
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      if (row0 + i * 16 >= p.M) continue;
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const floatx4 v = outputs(i, j);
        __builtin_memcpy(out + (size_t)(row0 + i * 16) * p.ldo + j * 16, &v, 16);
      }
    }
  }
}

// The same, each gate function in code of its own for outputs in bf16 and in fp32: chosen output by output it took as long as the gates themselves
template <bool GATED, int RM, int CN>
__device__ __forceinline__ void int8_epilogue(const intx4 (&acc)[RM][CN], int lane, int wm, int wn, int m0, int n0, const Int8Epilogue& p) {
#define I8_OUTPUTS(FN)                                                           \
  if (!GATED || p.out_dtype == JLLM_BF16)                                        \
    int8_outputs<GATED, FN, false>(acc, lane, wm, wn, m0, n0, p);                \
  else                                                                           \
    int8_outputs<GATED, FN, true>(acc, lane, wm, wn, m0, n0, p)
  if (!GATED || p.gate.fn == JLLM_GATE_SILU) {
    I8_OUTPUTS(JLLM_GATE_SILU);
  } else if (p.gate.fn == JLLM_GATE_GELU_TANH) {
    I8_OUTPUTS(JLLM_GATE_GELU_TANH);
  } else {
    I8_OUTPUTS(JLLM_GATE_SWISH_CLAMPED);
  }
#undef I8_OUTPUTS
}

// Above 64 KB a kernel's dynamic LDS has to be allowed first, on every device once
template <auto KERNEL>
static inline bool int8_allow_lds(int bytes) {
  static std::atomic<unsigned long long> allowed{0};
  int device = 0;
  if (hipGetDevice(&device) != hipSuccess) return false;
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return true;
  if (hipFuncSetAttribute((const void*)KERNEL, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return false;
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return true;
}
