// Rows of 8-bit integers with one fp32 scale each: made from rows of activations or weights, made by the RMSNorm that stands
// between two sublayers, and read back.
//
//   most = max_i |y[i]|,  scale = most / 127,  q[i] = round(y[i] * (127 / most)), halves to even, -127 .. 127
//   norm: h = x + add (fp32, written), y = (h * r) * gain, r = 1 / sqrt(mean(h^2) + eps)
//
// A row of zeros has scale 0 and zeros. A row with a NaN or an infinity has scale NaN and zeros, so that everything computed
// from it is NaN. Rows whose largest value lies below 2^-100 are multiplied by 2^100 first (exact), where 127 / most
// could be beyond fp32. Quotient and products are rounded to fp32 before they are rounded to whole numbers, as the formula reads: an exact half
// may fall to either side where 127 / most is no fp32 number.
//
// Bound by bytes: an entry is read once, and written once in one byte (the norm's h in four more). So a row stays in registers
// between its reduction and its rounding: eight neighbouring entries to a load (any alignment of an element), J loads to a
// thread, THREADS to a row. The last piece of a row whose width is no multiple of eight begins eight before the end
// and overlaps the one before; it counts what is new in it. Widths below 8 or above 32,768 take a loop that reads the row again.
//
// us inside a graph: norm with bf16 rows to add 8 x 4,096 3.3, 631 x 2,560 6.5, 8,192 x 5,120 87.7 (461 MB: 5.3 TB/s; a large copy reaches
// 5.1); bf16 rows made 8-bit 64 x 12,288 3.0, 8,192 x 5,120 22.8 (5.5 TB/s); read back into bf16 2.2 and 25.1. What few rows take is the
// launch and two chains of a load, a reduction and a store.
#include "common.h"

#define I8_LEVELS 127.0f

namespace {

struct RowsArgs {
  const void* x;     // [rows][width], fp32 for the norm
  const void* add;   // norm: what joins, or none
  const void* gain;  // norm
  float* sum;        // norm: where x + add goes (may be x)
  signed char* q;
  float* scale;
  int ldx, ld_add, ld_sum, ldq, width;
  float eps;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  T raw[8];
  __builtin_memcpy(raw, p, sizeof(raw));
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = ldf(raw, e);
}

// The largest of the magnitudes' bit patterns: the order of the numbers, with infinity and NaN above all
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = JLLM_WAVE / 2; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o, JLLM_WAVE));
  return v;
}

template <int NW>
__device__ __forceinline__ double row_sum(double v, double* red) {  // in a fixed order; `red` is this reduction's alone
#pragma unroll
  for (int o = JLLM_WAVE / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, JLLM_WAVE);
  if (NW == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) s += red[i];
  return s;
}

template <int NW>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t* red) {
  v = wave_umax(v);
  if (NW == 1) return v;
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t s = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) s = max(s, red[i]);
  return s;
}

struct Rounding {
  float pre, inv, scale;
};
__device__ __forceinline__ Rounding rounding_of(uint32_t most_bits) {
  const float most = __uint_as_float(most_bits);
  Rounding r;
  r.pre = most < 7.888609052210118e-31f ? 1.2676506002282294e30f : 1.0f;  // 2^-100, 2^100
  const bool number = most_bits < 0x7f800000u;
  r.inv = number && most_bits != 0 ? I8_LEVELS / (most * r.pre) : 0.f;
  r.scale = number ? most / I8_LEVELS : __uint_as_float(0x7fc00000u);
  return r;
}
// round(y * inv) in the low byte: 1.5 * 2^23 has steps of one, and its low byte is zero. `inv` zero: zeros, whatever y is.
__device__ __forceinline__ uint32_t rounded(float y, const Rounding& r) {
#pragma clang fp contract(off)
  const float t = (y * r.pre) * r.inv;
  return r.inv == 0.f ? 0u : __float_as_uint(t + 12582912.0f) & 0xffu;
}

// The norm's scale r, rounded once from 64 bits. Squares and their sum are in 64 bits, where the squares are exact and none overflows: the kernel waits
// for memory meanwhile, and a scale that is off by one unit turns whole numbers that lie near a half. Rows whose root mean square lies beyond 2^100
// or below 2^-100 are multiplied by a power of two first (exact, but for what is zero beside the row's largest): r itself may lie below
// fp32's normal numbers there, or beyond them. A row of zeros without an eps has no root: its entries stay zeros.
struct NormScale {
  float pre, r;
};
__device__ __forceinline__ NormScale rms_scale(double squares, int n, float eps) {
  const double mean = squares / n + (double)eps;
  const bool large = mean > 0x1p200, small = mean < 0x1p-200;
  const float r = (float)((large ? 0x1p32 : small ? 0x1p-64 : 1.0) / sqrt(mean));
  return {large ? 0x1p-32f : small ? 0x1p64f : 1.0f, mean == 0.0 ? 0.f : r};
}

// Every entry of a norm is (h * r) * gain, two roundings
__device__ __forceinline__ float normed(float h, NormScale s, float g) { return ((h * s.pre) * s.r) * g; }

template <bool NORM, bool ADD, typename TX, typename TA, typename TG, int J, int THREADS>
__global__ __launch_bounds__(THREADS) void int8_rows_kernel(RowsArgs p) {
  constexpr int NW = THREADS / 64;
  __shared__ double red_sum[NW];
  __shared__ uint32_t red_max[NW];
  const size_t row = blockIdx.x;
  const TX* x = (const TX*)p.x + row * p.ldx;
  const TA* add = ADD ? (const TA*)p.add + row * p.ld_add : nullptr;
  const TG* gain = (const TG*)p.gain;
  float* sum = ADD ? p.sum + row * p.ld_sum : nullptr;
  signed char* q = p.q + row * p.ldq;
  const int d = p.width, tid = threadIdx.x;
  if constexpr (J > 0) {
    const int pieces = (d + 7) >> 3;
    float v[J][8], g[J][8];
    int at[J];
    // everything is requested before the first use; beyond the row's end its last piece again
#pragma unroll
    for (int j = 0; j < J; ++j) {
      at[j] = min((tid + THREADS * j) * 8, d - 8);
      load8(x + at[j], v[j]);
    }
    if (ADD) {
      float a[J][8];
#pragma unroll
      for (int j = 0; j < J; ++j) load8(add + at[j], a[j]);
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += a[j][e];
    }
    if (NORM) {
#pragma unroll
      for (int j = 0; j < J; ++j) load8(gain + at[j], g[j]);
      double ss = 0.0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int first = (tid + THREADS * j) * 8;  // what lies below it in the piece belongs to the one before
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double h = at[j] + e >= first ? v[j][e] : 0.f;
          ss += h * h;
        }
      }
      ss = row_sum<NW>(ss, red_sum);
      const NormScale r = rms_scale(ss, d, p.eps);
      if (ADD) {  // behind the barrier: every thread has its overlapping entries of the old row
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (tid + THREADS * j < pieces) __builtin_memcpy(sum + at[j], v[j], 32);
      }
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] = normed(v[j][e], r, g[j][e]);
    }
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) most = max(most, magnitude(v[j][e]));
    most = row_max<NW>(most, red_max);
    const Rounding r = rounding_of(most);
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (tid + THREADS * j < pieces) {
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[h] = rounded(v[j][4 * h], r) | rounded(v[j][4 * h + 1], r) << 8 | rounded(v[j][4 * h + 2], r) << 16 | rounded(v[j][4 * h + 3], r) << 24;
        __builtin_memcpy(q + at[j], w, 8);
      }
    if (tid == 0) p.scale[row] = r.scale;
    return;
  } else {
    // A row of any width, entry by entry; a thread reads again what it alone wrote
    NormScale r{};
    if (NORM) {
      double ss = 0.0;
      for (int i = tid; i < d; i += THREADS) {
        float h = ldf(x, i);
        if (ADD) {
          h += ldf(add, i);
          sum[i] = h;
        }
        ss += (double)h * h;
      }
      r = rms_scale(row_sum<NW>(ss, red_sum), d, p.eps);
    }
    auto entry = [&](int i) { return NORM ? normed(ADD ? sum[i] : ldf(x, i), r, ldf(gain, i)) : ldf(x, i); };
    uint32_t most = 0;
    for (int i = tid; i < d; i += THREADS) most = max(most, magnitude(entry(i)));
    const Rounding to = rounding_of(row_max<NW>(most, red_max));
    for (int i = tid; i < d; i += THREADS) q[i] = (signed char)rounded(entry(i), to);
    if (tid == 0) p.scale[row] = to.scale;
  }
}

// A workgroup a row, in as many launches as the rows take
template <bool NORM, bool ADD, typename TX, typename TA, typename TG, int J, int THREADS>
int launch_rows_of(RowsArgs a, int rows, hipStream_t stream) {
  const int most = (int)jllm_most_groups(THREADS);
  for (; rows > 0; rows -= most) {
    int8_rows_kernel<NORM, ADD, TX, TA, TG, J, THREADS><<<min(rows, most), THREADS, 0, stream>>>(a);
    JLLM_CHECK_LAUNCH("int8_rows");
    if (rows <= most) break;
    const size_t n = (size_t)most;
    a.x = (const TX*)a.x + n * a.ldx;
    if (ADD) a.add = (const TA*)a.add + n * a.ld_add;
    if (ADD) a.sum += n * a.ld_sum;
    a.q += n * a.ldq;
    a.scale += n;
  }
  return 0;
}

// Threads of a row and pieces of a thread by width
template <bool NORM, bool ADD, typename TX, typename TA, typename TG>
int launch_rows(const RowsArgs& a, int rows, hipStream_t stream) {
#define I8_ROWS(J, THREADS) return launch_rows_of<NORM, ADD, TX, TA, TG, J, THREADS>(a, rows, stream)
  const int d = a.width;
  if (d < 8 || d > 32768) I8_ROWS(0, 256);
  if (d <= 512) I8_ROWS(1, 64);
  if (d <= 1024) I8_ROWS(2, 64);
  if (d <= 2048) I8_ROWS(1, 256);
  if (d <= 4096) I8_ROWS(2, 256);
  if (d <= 6144) I8_ROWS(3, 256);
  if (d <= 8192) I8_ROWS(4, 256);
  if (d <= 16384) I8_ROWS(2, 1024);
  if (d <= 24576) I8_ROWS(3, 1024);
  I8_ROWS(4, 1024);
#undef I8_ROWS
}

}  // namespace

extern "C" int jllm_quantize_rows(const void* x, int dtype, int ldx, int rows, int width, void* q, int ldq, float* scale, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || width > (1 << 30) || ldx < 0 || ldq < width) JLLM_FAIL("quantize_rows: rows of %d, %d and %d apart", width, ldx, ldq);
  RowsArgs a{x, nullptr, nullptr, nullptr, (signed char*)q, scale, ldx, 0, 0, ldq, width, 0.f};
  JLLM_DISPATCH_1(dtype, T, { return (launch_rows<false, false, T, float, float>(a, rows, stream)); })
}

extern "C" int jllm_rmsnorm_int8(const float* x, int ldx, const void* add, int add_dtype, int ld_add, float* sum, int ld_sum, int rows, int width,
                                 const void* gain, int gain_dtype, float eps, void* q, int ldq, float* scale, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || width > (1 << 30) || ldx < 0 || ldq < width) JLLM_FAIL("rmsnorm_int8: rows of %d, %d and %d apart", width, ldx, ldq);
  if ((add != nullptr) != (sum != nullptr)) JLLM_FAIL("rmsnorm_int8: rows to add and a place for the sum come together");
  if (add && (ld_add < 0 || ld_sum < width)) JLLM_FAIL("rmsnorm_int8: sums %d apart for rows of %d", ld_sum, width);
  RowsArgs a{x, add, gain, sum, (signed char*)q, scale, ldx, ld_add, ld_sum, ldq, width, eps};
  JLLM_DISPATCH_1(gain_dtype, TG, {
    if (!add) return (launch_rows<true, false, float, float, TG>(a, rows, stream));
    JLLM_DISPATCH_1(add_dtype, TA, { return (launch_rows<true, true, float, TA, TG>(a, rows, stream)); })
  })
}

// ---------------------------------------------------------------------------------------------------------
// out[m][i] = q[m][i] * scale[m], rounded once to the output's type; 8 neighbouring entries per thread, the last piece of a row
// overlapping the one before (it writes the same values).
template <typename TO, int V>
__global__ __launch_bounds__(256) void dequantize_rows_kernel(const signed char* __restrict__ q, int ldq, const float* __restrict__ scale, TO* __restrict__ out,
                                                              int ldo, int rows, int width, int pieces) {
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  const size_t row = i / (unsigned)pieces;
  if (row >= (size_t)rows) return;
  const int at = min((int)(i - row * pieces) * V, width - V);
  signed char v[V];
  __builtin_memcpy(v, q + row * ldq + at, V);
  const float s = scale[row];
  TO o[V];
#pragma unroll
  for (int e = 0; e < V; ++e) stf(o, e, (float)v[e] * s);
  __builtin_memcpy(out + row * ldo + at, o, sizeof(o));
}

extern "C" int jllm_dequantize_rows(const void* q, int ldq, const float* scale, int rows, int width, void* out, int out_dtype, int ldo, hipStream_t stream) {
  if (rows <= 0) return 0;
  if (width <= 0 || width > (1 << 30) || ldq < 0 || ldo < width) JLLM_FAIL("dequantize_rows: rows of %d, %d and %d apart", width, ldq, ldo);
  const int v = width < 8 ? 1 : 8, pieces = (width + v - 1) / v;
  const unsigned fit = jllm_most_groups(256) * 256u / (unsigned)pieces;
  const int most = fit > 0x7fffffffu ? 0x7fffffff : (int)fit;  // rows that one launch has threads for
  JLLM_DISPATCH_1(out_dtype, TO, {
    for (int first = 0; rows > 0; rows -= most, first += most) {
      const int n = min(rows, most);
      const unsigned groups = (unsigned)(((size_t)n * pieces + 255) / 256);
      const signed char* from = (const signed char*)q + (size_t)first * ldq;
      TO* to = (TO*)out + (size_t)first * ldo;
      if (v == 8)
        dequantize_rows_kernel<TO, 8><<<groups, 256, 0, stream>>>(from, ldq, scale + first, to, ldo, n, width, pieces);
      else
        dequantize_rows_kernel<TO, 1><<<groups, 256, 0, stream>>>(from, ldq, scale + first, to, ldo, n, width, pieces);
      JLLM_CHECK_LAUNCH("dequantize_rows");
      if (rows <= most) break;  // (first + most may not fit)
    }
  })
  return 0;
}
