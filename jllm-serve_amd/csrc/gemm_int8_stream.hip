// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for up to 64 rows of 8-bit integers (decode steps), bound by reading W
// from memory once.
//
// A workgroup owns `rows` weight rows (of each weight) and a range of K (gridDim.y of them), which its waves share in blocks of 128 bytes:
// wave w takes blocks w, w + WAVES, .. Both operands of a block go straight from memory into a ring of S blocks in LDS that belongs
// to the wave alone (8 rows of 128 bytes to an instruction, bank swizzle on the global side), so that nothing but the wave's own
// count of loads in flight stands between a load and its use, and no barrier before the end. Every wave multiplies all the
// activation rows by all the workgroup's weight rows over its blocks; the sums, whole numbers, meet in LDS.
//
// A compute unit's load pipe passes the activations, once per workgroup, as well as the weights: a workgroup should own about as
// many weight rows as there are activation rows, or more. Where that leaves compute units without one, K is cut over
// workgroups, and a second kernel adds the parts.
//
// us inside a graph over weights that no cache holds (in brackets the weights' way at the 6.2 TB/s of reading alone): 6,144 x 4,096 (4.1) at
// 1, 8, 32 and 64 rows 7.0, 7.1, 8.2, 10.7; gated 12,288 x 4,096 (16.2) 20.7, 20.6, 22.2, 24.9; 4,096 x 12,288 (8.1) 11.0, 10.9, 14.5, 17.5, the last
// in four parts; gated 17,408 x 5,120 (28.8) 35, 34.5, 38, 44.5. What is left is the launch and the first bytes (3), from some 32 rows on
// the load pipe, and with K cut the second launch (3 to 4). Measured and not taken: eight waves (the same or slower from 8 MB of weights on; 4,096 x
// 4,096 at one row 5.8 instead of 6.0), parts of K at few rows, one workgroup per compute unit where two fit, the next block's
// fragments read into a second set of registers while one multiplies (the same time where they fit, spills where not).
//
// Needs K % 16 == 0 and 16-byte aligned rows; any N, up to 64 rows.
#include "int8_mfma.h"
#include "int8_parts.h"
#include "lds_ring.h"

struct Stream8Args {
  const signed char *A, *W, *W2;
  int* partial;
  int lda, ldw, K, rows, blocks;  // weight rows per workgroup; blocks of K per part
  Int8Epilogue end;
};

template <int NI, int S>
__device__ __forceinline__ void i8_wait_block(int behind) {  // `behind` (< S) blocks behind the one that has to be here
  if (behind == S - 1) return wait_loads<(S - 1) * NI>();
  if (S > 2 && behind == S - 2) return wait_loads<(S > 2 ? S - 2 : 0) * NI>();
  if (S > 3 && behind == S - 3) return wait_loads<(S > 3 ? S - 3 : 0) * NI>();
  if (S > 4 && behind == S - 4) return wait_loads<(S > 4 ? S - 4 : 0) * NI>();
  if (S > 5 && behind == S - 5) return wait_loads<(S > 5 ? S - 5 : 0) * NI>();
  wait_loads<0>();
}

// blocks of NI KB in a wave's ring, out of all of the 160 KB: two workgroups share a compute unit where each still has two
constexpr int i8_slots(int ni, int waves) {
  const int shared = 80 / (waves * ni), fit = shared >= 2 ? shared : 160 / (waves * ni);
  return fit > 6 ? 6 : fit;
}

// NW: loads of 8 weight rows per block (of each weight), NA: of 8 activation rows
template <int NW, int NA, bool GATED, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gemm_int8_stream_kernel(Stream8Args p) {
  constexpr int CT = (NW + 1) / 2, MT = (NA + 1) / 2, MATS = GATED ? 2 : 1;  // tiles of 16 weight rows (of each weight), of 16 activation rows
  constexpr int NWT = MATS * NW, NI = NWT + NA;                             // loads of a block
  constexpr int S = i8_slots(NI, WAVES);
  static_assert(S >= 2 && (S - 1) * NI < 63, "the counter of loads in flight");
  static_assert(WAVES * MATS * CT * MT <= WAVES * S * NI, "the sums fit the rings");
  extern __shared__ __align__(1024) unsigned char smem[];  // [WAVES][S][NI KB]; afterwards the waves' sums
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int col = lane & 15, g = lane >> 4, M = p.end.M, N = p.end.N;
  const int n0 = blockIdx.x * p.rows;
  const int first = blockIdx.y * p.blocks, nblk = min((p.K + 127) / 128 - first, p.blocks);
  const int tail = p.K & 127;  // bytes of the last block of K, where it is not whole
  // workgroups walk K from different blocks, so that they do not all ask the same memory channels at once (rows often lie a multiple of
  // 4 KB apart; us, from the first block / so: 1 x 4,096 x 4,096 6.1 / 5.4, 8 x 12,288 x 4,096 gated 21.3 / 20.4, 8 x 4,096 x 12,288 12.2 / 11.1)
  const int turn = (int)((blockIdx.x * 3u) % (unsigned)nblk);
  // ---- the loads of a block: a scalar base that advances with the block and a byte offset per lane that never changes
  uint32_t goff[NI];
  const int lrow = lane >> 3, lslot = lane & 7;
#pragma unroll
  for (int c = 0; c < NI; ++c) {
    const bool of_w = c < NWT;
    const int r = (of_w ? c % NW : c - NWT) * 8 + lrow;
    const uint32_t at = of_w ? (uint32_t)(min(n0 + min(r, p.rows - 1), N - 1) - n0) * (uint32_t)p.ldw : (uint32_t)min(r, M - 1) * (uint32_t)p.lda;
    goff[c] = at + (uint32_t)((lslot ^ ring_swz(r)) * 16);
  }
  const unsigned char* wbase = (const unsigned char*)p.W + (size_t)n0 * p.ldw;
  const unsigned char* ubase = GATED ? (const unsigned char*)p.W2 + (size_t)n0 * p.ldw : nullptr;
  const unsigned char* ring = smem + (size_t)wave * S * NI * 1024;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const unsigned char*)ring;
  const int total = wave < nblk ? (nblk - wave + WAVES - 1) / WAVES : 0;
  // ---- outputs: a thread has items of four columns of a row. What an item needs beside its sums is on its way one item ahead, the first's
  // from here on (us, asked for behind the sums / so: 1 x 4,096 x 4,096 into the residual 5.8 / 5.15, 8 x 2,560 x 2,560 with a bias 4.5 / 3.85, 64 x 12,288 x
  // 4,096 gated 25.6 / 24.9)
  constexpr int ITEMS = (CT * MT + WAVES - 1) / WAVES;
  const bool whole_k = gridDim.y == 1;
  struct Item {
    int m, n, there;  // there <= 0: none
    float sa, sw[4], su[4];
    uint32_t bias[4];
    floatx4 was;
  };
  auto item_of = [&](int i) {
    const int item = threadIdx.x + i * WAVES * 64, t = item / (MT * 64), mt = item / 64 % MT, in = t * 16 + (item >> 4 & 3) * 4;
    Item it;
    it.m = mt * 16 + (item & 15), it.n = n0 + in;
    it.there = item < CT * MT * 64 && it.m < M ? min(4, min(N - it.n, p.rows - in)) : 0;
    if (whole_k && wave + i * WAVES < CT * MT) {
      const int m = min(it.m, M - 1);
      it.sa = p.end.scales.a[m];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int n = min(it.n + c, N - 1);
        it.sw[c] = p.end.scales.w[n];
        if (GATED) it.su[c] = p.end.scales.w2[n];
        if (!GATED && p.end.epilogue == 1) it.was[c] = ((const float*)p.end.out)[(size_t)m * p.end.ldo + n];
      }
      int8_load_bias(p.end, it.n, it.bias);
    }
    return it;
  };
  Item next = item_of(0);
  auto issue = [&](int i, int slot) {
    int b = wave + i * WAVES + turn;
    b = first + (b >= nblk ? b - nblk : b);
    const size_t kbytes = (size_t)b * 128;
    const bool cut = tail != 0 && (b + 1) * 128 > p.K;
#pragma unroll
    for (int c = 0; c < NI; ++c) {
      const unsigned char* base = (c >= NWT ? (const unsigned char*)p.A : GATED && c >= NW ? ubase : wbase) + kbytes;
      const uint32_t to = lds0 + (uint32_t)(slot * NI + c) * 1024u;
      if (cut) {  // pieces that are not there are zeros, of both operands
        const int r = (c < NWT ? c % NW : c - NWT) * 8 + lrow;
        load_to_lds_16((lslot ^ ring_swz(r)) * 16 < tail ? (const void*)(base + goff[c]) : (const void*)&int8_zeros, to);
      } else {
        load_to_lds_16(base, goff[c], to);
      }
    }
  };
#pragma unroll
  for (int i = 0; i < S; ++i)
    if (i < total) issue(i, i);
  // ---- fragments: lane l reads row l % 16, 16 of k at (l / 16) * 16 + 64 j: piece l / 16 + 4 j. Rows that no load fetched (of an odd
  // number of eights) are the last fetched eight again.
  intx4 acc[MATS][CT][MT];
#pragma unroll
  for (int u = 0; u < MATS; ++u)
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) acc[u][t][m] = intx4{0, 0, 0, 0};
  auto place = [&](int loads, int t) {  // of a lane's fragment of tile t among `loads` eights
    const int r = t * 16 + (loads - 2 * t == 1 ? col & 7 : col);
    return r * 128 + ((g ^ ring_swz(r)) << 4);
  };
  int slot = 0;
  for (int i = 0; i < total; ++i) {
    i8_wait_block<NI, S>(min(S - 1, total - 1 - i));
    const unsigned char* blk = ring + slot * NI * 1024;
    u32x4 a[MT][2], w[MATS][CT][2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {  // (piece + 4: bit 6 of the address)
#pragma unroll
      for (int m = 0; m < MT; ++m) a[m][j] = *(const u32x4*)(blk + NWT * 1024 + (place(NA, m) ^ (j * 64)));
#pragma unroll
      for (int u = 0; u < MATS; ++u)
#pragma unroll
        for (int t = 0; t < CT; ++t) w[u][t][j] = *(const u32x4*)(blk + u * NW * 1024 + (place(NW, t) ^ (j * 64)));
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot's last reads, before it is filled again
    __builtin_amdgcn_sched_barrier(0);
    if (i + S < total) issue(i + S, slot);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int u = 0; u < MATS; ++u)
#pragma unroll
        for (int t = 0; t < CT; ++t)
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[u][t][m] = mfma16_i8(w[u][t][j], a[m][j], acc[u][t][m]);
    if (++slot == S) slot = 0;
  }
  // ---- the waves' sums meet in LDS
  __syncthreads();  // every wave is done with its ring
  intx4(*red)[MATS][CT][MT][64] = (intx4(*)[MATS][CT][MT][64])smem;
#pragma unroll
  for (int u = 0; u < MATS; ++u)
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m) red[wave][u][t][m][lane] = acc[u][t][m];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const Item it = next;
    if (i + 1 < ITEMS) next = item_of(i + 1);
    if (it.there <= 0) continue;
    const int item = threadIdx.x + i * WAVES * 64, t = item / (MT * 64), mt = item / 64 % MT;
    intx4 sum[MATS];
#pragma unroll
    for (int u = 0; u < MATS; ++u) {
      sum[u] = intx4{0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < WAVES; ++w) sum[u] += red[w][u][t][mt][item & 63];
    }
    if (!whole_k) {
#pragma unroll
      for (int u = 0; u < MATS; ++u)
        int8_part_store(p.partial + ((size_t)blockIdx.y * MATS + u) * M * N, it.m, it.n, it.there, N, sum[u]);
    } else {
      const Int8RowScale sa = int8_row_scale(it.sa);
      floatx4 y;
#pragma unroll
      for (int c = 0; c < 4; ++c) y[c] = int8_output(sum[0][c], sa, it.sw[c], int8_bias(p.end, it.bias[c]));
      if (GATED) {
        floatx4 u;
#pragma unroll
        for (int c = 0; c < 4; ++c) u[c] = int8_output(sum[MATS - 1][c], sa, it.su[c], 0.f);
        y = int8_gated4(y, u, p.end.gate, p.end.out_dtype);
      }
      if (!GATED && p.end.epilogue == 1) y += it.was;
      int8_store4(p.end, it.m, it.n, it.there, y);
    }
  }
}

template <int NW, int NA, bool GATED>
static int launch_stream8(const Stream8Args& a, dim3 grid, hipStream_t stream) {
  // as many waves, up to four, as have two blocks each in their rings
  constexpr int NI = (GATED ? 2 : 1) * NW + NA, WAVES = i8_slots(NI, 4) >= 2 ? 4 : i8_slots(NI, 3) >= 2 ? 3 : 2, S = i8_slots(NI, WAVES);
  constexpr size_t smem = (size_t)S * WAVES * NI * 1024;
  if (!int8_allow_lds<gemm_int8_stream_kernel<NW, NA, GATED, WAVES>>((int)smem))
    JLLM_FAIL("gemm_int8_stream: cannot reserve %zu bytes of LDS", smem);
  gemm_int8_stream_kernel<NW, NA, GATED, WAVES><<<grid, WAVES * 64, smem, stream>>>(a);
  return 0;
}

template <int NA, bool GATED>
static int launch_stream8_rows(const Stream8Args& a, dim3 grid, hipStream_t stream) {
  const int eights = (a.rows + 7) / 8;
#define I8_EIGHTS(NW) if (eights <= NW) return launch_stream8<NW, NA, GATED>(a, grid, stream)
  I8_EIGHTS(1); I8_EIGHTS(2); I8_EIGHTS(3); I8_EIGHTS(4); I8_EIGHTS(6); I8_EIGHTS(8); I8_EIGHTS(9); I8_EIGHTS(10); I8_EIGHTS(12);
#undef I8_EIGHTS
  return 1;
}

template <bool GATED>
static int launch_stream8_batch(const Stream8Args& a, dim3 grid, hipStream_t stream) {
  const int M = a.end.M;
  if (M <= 8) return launch_stream8_rows<1, GATED>(a, grid, stream);
  if (M <= 16) return launch_stream8_rows<2, GATED>(a, grid, stream);
  if (M <= 32) return launch_stream8_rows<4, GATED>(a, grid, stream);
  if (M <= 48) return launch_stream8_rows<6, GATED>(a, grid, stream);
  return launch_stream8_rows<8, GATED>(a, grid, stream);
}

// `rows`: weight rows of each weight that a workgroup owns, up to 96.
// `parts` > 1 cuts K; `partial` then holds parts * (1 or, gated, 2) * M * N ints. Returns 0 when it ran, 1 when the shape is not one it takes,
// -1 on errors.
extern "C" int jllm_gemm_int8_stream(const void* A, int lda, const float* a_scale, const void* W, int ldw, const float* w_scale, const void* W2, int ldw2,
                                     const float* w2_scale, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int K,
                                     int epilogue, float gate_limit, int rows, int parts, int* partial, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (M > 64 || K <= 0 || K > I8_MOST_K || (K & 15) || (lda & 15) || (ldw & 15) || (W2 && ldw2 != ldw)) return 1;
  if (((uintptr_t)A & 15) || ((uintptr_t)W & 15) || ((uintptr_t)W2 & 15)) return 1;
  JLLM_TAKE_GATE("gemm_int8_stream", epilogue, gate_limit, gs);
  if (epilogue < 0 || epilogue > 2 || (epilogue == 2) != (W2 != nullptr)) JLLM_FAIL("gemm_int8_stream: epilogue %d", epilogue);
  if (epilogue == 1 && out_dtype != JLLM_F32) JLLM_FAIL("gemm_int8_stream: the accumulate epilogue adds into fp32");
  if (lda < 0 || ldw < 0 || ldo < N) JLLM_FAIL("gemm_int8_stream: rows %d, %d and %d apart", lda, ldw, ldo);
  if (rows < 1 || rows > 96) JLLM_FAIL("gemm_int8_stream: %d weight rows per workgroup (1 to 96)", rows);
  // a lane's place in an operand is a 32-bit byte offset from the workgroup's first row
  if ((unsigned)lda >= (1u << 25) || (unsigned)ldw >= (1u << 25)) return 1;
  const int blocks = (K + 127) / 128;
  parts = parts < 1 ? 1 : parts > blocks ? blocks : parts;
  const int each = (blocks + parts - 1) / parts;
  parts = (blocks + each - 1) / each;  // those that have any block
  const dim3 grid((N - 1) / rows + 1, parts);
  if (!jllm_grid_fits(grid, 256)) return 1;
  if (parts > 1 && (!partial || ((uintptr_t)partial & 15))) JLLM_FAIL("gemm_int8_stream: %d parts of K need a buffer for their sums", parts);
  const Stream8Args a{(const signed char*)A, (const signed char*)W, (const signed char*)W2, partial, lda, ldw, K, rows, each,
                      {{a_scale, w_scale, w2_scale}, bias, out, bias_dtype, out_dtype, ldo, M, N, epilogue, gs}};
  const int rc = W2 ? launch_stream8_batch<true>(a, grid, stream) : launch_stream8_batch<false>(a, grid, stream);
  if (rc != 0) return rc;
  JLLM_CHECK_LAUNCH("gemm_int8_stream");
  return parts > 1 ? int8_add_parts(partial, parts, a.end, W2 != nullptr, stream) : 0;
}
