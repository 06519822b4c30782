// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for rows of 8-bit integers in tiles of 64 x 64 to 128 x 128, for products
// of more than 64 rows that the large tiles would leave most compute units without (v_mfma_i32_16x16x64_i8).
//
// A wave owns RM x CN accumulators of 16 x 16, WGM x WGN waves a tile. K advances in stages of 128 bytes through a ring of NS stages
// in LDS, filled without registers (whole lines of 128 bytes, eight rows to an instruction, the bank swizzle applied on the global
// side). A stage's fragments are in registers before its multiplies begin; between these, evenly, a wave reads the next stage's into
// a second set and asks for its share of the stage that takes the place of the one it multiplies. One barrier a stage.
//
// What binds is the pipe through which a compute unit fills its LDS, and where there are few stages the launch, the first bytes and the sum
// of the parts. Two workgroups of 64 x 64 or 64 x 128 share a compute unit. us inside a graph: 128 x 6,144 x 4,096 11.9 (64 x 64), 487 23.0 (128 x
// 128; in 64 x 64 27.6), 320 x 12,288 x 4,096 gated 55.6 (64 x 128; the large tiles 43.7), 128 x 12,288 x 4,096 gated 28.5 (128 x 128), 1,000 x 2,048 x
// 2,048 10.8, 80 x 601 x 13,824 gated 13.4 (64 x 64 in six parts; with K whole 35.9). The scales requested at the start instead of in front of the
// outputs: the same or up to 6 % slower. Measured and not kept, since others were never far behind: 128 x 64, 128 x 128 by four waves in a ring of two, 128 x 256 and 256 x 128
// here (the large tiles' forms are 1 to 2 % faster).
//
// K may be cut over gridDim.z: the parts leave their whole-number sums, and a second kernel adds them and makes the outputs.
// Needs K % 16 == 0 and 16-byte aligned rows; any M and N.
#include <type_traits>
#include "int8_mfma.h"
#include "int8_parts.h"
#include "lds_ring.h"

#define T8_ROW_BYTES 128
#define T8_FENCE() __builtin_amdgcn_sched_barrier(0)

template <bool GATED, int RM, int CN, int WGM, int WGN, int NS>
__global__ __launch_bounds__(WGM* WGN * 64) void gemm_int8_tiled_kernel(Int8Args p) {
  constexpr int WAVES = WGM * WGN, TBM = WGM * RM * 16, TBN = WGN * CN * 16, STAGE = (TBM + TBN) * T8_ROW_BYTES;
  constexpr int LA = TBM / 8 / WAVES, L = LA + TBN / 8 / WAVES;  // load instructions (8 rows each) per wave and stage
  constexpr int NM = 2 * RM * CN, NR = 2 * (RM + CN);            // multiplies and LDS reads of a stage
  constexpr int EVERY = NS == 2 ? 1 : NM / L;                    // (a ring of two: what is asked for has to land within the stage)
  static_assert(LA * 8 * WAVES == TBM && (L - LA) * 8 * WAVES == TBN && EVERY >= 1, "every wave loads as many rows of either operand");
  static_assert(NS >= 2 && NS <= 6, "one stage being read, the others on their way");
  extern __shared__ __align__(1024) unsigned char smem[];
  const int M = p.end.M, N = p.end.N, tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int wm = wave / WGN, wn = wave % WGN;
  int row, col;
  int8_die_tile(blockIdx.x + blockIdx.y * gridDim.x, gridDim.y, gridDim.x, row, col);
  const int m0 = row * TBM, n0 = col * (GATED ? TBN / 2 : TBN);
  const int nk_all = (p.K + 127) / 128, nk_per = (nk_all + gridDim.z - 1) / gridDim.z, kt0 = blockIdx.z * nk_per;
  const int nk = max(0, min(nk_all, kt0 + nk_per) - kt0);
  const int tail = p.K & 127;  // bytes of the last stage of K, where it is not whole

  // ---- global side of the loads: the tile's start at its first stage and a 32-bit byte offset per lane that never changes
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const unsigned char* abase = (const unsigned char*)p.A + (size_t)m0 * p.lda + (size_t)kt0 * 128;
  const unsigned char* wbase[2] = {(const unsigned char*)p.W + (size_t)n0 * p.ldw + (size_t)kt0 * 128,
                                   (const unsigned char*)(GATED ? p.W2 : p.W) + (size_t)n0 * p.ldw + (size_t)kt0 * 128};
  const unsigned char* base[L];
  uint32_t off[L];
#pragma unroll
  for (int c = 0; c < L; ++c) {
    const int chunk = c < LA ? wave * LA + c : wave * (L - LA) + c - LA, r = chunk * 8 + (lane >> 3);
    const uint32_t piece = (uint32_t)(((lane & 7) ^ ring_swz(r)) * 16);
    if (c < LA) {
      base[c] = abase;
      off[c] = (uint32_t)min(r, M - 1 - m0) * (uint32_t)p.lda + piece;
    } else {  // gated: of a wave's CN blocks of 16 the first half is gate rows, the second the up rows of the same outputs
      const int block = chunk % (2 * CN) / 2;  // the same in all lanes
      const int n = GATED ? chunk / (2 * CN) * CN * 8 + block % (CN / 2) * 16 + (r & 15) : r;
      base[c] = wbase[GATED && block >= CN / 2];
      off[c] = (uint32_t)min(n, N - 1 - n0) * (uint32_t)p.ldw + piece;
    }
  }
  auto load = [&](int t, uint32_t slot, int c, bool whole) {  // the wave's load c of stage t into the slot at byte `slot`
    const unsigned char* from = base[c] + (size_t)t * 128;
    const uint32_t to = lds0 + slot + (c < LA ? (wave * LA + c) * 1024 : TBM * T8_ROW_BYTES + (wave * (L - LA) + c - LA) * 1024);
    if (!whole && tail && kt0 + t == nk_all - 1) {  // pieces that are not there are zeros, of both operands
      const int chunk = c < LA ? wave * LA + c : wave * (L - LA) + c - LA;
      const bool there = ((lane & 7) ^ (lane >> 3) ^ (chunk & 1)) * 16 < tail;
      load_to_lds_16(there ? (const void*)(from + off[c]) : (const void*)&int8_zeros, to);
      return;
    }
    load_to_lds_16(from, off[c], to);
  };
  auto landed = [&](int left) {  // until at most `left` stages of the wave's loads are on their way
    if (NS >= 6 && left >= 4) wait_loads<4 * L>();
    else if (NS >= 5 && left >= 3) wait_loads<3 * L>();
    else if (NS >= 4 && left >= 2) wait_loads<2 * L>();
    else if (left >= 1) wait_loads<L>();
    else wait_loads<0>();
  };
  auto meet = [&] {  // behind the wave's own reads: the stage that it has in registers now is free for the loads of all
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    T8_FENCE();
    __builtin_amdgcn_s_barrier();
    T8_FENCE();
  };

  // ---- LDS side: fragment of a block of 16 rows: row = block * 16 + lane % 16, piece = lane / 16 (16 of 64 k), + 4 for the stage's second 64
  // (bit 6 of the address); 16 rows further leaves ring_swz unchanged
  const int ra = wm * RM * 16 + (lane & 15), rb = wn * CN * 16 + (lane & 15);
  const int aread = ra * T8_ROW_BYTES + (((lane >> 4) ^ ring_swz(ra)) * 16);
  const int bread = TBM * T8_ROW_BYTES + rb * T8_ROW_BYTES + (((lane >> 4) ^ ring_swz(rb)) * 16);
  u32x4 fa[2][2][RM], fb[2][2][CN];  // [set][64 of k][block]
  auto read = [&](int set, uint32_t slot, int x) {  // read x of a stage, in the order of use
    const int kk = x / (RM + CN), y = x % (RM + CN);
    if (y < CN) fb[set][kk][y] = *(const u32x4*)(smem + slot + (bread ^ (kk * 64)) + y * 16 * T8_ROW_BYTES);
    else fa[set][kk][y - CN] = *(const u32x4*)(smem + slot + (aread ^ (kk * 64)) + (y - CN) * 16 * T8_ROW_BYTES);
  };
  intx4 acc[RM][CN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < CN; ++j) acc[i][j] = intx4{0, 0, 0, 0};

  // ---- prologue: every stage of the ring on its way, the first in registers, the second landed
#pragma unroll
  for (int s = 0; s < NS; ++s)
    if (s < nk) {
#pragma unroll
      for (int c = 0; c < L; ++c) load(s, s * STAGE, c, false);
    }
  if (nk >= NS) wait_loads<(NS - 1) * L>();
  else wait_loads<0>();
  meet();
#pragma unroll
  for (int x = 0; x < NR; ++x) read(0, 0, x);
  if (nk >= NS) wait_loads<(NS - 2) * L>();
  meet();
  // Stage t is multiplied from one set of registers while stage t + 1 (its slot: rs) is read into the other and stage t + NS loaded into
  // the slot of stage t (ws). At its end stage t + 2 has landed: each wave waits for its own loads, the barrier for all waves.
  uint32_t rs = STAGE, ws = 0;
  auto stage = [&](auto which, auto full, int t) {
    constexpr int SET = decltype(which)::value;
    constexpr bool FULL = decltype(full)::value;  // not among the last stages: every load is asked for, of a whole stage
    const int to_load = t + NS;
#pragma unroll
    for (int n = 0; n < NM; ++n) {
      const int kk = n / (RM * CN), i = n % (RM * CN) / CN, j = n % CN;
      // the weight fragment goes in as the first operand: a lane then owns four consecutive output columns of one row
      acc[i][j] = mfma16_i8(fb[SET][kk][j], fa[SET][kk][i], acc[i][j]);
      T8_FENCE();
      if (n < NR) {
        read(1 - SET, rs, n);
        T8_FENCE();
      }
      if (n == NM - 1) {
#pragma unroll
        for (int x = NM; x < NR; ++x) read(1 - SET, rs, x);
      }
      if (n % EVERY == EVERY / 2 && n / EVERY < L && (FULL || to_load < nk)) {
        load(to_load, ws, n / EVERY, FULL);
        T8_FENCE();
      }
    }
    landed(FULL ? NS - 2 : min(to_load, nk - 1) - (t + 2));
    meet();
    rs = rs == (NS - 1) * STAGE ? 0 : rs + STAGE;
    ws = ws == (NS - 1) * STAGE ? 0 : ws + STAGE;
  };
  int t = 0;
  for (; t + 1 < nk - NS - (tail ? 1 : 0); t += 2) {
    stage(std::integral_constant<int, 0>{}, std::true_type{}, t);
    stage(std::integral_constant<int, 1>{}, std::true_type{}, t + 1);
  }
  for (; t < nk; t += 2) {  // (the reads behind the last stage fetch some slot's bytes, which are never multiplied)
    stage(std::integral_constant<int, 0>{}, std::false_type{}, t);
    if (t + 1 < nk) stage(std::integral_constant<int, 1>{}, std::false_type{}, t + 1);
  }
  if (gridDim.z > 1)
    int8_partial<GATED>(acc, lane, wm, wn, m0, n0, p.partial, M, N);
  else
    int8_epilogue<GATED, RM, CN>(acc, lane, wm, wn, m0, n0, p.end);
}

template <bool GATED, int RM, int CN, int WGM, int WGN, int NS>
static int launch_int8_tiled(const Int8Args& a, int parts, hipStream_t stream) {
  constexpr int TBM = WGM * RM * 16, TBN = WGN * CN * 16, COLS = GATED ? TBN / 2 : TBN, LDS = (TBM + TBN) * T8_ROW_BYTES * NS;
  static_assert(LDS <= 160 * 1024, "the ring fits");
  const dim3 grid((a.end.N - 1) / COLS + 1, (a.end.M - 1) / TBM + 1, parts);
  if (!jllm_grid_fits(grid, WGM * WGN * 64)) return 1;
  if (!int8_allow_lds<gemm_int8_tiled_kernel<GATED, RM, CN, WGM, WGN, NS>>(LDS))
    JLLM_FAIL("gemm_int8_tiled: cannot reserve %d bytes of LDS", LDS);
  // No more of the ring than the stages there are and the one behind them, whose bytes are read and not used: then more workgroups share a compute
  // unit. us, the whole ring / so: 7,984 x 8,832 x 16 gated in fp32 113 / 91, 1,284 x 14,464 x 128 gated 34.3 / 28.4, in tiles of 64 x 64 52.5 / 35.1.
  const int stages = (a.K + 127) / 128, slots = min(NS, (stages + parts - 1) / parts + 1);
  gemm_int8_tiled_kernel<GATED, RM, CN, WGM, WGN, NS><<<grid, WGM * WGN * 64, (TBM + TBN) * T8_ROW_BYTES * slots, stream>>>(a);
  return 0;
}

// `tile`: rows * 1000 + columns of the output tile (gated: twice its outputs). `parts` > 1 cuts K into so many, in whole stages of 128;
// `partial` then holds parts * (1 or, gated, 2) * M * N ints. Returns 0 when it ran, 1 when the shape is not one it takes, -1 on errors.
extern "C" int jllm_gemm_int8_tiled(const void* A, int lda, const float* a_scale, const void* W, int ldw, const float* w_scale, const void* W2, int ldw2,
                                    const float* w2_scale, const void* bias, int bias_dtype, void* out, int out_dtype, int ldo, int M, int N, int K,
                                    int epilogue, float gate_limit, int tile, int parts, int* partial, hipStream_t stream) {
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || K > I8_MOST_K || (K & 15) || (lda & 15) || (ldw & 15) || (W2 && ldw2 != ldw)) return 1;
  if (((uintptr_t)A & 15) || ((uintptr_t)W & 15) || ((uintptr_t)W2 & 15)) return 1;
  JLLM_TAKE_GATE("gemm_int8_tiled", epilogue, gate_limit, gs);
  if (epilogue < 0 || epilogue > 2 || (epilogue == 2) != (W2 != nullptr)) JLLM_FAIL("gemm_int8_tiled: epilogue %d", epilogue);
  if (epilogue == 1 && out_dtype != JLLM_F32) JLLM_FAIL("gemm_int8_tiled: the accumulate epilogue adds into fp32");
  if (lda < 0 || ldw < 0 || ldo < N) JLLM_FAIL("gemm_int8_tiled: rows %d, %d and %d apart", lda, ldw, ldo);
  // a lane's place in an operand is a 32-bit byte offset from the tile's first row
  if ((unsigned)lda >= (1u << 24) || (unsigned)ldw >= (1u << 24)) return 1;
  const int stages = (K + 127) / 128;
  if (parts < 1) parts = 1;
  if (parts > 1 && (!partial || ((uintptr_t)partial & 15))) JLLM_FAIL("gemm_int8_tiled: %d parts of K need a buffer for their sums", parts);
  if (parts > 65535 || (parts > 1 && stages <= (stages + parts - 1) / parts * (parts - 1))) return 1;  // a part without any
  const Int8Args a{(const signed char*)A, (const signed char*)W, (const signed char*)W2, partial, lda, ldw, K,
                   {{a_scale, w_scale, w2_scale}, bias, out, bias_dtype, out_dtype, ldo, M, N, epilogue, gs}};
  int rc;
#define T8_CASE(CODE, ...) \
  case CODE: rc = W2 ? launch_int8_tiled<true, __VA_ARGS__>(a, parts, stream) : launch_int8_tiled<false, __VA_ARGS__>(a, parts, stream); break;
  switch (tile) {
    T8_CASE(64064, 2, 2, 2, 2, 4)
    T8_CASE(64128, 2, 4, 2, 2, 3)
    T8_CASE(128128, 2, 4, 4, 2, 5)
    default: JLLM_FAIL("gemm_int8_tiled: tiles of %d rows by %d columns are not built", tile / 1000, tile % 1000);
  }
#undef T8_CASE
  if (rc != 0) return rc;
  JLLM_CHECK_LAUNCH("gemm_int8_tiled");
  return parts > 1 ? int8_add_parts(partial, parts, a.end, W2 != nullptr, stream) : 0;
}
