// out[m][n] = a_scale[m] * w_scale[n] * sum_k A[m][k] W[n][k] for many rows of 8-bit integers, on the matrix cores
// (v_mfma_i32_16x16x64_i8).
//
//  * A workgroup of 8 waves owns a tile of 256 x 256 outputs (2 x 4 waves of 128 x 64), or of 192 x 256, 128 x 256 or 256 x 128.
//  * K advances in stages of 128 bytes, whole lines, eight rows to a load instruction. A stage is four units of LDS: each operand's first
//    half (for every wave the first half of its rows, of its columns) and second. Two units are a pair, which is what the ring in LDS
//    holds: even pairs the first halves A0 and B0 of a stage, odd ones its B1 and A1; five pairs of 32 KB are all of the 160 KB.
//  * Global -> LDS without registers, three to four pairs ahead, the bank swizzle applied on the global side (ring_swz).
//  * A wave multiplies half a stage between two barriers, A0 with B0 and B1, then A1 with both, its operands in registers when the half
//    begins except for B1; between the multiplies, evenly, stand the LDS reads of the next pair and its loads.
//  * A die takes a run of neighbouring tiles (int8_die_tile).
//
// That is the plan of the bf16 product's large tiles (gemm_pingpong.hip): in bytes and clocks an int8 stage of 128 is a bf16 stage of 64,
// so a product of half the bytes takes half the time. 8,192 x 17,408 x 5,120 gated 1,015 to 1,100 us by card, 2.65 to 2.9 POP/s
// (a library's 8,192 x 8,192 x 8,192 2.05 to 2.44, this one's 2.3 to 2.95; the matrix cores' peak at 2.4 GHz is 5.0): a half stage takes 1,190 clocks of
// the 1,024 that its multiplies take alone, at the 1.7 GHz that the chip's power leaves, and of a round's 111,000 clocks 16,000 lie beside its
// stages (first bytes, outputs).
//
// K may be cut over gridDim.z: the parts leave their whole-number sums, and a second kernel adds them and makes the outputs.
// Needs K % 16 == 0 and 16-byte aligned rows, K > 128; any M and N.
#include <type_traits>
#include "int8_mfma.h"
#include "int8_parts.h"
#include "lds_ring.h"

#define L8_ROW_BYTES 128  // a tile row in LDS: 8 pieces of 16 bytes
#define L8_WAVES 8
#define L8_FENCE() __builtin_amdgcn_sched_barrier(0)

// the ring of a tile of 32 FM rows for each of WGM waves and 64 columns for each of 8 / WGM
template <int FM, int WGM>
struct Int8Ring {
  static constexpr int WGN = L8_WAVES / WGM;
  static constexpr int A_UNIT = WGM * FM * 16 * L8_ROW_BYTES, B_UNIT = WGN * 32 * L8_ROW_BYTES, PAIR = A_UNIT + B_UNIT;
  static constexpr int PAIRS = 160 * 1024 / PAIR < 5 ? 160 * 1024 / PAIR : 5, BYTES = PAIRS * PAIR;
  static_assert(PAIRS >= 4, "one being read, one that must have landed, one on its way, one that others may still read");
};

// WGM x 8 / WGM waves of 32 FM rows by 64 columns each: the tile whose first row and first output are m0 and n0. Workgroup blockIdx.z
// of gridDim.z takes its part of K. `finish` gets the wave's accumulators.
template <bool GATED, int FM, int WGM, typename F>
__device__ __forceinline__ void int8_large_tile(const signed char* __restrict__ A, int lda, const signed char* __restrict__ W, const signed char* __restrict__ W2,
                                                int ldw, int M, int N, int K, int m0, int n0, F finish) {
  using Ring = Int8Ring<FM, WGM>;
  constexpr int WGN = Ring::WGN, NP = Ring::PAIRS, PAIR = Ring::PAIR;
  // load instructions (8 rows each) per wave and unit. Where A's unit is 12 or 4 of them, the first four waves take one more.
  constexpr int NA = WGM * FM * 2, LA = (NA + L8_WAVES - 1) / L8_WAVES, LA1 = NA * 2 / L8_WAVES - LA, LB = WGN * 4 / L8_WAVES;
  static_assert((LA + LA1) * L8_WAVES / 2 == NA && LA - LA1 <= 1, "the first four waves take LA, the others LA1");
  constexpr int L0 = LA + LB, L1 = LA1 + LB;
  constexpr int NM = 8 * FM, AHEAD = NP - 3;  // multiplies of half a stage; pairs that may be on their way at its end
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x;
  // the wave's number is the same in all its lanes: said so, its part of the tile and the places in LDS it fills stay in
  // scalar registers
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const bool first = wave < L8_WAVES / 2;
  const int wm = wave / WGN, wn = wave % WGN;
  const int nk_all = (K + L8_ROW_BYTES - 1) / L8_ROW_BYTES;
  const int nk_per = (nk_all + gridDim.z - 1) / gridDim.z;
  const int kt0 = blockIdx.z * nk_per;
  const int nk = max(0, min(nk_all, kt0 + nk_per) - kt0), pairs = 2 * nk;
  const int tail = K % L8_ROW_BYTES;  // bytes of the last stage, where it is not whole

  // ---- global side of the loads: an operand's start at this workgroup's first stage (the same in all lanes, advanced by scalar
  // arithmetic) plus a 32-bit byte offset per lane that never changes (row and piece; rows x row length < 4 GB: checked on the host)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const unsigned char* abase = (const unsigned char*)A + (size_t)kt0 * L8_ROW_BYTES;
  const unsigned char* wbase[2] = {(const unsigned char*)W + (size_t)kt0 * L8_ROW_BYTES,
                                   (const unsigned char*)(GATED ? W2 : W) + (size_t)kt0 * L8_ROW_BYTES};
  uint32_t aoff[2][LA], boff[2][LB];
  const int achunk = LA == LA1 || first ? wave * LA : L8_WAVES / 2 * LA + (wave - L8_WAVES / 2) * LA1;  // (the others' c = LA1 is never asked for)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int c = 0; c < LA; ++c) {
      const int r = (achunk + c) * 8 + (lane >> 3);  // row r of the unit: row r % 16 FM of the half of wave row r / 16 FM
      const int row = r / (FM * 16) * (FM * 32) + u * FM * 16 + r % (FM * 16);
      aoff[u][c] = (uint32_t)min(m0 + row, M - 1) * (uint32_t)lda + (uint32_t)(((lane & 7) ^ ring_swz(r)) * 16);
    }
#pragma unroll
    for (int c = 0; c < LB; ++c) {
      const int r = (wave * LB + c) * 8 + (lane >> 3);  // gated: B0 is the gate's rows, B1 the up weight's of the same outputs
      const int row = GATED ? n0 + r : n0 + (r >> 5) * 64 + u * 32 + (r & 31);
      boff[u][c] = (uint32_t)min(row, N - 1) * (uint32_t)ldw + (uint32_t)(((lane & 7) ^ ring_swz(r)) * 16);
    }
  }
  const uint32_t adst = lds0 + achunk * 8 * L8_ROW_BYTES, bdst = lds0 + Ring::A_UNIT + wave * LB * 8 * L8_ROW_BYTES;
  // Load l of pair p into the slot at byte `slot`; `whole`: not of a last stage that is cut
  auto load = [&](int p, uint32_t slot, int l, bool whole) {
    if (l >= LA1 && l < LA && !first) return;
    const unsigned char* base = (l < LA ? abase : wbase[p & 1]) + (size_t)(p >> 1) * L8_ROW_BYTES;
    const uint32_t off = l < LA ? aoff[p & 1][l < LA ? l : 0] : boff[p & 1][l < LA ? 0 : l - LA];
    const uint32_t to = (l < LA ? adst + l * 1024 : bdst + (l - LA) * 1024) + slot;
    if (!whole && tail && kt0 + (p >> 1) == nk_all - 1) {  // pieces that are not there are zeros, of both operands
      const int chunk = l < LA ? achunk + l : wave * LB + l - LA;
      const bool there = (((lane & 7) ^ (lane >> 3) ^ (chunk & 1)) * 16) < tail;
      load_to_lds_16(there ? (const void*)(base + off) : (const void*)&int8_zeros, to);
    } else {
      load_to_lds_16(base, off, to);
    }
  };
  auto landed = [&](int left) {  // until at most `left` pairs of the wave's loads are on their way
    if (LA == LA1 || first) {
      if (AHEAD >= 2 && left >= 2) wait_loads<2 * L0>();
      else if (left >= 1) wait_loads<L0>();
      else wait_loads<0>();
    } else {
      if (AHEAD >= 2 && left >= 2) wait_loads<2 * L1>();
      else if (left >= 1) wait_loads<L1>();
      else wait_loads<0>();
    }
  };

  // ---- LDS side: fragment of a block of 16 rows: row = block * 16 + lane % 16, piece = lane / 16 (16 of 64 k), + 4 for the
  // stage's second 64 (bit 6 of the address); 16 rows further leaves ring_swz unchanged
  const int ra = wm * FM * 16 + (lane & 15), rb = wn * 32 + (lane & 15);
  const int aread = ra * L8_ROW_BYTES + (((lane >> 4) ^ ring_swz(ra)) * 16);
  const int bread = Ring::A_UNIT + rb * L8_ROW_BYTES + (((lane >> 4) ^ ring_swz(rb)) * 16);
  u32x4 fa[2][2][FM], fb[2][2][2];  // [half of the rows, of the columns][64 of k][block]
  auto read_a = [&](int u, uint32_t slot, int x) {
    fa[u][x / FM][x % FM] = *(const u32x4*)(smem + slot + (aread ^ (x / FM * 64)) + x % FM * 16 * L8_ROW_BYTES);
  };
  auto read_b = [&](int u, uint32_t slot, int x) {
    fb[u][x / 2][x % 2] = *(const u32x4*)(smem + slot + (bread ^ (x / 2 * 64)) + x % 2 * 16 * L8_ROW_BYTES);
  };
  intx4 acc[2 * FM][4];
#pragma unroll
  for (int i = 0; i < 2 * FM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = intx4{0, 0, 0, 0};

  // ---- prologue: all pairs but one on their way, the first two landed, the first in registers
#pragma unroll
  for (int p = 0; p < NP - 1; ++p)
    if (p < pairs) {
#pragma unroll
      for (int l = 0; l < L0; ++l) load(p, p * PAIR, l, false);
    }
  landed(pairs >= NP - 1 ? AHEAD : 0);
  L8_FENCE();
  __builtin_amdgcn_s_barrier();
  L8_FENCE();
#pragma unroll
  for (int x = 0; x < 2 * FM; ++x) read_a(0, 0, x);
#pragma unroll
  for (int x = 0; x < 4; ++x) read_b(0, 0, x);
  // Half h of the whole product reads pair h + 1 (its slot: rs) and loads pair h + NP - 1 into the slot of pair h - 1 (ws), which
  // every wave had in registers, and multiplied, before the barrier behind half h - 1. At its end pair h + 2 has landed: each wave waits for
  // its own loads, the barrier for all waves.
  uint32_t rs = PAIR, ws = (NP - 1) * PAIR;
  auto half = [&](auto which, auto full, int t) {
    constexpr int H = decltype(which)::value;
    constexpr bool FULL = decltype(full)::value;  // not among the last stages: every load is asked for
    const int p = 2 * t + H + NP - 1;
#pragma unroll
    for (int n = 0; n < NM; ++n) {
      const int q = n / (NM / 2), kk = n / (NM / 4) % 2, i = n % (NM / 4) / 2, j = n % 2;
      acc[H * FM + i][q * 2 + j] = mfma16_i8(fb[q][kk][j], fa[H][kk][i], acc[H * FM + i][q * 2 + j]);
      L8_FENCE();
      // B1 is read first, used a quarter later; A0 of the next stage while A1 is multiplied, its B0 behind the last use of this one's
      if (n % 2 == 0) {
        const int x = n / 2;
        if (H == 0) {
          if (x < 4) read_b(1, rs, x);
          else if (x < 4 + 2 * FM) read_a(1, rs, x - 4);
        } else {
          if (x < 2 * FM) read_a(0, rs, x);
          else if (x < 2 * FM + 4) read_b(0, rs, x - 2 * FM);
        }
        L8_FENCE();
      }
      constexpr int EVERY = NM / L0;
      if (n % EVERY == EVERY / 2 && n / EVERY < L0 && (FULL || p < pairs)) {
        load(p, ws, n / EVERY, FULL);
        L8_FENCE();
      }
    }
    landed(FULL ? AHEAD : min(p, pairs - 1) - (2 * t + H + 2));
    L8_FENCE();
    __builtin_amdgcn_s_barrier();
    L8_FENCE();
    rs = rs == (NP - 1) * PAIR ? 0 : rs + PAIR;
    ws = ws == (NP - 1) * PAIR ? 0 : ws + PAIR;
  };
  int t = 0;
  for (; t < nk - (tail ? 3 : 2); ++t) {
    half(std::integral_constant<int, 0>{}, std::true_type{}, t);
    half(std::integral_constant<int, 1>{}, std::true_type{}, t);
  }
  for (; t < nk; ++t) {  // (the reads behind the last stage fetch some slot's bytes, which are never multiplied)
    half(std::integral_constant<int, 0>{}, std::false_type{}, t);
    half(std::integral_constant<int, 1>{}, std::false_type{}, t);
  }
  finish(acc, lane, wm, wn);
}

template <bool GATED, int FM, int WGM>
__global__ __launch_bounds__(L8_WAVES * 64) void gemm_int8_large_kernel(Int8Args p) {
  int row, col;
  int8_die_tile(blockIdx.x + blockIdx.y * gridDim.x, gridDim.y, gridDim.x, row, col);
  constexpr int TBM = WGM * FM * 32, TBN = L8_WAVES / WGM * 64;
  const int m0 = row * TBM, n0 = col * (GATED ? TBN / 2 : TBN);
  int8_large_tile<GATED, FM, WGM>(p.A, p.lda, p.W, p.W2, p.ldw, p.end.M, p.end.N, p.K, m0, n0, [&](auto& acc, int lane, int wm, int wn) {
    if (gridDim.z > 1)
      int8_partial<GATED>(acc, lane, wm, wn, m0, n0, p.partial, p.end.M, p.end.N);
    else
      int8_epilogue<GATED, 2 * FM, 4>(acc, lane, wm, wn, m0, n0, p.end);
  });
}

template <int FM, int WGM>
static int launch_int8_large(const Int8Args& a, int parts, hipStream_t stream) {
  constexpr int TBM = WGM * FM * 32, TBN = L8_WAVES / WGM * 64;
  const int cols = a.W2 ? TBN / 2 : TBN;
  const dim3 grid((a.end.N - 1) / cols + 1, (a.end.M - 1) / TBM + 1, parts);
  if (!jllm_grid_fits(grid, L8_WAVES * 64)) return 1;
  constexpr size_t smem = Int8Ring<FM, WGM>::BYTES;
  if (!(a.W2 ? int8_allow_lds<gemm_int8_large_kernel<true, FM, WGM>>((int)smem) : int8_allow_lds<gemm_int8_large_kernel<false, FM, WGM>>((int)smem)))
    JLLM_FAIL("gemm_int8_large: cannot reserve %zu bytes of LDS", smem);
  if (a.W2)
    gemm_int8_large_kernel<true, FM, WGM><<<grid, L8_WAVES * 64, smem, stream>>>(a);
  else
    gemm_int8_large_kernel<false, FM, WGM><<<grid, L8_WAVES * 64, smem, stream>>>(a);
  return 0;
}

// `tile`: rows * 1000 + columns of the output tile (gated: twice its outputs). `parts` > 1 cuts K into so many, in whole stages of 128;
// `partial` then holds parts * (1 or, gated, 2) * M * N ints. Returns 0 when it ran, 1 when the shape is not one it takes, -1 on errors.
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
  if (parts > 1 && (!partial || ((uintptr_t)partial & 15))) JLLM_FAIL("gemm_int8_large: %d parts of K need a buffer for their sums", parts);
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
  return parts > 1 ? int8_add_parts(partial, parts, a.end, W2 != nullptr, stream) : 0;
}
