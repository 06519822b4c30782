// The large tiles' way through K, for rows of bf16 and of 8-bit integers: a workgroup's operands through a ring of half stages in LDS (what
// it does, why, and what it measured stands in gemm_pingpong.hip; rows of 8-bit integers have twice the depth in the same bytes and
// clocks), and which tile a workgroup takes.
#pragma once
#include <type_traits>
#include "common.h"
#include "lds_ring.h"
#include "mfma.h"

#define PP_ROW_BYTES 128  // a tile row in LDS: a stage of 64 bf16 or 128 8-bit entries, 8 pieces of 16 bytes
#define PP_WAVES 8
#define PP_FENCE() __builtin_amdgcn_sched_barrier(0)

// the ring of a tile of 32 FM rows for each of WGM waves and 64 columns for each of 8 / WGM
template <int FM, int WGM>
struct PingpongRing {
  static constexpr int WGN = PP_WAVES / WGM;
  static constexpr int A_UNIT = WGM * FM * 16 * PP_ROW_BYTES, B_UNIT = WGN * 32 * PP_ROW_BYTES, PAIR = A_UNIT + B_UNIT;
  static constexpr int PAIRS = 160 * 1024 / PAIR < 5 ? 160 * 1024 / PAIR : 5, BYTES = PAIRS * PAIR;
  static_assert(PAIRS >= 4, "one being read, one that must have landed, one on its way, one that others may still read");
};

// What the operands' entries are. ANY_PIECES: K may end behind any 16 bytes of a stage (zeros stand behind it); else behind half a
// stage or a whole one.
struct PingpongBf16 {
  typedef bf16_t entry;
  typedef floatx4 acc;
  static constexpr bool ANY_PIECES = false;
  static __device__ __forceinline__ acc multiply(u32x4 a, u32x4 b, acc c) { return mfma16(a, b, c); }
};

// WGM x 8 / WGM waves of 32 FM rows by 64 columns each: the tile whose first row and first output are m0 and n0. Workgroup blockIdx.z
// of gridDim.z takes its part of K. `finish` gets the wave's accumulators.
template <typename E, bool GATED, int FM, int WGM, typename F>
__device__ __forceinline__ void pingpong_tile(const typename E::entry* __restrict__ A, int lda, const typename E::entry* __restrict__ W,
                                              const typename E::entry* __restrict__ W2, int ldw, int M, int N, int K, int m0, int n0, F finish) {
  constexpr uint32_t SIZE = sizeof(typename E::entry);
  constexpr int PP_BK = PP_ROW_BYTES / (int)SIZE;
  using Ring = PingpongRing<FM, WGM>;
  constexpr int WGN = Ring::WGN, NP = Ring::PAIRS, PAIR = Ring::PAIR;
  // load instructions (8 rows each) per wave and unit. Where A's unit is 12 or 4 of them, the first four waves take one more.
  constexpr int NA = WGM * FM * 2, LA = (NA + PP_WAVES - 1) / PP_WAVES, LA1 = NA * 2 / PP_WAVES - LA, LB = WGN * 4 / PP_WAVES;
  static_assert((LA + LA1) * PP_WAVES / 2 == NA && LA - LA1 <= 1, "the first four waves take LA, the others LA1");
  constexpr int L0 = LA + LB, L1 = LA1 + LB;
  constexpr int NM = 8 * FM, AHEAD = NP - 3;  // multiplies of half a stage; pairs that may be on their way at its end
  extern __shared__ __align__(1024) unsigned char smem[];
  const int tid = threadIdx.x;
  // the wave's number is the same in all its lanes: said so, its part of the tile and the places in LDS it fills stay in
  // scalar registers
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const bool first = wave < PP_WAVES / 2;
  const int wm = wave / WGN, wn = wave % WGN;
  const int nk_all = (K + PP_BK - 1) / PP_BK;
  const int nk_per = (nk_all + gridDim.z - 1) / gridDim.z;
  const int kt0 = blockIdx.z * nk_per;
  const int nk = max(0, min(nk_all, kt0 + nk_per) - kt0), pairs = 2 * nk;
  const bool half_k = !E::ANY_PIECES && (K & (PP_BK / 2)) != 0;  // the last stage of K is half as long
  const int tail = E::ANY_PIECES ? K * (int)SIZE % PP_ROW_BYTES : 0;  // bytes of the last stage, where it is not whole

  // ---- global side of the loads: an operand's start at this workgroup's first stage (the same in all lanes, advanced by scalar
  // arithmetic) plus a 32-bit byte offset per lane that never changes (row and piece; rows x row length < 4 GB: checked on the host)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)smem;
  const unsigned char* abase = (const unsigned char*)A + (size_t)kt0 * PP_ROW_BYTES;
  const unsigned char* wbase[2] = {(const unsigned char*)W + (size_t)kt0 * PP_ROW_BYTES,
                                   (const unsigned char*)(GATED ? W2 : W) + (size_t)kt0 * PP_ROW_BYTES};
  uint32_t aoff[2][LA], boff[2][LB];
  const int achunk = LA == LA1 || first ? wave * LA : PP_WAVES / 2 * LA + (wave - PP_WAVES / 2) * LA1;  // (the others' c = LA1 is never asked for)
#pragma unroll
  for (int u = 0; u < 2; ++u) {
#pragma unroll
    for (int c = 0; c < LA; ++c) {
      const int r = (achunk + c) * 8 + (lane >> 3);  // row r of the unit: row r % 16 FM of the half of wave row r / 16 FM
      const int row = r / (FM * 16) * (FM * 32) + u * FM * 16 + r % (FM * 16);
      aoff[u][c] = (uint32_t)min(m0 + row, M - 1) * (uint32_t)lda * SIZE + (uint32_t)(((lane & 7) ^ ring_swz(r)) * 16);
    }
#pragma unroll
    for (int c = 0; c < LB; ++c) {
      const int r = (wave * LB + c) * 8 + (lane >> 3);  // gated: B0 is the gate's rows, B1 the up weight's of the same outputs
      const int row = GATED ? n0 + r : n0 + (r >> 5) * 64 + u * 32 + (r & 31);
      boff[u][c] = (uint32_t)min(row, N - 1) * (uint32_t)ldw * SIZE + (uint32_t)(((lane & 7) ^ ring_swz(r)) * 16);
    }
  }
  const uint32_t adst = lds0 + achunk * 8 * PP_ROW_BYTES, bdst = lds0 + Ring::A_UNIT + wave * LB * 8 * PP_ROW_BYTES;
  // Load l of pair p into the slot at byte `slot`. Of a last stage of 32 the lanes of its second half read the first again, which
  // is never multiplied; `whole`: not that stage. (Bit 2 of a lane's piece is that of lane ^ lane / 8, whatever the row.)
  const uint32_t second = (uint32_t)((lane ^ (lane >> 3)) & 4) * 16;
  auto load = [&](int p, uint32_t slot, int l, bool whole) {
    const size_t kbytes = (size_t)(p >> 1) * PP_ROW_BYTES;
    const uint32_t back = !whole && half_k && kt0 + (p >> 1) == nk_all - 1 ? second : 0u;
    if constexpr (E::ANY_PIECES) {
      if (!whole && tail && kt0 + (p >> 1) == nk_all - 1) {  // pieces that are not there are zeros, of both operands
        const int chunk = l < LA ? achunk + l : wave * LB + l - LA;
        const bool there = (((lane & 7) ^ (lane >> 3) ^ (chunk & 1)) * 16) < tail;
        const unsigned char* from = l < LA ? abase + kbytes + aoff[p & 1][l < LA ? l : 0] : wbase[p & 1] + kbytes + boff[p & 1][l < LA ? 0 : l - LA];
        if (l >= LA1 && l < LA && !first) return;
        load_to_lds_16(there ? (const void*)from : E::zeros(), (l < LA ? adst + l * 1024 : bdst + (l - LA) * 1024) + slot);
        return;
      }
    }
    if (l < LA) {
      if (l >= LA1 && !first) return;
      load_to_lds_16(abase + kbytes, aoff[p & 1][l] - back, adst + slot + l * 1024);
    } else {
      load_to_lds_16(wbase[p & 1] + kbytes, boff[p & 1][l - LA] - back, bdst + slot + (l - LA) * 1024);
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

  // ---- LDS side: fragment of a block of 16 rows: row = block * 16 + lane % 16, piece = lane / 16 (16 bytes: 8 of 32 k), + 4 for the
  // stage's second 32 (bit 6 of the address); 16 rows further leaves ring_swz unchanged
  const int ra = wm * FM * 16 + (lane & 15), rb = wn * 32 + (lane & 15);
  const int aread = ra * PP_ROW_BYTES + (((lane >> 4) ^ ring_swz(ra)) * 16);
  const int bread = Ring::A_UNIT + rb * PP_ROW_BYTES + (((lane >> 4) ^ ring_swz(rb)) * 16);
  u32x4 fa[2][2][FM], fb[2][2][2];  // [half of the rows, of the columns][32 of k][block]
  auto read_a = [&](int u, uint32_t slot, int x) {
    fa[u][x / FM][x % FM] = *(const u32x4*)(smem + slot + (aread ^ (x / FM * 64)) + x % FM * 16 * PP_ROW_BYTES);
  };
  auto read_b = [&](int u, uint32_t slot, int x) {
    fb[u][x / 2][x % 2] = *(const u32x4*)(smem + slot + (bread ^ (x / 2 * 64)) + x % 2 * 16 * PP_ROW_BYTES);
  };
  typename E::acc acc[2 * FM][4];
#pragma unroll
  for (int i = 0; i < 2 * FM; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = typename E::acc{};

  // ---- prologue: all pairs but one on their way, the first two landed, the first in registers
#pragma unroll
  for (int p = 0; p < NP - 1; ++p)
    if (p < pairs) {
#pragma unroll
      for (int l = 0; l < L0; ++l) load(p, p * PAIR, l, false);
    }
  landed(pairs >= NP - 1 ? AHEAD : 0);
  PP_FENCE();
  __builtin_amdgcn_s_barrier();
  PP_FENCE();
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
      if (FULL || !(kk && half_k && kt0 + t == nk_all - 1)) acc[H * FM + i][q * 2 + j] = E::multiply(fb[q][kk][j], fa[H][kk][i], acc[H * FM + i][q * 2 + j]);
      PP_FENCE();
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
        PP_FENCE();
      }
      constexpr int EVERY = NM / L0;
      if (n % EVERY == EVERY / 2 && n / EVERY < L0 && (FULL || p < pairs)) {
        load(p, ws, n / EVERY, FULL);
        PP_FENCE();
      }
    }
    landed(FULL ? AHEAD : min(p, pairs - 1) - (2 * t + H + 2));
    PP_FENCE();
    __builtin_amdgcn_s_barrier();
    PP_FENCE();
    rs = rs == (NP - 1) * PAIR ? 0 : rs + PAIR;
    ws = ws == (NP - 1) * PAIR ? 0 : ws + PAIR;
  };
  int t = 0;
  for (; t < nk - (half_k || tail ? 3 : 2); ++t) {
    half(std::integral_constant<int, 0>{}, std::true_type{}, t);
    half(std::integral_constant<int, 1>{}, std::true_type{}, t);
  }
  for (; t < nk; ++t) {  // (the reads behind the last stage fetch some slot's bytes, which are never multiplied)
    half(std::integral_constant<int, 0>{}, std::false_type{}, t);
    half(std::integral_constant<int, 1>{}, std::false_type{}, t);
  }
  finish(acc, lane, wm, wn);
}

// Which tile workgroup b of rows x cols takes: workgroups b, b + 8, b + 16 .. share a die, which gets a run of neighbouring tiles,
// in bands of four columns, row by row inside a band
__device__ __forceinline__ void die_tile(int b, int rows, int cols, int& row, int& col) {
  const int tiles = rows * cols, each = tiles >> 3, more = tiles & 7, die = b & 7;
  const int i = die * each + min(die, more) + (b >> 3);
  const int band = i / (4 * rows), r = i - band * 4 * rows, width = min(4, cols - band * 4);
  row = r / width;
  col = band * 4 + r - row * width;
}
