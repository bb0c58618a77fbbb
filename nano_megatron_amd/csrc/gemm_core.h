// The pipelined core of the bf16 matrix products: operand tiles streamed into
// LDS, fragments, and the K loop of one output tile (gemm.hip describes the
// layouts).
#pragma once

#include <type_traits>

#include "common.h"
#include "lds_dma.h"

namespace nmb {
namespace {

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ bf16x8 ld8(const bf16* p) { return *reinterpret_cast<const bf16x8*>(p); }

// 16-byte chunk slots of the K-contiguous tile.  64-deep K tiles (128-byte
// rows, 8 chunks): row r keeps chunk c in slot c ^ (r & 7).  32-deep K tiles
// (64-byte rows, 4 chunks): slot c ^ ((r >> 1) & 3).  With these a fragment
// read (16 rows x 16 bytes in each group of 16 lanes) has no LDS bank
// conflicts on gfx950 (SQ_LDS_BANK_CONFLICT reads zero; c ^ (r & 3), no
// swizzle, and ((r >> 1) & 3) ^ ((r >> 3) & 1) give two-way conflicts).
template <int BKT>
__device__ __forceinline__ int kc_swizzle(int r) {
  return BKT == 64 ? (r & 7) : ((r >> 1) & 3);
}
// 32-byte pair slots of the M/N-contiguous tile: k row k keeps pair p in slot
// p ^ rc_swizzle(k), so that the 8 k rows of a half-wave transposed read
// (k .. k + 3 and k + 8 .. k + 11) land on distinct banks.
__device__ __forceinline__ int rc_swizzle(int k) { return (k & 3) | ((k >> 1) & 4); }

// One wave's share of the loads of an R-row operand tile per BKT-deep K tile:
// R * BKT / 512 load instructions of 1 KB (64 lanes x 16 B), spread over NW
// waves.
template <int R, bool KC, int BKT, int NW>
struct Loader {
  static constexpr int kPer = R * BKT / (512 * NW);
  static constexpr int kCpr = BKT / 8;   // K-contiguous: 16-byte chunks per row
  static constexpr int kRpi = 64 / kCpr; // K-contiguous: rows per instruction
  static constexpr int kChunks = R / 8;  // M/N-contiguous: 16-byte chunks per k row
  static_assert(kPer >= 1 && R * BKT % (512 * NW) == 0, "tile must split evenly over the waves");
  static_assert(KC || R == 128 || R == 256, "M/N-contiguous tiles have 128 or 256 columns");
  i32x4 rsrc;
  uint32_t off[kPer];  // byte offset at k0 = 0, kOOB for an invalid row / column
  int kin[kPer];       // k index (within the K tile) where this lane's chunk starts
  uint32_t kstride;    // bytes per unit of k

  // base: element (row0, k 0) of the tile (K-contiguous) or (k 0, col0)
  // (M/N-contiguous); valid: rows (K-contiguous) or columns of the tile inside
  // the matrix; bytes: extent of the matrix from base.
  __device__ void init(const bf16* base, int64_t ld, int valid, uint32_t bytes, int wave, int lane) {
    rsrc = make_rsrc(base, bytes);
    kstride = KC ? 2u : static_cast<uint32_t>(2 * ld);
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = wave * kPer + j;
      if (KC) {
        // instruction i fills rows kRpi i ..; lane p: row kRpi i + p / kCpr, slot p % kCpr
        const int r = kRpi * i + lane / kCpr;
        const int c = (lane % kCpr) ^ kc_swizzle<BKT>(r);
        kin[j] = 8 * c;
        off[j] = r < valid ? static_cast<uint32_t>((r * ld + 8 * c) * 2) : kOOB;
      } else {
        const int q = 64 * i + lane;
        const int kr = q / kChunks, s = q % kChunks;
        const int c = s ^ (2 * rc_swizzle(kr));  // pair swizzle keeps the chunk's low bit
        kin[j] = kr;
        off[j] = 8 * c < valid ? static_cast<uint32_t>((kr * ld + 8 * c) * 2) : kOOB;
      }
    }
  }

  // SwiGLU tiles (K-contiguous [2F, K] weights, gate rows then up rows): tile
  // row r reads gate (r & 32 clear) or up row j0 + 32 (r / 64) + r % 32, so a
  // wave's 64 columns hold 32 gate columns and the matching 32 up columns.
  __device__ void init_pairs(const bf16* base, int64_t ld, int f, int j0, uint32_t bytes, int wave,
                             int lane) {
    static_assert(KC, "paired rows need K-contiguous weights");
    rsrc = make_rsrc(base, bytes);
    kstride = 2u;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int i = wave * kPer + j;
      const int r = kRpi * i + lane / kCpr;
      const int c = (lane % kCpr) ^ kc_swizzle<BKT>(r);
      const int col = j0 + 32 * (r >> 6) + (r & 31);
      const int64_t row = col + ((r >> 5) & 1) * static_cast<int64_t>(f);
      kin[j] = 8 * c;
      off[j] = col < f ? static_cast<uint32_t>((row * ld + 8 * c) * 2) : kOOB;
    }
  }

  // Loads K tile [k0, k0 + BKT) (zeros at and past k_end) with scalar arithmetic
  // only for a whole K tile: m0 is the LDS byte address of this wave's first
  // 1 KB of the tile (uniform) and the K advance rides in the instruction's
  // scalar offset; a partial last K tile zeroes its chunks past k_end per lane.
  __device__ __forceinline__ void issue_s(uint32_t m0, int k0, int k_end) const {
    const uint32_t koff = static_cast<uint32_t>(k0) * kstride;
    if (k0 + BKT <= k_end) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) load_lds16s(rsrc, m0 + 1024u * j, off[j], koff);
    } else {
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const bool ok = off[j] != kOOB && k0 + kin[j] < k_end;
        load_lds16s(rsrc, m0 + 1024u * j, ok ? off[j] : kOOB, koff);
      }
    }
  }
  // Load j of issue_s alone, any K tile (past k_end: zeros), without a branch.
  // The scalar offset stays inside the matrix: the hardware takes it off
  // num_records before the range check of the lane's offset.
  __device__ __forceinline__ void issue_one(int j, uint32_t m0, int k0, int k_end) const {
    const bool ok = off[j] != kOOB && k0 + kin[j] < k_end;
    const uint32_t koff = k0 < k_end ? static_cast<uint32_t>(k0) * kstride : 0u;
    load_lds16s(rsrc, m0 + 1024u * j, ok ? off[j] : kOOB, koff);
  }
};

// Per-lane LDS offsets (elements) of the MFMA fragments of T 16-row groups of
// an R-row operand tile, starting at tile row row0: fragment t of k32 step kk
// gives lane l op[row0 + 16 t + l % 16][kk + 8 (l / 16) .. + 7].
template <int R, bool KC, int T, int BKT>
struct Frags {
  // K-contiguous: one offset (the swizzle depends on l % 16 only; the group
  // offset 16 t BKT is an immediate, and for kk = 32 the chunk (4 + g) ^ x is
  // (g ^ x) ^ 4).  M/N-contiguous: the two transposed reads of each fragment
  // (the swizzle does not depend on k bit 5).
  int off[KC ? 1 : 2 * T];

  __device__ void init(int row0, int lane) {
    const int l16 = lane & 15, g = lane >> 4;
    if (KC) {
      off[0] = (row0 + l16) * BKT + 8 * (g ^ kc_swizzle<BKT>(l16));
    } else {
#pragma unroll
      for (int t = 0; t < T; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          // lane p of group g: k row 8 g + 4 h + p / 4, columns 16 pair + 4 (p & 3) .. + 3
          const int k = 8 * g + 4 * h + (l16 >> 2);
          const int pair = (row0 >> 4) + t;
          off[2 * t + h] = k * R + 16 * (pair ^ rc_swizzle(k)) + 4 * (l16 & 3);
        }
    }
  }

  __device__ __forceinline__ bf16x8 get(const bf16* tile, int t, int kk) const {
    if (KC) return ld8(tile + t * 16 * BKT + (kk ? (off[0] ^ 32) : off[0]));
    return ld_tr(tile + off[2 * t] + kk * R, tile + off[2 * t + 1] + kk * R);
  }
};

// LDS stages of a configuration (K tiles in flight + 1) within the
// workgroup's share of 160 KB.
template <int TBM, int TBN, int NW, int BKT>
struct Stages {
  static constexpr int kStageBytes = (TBM + TBN) * BKT * 2;
  static constexpr int kBudget = NW == 4 ? 80 * 1024 : 160 * 1024;
  static constexpr int S = kBudget / kStageBytes >= 4 ? 4 : kBudget / kStageBytes;
  static_assert(S >= 2, "two LDS stages at least");
};

// Byte offsets of K-tile stage st of the A and B operand tiles from sA and
// sB: consecutive stages.
template <int TBM, int TBN, int BKT>
struct LinearStages {
  __device__ static uint32_t a(int st) { return static_cast<uint32_t>(st) * (TBM * BKT * 2u); }
  __device__ static uint32_t b(int st) { return static_cast<uint32_t>(st) * (TBN * BKT * 2u); }
};

// Called at the start of every K tile, after the barrier (no-op).
struct NoHook {
  __device__ void operator()(int, int) const {}
};

__device__ __forceinline__ const bf16* at_byte(const void* base, uint32_t off) {
  return reinterpret_cast<const bf16*>(reinterpret_cast<const char*>(base) + off);
}

// This wave's LDS reads have completed and its loads but the latest `later`
// have landed; then the workgroup's barrier.  One asm statement, so that no LDS
// read moves between the wait and the barrier.
template <int later>
__device__ __forceinline__ void wait_tiles() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(later) : "memory");
}

// The K loop of one tile: acc[i][j] += the wave's 16 x 16 MFMA tiles of
// op(A) op(B) over [k_begin, k_end), the operands streamed through the S LDS
// stages (at sA + Map::a(stage), sB + Map::b(stage)) by the loaders (the
// wave tile at rows wm, columns wn).  The first `pre` K tiles may have been
// issued by the caller already (into their stages, by the same loaders, with
// nothing issued after them); hook(kt, nk) runs at the start of each K tile,
// after the barrier.  Returns with every load of the loop complete; the other
// waves may still read the last stage.
template <int TBM, int TBN, int NW, int BKT, bool A_KC, bool B_KC, int TM, int TN,
          class Map = LinearStages<TBM, TBN, BKT>, class Hook = NoHook, bool PIPE = BKT == 64>
__device__ __forceinline__ void k_loop(const Loader<TBM, A_KC, BKT, NW>& la,
                                       const Loader<TBN, B_KC, BKT, NW>& lb, bf16 (*sA)[TBM * BKT],
                                       bf16 (*sB)[TBN * BKT], f32x4 (&acc)[TM][TN], int wm, int wn,
                                       int k_begin, int k_end, int wave, int lane, int pre = 0,
                                       const Hook& hook = Hook{}) {
  constexpr int KSTEPS = BKT / 32;
  constexpr int S = Stages<TBM, TBN, NW, BKT>::S;
  Frags<TBM, A_KC, TM, BKT> fra;
  Frags<TBN, B_KC, TN, BKT> frb;
  fra.init(wm, lane);
  frb.init(wn, lane);

  constexpr int kLoadsA = Loader<TBM, A_KC, BKT, NW>::kPer;
  constexpr int kLoads = kLoadsA + Loader<TBN, B_KC, BKT, NW>::kPer;
  const int nk = (k_end - k_begin + BKT - 1) / BKT;
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const uint32_t a_lds = lds_offset(&sA[0][0]) + 1024u * wave_u * Loader<TBM, A_KC, BKT, NW>::kPer;
  const uint32_t b_lds = lds_offset(&sB[0][0]) + 1024u * wave_u * Loader<TBN, B_KC, BKT, NW>::kPer;
  auto issue = [&](int kt) {
    const int st = kt % S;
    la.issue_s(a_lds + Map::a(st), k_begin + kt * BKT, k_end);
    lb.issue_s(b_lds + Map::b(st), k_begin + kt * BKT, k_end);
  };
  if constexpr (PIPE) {
    // S K tiles in flight and the fragments of the next 32-deep step always
    // being read while the MFMAs of this one run, across the K tiles too: with
    // the second step's fragments in registers a K tile's stage is free, so the
    // one barrier per K tile stands between the two steps, the loads of tile
    // kt + S go out behind it, one after every few MFMAs, and a tile has a
    // whole iteration to arrive.  (Reading both steps after the barrier left
    // the MFMAs waiting for the first step's reads in every K tile and the fill
    // half an iteration: a K tile took 1.5 us against 0.85 us of MFMAs.  With
    // the loads all right behind the barrier, or the reads placed by scheduling
    // hints, 1-4% slower.)  Loads past the last K tile are issued as well, out
    // of range (zeros into a stage nobody reads), so that the waits are constant
    // and the loop has no branch; with a hook, whose loads own the other stages
    // by then, they are not.  Measured on 256 x 256 tiles, before -> after in one
    // run: 8192^3 NT 925 -> 822 us, 2048 x 50304 x 1536 NT 360 -> 320, 2048 x
    // 768 x 50304 NN in 8 K splits 180 -> 159, 50304 x 768 x 2048 TN 178 -> 164,
    // 8192 x 11264 x 2048 NT 318 -> 309, 8192 x 2048 x 5632 NT 146 -> 142; on
    // the 256 x 128 tiles (whose 8 fragment reads per 16 MFMAs bound them by
    // LDS) 0-9%; the fused gate/up backward below 8192 x 5632 x 2048 607 -> 575.
    constexpr bool kTail = std::is_same_v<Hook, NoHook>;
    static_assert(KSTEPS == 2 && (kTail || S == 2), "two steps; a hook's loads follow the last wait");
    if (nk <= 0) return;  // K = 0: no stage was filled, acc stays as it is
    auto read_a = [&](int st, int i, int k) { return fra.get(at_byte(&sA[0][0], Map::a(st)), i, k); };
    auto read_b = [&](int st, int j, int k) { return frb.get(at_byte(&sB[0][0], Map::b(st)), j, k); };
    bf16x8 fa0[TM], fb0[TN], fa1[TM], fb1[TN];
#pragma unroll
    for (int p = 0; p < S; ++p)
      if (p >= pre && p < nk) issue(p);
    if (nk >= S) wait_tiles<(S - 1) * kLoads>();
    else wait_tiles<0>();
    hook(0, nk);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb0[j] = read_b(0, j, 0);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa0[i] = read_a(0, i, 0);
    for (int kt = 0; kt + 1 < nk; ++kt) {
      const int st = kt % S;
#pragma unroll
      for (int j = 0; j < TN; ++j) fb1[j] = read_b(st, j, 32);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb0[j], fa0[i], acc[i][j]);
        fa1[i] = read_a(st, i, 32);
      }
      __builtin_amdgcn_sched_barrier(0);
      wait_tiles<(S - 2) * kLoads>();
      hook(kt + 1, nk);
      const int sn = (kt + 1) % S, k0 = k_begin + (kt + S) * BKT;
#pragma unroll
      for (int j = 0; j < TN; ++j) fb0[j] = read_b(sn, j, 0);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb1[j], fa1[i], acc[i][j]);
        fa0[i] = read_a(sn, i, 0);
        if (kTail || kt + S < nk) {
          // this row's share of the loads (stage (kt + S) % S)
#pragma unroll
          for (int l = 0; l < kLoads; ++l) {
            if (l * TM / kLoads == i) {
              if (l < kLoadsA) la.issue_one(l, a_lds + Map::a(st), k0, k_end);
              else lb.issue_one(l - kLoadsA, b_lds + Map::b(st), k0, k_end);
            }
          }
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int sl = (nk - 1) % S;
#pragma unroll
    for (int j = 0; j < TN; ++j) fb1[j] = read_b(sl, j, 32);
#pragma unroll
    for (int i = 0; i < TM; ++i) fa1[i] = read_a(sl, i, 32);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb0[j], fa0[i], acc[i][j]);
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb1[j], fa1[i], acc[i][j]);
    if constexpr (kTail) wait_vmcnt<0>();  // the loads past the end, before the stages are used again
  } else {
    // S - 1 K tiles in flight.  Each K tile kt: wait until this wave's loads of
    // tile kt have landed (those of later tiles may stay in flight), barrier
    // (everyone's have; everyone is done with the stage read last iteration),
    // all fragment reads, the loads of tile kt + S - 1 into that freed stage,
    // then the MFMAs.
#pragma unroll
    for (int p = 0; p < S - 1; ++p)
      if (p >= pre && p < nk) issue(p);
    for (int kt = 0; kt < nk; ++kt) {
      // tiles issued after tile kt: min(nk - 1, kt + S - 2) - kt
      const int after = min(nk - 1, kt + S - 2) - kt;
      if (after >= 2) wait_vmcnt<2 * kLoads>();
      else if (after == 1) wait_vmcnt<kLoads>();
      else wait_vmcnt<0>();
      lds_barrier();
      hook(kt, nk);
      const int st = kt % S;
      const bf16* ta = at_byte(&sA[0][0], Map::a(st));
      const bf16* tb = at_byte(&sB[0][0], Map::b(st));
      bf16x8 fa[KSTEPS][TM], fb[KSTEPS][TN];
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ++ks) {
#pragma unroll
        for (int j = 0; j < TN; ++j) fb[ks][j] = frb.get(tb, j, 32 * ks);
#pragma unroll
        for (int i = 0; i < TM; ++i) fa[ks][i] = fra.get(ta, i, 32 * ks);
      }
      if constexpr (KSTEPS == 2) {
        // The wave issues in order and a full LDS queue stalls it, MFMAs
        // included: let the step-0 MFMAs start after the step-0 reads and put one
        // step-1 read between every two of them (scheduling hints only).
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb[0][j], fa[0][i], acc[i][j]);
        constexpr int R = TM + TN;
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);  // step-0 LDS reads
#pragma unroll
        for (int r = 0; r < R; ++r) {
          __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);  // two MFMAs
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one step-1 LDS read
        }
        if constexpr (TM * TN > 2 * R) __builtin_amdgcn_sched_group_barrier(0x008, TM * TN - 2 * R, 0);
        if (kt + S - 1 < nk) issue(kt + S - 1);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb[1][j], fa[1][i], acc[i][j]);
      } else {
        if (kt + S - 1 < nk) issue(kt + S - 1);
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) acc[i][j] = mfma16(fb[0][j], fa[0][i], acc[i][j]);
      }
    }
  }
}

}  // namespace
}  // namespace nmb
