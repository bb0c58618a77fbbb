// What the tiled kernels of scored attention (bf16) share: tiles of 64 rows in
// LDS, scores from products, spans of a tile of rows.
#pragma once

#include "attention_scored.h"
#include "lds_dma.h"

namespace nmb {
namespace {

__device__ __forceinline__ f32x4 mfma16(const bf16x8& a, const bf16x8& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ f32x4 zero4() { return f32x4{0.f, 0.f, 0.f, 0.f}; }

__device__ __forceinline__ bf16x8 zero8() {
  bf16x8 z;
#pragma unroll
  for (int i = 0; i < 8; ++i) z[i] = static_cast<bf16>(0.f);
  return z;
}

// columns col .. col + 7 of a row of D (a multiple of 8); zeros past D or where !ok
__device__ __forceinline__ bf16x8 row_frag(const bf16* row, int col, int D, bool ok) {
  return ok && col < D ? *reinterpret_cast<const bf16x8*>(row + col) : zero8();
}

// exp2 as the bare v_exp_f32 (results below 2^-126 are 0: no weight beside the others of a row)
__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// 64 rows x D columns (64 or 128; rows of fewer columns are padded with zeros)
// of bf16 in LDS, row-major with the 16-byte chunk c of row r at c ^ swz(r):
// rows and columns of it are then read as MFMA operands without bank conflicts.
template <int D>
struct RowTile {
  static constexpr int kElems = 64 * D;
  __device__ static int swz(int r) { return D == 64 ? (r & 7) : 2 * (r & 7); }
  __device__ static int at(int r, int col) { return r * D + 8 * ((col >> 3) ^ swz(r)) + (col & 7); }
  // row r, columns col .. col + 7
  __device__ static bf16x8 row8(const bf16* t, int r, int col) {
    return *reinterpret_cast<const bf16x8*>(t + at(r, col));
  }
  // column c0 + l16, rows r0 + 4g .. +3 and r0 + 16 + 4g .. +3: the order in
  // which two 16 x 16 score tiles hold their rows
  __device__ static bf16x8 col8(const bf16* t, int r0, int c0, int l16, int g) {
    const int r = r0 + 4 * g + (l16 >> 2), cc = c0 + 4 * (l16 & 3);
    return ld_tr(t + at(r, cc), t + at(r + 16, cc));
  }
};

// One wave's share (of NW) of loading a tile of ROWS rows straight from memory into LDS.
template <int D, int NW, int ROWS = 64>
struct RowLoader {
  static constexpr int P = ROWS * D * 2 / 1024 / NW;  // 1 KB loads per wave and tile
  static_assert(P >= 1 && ROWS * D * 2 % (1024 * NW) == 0, "a tile splits evenly over the waves");
  uint32_t off[P];  // bytes from the tile's first row; kOOB past the head dim
  int row[P];

  __device__ void init(int64_t stride, int head_dim, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int e = (1024 * (wave * P + j) + 16 * lane) / 2;  // element of the tile
      const int r = e / D, c = ((e % D) / 8) ^ RowTile<D>::swz(r);
      row[j] = r;
      off[j] = 8 * c < head_dim ? static_cast<uint32_t>(r * stride * 2) + 16u * static_cast<uint32_t>(c) : kOOB;
    }
  }
  // the ROWS rows from `first` to LDS byte m0 (of this wave's share) on: the first n
  // (<= 0: none) are read, the others become zeros.  The address is formed in 64 bits,
  // so a tensor may be of any size.
  __device__ __forceinline__ void issue(const bf16* first, uint32_t m0, int n) const {
    const i32x4 rs = make_rsrc(first, 0x7fffffffu);
    if (n >= ROWS) {
#pragma unroll
      for (int j = 0; j < P; ++j) load_lds16s(rs, m0 + 1024u * j, off[j], 0u);
    } else {
#pragma unroll
      for (int j = 0; j < P; ++j) load_lds16s(rs, m0 + 1024u * j, row[j] < n ? off[j] : kOOB, 0u);
    }
  }
};

// LDS byte address of this wave's share of stage 0 of a ring of tiles
template <class Load>
__device__ __forceinline__ uint32_t share_of(const bf16* stages, int wave) {
  return __builtin_amdgcn_readfirstlane(lds_offset(stages)) + 1024u * static_cast<uint32_t>(wave * Load::P);
}

// The tiles of 64 consecutive rows of two tensors (K and V) through a ring of STAGES places
// in LDS, the last tile first where DOWN; past the end zeros are loaded, so that every wait
// counts alike.
template <int D, int NW, int STAGES, bool DOWN>
struct PairStream {
  using Load = RowLoader<D, NW>;
  static constexpr uint32_t kStage = RowTile<D>::kElems * 2;  // bytes
  Load la, lb;
  const bf16 *pa, *pb;    // first row of the next tile
  int64_t step_a, step_b; // 64 rows
  uint32_t a0, b0, at;    // this wave's share of stage 0; byte offset of the next stage
  int rows, left;         // of the next tile (not DOWN: from there on); > 0 while there is one

  __device__ __forceinline__ void init(const bf16* a, int64_t sa, const bf16* b, int64_t sb, int n, int head_dim,
                                       const bf16* lds_a, const bf16* lds_b, int wave, int lane) {
    la.init(sa, head_dim, wave, lane);
    lb.init(sb, head_dim, wave, lane);
    step_a = 64 * sa;
    step_b = 64 * sb;
    pa = a;
    pb = b;
    if constexpr (DOWN) {
      left = (n + 63) / 64;
      rows = n - 64 * (left - 1);
      pa += (left - 1) * step_a;
      pb += (left - 1) * step_b;
    } else {
      left = rows = n;
    }
    a0 = share_of<Load>(lds_a, wave);
    b0 = share_of<Load>(lds_b, wave);
    at = 0;
  }
  __device__ __forceinline__ void issue() {
    const i32x4 ra = make_rsrc(pa, 0x7fffffffu), rb = make_rsrc(pb, 0x7fffffffu);
    const int n = left > 0 ? rows : 0;
    if (n >= 64) {
#pragma unroll
      for (int j = 0; j < Load::P; ++j) load_lds16s(ra, a0 + at + 1024u * j, la.off[j], 0u);
#pragma unroll
      for (int j = 0; j < Load::P; ++j) load_lds16s(rb, b0 + at + 1024u * j, lb.off[j], 0u);
    } else {
#pragma unroll
      for (int j = 0; j < Load::P; ++j) load_lds16s(ra, a0 + at + 1024u * j, la.row[j] < n ? la.off[j] : kOOB, 0u);
#pragma unroll
      for (int j = 0; j < Load::P; ++j) load_lds16s(rb, b0 + at + 1024u * j, lb.row[j] < n ? lb.off[j] : kOOB, 0u);
    }
    if constexpr (DOWN) {
      pa -= step_a;
      pb -= step_b;
      rows = 64;
      --left;
    } else {
      pa += step_a;
      pb += step_b;
      left = rows -= 64;
    }
    at = at + kStage == STAGES * kStage ? 0 : at + kStage;
  }
};

// the next of STAGES places
template <int STAGES>
__device__ __forceinline__ int next_stage(int st) { return st + 1 == STAGES ? 0 : st + 1; }

// This wave's loads but the latest N have landed and its LDS reads are done;
// then the workgroup's barrier.  One statement, so that nothing moves between.
template <int N>
__device__ __forceinline__ void tile_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// How a score is formed, known when a kernel is compiled: with a cap, with a
// distance bias, and whether scores need no running maximum.  They need none where a
// cap bounds them by kFixedMax in base 2: weights 2^(x - m) with m the largest bias of a
// row's keys (fixed_max) are at most 2^80 and their sums over 2^30 keys within fp32; the
// key of that bias has a weight of 2^-80 at least; and relative precision does not
// depend on the exponent.
template <bool CAP_, bool BIAS_, bool FIXED_>
struct Mode {
  static constexpr bool CAP = CAP_, BIAS = BIAS_, FIXED = FIXED_;
};
constexpr float kFixedMax = 80.f;

// The largest bias of the keys `seen` from position pos: 0, the nearest key's (see
// bias_pos), or with a negative slope that of the furthest.
__device__ __forceinline__ float fixed_max(float slope2, float pos, const Span& seen) {
  const float far = fmaxf(fabsf(pos - static_cast<float>(seen.lo)), fabsf(pos - static_cast<float>(seen.hi - 1)));
  return slope2 < 0.f && seen.hi > seen.lo ? -slope2 * far : 0.f;
}

// The capped score in base 2, A tanh(y) = A - 2 A / (1 + e^(2 y)) with A =
// cap_out and e^(2 y) = 2^(cap_in s): two of the hardware's transcendentals
// (8 cycles a wave each here) and three plain operations.  It is off by a few
// 2^-24 A, absolutely; that is what the exponential needs.  t = 1 / (1 +
// e^(2 y)) gives the derivative 1 - tanh^2 = 4 t (1 - t) too.
__device__ __forceinline__ float cap_t(const ScoredShape& p, float s) {
  return __builtin_amdgcn_rcpf(1.f + fast_exp2(s * p.cap_in));
}

// Where every distance of a tile is >= 0 its bias is linear in the row: a part that is the
// same in every tile, slope2 (16 i + e) of row 16 i + e, and one that is the same for all
// rows.  Without a cap the products' sums start from the first, divided by the scale c, and
// one operation a score is left (4 x 32 heads of 2048: forward 112.7 -> 111.2 us, backward
// 322 -> 318).
template <class M>
constexpr bool kBiasInProduct = M::BIAS && !M::CAP;
template <class M, int N>
__device__ __forceinline__ void bias_start(const ScoredShape& p, float slope2, f32x4 (&start)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) start[i][e] = kBiasInProduct<M> ? slope2 / p.c * (16.f * i + e) : 0.f;
}

// Scores of N consecutive groups of four rows of the other side, 16 apart, from raw
// products (whose sums started from bias_start's values): x[4 i + e] = off + score of
// s[i][e], at distance dist - (16 i + e), t the cap's t where there is one; behind: no
// distance is negative.
template <class M, int N>
__device__ __forceinline__ void tile_scores(const ScoredShape& p, const f32x4 (&s)[N], float off, float slope2,
                                            float dist, bool behind, float (&x)[4 * N], float (&t)[4 * N]) {
  if constexpr (M::CAP) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) t[4 * i + e] = cap_t(p, s[i][e]);
  }
  auto last = [&](int n, float c) {
    return M::CAP ? fmaf(-2.f * p.cap_out, t[n], c) : fmaf(s[n >> 2][n & 3], p.c, c);
  };
  if constexpr (M::BIAS) {
    if (behind) {
      const float base = fmaf(-slope2, dist, off);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if constexpr (kBiasInProduct<M>) {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[4 * i + e] = last(4 * i + e, base);
          continue;
        }
        const float row = fmaf(slope2, 16.f * i, base);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[4 * i + e] = last(4 * i + e, e == 0 ? row : fmaf(slope2, e, row));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          x[4 * i + e] = fmaf(-slope2, fabsf(dist - static_cast<float>(16 * i + e)),
                              last(4 * i + e, kBiasInProduct<M> ? fmaf(-slope2, 16.f * i + e, off) : off));
    }
  } else {
#pragma unroll
    for (int n = 0; n < 4 * N; ++n) x[n] = last(n, off);
  }
}

// x of the rows 16 (n / 4) + n % 4 below lo (from hi on) becomes v.  Called under a
// condition that is the same for the wave and mostly false: the empty statement keeps the
// compiler from running the selects always.
template <int N>
__device__ __forceinline__ void hide_below(float (&x)[N], int lo, float v) {
  asm volatile("");
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = 16 * (n >> 2) + (n & 3) < lo ? v : x[n];
}
template <int N>
__device__ __forceinline__ void hide_from(float (&x)[N], int hi, float v) {
  asm volatile("");
#pragma unroll
  for (int n = 0; n < N; ++n) x[n] = 16 * (n >> 2) + (n & 3) >= hi ? v : x[n];
}

struct ColSpan {   // of 16 consecutive rows (queries or keys)
  Span mine;       // this lane's row
  int lo_min, lo_max, hi_min, hi_max;
};

// spans are non-decreasing, so the extremes are those of the first and last row
__device__ __forceinline__ ColSpan col_span(const Span& s) {
  ColSpan c;
  c.mine = s;
  c.lo_min = __builtin_amdgcn_readlane(s.lo, 0);
  c.hi_min = __builtin_amdgcn_readlane(s.hi, 0);
  c.lo_max = __builtin_amdgcn_readlane(s.lo, 15);
  c.hi_max = __builtin_amdgcn_readlane(s.hi, 15);
  return c;
}

// Workgroup of a 1-D grid -> a tile of a head, tile by tile over all heads: under a causal
// mask tiles differ in work, and the last ones to start should be the lightest, whichever
// head is theirs (in head order 4 x 32 heads x 2048 tokens took 171 us forward where its
// share of a larger batch takes 152).  Workgroups go round-robin over the 8 XCDs, each with
// an L2 of its own: where the heads divide by 8, each XCD takes an eighth of them.
struct HeadTile {
  int head, tile;  // tile counts from 0
};
__device__ __forceinline__ HeadTile head_tile(int heads) {
  const int l = static_cast<int>(blockIdx.x);
  if (heads % 8 != 0) return HeadTile{l % heads, l / heads};
  const int per = heads / 8, j = l / 8;
  return HeadTile{l % 8 * per + j % per, j / per};
}

// the same, consecutive items on one XCD
__device__ __forceinline__ int xcd_item(int items, int per_xcd) {
  const int l = static_cast<int>(blockIdx.x);
  const int w = (l % 8) * per_xcd + l / 8;
  return w < items ? w : -1;
}

}  // namespace
}  // namespace nmb
