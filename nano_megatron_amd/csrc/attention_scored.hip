// Attention with capped scores, a distance bias and interval masks (documents,
// prefix, window), forward and backward, for gfx950.  attention_scored.h holds
// the mathematics.
#include <algorithm>
#include <type_traits>

#include "attention_scored_tiles.h"

namespace nmb {
namespace {

// ------------------------------------------------------------ documents
// {start, end} of the run of equal ids that each token lies in ({start, ~end}
// where the id is negative).  A workgroup per row: the start of a token's run
// is the largest start of a run at or before it, the end the smallest after
// it, each by a scan over the row, forwards then backwards, 1,024 threads of 8
// tokens at a time.  Bound by the latency of its loads and scans: 7 us for 16 x 512
// tokens, 11 for 8192 in a row, once for all layers that read them.
constexpr int kRunThreads = 1024, kRunTokens = 8;

// inclusive scan of v over the workgroup, larger (MAX) or smaller value kept
template <bool MAX>
__device__ __forceinline__ int block_scan(int v, int* sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int u = __shfl_up(v, d, 64);
    if (lane >= d) v = MAX ? max(v, u) : min(v, u);
  }
  __syncthreads();  // sh may still be read from the last scan
  if (lane == 63) sh[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v = MAX ? max(v, sh[w]) : min(v, sh[w]);
  return v;
}

__global__ __launch_bounds__(kRunThreads) void document_runs_kernel(const int32_t* __restrict__ docs, int64_t stride,
                                                                    int n, int2* __restrict__ runs) {
  __shared__ int sh[kRunThreads / 64];
  __shared__ int carry;
  const int32_t* d = docs + blockIdx.x * stride;
  int2* out = runs + static_cast<int64_t>(blockIdx.x) * n;
  constexpr int kChunk = kRunThreads * kRunTokens;
  const int chunks = (n + kChunk - 1) / kChunk;
  const int tid = static_cast<int>(threadIdx.x);
  int before = 0;  // start of the run that the last chunk ended in
  for (int c = 0; c < chunks; ++c) {
    const int t0 = c * kChunk + tid * kRunTokens;
    int start[kRunTokens], last = -1;
#pragma unroll
    for (int e = 0; e < kRunTokens; ++e) {
      const int t = t0 + e;
      if (t < n && (t == 0 || d[t] != d[t - 1])) last = t;
      start[e] = last;
    }
    const int incl = block_scan<true>(last, sh);
    int prev = __shfl_up(incl, 1, 64);
    if ((tid & 63) == 0) prev = tid == 0 ? -1 : -2;
    __syncthreads();
    if (prev == -2) {  // the first lane of a later wave: the scan up to the wave before
      prev = -1;
      for (int w = 0; w < tid >> 6; ++w) prev = max(prev, sh[w]);
    }
    prev = max(prev, before);
#pragma unroll
    for (int e = 0; e < kRunTokens; ++e)
      if (t0 + e < n) out[t0 + e].x = max(start[e], prev);
    if (tid == kRunThreads - 1) carry = max(incl, before);
    __syncthreads();
    before = carry;
  }
  int after = n;  // end of the run that the chunk behind starts in the middle of
  for (int c = chunks - 1; c >= 0; --c) {
    // thread 0 takes the last tokens of the chunk
    const int t0 = c * kChunk + (kRunThreads - 1 - tid) * kRunTokens;
    int end[kRunTokens], next = n;
    int32_t id[kRunTokens + 1];
#pragma unroll
    for (int e = 0; e <= kRunTokens; ++e) id[e] = t0 + e < n ? d[t0 + e] : 0;
#pragma unroll
    for (int e = kRunTokens - 1; e >= 0; --e) {
      const int t = t0 + e;
      if (t + 1 < n && id[e] != id[e + 1]) next = t + 1;
      end[e] = next;
    }
    const int incl = block_scan<false>(next, sh);
    int prev = __shfl_up(incl, 1, 64);
    if ((tid & 63) == 0) prev = tid == 0 ? n : -2;
    __syncthreads();
    if (prev == -2) {
      prev = n;
      for (int w = 0; w < tid >> 6; ++w) prev = min(prev, sh[w]);
    }
    prev = min(prev, after);
#pragma unroll
    for (int e = 0; e < kRunTokens; ++e) {
      const int t = t0 + e, y = min(end[e], prev);
      if (t < n) out[t].y = id[e] < 0 ? ~y : y;
    }
    if (tid == kRunThreads - 1) carry = min(incl, after);
    __syncthreads();
    after = carry;
  }
}

// ------------------------------------------------------------ forward
// bf16.  A workgroup owns 16 NW queries of one head, 16 a wave.  The key tiles that
// any of them sees stream through LDS.  S^T = K Q^T puts all scores of a query in the
// lanes l, l + 16, l + 32, l + 48, where the statistics are plain registers, and exp2
// of them is, rounded to bf16, the operand of O^T += V^T P as it stands (the 32-deep
// index of that product runs over the keys in the order the scores hold them).
// Sums, maxima and outputs stay fp32; the probabilities are operands of the bf16 matrix
// instruction.  LOW, for training: as two terms, p and what its rounding cut off, because
// the backward's dP - delta cancels where one key has nearly all the weight and takes delta
// from this output (dq and dk off by 2.35e-3 of their norm; with one term 2.55e-3, and the
// rounding of dS and of the result alone give 2.35e-3).  Otherwise one term, rounded by half
// a step (2^-8), divided by the sum of the rounded ones, which a row of ones in the same
// product gives: a key that outweighs the others then has weight 1 exactly.  Two terms
// and one, us: 4 x 32 heads of 2048 with a distance bias 136 and 112, 16 heads of 128 x 8192
// in documents 194 and 156, 16 x 16 heads x 512 28.9 and 24.8.
// D: columns of the tiles in LDS, DC: those that enter the products.  Head dims of 65 to 96
// lie in tiles of 128 and leave out the last quarter of their zeros (2 x 16 heads of 80 x
// 2048: forward 59 -> 52.6 us, backward 212 -> 179).
// Four waves a SIMD at D <= 64; at D 128 the registers for that are too few to read
// operands ahead of their products: two take 155 us and four 166 (8192 queries of 16
// heads in documents).
template <int D, int NW, class M, bool LOW, int DC = D>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 2) void scored_fwd_kernel(
    ScoredShape p, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v,
    bf16* __restrict__ o, bf16* __restrict__ o_low, float* __restrict__ lse2, int n_qt) {
  constexpr int BQ = 16 * NW, KS = DC / 32, DT = DC / 16;
  constexpr int kStages = 2;
  // The last keys first where a maximum is followed: a causal query's nearest lie there,
  // with a distance bias its largest scores, and the maximum moves little after them (4 x 32
  // heads of 2048 queries: 113 us, in the other order 121; without one the order of memory,
  // 16 x 16 heads x 512 in documents 24.7 us, 26.0 in the other).
  constexpr bool kDown = !M::FIXED;
  using Tile = RowTile<D>;
  using Load = RowLoader<D, NW>;
  __shared__ __attribute__((aligned(1024))) bf16 sK[kStages][Tile::kElems];
  __shared__ __attribute__((aligned(1024))) bf16 sV[kStages][Tile::kElems];
  const HeadTile ht = head_tile(p.B * p.Hq);
  const int q0 = (n_qt - 1 - ht.tile) * BQ;  // the most keys first
  const int b = ht.head / p.Hq, h = ht.head % p.Hq, hk = h / (p.Hq / p.Hkv);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int l16 = lane & 15, g = lane >> 4;
  const RowView r = row_view(p, b);
  const float slope2 = M::BIAS ? slope2_of(p, h) : 0.f;

  const int i = min(q0 + 16 * wave + l16, p.Sq - 1);
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    qf[ks] = row_frag(q + b * p.q_sb + i * p.q_ss + h * p.q_sh, ks * 32 + g * 8, p.D, true);
  const ColSpan span = col_span(seen_keys(p, r, i));
  const float pos = M::BIAS ? bias_pos(p, r, i) : 0.f;
  const float first_pos = __shfl(pos, 0, 16);
  f32x4 start[4];
  bias_start<M, 4>(p, slope2, start);
  float m = M::FIXED && M::BIAS ? fixed_max(slope2, pos, span.mine) : 0.f, l = 0.f;  // weights are 2^(x - m)
  bool empty = true;       // the row has seen no score yet
  f32x4 acc[DT], rounded = zero4();  // O^T, and the sum of the rounded probabilities in every lane
  bf16x8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = static_cast<bf16>(1.f);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero4();
  const int k_lo = __builtin_amdgcn_readfirstlane(seen_keys(p, r, q0).lo);
  const int k_hi = __builtin_amdgcn_readfirstlane(seen_keys(p, r, min(q0 + BQ, p.Sq) - 1).hi);
  // everything above has landed before the first tile is on its way: the
  // compiler counts only its own loads and would wait for all
  wait_vmcnt<0>();
  PairStream<D, NW, kStages, kDown> in;
  in.init(k + b * p.k_sb + hk * p.k_sh + k_lo * p.k_ss, p.k_ss, v + b * p.v_sb + hk * p.v_sh + k_lo * p.v_ss, p.v_ss,
          k_hi - k_lo, p.D, sK[0], sV[0], wave, lane);
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) in.issue();

  const int tiles = (k_hi - k_lo + 63) / 64;
  int st = 0;
  for (int n = 0; n < tiles; ++n, st = next_stage<kStages>(st)) {
    const int k0 = k_lo + 64 * (kDown ? tiles - 1 - n : n);
    // this wave's loads of this tile have landed, after the barrier everyone's; and
    // nobody reads the stage of the tile before any more
    tile_barrier<(kStages - 2) * 2 * Load::P>();
    in.issue();
    if (k0 >= span.hi_max || k0 + 64 <= span.lo_min || q0 + 16 * wave >= p.Sq) continue;
    const bf16* tk = sK[st];
    const bf16* tv = sV[st];
    f32x4 s[4];
#pragma unroll
    for (int mk = 0; mk < 4; ++mk) s[mk] = start[mk];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int mk = 0; mk < 4; ++mk) s[mk] = mfma16(Tile::row8(tk, mk * 16 + l16, ks * 32 + g * 8), qf[ks], s[mk]);
    // lane: key k0 + 16 mk + 4 g + e of its query
    float x[16], t[16];
    tile_scores<M>(p, s, (M::CAP ? p.cap_out : 0.f) - m, slope2, pos - static_cast<float>(k0 + 4 * g),
                   __builtin_amdgcn_readfirstlane(first_pos >= static_cast<float>(k0 + 63)), x, t);
    if (k0 < span.lo_max) hide_below<16>(x, span.mine.lo - k0 - 4 * g, -__builtin_inff());
    if (k0 + 64 > span.hi_min) hide_from<16>(x, span.mine.hi - k0 - 4 * g, -__builtin_inff());
    if constexpr (!M::FIXED) {
      // m follows the row's maximum only when a tile's exceeds it by 8 (until then the
      // weights are at most 2^8, which fp32 sums can hold), or, before the row has any
      // weight, when it lies below it by 8
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, x[e]);
      if (__any((top > 8.f) | empty)) {
        top = xor32_max(xor16_max(top));
        const bool move = (top > 8.f) | (empty & (top < -8.f) & (top > -__builtin_inff()));
        const float shift = move ? top : 0.f;
        const float alpha = move && !empty ? fast_exp2(-top) : 1.f;
        empty = empty & !(top > -__builtin_inff());
        m += shift;
        l *= alpha;
        rounded *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] -= shift;
      }
    }
    bf16x8 pf[2], pl[2];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float weight = fast_exp2(x[e]);
      l += weight;
      pf[e >> 3][e & 7] = static_cast<bf16>(weight);
      if constexpr (LOW) pl[e >> 3][e & 7] = static_cast<bf16>(weight - static_cast<float>(pf[e >> 3][e & 7]));
    }
    if constexpr (!LOW) {
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) rounded = mfma16(ones, pf[s2], rounded);
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bf16x8 a0 = Tile::col8(tv, 0, dt * 16, l16, g), a1 = Tile::col8(tv, 32, dt * 16, l16, g);
      acc[dt] = mfma16(a0, pf[0], acc[dt]);
      acc[dt] = mfma16(a1, pf[1], acc[dt]);
      if constexpr (LOW) {
        acc[dt] = mfma16(a0, pl[0], acc[dt]);
        acc[dt] = mfma16(a1, pl[1], acc[dt]);
      }
    }
  }
  wait_vmcnt<0>();  // no load may still write this workgroup's LDS when it ends
  const bool mine = q0 + 16 * wave + l16 < p.Sq;
  const float sum = xor32_sum(xor16_sum(l));
  // a visible score that is not a number (hidden ones are replaced) has lost its row
  const bool lost = sum != sum && fabsf(start[3][3]) < __builtin_inff();
  const float all = LOW ? sum : rounded[0], inv = lost ? sum : all > 0.f ? 1.f / all : 0.f;
  bool fine = sum < __builtin_inff();
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) fine = fine && fabsf(acc[dt][e]) < __builtin_inff();
  fine = fine || lost;
  const uint32_t bad = named_rows(__ballot(!fine && mine));
  if (mine && (bad >> l16 & 1) == 0) {
    const int64_t at = b * p.o_sb + i * p.o_ss + h * p.o_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float full = acc[dt][e] * inv;
        x[e] = static_cast<bf16>(full);
        y[e] = static_cast<bf16>(full - static_cast<float>(x[e]));
      }
      if (dt * 16 + g * 4 < p.D) {
        *reinterpret_cast<bf16x4*>(o + at + dt * 16 + g * 4) = x;
        if (o_low != nullptr) *reinterpret_cast<bf16x4*>(o_low + at + dt * 16 + g * 4) = y;
      }
    }
    if (g == 0)
      lse2[(static_cast<int64_t>(b) * p.Hq + h) * p.Sq + i] =
          lost ? sum : sum > 0.f ? m + log2f(sum) : -__builtin_inff();
  }
  for (uint32_t left = bad; left != 0; left &= left - 1)  // not finite: on the visible keys alone
    scored_row_fwd(p, q, k, v, o, o_low, lse2, b, h, q0 + 16 * wave + __ffs(left) - 1, lane);
}

// ------------------------------------------------------------ few queries
// For a few queries against many keys the keys and values are read once and that is
// what bounds it (one token each of 32 sequences, 32 / 8 heads of 128, 8,192 keys less
// a quarter: 157 us for 806 MB, 5.1 TB/s).  The rows of a tile are 16 (query, head) pairs of one KV head's
// group, so that a group reads its keys once; a workgroup takes a share of their keys
// and each of its waves every NW-th tile of 32 of them, with tiles, maximum, sum and
// output of its own (no barrier in the loop: 8 or 16 KB a wave in flight while as much
// is computed), merged through LDS at the end.  With `splits` > 1 workgroups per row
// tile the merged {O, m, l} go to `partial` and scored_few_merge_kernel joins them.
// The probabilities enter the product as two bf16 terms (the matrix unit is idle here).
constexpr int kFewKeys = 32;
constexpr int kFewSplits = 64;  // at most

// where a workgroup's rows lie: row n of a row tile is query n / group, head n % group
struct FewRows {
  int b, hk, row0, rows, group;  // rows: of this KV head, over all row tiles
  __device__ __forceinline__ int query(int n) const { return min(row0 + n, rows - 1) / group; }
  __device__ __forceinline__ int head(int n) const { return hk * group + min(row0 + n, rows - 1) % group; }
};
__device__ __forceinline__ FewRows few_rows(const ScoredShape& p, int tile, int n_rt) {
  FewRows f;
  f.group = p.Hq / p.Hkv;
  f.rows = f.group * p.Sq;
  f.row0 = tile % n_rt * 16;
  f.hk = tile / n_rt % p.Hkv;
  f.b = tile / n_rt / p.Hkv;
  return f;
}

// Outputs of 16 rows from {O, m, l} of W parts: get(w, n, d) four elements of O of row
// n, stat(w, n, &m, &l) its statistics (m in base 2).  All threads of the workgroup.
template <int D, class M, class Get, class Stat>
__device__ __forceinline__ void few_finish(const ScoredShape& p, const FewRows& f, const bf16* q, const bf16* k,
                                           const bf16* v, bf16* o, bf16* o_low, float* lse2, int parts, uint32_t* bad,
                                           const Get& get, const Stat& stat) {
  if (threadIdx.x == 0) *bad = 0;
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * (D / 4); x += blockDim.x) {
    const int n = x / (D / 4), d = x % (D / 4) * 4;
    if (f.row0 + n >= f.rows || d >= p.D) continue;  // (columns past D need not have been summed)
    float top = -__builtin_inff();
    for (int w = 0; w < parts; ++w) {
      float m, l;
      stat(w, n, m, l);
      top = fmaxf(top, m);
    }
    float sum = 0.f;
    f32x4 acc = zero4();
#pragma unroll 4
    for (int w = 0; w < parts; ++w) {
      float m, l;
      stat(w, n, m, l);
      const float a = m == -__builtin_inff() ? 0.f : fast_exp2(m - top);
      sum = fmaf(a, l, sum);
      const f32x4 part = get(w, n, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(a, part[e], acc[e]);
    }
    const bool lost = sum != sum;  // as in the kernel above
    const float inv = lost ? sum : sum > 0.f ? 1.f / sum : 0.f;
    bf16x4 hi, lo;
    bool fine = sum < __builtin_inff();
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      fine = fine && fabsf(acc[e]) < __builtin_inff();
      hi[e] = static_cast<bf16>(acc[e] * inv);
      lo[e] = static_cast<bf16>(acc[e] * inv - static_cast<float>(hi[e]));
    }
    if (!fine && !lost) atomicOr(bad, 1u << n);
    const int i = f.query(n), h = f.head(n);
    const int64_t at = f.b * p.o_sb + i * p.o_ss + h * p.o_sh + d;
    *reinterpret_cast<bf16x4*>(o + at) = hi;
    if (o_low != nullptr) *reinterpret_cast<bf16x4*>(o_low + at) = lo;
    if (d == 0)
      lse2[(static_cast<int64_t>(f.b) * p.Hq + h) * p.Sq + i] =
          lost ? sum : sum > 0.f ? top + log2f(sum) : -__builtin_inff();
  }
  __syncthreads();  // the stores above are done before a row is written again
  const int waves = static_cast<int>(blockDim.x) / 64, wave = static_cast<int>(threadIdx.x) / 64;
  for (uint32_t left = *bad; left != 0; left &= left - 1) {
    const int n = __ffs(left) - 1;
    if (n % waves == wave)
      scored_row_fwd(p, q, k, v, o, o_low, lse2, f.b, f.head(n), f.query(n), static_cast<int>(threadIdx.x & 63));
  }
}

template <int D, int NW, class M, int DC = D>
__global__ __launch_bounds__(64 * NW, 1) void scored_few_kernel(
    ScoredShape p, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v,
    bf16* __restrict__ o, bf16* __restrict__ o_low, float* __restrict__ lse2, float* __restrict__ partial, int n_rt,
    int splits, int items, int per_xcd) {
  constexpr int KS = DC / 32, DT = DC / 16, BK = kFewKeys, kTile = BK * D;
  using Tile = RowTile<D>;
  using Load = RowLoader<D, 1, BK>;
  constexpr int kLdO = D + 4;
  __shared__ __attribute__((aligned(1024))) bf16 lds[NW][2][2][kTile];  // [wave][stage][K, V]
  __shared__ float sM[NW][16], sL[NW][16];
  __shared__ uint32_t bad;
  static_assert(sizeof(float) * NW * 16 * kLdO <= sizeof(lds), "the outputs take the tiles' place");
  const int item = xcd_item(items, per_xcd);
  if (item < 0) return;
  const int split = item % splits;
  const FewRows f = few_rows(p, item / splits, n_rt);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int l16 = lane & 15, g = lane >> 4;
  const RowView r = row_view(p, f.b);
  const int i = f.query(l16), h = f.head(l16);
  const float slope2 = M::BIAS ? slope2_of(p, h) : 0.f;
  const float pos = M::BIAS ? bias_pos(p, r, i) : 0.f;
  const ColSpan span = col_span(seen_keys(p, r, i));
  bf16x8 qf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
    qf[ks] = row_frag(q + f.b * p.q_sb + i * p.q_ss + h * p.q_sh, ks * 32 + g * 8, p.D, true);
  float m = !M::FIXED ? -__builtin_inff() : M::BIAS ? fixed_max(slope2, pos, span.mine) : 0.f, l = 0.f;
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero4();
  const int tiles = (span.hi_max - span.lo_min + BK - 1) / BK;
  const int t_end = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / splits);
  const int t_begin = static_cast<int>(static_cast<int64_t>(tiles) * split / splits) + wave;
  const bf16* kb = k + f.b * p.k_sb + f.hk * p.k_sh;
  const bf16* vb = v + f.b * p.v_sb + f.hk * p.v_sh;
  wait_vmcnt<0>();
  Load lk, lv;
  lk.init(p.k_ss, p.D, 0, lane);
  lv.init(p.v_ss, p.D, 0, lane);
  auto issue = [&](int t, int st) {
    const int k0 = span.lo_min + BK * t, n = t < t_end ? span.hi_max - k0 : 0;
    lk.issue(kb + k0 * p.k_ss, share_of<Load>(lds[wave][st][0], 0), n);
    lv.issue(vb + k0 * p.v_ss, share_of<Load>(lds[wave][st][1], 0), n);
  };
  issue(t_begin, 0);
  issue(t_begin + NW, 1);
  int st = 0;
  for (int t = t_begin; t < t_end; t += NW, st ^= 1) {
    wait_vmcnt<2 * Load::P>();
    asm volatile("" ::: "memory");
    const bf16* tk = lds[wave][st][0];
    const bf16* tv = lds[wave][st][1];
    const int k0 = span.lo_min + BK * t;
    f32x4 s[2] = {zero4(), zero4()};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int mk = 0; mk < 2; ++mk) s[mk] = mfma16(Tile::row8(tk, mk * 16 + l16, ks * 32 + g * 8), qf[ks], s[mk]);
    float x[8];
    const float dist = pos - static_cast<float>(k0 + 4 * g);
    const int lo = span.mine.lo - k0 - 4 * g, hi = span.mine.hi - k0 - 4 * g;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = 16 * (e >> 2) + (e & 3);
      const float raw = s[e >> 2][e & 3];
      x[e] = M::CAP ? fmaf(-2.f * p.cap_out, cap_t(p, raw), p.cap_out) : raw * p.c;
      if constexpr (M::BIAS) x[e] = fmaf(-slope2, fabsf(dist - static_cast<float>(at)), x[e]);
      x[e] = at < lo || at >= hi ? -__builtin_inff() : x[e];
    }
    float off = m;
    if constexpr (!M::FIXED) {
      float top = x[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, x[e]);
      top = xor32_max(xor16_max(top));
      const bool grow = top > m && (m == -__builtin_inff() || top - m > 8.f);
      if (__any(grow)) {
        const float alpha = grow ? fast_exp2(m - top) : 1.f;
        m = grow ? top : m;
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      off = m == -__builtin_inff() ? 0.f : m;
    }
    bf16x8 ph, pl;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float w = fast_exp2(x[e] - off);
      l += w;
      ph[e] = static_cast<bf16>(w);
      pl[e] = static_cast<bf16>(w - static_cast<float>(ph[e]));
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const bf16x8 vv = Tile::col8(tv, 0, dt * 16, l16, g);
      acc[dt] = mfma16(vv, ph, acc[dt]);
      acc[dt] = mfma16(vv, pl, acc[dt]);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this stage has been read
    issue(t + 2 * NW, st);
  }
  wait_vmcnt<0>();
  __syncthreads();  // the tiles' place is free in every wave's part
  float* sO = reinterpret_cast<float*>(&lds[0][0][0][0]);
  l = xor32_sum(xor16_sum(l));
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
    *reinterpret_cast<f32x4*>(sO + (wave * 16 + l16) * kLdO + dt * 16 + 4 * g) = acc[dt];
  if (g == 0) {
    sM[wave][l16] = m;
    sL[wave][l16] = l;
  }
  __syncthreads();
  auto get = [&](int w, int n, int d) { return *reinterpret_cast<const f32x4*>(sO + (w * 16 + n) * kLdO + d); };
  auto stat = [&](int w, int n, float& mm, float& ll) {
    mm = sM[w][n];
    ll = sL[w][n];
  };
  if (splits == 1) {
    few_finish<D, M>(p, f, q, k, v, o, o_low, lse2, NW, &bad, get, stat);
    return;
  }
  // one {O [16][D], m [16], l [16]} of the workgroup
  float* out = partial + static_cast<int64_t>(item) * (16 * D + 32);
  for (int x = threadIdx.x; x < 16 * (D / 4); x += 64 * NW) {
    const int n = x / (D / 4), d = x % (D / 4) * 4;
    float top = -__builtin_inff(), sum = 0.f;
    f32x4 a4 = zero4();
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, sM[w][n]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = sM[w][n] == -__builtin_inff() ? 0.f : fast_exp2(sM[w][n] - top);
      sum = fmaf(a, sL[w][n], sum);
      const f32x4 part = get(w, n, d);
#pragma unroll
      for (int e = 0; e < 4; ++e) a4[e] = fmaf(a, part[e], a4[e]);
    }
    *reinterpret_cast<f32x4*>(out + n * D + d) = a4;
    if (d == 0) {
      out[16 * D + n] = top;
      out[16 * D + 16 + n] = sum;
    }
  }
}

// a workgroup per row tile
template <int D, class M>
__global__ __launch_bounds__(256) void scored_few_merge_kernel(ScoredShape p, const bf16* q, const bf16* k,
                                                               const bf16* v, bf16* o, bf16* o_low, float* lse2,
                                                               const float* __restrict__ partial, int n_rt,
                                                               int splits) {
  __shared__ uint32_t bad;
  __shared__ float sS[kFewSplits][32];  // m and l of the rows
  const FewRows f = few_rows(p, static_cast<int>(blockIdx.x), n_rt);
  const float* from = partial + static_cast<int64_t>(blockIdx.x) * splits * (16 * D + 32);
  for (int x = threadIdx.x; x < 32 * splits; x += 256) sS[x / 32][x % 32] = from[x / 32 * (16 * D + 32) + 16 * D + x % 32];
  __syncthreads();
  few_finish<D, M>(
      p, f, q, k, v, o, o_low, lse2, splits, &bad,
      [&](int w, int n, int d) {
        return *reinterpret_cast<const f32x4*>(from + w * (16 * D + 32) + n * D + d);
      },
      [&](int w, int n, float& m, float& l) {
        m = sS[w][n];
        l = sS[w][16 + n];
      });
}

// ------------------------------------------------------------ backward
// dS = P (dP - delta) (1 - tanh^2), P = 2^(x - lse2), in two kernels that each
// form the scores again: dQ by query tiles, dK and dV by key tiles; so nothing
// is added up by atomics and a gradient has one order of its sums.  P and dS
// are rounded to bf16 (half a step, 2^-8) as operands of the next product.

// dS of weight P and dP - delta, without the factor 4 of 1 - tanh^2 = 4 t (1 - t)
template <class M>
__device__ __forceinline__ float score_grad(float pv, float dp, float t) {
  return M::CAP ? pv * dp * fmaf(-t, t, t) : pv * dp;
}
template <class M>
__device__ __forceinline__ float grad_scale(const ScoredShape& p) {
  return M::CAP ? 4.f * p.scale : p.scale;
}

// dQ, tiled as the forward.  First the statistics of the workgroup's queries,
// which the next kernel reads too: nl2 (-inf for a row that sees nothing: every
// P is 0) and ndelta = -rowsum(dO o), the start of the dP products' sums.  o_low (the
// part of o that its rounding cut off, if given) goes into that sum: dP - delta
// cancels where one key has nearly all the weight, and half a step of o in delta
// would be most of what is left (dQ and dK 2.5 times further from 64 bits).  Three
// products a tile and one exponential a score: 138 us for 4 x 32 heads of 2048 with a
// distance bias, 226 for 16 heads of 128 x 8192 in documents.  No unit is busy all the time
// (counters, of all cycles: matrix unit 35 and 30%, VALU issue 40 and 32%, LDS 36 and 30%,
// at the 256 bytes a clock that a loop of such reads reaches): a tile's products, exponentials
// and products follow each other, and four waves a SIMD (D 128: two) do not fill each
// other's gaps.
template <int D, int NW, class M, int DC = D>
__global__ __launch_bounds__(64 * NW, D == 64 || NW == 8 ? 4 : 2) void scored_dq_kernel(
    ScoredShape p, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v,
    const bf16* __restrict__ o, const bf16* __restrict__ o_low, const bf16* __restrict__ dout,
    const float* __restrict__ lse2, float* __restrict__ nl2_out, float* __restrict__ nd_out, bf16* __restrict__ dq,
    int n_qt) {
  constexpr int BQ = 16 * NW, KS = DC / 32, DT = DC / 16;
  constexpr int kStages = 2;
  using Tile = RowTile<D>;
  using Load = RowLoader<D, NW>;
  __shared__ __attribute__((aligned(1024))) bf16 sK[kStages][Tile::kElems];
  __shared__ __attribute__((aligned(1024))) bf16 sV[kStages][Tile::kElems];
  const HeadTile ht = head_tile(p.B * p.Hq);
  const int q0 = (n_qt - 1 - ht.tile) * BQ;
  const int b = ht.head / p.Hq, h = ht.head % p.Hq, hk = h / (p.Hq / p.Hkv);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int l16 = lane & 15, g = lane >> 4;
  const RowView r = row_view(p, b);
  const float slope2 = M::BIAS ? slope2_of(p, h) : 0.f;
  const int64_t stat = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;

  const int i = min(q0 + 16 * wave + l16, p.Sq - 1);
  const bool mine = q0 + 16 * wave + l16 < p.Sq;
  const int64_t at = b * p.o_sb + i * p.o_ss + h * p.o_sh;
  bf16x8 qf[KS], df[KS];
  float part = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    qf[ks] = row_frag(q + b * p.q_sb + i * p.q_ss + h * p.q_sh, ks * 32 + g * 8, p.D, true);
    df[ks] = row_frag(dout + at, ks * 32 + g * 8, p.D, true);
    const bf16x8 of = row_frag(o + at, ks * 32 + g * 8, p.D, true);
    const bf16x8 ol = row_frag(o_low + at, ks * 32 + g * 8, p.D, o_low != nullptr);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      part = fmaf(static_cast<float>(df[ks][e]), static_cast<float>(of[e]) + static_cast<float>(ol[e]), part);
  }
  const float nd = -xor32_sum(xor16_sum(part));
  const float l2 = lse2[stat + i];
  const float nl2 = l2 == -__builtin_inff() ? l2 : p.cap_out - l2;
  if (mine && g == 0) {
    nl2_out[stat + i] = nl2;
    nd_out[stat + i] = nd;
  }
  const ColSpan span = col_span(seen_keys(p, r, i));
  const float pos = M::BIAS ? bias_pos(p, r, i) : 0.f;
  const float first_pos = __shfl(pos, 0, 16);
  f32x4 acc[DT], start[2];
  bias_start<M, 2>(p, slope2, start);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = zero4();
  const int k_lo = __builtin_amdgcn_readfirstlane(seen_keys(p, r, q0).lo);
  const int k_hi = __builtin_amdgcn_readfirstlane(seen_keys(p, r, min(q0 + BQ, p.Sq) - 1).hi);
  wait_vmcnt<0>();
  PairStream<D, NW, kStages, false> in;
  in.init(k + b * p.k_sb + hk * p.k_sh + k_lo * p.k_ss, p.k_ss, v + b * p.v_sb + hk * p.v_sh + k_lo * p.v_ss, p.v_ss,
          k_hi - k_lo, p.D, sK[0], sV[0], wave, lane);
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) in.issue();

  int st = 0;
  for (int k0 = k_lo; k0 < k_hi; k0 += 64, st = next_stage<kStages>(st)) {
    tile_barrier<(kStages - 2) * 2 * Load::P>();
    in.issue();
    if (k0 >= span.hi_max || k0 + 64 <= span.lo_min || q0 + 16 * wave >= p.Sq) continue;
    const bf16* tk = sK[st];
    const bf16* tv = sV[st];
    const bool behind = __builtin_amdgcn_readfirstlane(first_pos >= static_cast<float>(k0 + 63));
    const float dist = pos - static_cast<float>(k0 + 4 * g);
    // 32 keys at a time: S^T and dP^T, then dS as the operand of the last product
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      f32x4 s[2], dp[2];
#pragma unroll
      for (int m2 = 0; m2 < 2; ++m2) {
        s[m2] = start[m2];
        dp[m2] = f32x4{nd, nd, nd, nd};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          s[m2] = mfma16(Tile::row8(tk, 32 * s2 + 16 * m2 + l16, ks * 32 + g * 8), qf[ks], s[m2]);
          dp[m2] = mfma16(Tile::row8(tv, 32 * s2 + 16 * m2 + l16, ks * 32 + g * 8), df[ks], dp[m2]);
        }
      }
      float x[8], t[8], ds[8];
      tile_scores<M>(p, s, nl2, slope2, dist - 32.f * s2, behind, x, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) ds[e] = score_grad<M>(fast_exp2(x[e]), dp[e >> 2][e & 3], t[e]);
      if (k0 < span.lo_max) hide_below<8>(ds, span.mine.lo - k0 - 4 * g - 32 * s2, 0.f);
      if (k0 + 64 > span.hi_min) hide_from<8>(ds, span.mine.hi - k0 - 4 * g - 32 * s2, 0.f);
      bf16x8 dsf;
#pragma unroll
      for (int e = 0; e < 8; ++e) dsf[e] = static_cast<bf16>(ds[e]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma16(Tile::col8(tk, 32 * s2, dt * 16, l16, g), dsf, acc[dt]);
    }
  }
  wait_vmcnt<0>();
  const float f = grad_scale<M>(p);
  bool fine = true;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) fine = fine && fabsf(acc[dt][e]) < __builtin_inff();
  const uint32_t bad = named_rows(__ballot(!fine && mine));
  if (mine && (bad >> l16 & 1) == 0) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = static_cast<bf16>(acc[dt][e] * f);
      if (dt * 16 + g * 4 < p.D) *reinterpret_cast<bf16x4*>(dq + at + dt * 16 + g * 4) = x;
    }
  }
  for (uint32_t left = bad; left != 0; left &= left - 1) {
    const int n = __ffs(left) - 1, row = q0 + 16 * wave + n;
    scored_row_dq(p, q, k, v, dout, lse2[stat + row], __shfl(nd, n, 64), dq, b, h, row, lane);
  }
}

// As tile_scores for one key and 8 queries: rows 4 g + e and 16 + 4 g + e from position
// `first` on, off their nl2 and the distance from their position, beyond the keys counted
// from the nearest of them as in bias_pos.  ahead: every position lies among the keys and
// not before this one.
template <class M>
__device__ __forceinline__ void query_scores(const ScoredShape& p, const f32x4 (&s)[2], const f32x4 (&nl2)[2],
                                             float slope2, float first, float key, bool ahead, float (&x)[8],
                                             float (&t)[8]) {
  float bias[8];
  if constexpr (M::BIAS) {
    if (ahead) {
      const float base = -slope2 * (first - key);
#pragma unroll
      for (int e = 0; e < 8; ++e) bias[e] = fmaf(-slope2, static_cast<float>(16 * (e >> 2) + (e & 3)), base);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float at = first + static_cast<float>(16 * (e >> 2) + (e & 3));
        bias[e] = -slope2 * fabsf(fminf(fmaxf(at, 0.f), static_cast<float>(p.Sk - 1)) - key);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float off = M::BIAS ? nl2[e >> 2][e & 3] + bias[e] : nl2[e >> 2][e & 3];
    if constexpr (M::CAP) {
      t[e] = cap_t(p, s[e >> 2][e & 3]);
      x[e] = fmaf(-2.f * p.cap_out, t[e], off);
    } else {
      x[e] = fmaf(s[e >> 2][e & 3], p.c, off);
    }
  }
}

// dK and dV.  A workgroup owns 16 NW keys of a KV head, 16 a wave, and walks the 64-query
// tiles that see any of them, of every query head of the group: the products are those of
// the forward with queries and keys exchanged (S = Q K^T, a lane holding one key's
// scores).  `splits` workgroups share that walk where there are few keys; their fp32 sums
// go to `partial` ([split][row of the batch, KV head, key][dK | dV][D]) and are added in
// split order by scored_reduce_kernel.  Four products a tile: 195 us for 4 x 32 heads of
// 2048 with a distance bias and 8 KV heads, 14 to add the parts up; 318 and 23 for 16 / 4
// heads of 128 x 8192 in documents.  As in dQ no unit is busy all the time (matrix unit 31
// and 29%, VALU issue 42 and 26%, LDS 38 and 33%).
template <int D, int NW, class M, int DC = D>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 2) void scored_dkdv_kernel(
    ScoredShape p, const bf16* __restrict__ q, const bf16* __restrict__ k, const bf16* __restrict__ v,
    const bf16* __restrict__ dout, const float* __restrict__ lse2, const float* __restrict__ nl2,
    const float* __restrict__ nd, bf16* __restrict__ dk, bf16* __restrict__ dv, float* __restrict__ partial,
    int splits) {
  constexpr int BK = 16 * NW, KS = DC / 32, DT = DC / 16;
  constexpr int kStages = D == 64 ? 2 : 4;
  using Tile = RowTile<D>;
  using Load = RowLoader<D, NW>;
  constexpr int kLoads = 2 * Load::P + 1;  // Q, dO, and one of the two row statistics
  __shared__ __attribute__((aligned(1024))) bf16 sQ[kStages][Tile::kElems];
  __shared__ __attribute__((aligned(1024))) bf16 sD[kStages][Tile::kElems];
  __shared__ __attribute__((aligned(256))) float sStat[kStages][NW][64];
  // under a causal mask the first keys have the most queries
  const HeadTile ht = head_tile(p.B * p.Hkv);
  const int part = ht.tile % splits, kt0 = ht.tile / splits * BK, hk = ht.head % p.Hkv, b = ht.head / p.Hkv;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int l16 = lane & 15, g = lane >> 4;
  const int group = p.Hq / p.Hkv;
  const RowView r = row_view(p, b);

  const int key = min(kt0 + 16 * wave + l16, p.Sk - 1);
  bf16x8 kf[KS], vf[KS];
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    kf[ks] = row_frag(k + b * p.k_sb + key * p.k_ss + hk * p.k_sh, ks * 32 + g * 8, p.D, true);
    vf[ks] = row_frag(v + b * p.v_sb + key * p.v_ss + hk * p.v_sh, ks * 32 + g * 8, p.D, true);
  }
  const ColSpan span = col_span(seen_by(p, r, key));
  const float keyf = static_cast<float>(key);
  f32x4 ka[DT], va[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ka[dt] = va[dt] = zero4();
  const int q_lo = __builtin_amdgcn_readfirstlane(seen_by(p, r, kt0).lo);
  const int q_hi = __builtin_amdgcn_readfirstlane(seen_by(p, r, min(kt0 + BK, p.Sk) - 1).hi);
  const int n_qt = (q_hi - q_lo + 63) / 64;  // per query head
  const int64_t walk = static_cast<int64_t>(n_qt) * group;
  const int first = static_cast<int>(walk * part / splits), total = static_cast<int>(walk * (part + 1) / splits) - first;
  wait_vmcnt<0>();
  // Walk tile n is 64 queries of one head: the heads' tiles one head after the other.
  // `q_at` walks for the loads (pointers to the next tile's rows), c_h / c_t for the
  // products.
  Load lq, ld;
  lq.init(p.q_ss, p.D, wave, lane);
  ld.init(p.o_ss, p.D, wave, lane);
  const uint32_t q_lds = share_of<Load>(sQ[0], wave), d_lds = share_of<Load>(sD[0], wave);
  constexpr uint32_t kStageBytes = Tile::kElems * 2;
  int l_h = 0, l_t = 0;
  if (total > 0) l_h = first / n_qt, l_t = first % n_qt;
  int c_h = hk * group + l_h, c_t = l_t;
  const bf16 *q_head = q + b * p.q_sb + c_h * p.q_sh + q_lo * p.q_ss;
  const bf16 *d_head = dout + b * p.o_sb + c_h * p.o_sh + q_lo * p.o_ss;
  const float* s_head = ((wave & 1) ? nd : nl2) + (static_cast<int64_t>(b) * p.Hq + c_h) * p.Sq + q_lo;
  const bf16 *q_at = q_head + 64 * l_t * p.q_ss, *d_at = d_head + 64 * l_t * p.o_ss;
  const float* s_at = s_head + 64 * l_t;
  int issued = 0, l_st = 0, l_left = q_hi - q_lo - 64 * l_t;
  auto issue = [&]() {
    const int n = issued < total ? l_left : 0;
    lq.issue(q_at, q_lds + l_st * kStageBytes, n);
    ld.issue(d_at, d_lds + l_st * kStageBytes, n);
    load_lds4(make_rsrc(s_at, 256), &sStat[l_st][wave][0], lane < n ? 4u * static_cast<uint32_t>(lane) : kOOB);
    ++issued;
    l_st = next_stage<kStages>(l_st);
    q_at += 64 * p.q_ss;
    d_at += 64 * p.o_ss;
    s_at += 64;
    l_left -= 64;
    if (l_left <= 0) {  // the next head
      q_head += p.q_sh;
      d_head += p.o_sh;
      s_head += p.Sq;
      q_at = q_head;
      d_at = d_head;
      s_at = s_head;
      l_left = q_hi - q_lo;
    }
  };
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) issue();

  int st = 0;
  for (int it = 0; it < total; ++it, st = next_stage<kStages>(st)) {
    tile_barrier<(kStages - 2) * kLoads>();
    issue();
    const bf16* tq = sQ[st];
    const bf16* td = sD[st];
    const float* sL = sStat[st][0];
    const float* sN = sStat[st][1];
    const int q0 = q_lo + 64 * c_t;
    const float slope2 = M::BIAS ? slope2_of(p, c_h) : 0.f;
    if (++c_t == n_qt) c_t = 0, ++c_h;
    if (q0 >= span.hi_max || q0 + 64 <= span.lo_min || kt0 + 16 * wave >= p.Sk) continue;
    // the queries' positions: of this lane's first, and whether all lie among the keys
    // and none before one of the workgroup's
    const int64_t pos0 = r.offset + q0;
    const float first_pos = static_cast<float>(pos0 + 4 * g);
    const bool ahead = pos0 >= kt0 + BK - 1 && pos0 + 64 <= p.Sk;
    // 32 queries at a time
#pragma unroll
    for (int s2 = 0; s2 < 2; ++s2) {
      f32x4 s[2], dp[2], l4[2];
#pragma unroll
      for (int m2 = 0; m2 < 2; ++m2) {
        const int row = 32 * s2 + 16 * m2;
        l4[m2] = *reinterpret_cast<const f32x4*>(sL + row + 4 * g);
        s[m2] = zero4();
        dp[m2] = *reinterpret_cast<const f32x4*>(sN + row + 4 * g);
      }
#pragma unroll
      for (int m2 = 0; m2 < 2; ++m2)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const bf16x8 aq = Tile::row8(tq, 32 * s2 + 16 * m2 + l16, ks * 32 + g * 8);
          const bf16x8 ad = Tile::row8(td, 32 * s2 + 16 * m2 + l16, ks * 32 + g * 8);
          s[m2] = mfma16(aq, kf[ks], s[m2]);
          dp[m2] = mfma16(ad, vf[ks], dp[m2]);
        }
      float x[8], t[8], pv[8], ds[8];
      query_scores<M>(p, s, l4, slope2, first_pos + 32.f * s2, keyf, ahead, x, t);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pv[e] = fast_exp2(x[e]);
        ds[e] = score_grad<M>(pv[e], dp[e >> 2][e & 3], t[e]);
      }
      const int from = q0 + 32 * s2 + 4 * g;
      if (q0 < span.lo_max) {
        hide_below<8>(pv, span.mine.lo - from, 0.f);
        hide_below<8>(ds, span.mine.lo - from, 0.f);
      }
      if (q0 + 64 > span.hi_min) {
        hide_from<8>(pv, span.mine.hi - from, 0.f);
        hide_from<8>(ds, span.mine.hi - from, 0.f);
      }
      bf16x8 pa, da;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        pa[e] = static_cast<bf16>(pv[e]);
        da[e] = static_cast<bf16>(ds[e]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const bf16x8 bd = Tile::col8(td, 32 * s2, dt * 16, l16, g);
        const bf16x8 bq = Tile::col8(tq, 32 * s2, dt * 16, l16, g);
        va[dt] = mfma16(bd, pa, va[dt]);
        ka[dt] = mfma16(bq, da, ka[dt]);
      }
    }
  }
  wait_vmcnt<0>();
  // lane: dK^T and dV^T [d = 16 dt + 4 g + e][its key]
  const float f = grad_scale<M>(p);
  const bool mine = kt0 + 16 * wave + l16 < p.Sk;
  if (splits > 1) {
    if (!mine) return;
    float* row = partial + (((static_cast<int64_t>(part) * p.B + b) * p.Hkv + hk) * p.Sk + key) * (2 * D) + 4 * g;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      *reinterpret_cast<f32x4*>(row + 16 * dt) = ka[dt] * f;
      *reinterpret_cast<f32x4*>(row + D + 16 * dt) = va[dt];
    }
    return;
  }
  bool fine = true;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int e = 0; e < 4; ++e) fine = fine && fabsf(ka[dt][e]) < __builtin_inff() && fabsf(va[dt][e]) < __builtin_inff();
  const uint32_t bad = named_rows(__ballot(!fine && mine));
  if (mine && (bad >> l16 & 1) == 0) {
    const int64_t at = b * p.g_sb + key * p.g_ss + hk * p.g_sh;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x4 x, y;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[e] = static_cast<bf16>(ka[dt][e] * f);
        y[e] = static_cast<bf16>(va[dt][e]);
      }
      if (dt * 16 + g * 4 < p.D) {
        *reinterpret_cast<bf16x4*>(dk + at + dt * 16 + g * 4) = x;
        *reinterpret_cast<bf16x4*>(dv + at + dt * 16 + g * 4) = y;
      }
    }
  }
  for (uint32_t left = bad; left != 0; left &= left - 1)
    scored_row_dkdv(p, q, k, v, dout, lse2, nd, dk, dv, b, hk, kt0 + 16 * wave + __ffs(left) - 1, lane);
}

// dK and dV of shared walks: the sums of the splits in their order.  A wavefront
// takes 256 / D rows (dK and dV of a key are one row of 2 D), 8 elements a lane; a
// row that is not finite is run again as in the kernels above.
template <int D>
__global__ __launch_bounds__(256) void scored_reduce_kernel(ScoredShape p, const float* __restrict__ partial,
                                                            int splits, int64_t rows, const bf16* q, const bf16* k,
                                                            const bf16* v, const bf16* dout, const float* lse2,
                                                            const float* nd, bf16* dk, bf16* dv) {
  constexpr int LPR = D / 4;  // lanes per row
  const int lane = threadIdx.x & 63;
  const int64_t row0 = (static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6)) * (64 / LPR);
  const int64_t row = row0 + lane / LPR;
  const int d = lane % LPR * 8;  // of the 2 D
  const bool ok = row < rows && d % D < p.D;  // (columns past D need not have been summed)
  float x[8] = {};
  if (ok)
#pragma unroll 2
    for (int s = 0; s < splits; ++s) {
      const f32x4* from = reinterpret_cast<const f32x4*>(partial + (s * rows + row) * (2 * D) + d);
      const f32x4 lo = from[0], hi = from[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += lo[e], x[4 + e] += hi[e];
    }
  bool fine = true;
#pragma unroll
  for (int e = 0; e < 8; ++e) fine = fine && fabsf(x[e]) < __builtin_inff();
  const uint64_t bad = __ballot(ok && !fine);
  constexpr uint64_t kRow = LPR == 64 ? ~uint64_t{0} : (uint64_t{1} << (LPR % 64)) - 1;
  auto where = [&](int64_t n, int& b, int& hk, int& key) {
    key = static_cast<int>(n % p.Sk);
    hk = static_cast<int>(n / p.Sk % p.Hkv);
    b = static_cast<int>(n / p.Sk / p.Hkv);
  };
  int b, hk, key;
  if (ok && (bad >> (lane / LPR * LPR) & kRow) == 0) {
    where(row, b, hk, key);
    bf16x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = static_cast<bf16>(x[e]);
    bf16* to = (d < D ? dk : dv) + b * p.g_sb + key * p.g_ss + hk * p.g_sh + d % D;
    __builtin_memcpy(to, &y, 16);
  }
  for (int n = 0; n < 64 / LPR; ++n)
    if ((bad >> (n * LPR) & kRow) != 0) {
      where(row0 + n, b, hk, key);
      scored_row_dkdv(p, q, k, v, dout, lse2, nd, dk, dv, b, hk, key, lane);
    }
}

// ------------------------------------------------------------ host side
int fill_scored(ScoredShape* p, const nmb_scores* sc, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk,
                int64_t D, const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* os,
                const int64_t* gs, const void* q, const void* k, const void* v, const void* o, int dtype) {
  NMB_REQUIRE(sc != nullptr && qs != nullptr && ks != nullptr && vs != nullptr && os != nullptr,
              "scored attention: null argument");
  NMB_REQUIRE(B >= 0 && Hq > 0 && Hkv > 0 && Sq >= 0 && Sk >= 0 && D > 0, "scored attention: invalid shape");
  NMB_REQUIRE(Hq % Hkv == 0, "query heads (%lld) must be divisible by KV heads (%lld)", (long long)Hq,
              (long long)Hkv);
  NMB_REQUIRE(B <= 65535 && Hq <= 65535 && Sq <= 0x3fffffff && Sk <= 0x3fffffff,
              "scored attention: shape exceeds the launch grid");
  NMB_REQUIRE_SUPPORTED(dtype == NMB_BF16 || dtype == NMB_F32, "scored attention: unsupported dtype code %d", dtype);
  NMB_REQUIRE_SUPPORTED(D <= 128, "scored attention: head_dim must be <= 128, got %lld", (long long)D);
  // 2^-20 of the cap is what a capped score is off by, and 2 log2(e) / cap overflows for the smallest
  NMB_REQUIRE((sc->scale <= 0.f || (sc->scale >= 1e-30f && sc->scale <= 1e30f)) && (sc->cap == 0.f || (sc->cap >= 1e-3f && sc->cap <= 1e4f)),
              "scored attention: scale must lie within 1e-30 and 1e30 (or be <= 0), cap within 1e-3 and 1e4 (or be 0)");
  NMB_REQUIRE_SUPPORTED(sc->slopes == nullptr || Sk <= (1 << 24),
                        "scored attention: a distance bias needs at most 2^24 keys (positions in fp32)");
  NMB_REQUIRE(sc->window >= 0, "scored attention: window must be >= 0 (0: none)");
  NMB_REQUIRE(sc->prefix == nullptr || sc->causal, "scored attention: a prefix needs causal");
  NMB_REQUIRE(llabs(sc->q_offset) <= (int64_t{1} << 40), "scored attention: q_offset out of range");
  NMB_REQUIRE((reinterpret_cast<uintptr_t>(sc->runs) & 7) == 0, "scored attention: runs must be 8-byte aligned");
  for (int i = 0; i < 3; ++i)
    NMB_REQUIRE(qs[i] >= 0 && ks[i] >= 0 && vs[i] >= 0 && os[i] >= 0 && (gs == nullptr || gs[i] >= 0),
                "scored attention: negative stride");
  if (dtype == NMB_BF16) {
    // 16-byte rows; a tile of 64 of them within 2 GiB
    NMB_REQUIRE_SUPPORTED(D % 8 == 0, "scored attention (bf16): head_dim must be a multiple of 8, got %lld", (long long)D);
    for (int i = 0; i < 3; ++i)
      NMB_REQUIRE_SUPPORTED(qs[i] % 8 == 0 && ks[i] % 8 == 0 && vs[i] % 8 == 0 && os[i] % 8 == 0 &&
                                (gs == nullptr || gs[i] % 8 == 0),
                            "scored attention (bf16): strides must be multiples of 8 elements");
    NMB_REQUIRE_SUPPORTED(qs[1] < (1 << 23) && ks[1] < (1 << 23) && vs[1] < (1 << 23) && os[1] < (1 << 23),
                          "scored attention (bf16): token strides must be below 2^23 elements");
    for (const void* t : {q, k, v, o})
      NMB_REQUIRE(aligned16(t), "scored attention (bf16): tensors must be 16-byte aligned");
  }
  p->B = static_cast<int>(B);
  p->Hq = static_cast<int>(Hq);
  p->Hkv = static_cast<int>(Hkv);
  p->Sq = static_cast<int>(Sq);
  p->Sk = static_cast<int>(Sk);
  p->D = static_cast<int>(D);
  p->q_sb = qs[0], p->q_ss = qs[1], p->q_sh = qs[2];
  p->k_sb = ks[0], p->k_ss = ks[1], p->k_sh = ks[2];
  p->v_sb = vs[0], p->v_ss = vs[1], p->v_sh = vs[2];
  p->o_sb = os[0], p->o_ss = os[1], p->o_sh = os[2];
  p->g_sb = p->g_ss = p->g_sh = 0;
  if (gs != nullptr) p->g_sb = gs[0], p->g_ss = gs[1], p->g_sh = gs[2];
  const double scale = sc->scale > 0.f ? sc->scale : 1.0 / sqrt(static_cast<double>(D));
  const double log2e = 1.4426950408889634074;
  p->scale = static_cast<float>(scale);
  p->c = static_cast<float>(scale * log2e);
  p->cap_in = sc->cap > 0.f ? static_cast<float>(2.0 * log2e * scale / sc->cap) : 0.f;
  p->cap_out = sc->cap > 0.f ? static_cast<float>(sc->cap * log2e) : 0.f;
  p->causal = sc->causal ? 1 : 0;
  p->window = std::min(sc->window, int64_t{1} << 42);  // further than any two positions
  p->q_offset = sc->q_offset;
  p->slopes = sc->slopes;
  p->offsets = sc->offsets;
  p->prefix = sc->prefix;
  p->runs = reinterpret_cast<const int2*>(sc->runs);
  return NMB_OK;
}

// f(Mode): the compiled way of forming scores for p
template <class F>
void with_mode(const ScoredShape& p, F&& f) {
  const bool bias = p.slopes != nullptr;
  if (p.cap_out > kFixedMax) f(Mode<true, true, false>{});  // (without slopes: a bias of 0)
  else if (p.cap_out > 0.f && bias) f(Mode<true, true, true>{});
  else if (p.cap_out > 0.f) f(Mode<true, false, true>{});
  else if (bias) f(Mode<false, true, false>{});
  else f(Mode<false, false, false>{});
}

void grid_of(int64_t items, int* per_xcd, dim3* grid) {
  *per_xcd = static_cast<int>((items + 7) / 8);
  *grid = dim3(static_cast<unsigned>(*per_xcd) * 8u);
}

// Queries of a workgroup of the tiled kernels, 16 a wave: 64 while there are at most 1,024
// tiles of them (the GPU holds 1,024 or 512 such workgroups at once), then 128, which read
// the keys half as often.  Forward without and with gradients (one and two terms of P) /
// backward, us, 64 and 128 queries: 2 x 16 heads x 1024 (512 tiles) 18.0, 22.0 / 56 and 23.7,
// 26.9 / 62; 2 x 16 x 2048 (1,024) 38.4, 47.6 / 121 and 44.7, 55.6 / 127; 3 x 16 x 2048 (1,536)
// 50.7, 63.2 / 147 and 57.5, 66.4 / 154; 16 x 16 x 512 in documents (2,048) 22.8, 28.6 / 71
// and 23.2, 30.4 / 74; 4 x 32 x 2048 with a distance bias (4,096) 107.6, 135 / 324 and 105.9,
// 137 / 325; heads of 128: 2 x 16 x 2048 (1,024) 59.8, 75.6 / 188 and 59.4, 77.1 / 192, 16 x
// 8192 (2,048) 372, 463 / 1184 and 339, 424 / 1136.  (Between 1,024 and 2,048 tiles 64 would
// be the better number up to a head dim of 64.)
int queries_per_workgroup(const ScoredShape& p) {
  return (p.Sq + 63) / 64 * static_cast<int64_t>(p.Hq) * p.B <= 1024 ? 64 : 128;
}

int tiles_fwd_launch(const ScoredShape& p, const bf16* q, const bf16* k, const bf16* v, bf16* o, bf16* o_low, float* lse2,
                     hipStream_t stream) {
  const int64_t heads = static_cast<int64_t>(p.Hq) * p.B;
  const int bq = queries_per_workgroup(p);
  const int n_qt = (p.Sq + bq - 1) / bq;
  NMB_REQUIRE(n_qt * heads < (int64_t{1} << 30), "attn_scored_fwd: problem too large for one launch");
  const dim3 grid(static_cast<unsigned>(n_qt * heads));
  with_mode(p, [&](auto mode) {
    using M = decltype(mode);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(4 * bq), 0, stream, p, q, k, v, o, o_low, lse2, n_qt);
    };
    auto with_low = [&](auto low) {
      constexpr bool LOW = decltype(low)::value;
      if (p.D <= 64) {
        if (bq == 64) go(scored_fwd_kernel<64, 4, M, LOW>); else go(scored_fwd_kernel<64, 8, M, LOW>);
      } else if (p.D <= 96) {
        if (bq == 64) go(scored_fwd_kernel<128, 4, M, LOW, 96>); else go(scored_fwd_kernel<128, 8, M, LOW, 96>);
      } else {
        if (bq == 64) go(scored_fwd_kernel<128, 4, M, LOW>); else go(scored_fwd_kernel<128, 8, M, LOW>);
      }
    };
    if (o_low != nullptr) with_low(std::true_type{}); else with_low(std::false_type{});
  });
  NMB_CHECK_LAUNCH("attn_scored_fwd");
  return NMB_OK;
}

// Few queries: row tiles of 16 (query, head) pairs and workgroups per row tile.  Taken for
// up to 16 queries, whose tiles of 64 would be mostly empty, and where the tiled kernel has
// at most 64 workgroups, a quarter of the CUs, so that the keys are better shared (each row
// tile reads them again).  Forward, us, tiled without and with gradients / few (two terms of P
// in both): up to 16 queries: 32 sequences x 32 / 8 heads x 1 on 512 keys 13.3, 14.2 / 8.1, 64 x
// 32 / 8 x 4 on 512 34.3, 44.0 / 19.3, 8 x 32 / 8 heads of 128 x 16 on 2048 36.8, 42.7 / 40.1;
// more: 8 workgroups (8 heads x 40 on 8192) 98, 121 / 11.7, 32 (4 x 8 heads of 128 x 40 on
// 4096) 70, 82 / 33, 64 (4 heads x 1024) 15.9, 19.2 / 9.0, 80 (8 heads of 128 x 640) 15.3, 18.0 /
// 16.7, 96 (2 x 24 heads x 100 on 1000, 16 heads x 384) 15.9, 19.2 / 16.1 and 8.6, 10.1 / 10.9,
// 128 (8 x 16 heads of 128 x 64 on 4096) 72, 85 / 100.  The first rule loses where there are
// many sequences and a group's rows leave the row tiles mostly empty on few keys: 64 x 32 heads
// of their own x 1 to 16 on 512 keys 45, 50 / 58 to 66.
struct FewPlan {
  bool use;
  int n_rt, splits;
  int64_t tiles;
  size_t bytes;
};
FewPlan few_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int dtype) {
  FewPlan f{false, 0, 1, 0, 0};
  if (dtype != NMB_BF16 || Sq == 0 || B == 0 || (Sq > 16 && (Sq + 63) / 64 * Hq * B > 64)) return f;
  f.use = true;
  f.n_rt = static_cast<int>((Hq / Hkv * Sq + 15) / 16);
  f.tiles = static_cast<int64_t>(f.n_rt) * Hkv * B;
  // four workgroups per CU in all, none below 4 key tiles a wave.  With at least 1, 2, 4 and
  // 8, us: one token of 16 heads on 400 keys 7.2 each, on 700 8.7, 7.9, 7.9, 7.9 (one chain of
  // loads, shared or not), on 1500 9.0, 10.3, 10.5, 10.5; of 32 / 8 heads of 128 on 700 10.0,
  // 10.9, 11.7, 11.7, on 2000 10.8, 11.5, 14.3, 22.2; 16 of 2 x 16 heads of 128 on 3000 31.8,
  // 25.0, 18.8, 23.2; of 4 x 8 heads of 80 on 8192 37.9, 37.8, 27.6, 20.9; 5 of 6 x 32 on 5001
  // 47.1, 47.3, 45.7, 47.0
  const int64_t per = 4 * kFewKeys * (D <= 64 ? 8 : 4);
  f.splits = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({1024 / f.tiles, Sk / per, kFewSplits})));
  if (f.splits > 1) f.bytes = static_cast<size_t>(f.tiles) * f.splits * (16 * (D <= 64 ? 64 : 128) + 32) * sizeof(float);
  return f;
}

int few_fwd_launch(const ScoredShape& p, const bf16* q, const bf16* k, const bf16* v, bf16* o, bf16* o_low,
                   float* lse2, float* partial, const FewPlan& f, hipStream_t stream) {
  NMB_REQUIRE(f.tiles * f.splits < (int64_t{1} << 30), "attn_scored_fwd: problem too large for one launch");
  const int items = static_cast<int>(f.tiles * f.splits);
  int per;
  dim3 grid;
  grid_of(items, &per, &grid);
  with_mode(p, [&](auto mode) {
    using M = decltype(mode);
    auto go = [&](auto kernel, int threads) {
      hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, stream, p, q, k, v, o, o_low, lse2, partial, f.n_rt, f.splits,
                         items, per);
    };
    if (p.D <= 64) go(scored_few_kernel<64, 8, M>, 512);
    else if (p.D <= 96) go(scored_few_kernel<128, 4, M, 96>, 256);
    else go(scored_few_kernel<128, 4, M>, 256);
    if (f.splits > 1) {
      const dim3 rows(static_cast<unsigned>(f.tiles));
      if (p.D <= 64)
        hipLaunchKernelGGL((scored_few_merge_kernel<64, M>), rows, dim3(256), 0, stream, p, q, k, v, o, o_low, lse2,
                           partial, f.n_rt, f.splits);
      else
        hipLaunchKernelGGL((scored_few_merge_kernel<128, M>), rows, dim3(256), 0, stream, p, q, k, v, o, o_low, lse2,
                           partial, f.n_rt, f.splits);
    }
  });
  NMB_CHECK_LAUNCH("attn_scored_fwd(few)");
  return NMB_OK;
}

// Keys of a workgroup of the dK/dV kernel, and the workgroups that share the walk over
// their queries: enough for two rounds of the GPU's slots (two workgroups share a CU at D <=
// 64, one at D 128), none with a walk below 8 tiles; four rounds, which even out walks that
// documents leave of any length, where each is then still 128 tiles, beside which adding up
// the parts is little.  Backward, us, two and four rounds (walks of four): 16 / 4 heads of 128
// in documents of ~2000 x 4096 213 and 240 (32 tiles), x 6144 284 and 294 (72), of ~3000 x 8192
// 424 and 415 (128); 32 / 4 heads of 64 in documents of ~1000 x 8192 306 and 300 (128), of ~500
// x 16384 568 and 509 (512); 4 x 32 / 8 heads of 64 x 2048 of ~700 261 and 283 (32), 4 x 16
// heads of 128 x 1024 112 and 157 (8).
constexpr int kKeysPerWorkgroup = 128;
int dkdv_splits(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D) {
  const int64_t items = (Sk + kKeysPerWorkgroup - 1) / kKeysPerWorkgroup * Hkv * B;
  const int64_t walk = Hq / Hkv * ((Sq + 63) / 64), slots = D <= 64 ? 512 : 256;
  const int64_t want = (walk * items >= 128 * 4 * slots ? 4 : 2) * slots;
  if (items == 0 || items >= want) return 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({(want + items / 2) / items, walk / 8, 8})));
}

struct BwdSpace {
  size_t stats, total;  // bytes of nl2 and ndelta; with the partial sums of `splits` behind
  int splits;
};
BwdSpace bwd_space(int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk, int64_t D, int dtype) {
  BwdSpace s;
  const size_t row = static_cast<size_t>(B) * Hq * Sq * sizeof(float);
  s.splits = dtype == NMB_BF16 ? dkdv_splits(B, Hq, Hkv, Sq, Sk, D) : 1;
  s.stats = dtype == NMB_BF16 ? (2 * row + 255) / 256 * 256 : row;
  s.total = s.stats;
  if (s.splits > 1) s.total += static_cast<size_t>(s.splits) * B * Hkv * Sk * 2 * (D <= 64 ? 64 : 128) * sizeof(float);
  return s;
}

int tiles_bwd_launch(const ScoredShape& p, const bf16* q, const bf16* k, const bf16* v, const bf16* o, const bf16* o_low,
                     const bf16* dout, const float* lse2, bf16* dq, bf16* dk, bf16* dv, char* ws, const BwdSpace& space,
                     hipStream_t stream) {
  float* nl2 = reinterpret_cast<float*>(ws);
  float* nd = nl2 + static_cast<int64_t>(p.B) * p.Hq * p.Sq;
  float* partial = reinterpret_cast<float*>(ws + space.stats);
  if (p.Sq > 0) {
    const int64_t heads = static_cast<int64_t>(p.Hq) * p.B;
    const int bq = queries_per_workgroup(p);
    const int n_qt = (p.Sq + bq - 1) / bq;
    NMB_REQUIRE(n_qt * heads < (int64_t{1} << 30), "attn_scored_bwd: problem too large for one launch");
    const dim3 grid(static_cast<unsigned>(n_qt * heads));
    with_mode(p, [&](auto mode) {
      using M = decltype(mode);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(4 * bq), 0, stream, p, q, k, v, o, o_low, dout, lse2, nl2, nd, dq, n_qt);
      };
      if (p.D <= 64) {
        if (bq == 64) go(scored_dq_kernel<64, 4, M>); else go(scored_dq_kernel<64, 8, M>);
      } else if (p.D <= 96) {
        if (bq == 64) go(scored_dq_kernel<128, 4, M, 96>); else go(scored_dq_kernel<128, 8, M, 96>);
      } else {
        if (bq == 64) go(scored_dq_kernel<128, 4, M>); else go(scored_dq_kernel<128, 8, M>);
      }
    });
    NMB_CHECK_LAUNCH("attn_scored_bwd(dq)");
  }
  if (p.Sk > 0) {
    const int n_kt = (p.Sk + kKeysPerWorkgroup - 1) / kKeysPerWorkgroup;
    const int64_t wide = static_cast<int64_t>(n_kt) * p.Hkv * p.B * space.splits;
    NMB_REQUIRE(wide < (int64_t{1} << 30), "attn_scored_bwd: problem too large for one launch");
    const dim3 grid(static_cast<unsigned>(wide));
    with_mode(p, [&](auto mode) {
      using M = decltype(mode);
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(512), 0, stream, p, q, k, v, dout, lse2, nl2, nd, dk, dv, partial,
                           space.splits);
      };
      if (p.D <= 64) go(scored_dkdv_kernel<64, 8, M>);
      else if (p.D <= 96) go(scored_dkdv_kernel<128, 8, M, 96>);
      else go(scored_dkdv_kernel<128, 8, M>);
    });
    NMB_CHECK_LAUNCH("attn_scored_bwd(dkdv)");
    if (space.splits > 1) {
      const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.Sk;
      const int64_t blocks = (rows * (p.D <= 64 ? 16 : 32) + 255) / 256;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, p, partial, space.splits,
                           rows, q, k, v, dout, lse2, nd, dk, dv);
      };
      if (p.D <= 64) go(scored_reduce_kernel<64>); else go(scored_reduce_kernel<128>);
      NMB_CHECK_LAUNCH("attn_scored_bwd(reduce)");
    }
  }
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

using nmb::ScoredShape;

extern "C" int nmb_document_runs(const int32_t* documents, int64_t batch_stride, int64_t batch, int64_t tokens,
                                 int32_t* runs, hipStream_t stream) {
  NMB_REQUIRE(batch >= 0 && tokens >= 0 && batch_stride >= 0 && batch <= 0x7fffffff && tokens <= 0x3fffffff,
              "document_runs: invalid shape");
  if (batch == 0 || tokens == 0) return NMB_OK;
  NMB_REQUIRE(documents != nullptr && runs != nullptr, "document_runs: null argument");
  NMB_REQUIRE((reinterpret_cast<uintptr_t>(runs) & 7) == 0, "document_runs: runs must be 8-byte aligned");
  hipLaunchKernelGGL(nmb::document_runs_kernel, dim3(static_cast<unsigned>(batch)), dim3(nmb::kRunThreads), 0, stream,
                     documents, batch_stride, static_cast<int>(tokens), reinterpret_cast<int2*>(runs));
  NMB_CHECK_LAUNCH("document_runs");
  return NMB_OK;
}

extern "C" int nmb_attn_scored_workspace_bytes(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t seq_q,
                                               int64_t seq_k, int64_t head_dim, int dtype, size_t* forward,
                                               size_t* backward) {
  NMB_REQUIRE(batch >= 0 && q_heads > 0 && kv_heads > 0 && seq_q >= 0 && seq_k >= 0 && head_dim > 0,
              "attn_scored_workspace_bytes: invalid shape");
  if (forward != nullptr)
    *forward = q_heads % kv_heads == 0
                   ? nmb::few_plan(batch, q_heads, kv_heads, seq_q, seq_k, head_dim, dtype).bytes
                   : 0;
  if (backward != nullptr)
    *backward = nmb::bwd_space(batch, q_heads, kv_heads, seq_q, seq_k, head_dim, dtype).total;
  return NMB_OK;
}

extern "C" int nmb_attn_scored_fwd(const void* q, const void* k, const void* v, void* o, void* o_low, float* lse2, int64_t batch,
                                   int64_t q_heads, int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* o_strides, const nmb_scores* scores, int dtype, void* workspace,
                                   size_t workspace_bytes, hipStream_t stream) {
  ScoredShape p;
  const int st = nmb::fill_scored(&p, scores, batch, q_heads, kv_heads, seq_q, seq_k, head_dim, q_strides, k_strides,
                                  v_strides, o_strides, nullptr, q, k, v, o, dtype);
  if (st != NMB_OK) return st;
  if (batch == 0 || seq_q == 0) return NMB_OK;
  NMB_REQUIRE(q != nullptr && o != nullptr && lse2 != nullptr && (seq_k == 0 || (k != nullptr && v != nullptr)),
              "attn_scored_fwd: null tensor");
  NMB_REQUIRE(nmb::aligned16(o_low), "scored attention (bf16): tensors must be 16-byte aligned");
  const nmb::FewPlan few = nmb::few_plan(batch, q_heads, kv_heads, seq_q, seq_k, head_dim, dtype);
  NMB_REQUIRE(workspace_bytes >= few.bytes && (few.bytes == 0 || workspace != nullptr) && nmb::aligned16(workspace),
              "attn_scored_fwd: a 16-byte aligned workspace of %zu bytes is needed, got %zu", few.bytes, workspace_bytes);
  if (few.use)
    return nmb::few_fwd_launch(p, static_cast<const nmb::bf16*>(q), static_cast<const nmb::bf16*>(k),
                               static_cast<const nmb::bf16*>(v), static_cast<nmb::bf16*>(o),
                               static_cast<nmb::bf16*>(o_low), lse2, static_cast<float*>(workspace), few, stream);
  if (dtype == NMB_BF16)
    return nmb::tiles_fwd_launch(p, static_cast<const nmb::bf16*>(q), static_cast<const nmb::bf16*>(k),
                                 static_cast<const nmb::bf16*>(v), static_cast<nmb::bf16*>(o), static_cast<nmb::bf16*>(o_low),
                                 lse2, stream);
  return nmb::scored_f32_fwd(p, static_cast<const float*>(q), static_cast<const float*>(k),
                             static_cast<const float*>(v), static_cast<float*>(o), lse2, stream);
}

extern "C" int nmb_attn_scored_bwd(const void* q, const void* k, const void* v, const void* o, const void* o_low,
                                   const void* dout,
                                   const float* lse2, void* dq, void* dk, void* dv, int64_t batch, int64_t q_heads,
                                   int64_t kv_heads, int64_t seq_q, int64_t seq_k, int64_t head_dim,
                                   const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                   const int64_t* o_strides, const int64_t* dkv_strides, const nmb_scores* scores,
                                   int dtype, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  ScoredShape p;
  NMB_REQUIRE(dkv_strides != nullptr, "attn_scored_bwd: null argument");
  const int st = nmb::fill_scored(&p, scores, batch, q_heads, kv_heads, seq_q, seq_k, head_dim, q_strides, k_strides,
                                  v_strides, o_strides, dkv_strides, q, k, v, o, dtype);
  if (st != NMB_OK) return st;
  if (batch == 0 || (seq_q == 0 && seq_k == 0)) return NMB_OK;
  NMB_REQUIRE(seq_q == 0 || (q != nullptr && o != nullptr && dout != nullptr && lse2 != nullptr && dq != nullptr),
              "attn_scored_bwd: null tensor");
  NMB_REQUIRE(seq_k == 0 || (k != nullptr && v != nullptr && dk != nullptr && dv != nullptr),
              "attn_scored_bwd: null tensor");
  const nmb::BwdSpace space = nmb::bwd_space(batch, q_heads, kv_heads, seq_q, seq_k, head_dim, dtype);
  NMB_REQUIRE(workspace_bytes >= space.total && (space.total == 0 || workspace != nullptr),
              "attn_scored_bwd: workspace of %zu bytes is smaller than the %zu required", workspace_bytes, space.total);
  NMB_REQUIRE(nmb::aligned16(workspace), "attn_scored_bwd: the workspace must be 16-byte aligned");
  float* ndelta = static_cast<float*>(workspace);
  if (dtype == NMB_BF16) {
    using nmb::bf16;
    for (const void* t : {o_low, dout, static_cast<const void*>(dq), static_cast<const void*>(dk), static_cast<const void*>(dv)})
      NMB_REQUIRE(nmb::aligned16(t), "scored attention (bf16): tensors must be 16-byte aligned");
    return nmb::tiles_bwd_launch(p, static_cast<const bf16*>(q), static_cast<const bf16*>(k),
                                 static_cast<const bf16*>(v), static_cast<const bf16*>(o),
                                 static_cast<const bf16*>(o_low), static_cast<const bf16*>(dout), lse2, static_cast<bf16*>(dq), static_cast<bf16*>(dk),
                                 static_cast<bf16*>(dv), static_cast<char*>(workspace), space, stream);
  }
  return nmb::scored_f32_bwd(p, static_cast<const float*>(q), static_cast<const float*>(k),
                             static_cast<const float*>(v), static_cast<const float*>(o),
                             static_cast<const float*>(dout), lse2, ndelta, static_cast<float*>(dq),
                             static_cast<float*>(dk), static_cast<float*>(dv), stream);
}
