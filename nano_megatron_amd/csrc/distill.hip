// The LM head's loss against the largest logits of a teacher, for gfx950: no counterpart in
// the reference (its head and loss: tensor_parallel/layers.py:207-214, cross_entropy.py:30-86).
//
//   s = x w^T;  p = softmax of a row's present teacher logits t / T;  q = softmax(s / T)
//   loss = T^2 sum_k p_k (log p_k - log q[id_k]) + c (log sum exp s - s_y)
//   dL/ds = grad (T [present] (q - p) + c [used] (softmax(s) - [y]))
//
// bf16, as head.hip: the exponential sums of both softmaxes are the epilogue of the product's
// tiles, in fp32 and with logits neither rounded nor written, and the backward forms the
// tiles again and writes only the gradient.  Both softmaxes share one running maximum, that of
// s, and everything is kept relative to it: the loss is a sum of differences.  Exponentials are
// 2^(s k - o) with whole numbers o, so one fma forms the exponent with one rounding, of the
// small difference, and sums are moved from one o to another exactly.
// The few logits that a row's teacher names (and its target's) are formed a second time, row by
// row, from the rows of w that they point to (distill_pick_kernel), in the product's own order
// of sums (for few rows in four shares of it), and kept in fp32: the epilogues so need no search
// for them, and the backward writes their gradients, rounded once, over what the product wrote
// (distill_entries_kernel).
// dL/ds is rounded to bf16 once, as the operand that it is of the two products behind it, dx =
// G w and dw = G^T x, on bf16 matrix instructions: a rounding of 1.7e-3 of its size (the root of
// the mean square over the values of a step of 2^-8), beside the results' own of as much, so dx
// and dw are 2.4e-3 off, 1.7e-3 with G in 32 bits.  As two bf16 terms it would keep 16 bits for twice
// the work of both products (1.1 of 2.5 ms at 8192 x 50304 x 768); fp32 tensors keep 32 throughout.
// fp32: row kernels over stored logits, then the same joining and writing over.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "gemm_core.h"
#include "head_plan.h"

namespace nmb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int64_t kMostEntries = 1024;

struct Teacher {
  const void* logits;
  const void* ids;
  int64_t ldt, ldi;
  const int64_t* targets;  // null: none
  int64_t ignore_index;
  int top;          // entries of a row
  bool wide, bf16;  // 8-byte ids, bf16 logits
  float temperature, scale_t, weight;  // scale_t: log2(e) / T
  int vocab;

  __device__ __forceinline__ int64_t id(int64_t row, int k) const {
    const int64_t at = row * ldi + k;
    return wide ? static_cast<const int64_t*>(ids)[at] : static_cast<const int32_t*>(ids)[at];
  }
  __device__ __forceinline__ float logit(int64_t row, int k) const {
    const int64_t at = row * ldt + k;
    return bf16 ? to_f32(static_cast<const nmb::bf16*>(logits)[at]) : static_cast<const float*>(logits)[at];
  }
  // -1 without targets.  Read where every lane passes: a load whose address is one for the
  // wavefront is scalar, and behind a condition of lanes is made for none of them too.
  __device__ __forceinline__ int64_t target(int64_t row) const { return targets != nullptr ? targets[row] : -1; }
  // entries with the target's, which is the last
  __device__ __host__ __forceinline__ int entries() const { return top + (targets != nullptr); }
};

struct DistillArgs {
  const bf16* x;
  const bf16* w;
  int64_t ldx, ldw;
  int rows, vocab, hidden;
  float scale_a, scale_b;  // log2(e) / T, log2(e)
  // forward
  float* tile_max;  // [tiles_n][rows], and the sums of both softmaxes
  float* tile_a;
  float* tile_b;
  // backward
  const float* stats;  // [4][stats_ld]: maximum, log2 of both sums, whether a teacher's entry is there
  int64_t stats_ld;
  const int64_t* targets;
  int64_t ignore_index;
  float temperature, weight;
  const float* grad;
  bf16* g;
  int64_t ldg;
  bool past_cache;
  int tiles_m, tiles_n, per_xcd;
  int first_n;  // the launch's first column of tiles
};

// The two factors of a row's gradient: grad T [present] and grad c [used].  A row with a bad id
// (some is NaN then) or target has NaN, as its loss does.
struct Factors {
  float a, b;
};
__device__ __forceinline__ Factors factors(float grad, float some, float temperature, float weight, int64_t target,
                                           int64_t ignore_index, int vocab) {
  // an absent part is 0 whatever the gradient holds
  const float b = target < 0 || target >= vocab ? __builtin_nanf("") : grad * weight;
  return Factors{some == 0.f ? 0.f : grad * temperature * some, target != ignore_index ? b : 0.f};
}

// The whole number at or above s k: sums of a row's exponentials are relative to that of its
// largest logit.
__device__ __forceinline__ float whole_above(float top, float k) {
  return top == -__builtin_inff() ? 0.f : ceilf(top * k);
}
// A sum relative to one maximum's, relative to a larger one's: a power of two.  (Without a
// maximum it is a sum of nothing.)
__device__ __forceinline__ float moved(float sum, float from, float to, float k) {
  const float by = from == -__builtin_inff() ? 0.f : whole_above(from, k) - whole_above(to, k);
  return sum * __builtin_amdgcn_exp2f(by);
}
// 2^(s k - (top k + l2)) = 2^(s k - whole) rest: what a row subtracts, without its rounding
struct Shift {
  float whole, rest;
};
__device__ __forceinline__ Shift shift_of(float top, float k, float l2) {
  const float t = top * k, low = fmaf(top, k, -t), whole = rintf(t + l2);
  return Shift{whole, __builtin_amdgcn_exp2f((whole - t) - l2 - low)};
}

// Minus infinity in the columns past the vocabulary.  One branch of the workgroup: as a
// condition of every element it would cost the other tiles a third of their epilogue.
template <int TM, int TN>
__device__ __forceinline__ void hide_columns(f32x4 (&acc)[TM][TN], int col0, int vocab) {
  asm volatile("");  // (or it becomes such a condition)
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][j][e] = col0 + 16 * j + e < vocab ? acc[i][j][e] : -__builtin_inff();
}

// One of the product's tiles: 4 tile rows at a time, the rows fastest, as in gemm.hip.
struct Tile {
  int m0, n, n0;
};
template <int TBM, int TBN>
__device__ __forceinline__ Tile tile_of(const DistillArgs& a, int item) {
  constexpr int GM = 4;
  const int grp = item / (GM * a.tiles_n);
  const int gsize = min(a.tiles_m - grp * GM, GM);
  const int r = item - grp * GM * a.tiles_n;
  const int n = a.first_n + r / gsize;
  return Tile{(grp * GM + r % gsize) * TBM, n, n * TBN};
}
// Its operands.
template <int TBM, int TBN, int NW, int BKT>
__device__ __forceinline__ void load_from(const DistillArgs& a, const Tile& t, Loader<TBM, true, BKT, NW>& la,
                                          Loader<TBN, true, BKT, NW>& lb, int wave, int lane) {
  const int va = min(TBM, a.rows - t.m0), vb = min(TBN, a.vocab - t.n0);
  la.init(a.x + static_cast<int64_t>(t.m0) * a.ldx, a.ldx, va, static_cast<uint32_t>(((va - 1) * a.ldx + a.hidden) * 2),
          wave, lane);
  lb.init(a.w + static_cast<int64_t>(t.n0) * a.ldw, a.ldw, vb, static_cast<uint32_t>(((vb - 1) * a.ldw + a.hidden) * 2),
          wave, lane);
}
template <int TBM, int TBN, int NW>
struct Waves {  // the shares of a tile's wavefronts, as head.hip's
  static constexpr int N = NW == 4 ? (TBN == 64 ? 1 : 2) : (TBN == 256 ? 4 : 2);
  static constexpr int M = NW / N, WM = TBM / M, WN = TBN / N, TM = WM / 16, TN = WN / 16;
};

// The exponential sums.  TWO: the softmaxes differ (T is not 1 and there are targets).
// A workgroup takes one tile after the other, and the next one's first K tiles are loaded under
// the epilogue of this one: every stage is free by then, and the sums have LDS of their own
// (8192 x 50304 x 768 with the entries' logits 708 -> 691 us with two softmaxes, 646 -> 634 with
// one).  What bounds it: the matrix unit is busy 50% of the time (in the plain products of dx and
// dw 53 and 58%), and the epilogue's exponentials take four times as long as other instructions:
// with the products these issue for 44% of it.
template <int TBM, int TBN, int NW, int BKT, bool TWO>
__device__ __forceinline__ void sums_of(const DistillArgs& a, int block, int blocks) {
  using W = Waves<TBM, TBN, NW>;
  constexpr int S = Stages<TBM, TBN, NW, BKT>::S;
  static_assert(BKT == 64, "all stages are filled ahead");
  __shared__ __attribute__((aligned(1024))) bf16 sA[S][TBM * BKT];
  __shared__ __attribute__((aligned(1024))) bf16 sB[S][TBN * BKT];
  __shared__ float red_max[W::N * TBM], red_a[W::N * TBM], red_b[TWO ? W::N * TBM : 1];

  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave / W::N) * W::WM, wn = (wave % W::N) * W::WN;
  const int l16 = lane & 15, q4 = lane >> 4;
  // the tiles of this XCD, and this workgroup's among them
  const int begin = (block % 8) * a.per_xcd;
  const int end = min(begin + a.per_xcd, a.tiles_m * a.tiles_n), step = blocks / 8;
  int item = begin + block / 8, loaded = 0;
  if (item >= end) return;
  Loader<TBM, true, BKT, NW> la;
  Loader<TBN, true, BKT, NW> lb;
  Tile tile = tile_of<TBM, TBN>(a, item);
  load_from(a, tile, la, lb, wave, lane);
  while (true) {
    f32x4 acc[W::TM][W::TN];
#pragma unroll
    for (int i = 0; i < W::TM; ++i)
#pragma unroll
      for (int j = 0; j < W::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    k_loop<TBM, TBN, NW, BKT, true, true, W::TM, W::TN>(la, lb, sA, sB, acc, wm, wn, 0, a.hidden, wave, lane, loaded);
    wait_tiles<0>();  // every wave is done with the operand stages
    const Tile now = tile;
    item += step;
    if (item < end) {
      tile = tile_of<TBM, TBN>(a, item);
      load_from(a, tile, la, lb, wave, lane);
      loaded = S;
      const int wave_u = __builtin_amdgcn_readfirstlane(wave);
      const uint32_t a_lds = lds_offset(&sA[0][0]) + 1024u * wave_u * Loader<TBM, true, BKT, NW>::kPer;
      const uint32_t b_lds = lds_offset(&sB[0][0]) + 1024u * wave_u * Loader<TBN, true, BKT, NW>::kPer;
#pragma unroll
      for (int p = 0; p < S; ++p)
        if (p * BKT < a.hidden) {
          la.issue_s(a_lds + LinearStages<TBM, TBN, BKT>::a(p), p * BKT, a.hidden);
          lb.issue_s(b_lds + LinearStages<TBM, TBN, BKT>::b(p), p * BKT, a.hidden);
        }
    }

    // acc[i][j][e] = s[m0 + wm + 16 i + l16][n0 + wn + 16 j + 4 q4 + e]
    if (now.n0 + TBN > a.vocab) hide_columns<W::TM, W::TN>(acc, now.n0 + wn + 4 * q4, a.vocab);
#pragma unroll
    for (int i = 0; i < W::TM; ++i) {
      const int lr = wm + 16 * i + l16;
      float top = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < W::TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, acc[i][j][e]);
      top = xor32_max(xor16_max(top));
      const float oa = whole_above(top, a.scale_a), ob = TWO ? whole_above(top, a.scale_b) : 0.f;
      float sa = 0.f, sb = 0.f;
#pragma unroll
      for (int j = 0; j < W::TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sa += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.scale_a, -oa));
          if constexpr (TWO) sb += __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.scale_b, -ob));
        }
      sa = xor32_sum(xor16_sum(sa));
      if constexpr (TWO) sb = xor32_sum(xor16_sum(sb));
      if (q4 == 0) {
        const int at = (wave % W::N) * TBM + lr;
        red_max[at] = top;
        red_a[at] = sa;
        if constexpr (TWO) red_b[at] = sb;
      }
    }
    // (not __syncthreads, which may wait for the loads)
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int lr = static_cast<int>(threadIdx.x), m = now.m0 + lr;
    if (lr < TBM && m < a.rows) {
      float top = -__builtin_inff(), sa = 0.f, sb = 0.f;
#pragma unroll
      for (int w = 0; w < W::N; ++w) top = fmaxf(top, red_max[w * TBM + lr]);
#pragma unroll
      for (int w = 0; w < W::N; ++w) {
        const float most = red_max[w * TBM + lr];
        sa += moved(red_a[w * TBM + lr], most, top, a.scale_a);
        if constexpr (TWO) sb += moved(red_b[w * TBM + lr], most, top, a.scale_b);
      }
      const int64_t at = static_cast<int64_t>(now.n) * a.rows + m;
      a.tile_max[at] = top;
      a.tile_a[at] = sa;
      if constexpr (TWO) a.tile_b[at] = sb;
    }
    if (item >= end) break;
    wait_vmcnt<0>();  // k_loop counts its own loads alone
  }
}
template <int TBM, int TBN, int NW, int BKT, bool TWO>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void distill_sums_kernel(DistillArgs a) {
  sums_of<TBM, TBN, NW, BKT, TWO>(a, static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
}

// The gradient.  Two workgroups a CU overlap one's epilogue with the other's products; what
// bounds it is those (matrix unit 40%) and the 824 MB that it writes past the cache (8192 x 50304 x
// 768 with the entries' part 782 us with two softmaxes, 758 with one).
template <int TBM, int TBN, int NW, int BKT, bool TWO>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void distill_grad_kernel(DistillArgs a) {
  using W = Waves<TBM, TBN, NW>;
  constexpr int S = Stages<TBM, TBN, NW, BKT>::S;
  __shared__ __attribute__((aligned(1024))) bf16 sA[S][TBM * BKT];
  __shared__ __attribute__((aligned(1024))) bf16 sB[S][TBN * BKT];
  const int L = static_cast<int>(blockIdx.x);
  const int item = (L % 8) * a.per_xcd + L / 8;
  if (item >= a.tiles_m * a.tiles_n) return;
  const Tile tile = tile_of<TBM, TBN>(a, item);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave / W::N) * W::WM, wn = (wave % W::N) * W::WN;
  const int l16 = lane & 15, q4 = lane >> 4;
  Loader<TBM, true, BKT, NW> la;
  Loader<TBN, true, BKT, NW> lb;
  load_from(a, tile, la, lb, wave, lane);
  f32x4 acc[W::TM][W::TN];
#pragma unroll
  for (int i = 0; i < W::TM; ++i)
#pragma unroll
    for (int j = 0; j < W::TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  k_loop<TBM, TBN, NW, BKT, true, true, W::TM, W::TN>(la, lb, sA, sB, acc, wm, wn, 0, a.hidden, wave, lane);

  constexpr int RPA = (S * TBM * BKT) / TBN;  // tile rows that fit in sA, the rest in sB
  static_assert(RPA + S * BKT >= TBM, "the bf16 tile fits in the operand stages");
  auto tile_at = [&](int row, int c) -> bf16* {  // element (row, c), c a multiple of 4
    bf16* rp = row < RPA ? &sA[0][0] + row * TBN : &sB[0][0] + (row - RPA) * TBN;
    return rp + 8 * ((c >> 3) ^ (row & (TBN == 64 ? 7 : 15))) + (c & 4);
  };
  __syncthreads();  // every wave is done with the operand stages
  // past the vocabulary the gradient is 0
  if (tile.n0 + TBN > a.vocab) hide_columns<W::TM, W::TN>(acc, tile.n0 + wn + 4 * q4, a.vocab);
#pragma unroll
  for (int i = 0; i < W::TM; ++i) {
    const int lr = wm + 16 * i + l16, m = min(tile.m0 + lr, a.rows - 1);
    const float top = a.stats[m], la2 = a.stats[a.stats_ld + m], some = a.stats[3 * a.stats_ld + m];
    const float lb2 = TWO ? a.stats[2 * a.stats_ld + m] : 0.f;
    const int64_t target = a.targets != nullptr ? a.targets[m] : a.ignore_index;
    const Factors f = factors(a.grad[m], some, a.temperature, a.weight, target, a.ignore_index, a.vocab);
    const Shift sa = shift_of(top, a.scale_a, la2), sb = TWO ? shift_of(top, a.scale_b, lb2) : Shift{0.f, 0.f};
    const float fa = (TWO ? f.a : f.a + f.b) * sa.rest, fb = f.b * sb.rest;
    const uint32_t used = f.a == 0.f && f.b == 0.f ? 0u : ~0u;  // rows without any part may hold anything
#pragma unroll
    for (int j = 0; j < W::TN; ++j) {
      bf16x4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float g = fa * __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.scale_a, -sa.whole));
        if constexpr (TWO) g = fmaf(fb, __builtin_amdgcn_exp2f(fmaf(acc[i][j][e], a.scale_b, -sb.whole)), g);
        out[e] = static_cast<bf16>(g);
      }
      uint2 bits;
      __builtin_memcpy(&bits, &out, 8);
      *reinterpret_cast<uint2*>(tile_at(lr, wn + 16 * j + 4 * q4)) = uint2{bits.x & used, bits.y & used};
    }
  }
  __syncthreads();
  constexpr int LPR = TBN / 8, RPI = 64 / LPR, ROWS_PER_WAVE = TBM / NW;
  static_assert(ROWS_PER_WAVE % RPI == 0, "whole store instructions per wave");
  const int sl = lane % LPR;
#pragma unroll
  for (int it = 0; it < ROWS_PER_WAVE / RPI; ++it) {
    const int row = wave * ROWS_PER_WAVE + it * RPI + lane / LPR;
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(tile_at(row, 8 * sl));
    const int m = tile.m0 + row, n = tile.n0 + 8 * sl;
    if (m >= a.rows || n >= a.vocab) continue;
    bf16x8* out = reinterpret_cast<bf16x8*>(a.g + m * a.ldg + n);
    if (a.past_cache) {  // as in head.hip
      __builtin_nontemporal_store(v, out);
      asm volatile("");
    } else {
      *out = v;
    }
  }
}

// The logits of a row's entries: 32 of them a wavefront, whose rows of w are the first operand
// of the matrix instruction and x's row, in every column, the second.  What bounds it: the rows
// of w, 648 of 805 MB past the L2 caches (8192 x 768 with 65 entries, 110 us).  SPLIT, up to a
// wavefront's worth a SIMD: a workgroup's four wavefronts share out the hidden size instead, and
// add up in LDS (the whole forward, hidden 768, vocabulary 8,192, 20 entries, without and with
// it, us: 96 rows 18.1 and 15.0, 300 24.3 and 22.2, 700 27.6 and 27.2, 1,000 28.5 and 29.3).
constexpr int64_t kFewItems = 1024;
template <bool SPLIT>
__device__ __forceinline__ void pick(const DistillArgs& a, const Teacher& t, float* __restrict__ picked, int passes,
                                     int64_t block) {
  __shared__ float s_part[SPLIT ? 4 : 1][2][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = SPLIT ? block : block * 4 + wave;
  const int64_t row = item / passes;
  if (row >= a.rows) return;  // (SPLIT: never)
  const int first = static_cast<int>(item - row * passes) * 32;
  const int lane = threadIdx.x & 63, l16 = lane & 15, q4 = lane >> 4;
  const int entries = t.entries();
  const int64_t target = t.target(row);
  const bf16* wr[2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int k = first + 16 * n + l16;
    int64_t id = -1;
    if (k < t.top) id = t.id(row, k);
    else if (k < entries) id = target;
    wr[n] = a.w + (id >= 0 && id < a.vocab ? id : 0) * a.ldw;  // absent: any row, its value unused
  }
  const bf16* xr = a.x + row * a.ldx;
  const int steps = (a.hidden + 31) / 32, share = SPLIT ? (steps + 3) / 4 : steps;
  const int k_begin = SPLIT ? wave * share * 32 : 0, k_end = min(a.hidden, k_begin + share * 32);
  f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
  // N groups of 16: eight steps' loads are under way at a time
  auto products = [&](auto groups) {
    constexpr int N = decltype(groups)::value, U = 8;
    for (int k0 = k_begin; k0 < k_end; k0 += 32 * U) {
      bf16x8 xv[U], wv[N][U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // a lane's eight lie inside its range or past it: then the row's last, times zero
        const int k = k0 + 32 * u + 8 * q4, at = min(k, a.hidden - 8);
#pragma unroll
        for (int n = 0; n < N; ++n) wv[n][u] = ld8(wr[n] + at);
        const bf16x8 x = ld8(xr + at);
        xv[u] = k < k_end ? x : bf16x8{};
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[n] = mfma16(wv[n][u], xv[u], acc[n]);
    }
  };
  if (first + 16 < entries) products(std::integral_constant<int, 2>{});
  else products(std::integral_constant<int, 1>{});
  // acc[n][e]: entry 16 n + 4 q4 + e, in every column
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float v = l16 == 0 ? acc[n][0] : l16 == 1 ? acc[n][1] : l16 == 2 ? acc[n][2] : acc[n][3];
    const int k = first + 16 * n + 4 * q4 + l16;
    if constexpr (SPLIT) {
      s_part[wave][n][lane] = v;
      __syncthreads();
      v = (s_part[0][n][lane] + s_part[1][n][lane]) + (s_part[2][n][lane] + s_part[3][n][lane]);
      if (wave != n) continue;
    }
    if (l16 < 4 && k < entries) picked[row * entries + k] = v;
  }
}
template <bool SPLIT>
__global__ __launch_bounds__(256) void distill_pick_kernel(DistillArgs a, Teacher t, float* __restrict__ picked,
                                                           int passes) {
  pick<SPLIT>(a, t, picked, passes, blockIdx.x);
}

// Both in one launch, for 64 x 64 tiles and few items, where two launches' starts and ends are a
// good part of the time: the first sums_blocks workgroups take tiles, the others an item of the
// entries' logits each (the whole forward, us, two launches and one: 96 x 8192 x 768 with 20
// entries 15.4 and 12.2, 300 rows 23.0 and 18.4, 512 25.2 and 23.9; 64 x 50304 x 768 with 64
// entries 35.6 and 30.5; items first are within 3% either way).
template <bool TWO>
__global__ __launch_bounds__(256, 2) void distill_few_kernel(DistillArgs a, Teacher t, float* __restrict__ picked,
                                                             int passes, int sums_blocks) {
  const int block = static_cast<int>(blockIdx.x);
  if (block < sums_blocks) sums_of<64, 64, 4, 64, TWO>(a, block, sums_blocks);
  else pick<true>(a, t, picked, passes, block - sums_blocks);
}

// A row's teacher, read by LANES lanes, PER entries of each at a time.
__device__ __forceinline__ bool present(const Teacher& t, int64_t row, int k, float& v, int64_t& id) {
  id = -1;
  v = -__builtin_inff();
  if (k >= t.top) return false;
  id = t.id(row, k);
  v = t.logit(row, k);  // (of an absent entry too: both loads are under way at once)
  return id >= 0 && v != -__builtin_inff();
}

template <int LANES, int PER>
struct Entries {
  float v[PER];
  int64_t id[PER];
  bool there[PER];

  __device__ __forceinline__ void load(const Teacher& t, int64_t row, int k0, int lane) {
#pragma unroll
    for (int j = 0; j < PER; ++j) there[j] = present(t, row, k0 + lane + LANES * j, v[j], id[j]);
  }
};

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  if constexpr (LANES == 64) return wave_sum(v);
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  return v + dpp<0x140>(v);
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  if constexpr (LANES == 64) return wave_max(v);
  v = fmaxf(v, dpp<0xB1>(v));
  v = fmaxf(v, dpp<0x4E>(v));
  v = fmaxf(v, dpp<0x141>(v));
  return fmaxf(v, dpp<0x140>(v));
}

// The maximum of a row's present logits and the sum of their exponentials at T; use(entry, e)
// is called for each with its exponential.  The first LANES * PER entries are read once.
struct Soft {
  float top, sum;
  bool bad;  // an id past the vocabulary, a logit that is not a number
};
template <int LANES, int PER, class Use>
__device__ __forceinline__ Soft soft_of(const Teacher& t, int64_t row, int lane, const Use& use) {
  static_assert(LANES == 16 || LANES == 64, "a row of DPP lanes or a wavefront");
  Entries<LANES, PER> first;
  first.load(t, row, 0, lane);
  Soft s{-__builtin_inff(), 0.f, false};
  float bad = 0.f;
  auto look = [&](const Entries<LANES, PER>& e) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (e.there[j]) {
        s.top = fmaxf(s.top, e.v[j]);
        if (e.id[j] >= t.vocab || !(e.v[j] < __builtin_inff())) bad = 1.f;
      }
  };
  look(first);
  for (int k0 = LANES * PER; k0 < t.top; k0 += LANES * PER) {
    Entries<LANES, PER> e;
    e.load(t, row, k0, lane);
    look(e);
  }
  s.top = lanes_max<LANES>(s.top);
  s.bad = lanes_max<LANES>(bad) != 0.f;
  auto add = [&](const Entries<LANES, PER>& e, int k0) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (k0 + lane + LANES * j < t.top) {
        const float x = e.there[j] ? __builtin_amdgcn_exp2f((e.v[j] - s.top) * t.scale_t) : 0.f;
        s.sum += x;
        use(k0 + lane + LANES * j, e.there[j], e.id[j], e.v[j] - s.top, x);
      }
  };
  add(first, 0);
  for (int k0 = LANES * PER; k0 < t.top; k0 += LANES * PER) {
    Entries<LANES, PER> e;
    e.load(t, row, k0, lane);
    add(e, k0);
  }
  s.sum = lanes_sum<LANES>(s.sum);
  return s;
}

// Joins the tiles of 16 rows a workgroup, in an order that depends on their number alone, and
// forms the rows' losses, 16 lanes a row.  two: tile_b holds sums of its own.
__global__ __launch_bounds__(256) void distill_merge_kernel(const float* __restrict__ tile_max,
                                                            const float* __restrict__ tile_a,
                                                            const float* __restrict__ tile_b, int tiles, int64_t rows,
                                                            bool two, Teacher t, const float* __restrict__ picked,
                                                            float* __restrict__ loss, float* __restrict__ stats,
                                                            int64_t stats_ld) {
  __shared__ float s_max[16][17], s_a[16][17], s_b[16][17], s_top[16], s_la[16], s_lb[16];
  {
    const int n = threadIdx.x & 15, part = threadIdx.x >> 4;  // row, share of its tiles
    const int64_t m = min(static_cast<int64_t>(blockIdx.x) * 16 + n, rows - 1);
    float top = -__builtin_inff(), sa = 0.f, sb = 0.f;
    constexpr int PER = 8;  // tiles' loads under way at a time
    for (int k0 = part; k0 < tiles; k0 += 16 * PER) {
      float tm[PER], ta[PER], tb[PER], most = top;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int64_t at = min(k0 + 16 * j, tiles - 1) * rows + m;
        tm[j] = tile_max[at];
        ta[j] = tile_a[at];
        tb[j] = two ? tile_b[at] : 0.f;
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) most = fmaxf(most, tm[j]);
      sa = moved(sa, top, most, t.scale_t);
      sb = moved(sb, top, most, kLog2e);
      top = most;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (k0 + 16 * j < tiles) {
          sa += moved(ta[j], tm[j], top, t.scale_t);
          sb += moved(tb[j], tm[j], top, kLog2e);
        }
    }
    s_max[part][n] = top;
    s_a[part][n] = sa;
    s_b[part][n] = sb;
    __syncthreads();
    if (part == 0) {
#pragma unroll
      for (int k = 0; k < 16; ++k) top = fmaxf(top, s_max[k][n]);
      sa = sb = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        sa += moved(s_a[k][n], s_max[k][n], top, t.scale_t);  // (of a share without tiles: 0)
        sb += moved(s_b[k][n], s_max[k][n], top, kLog2e);
      }
      s_top[n] = top;
      s_la[n] = log2f(sa) + fmaf(-top, t.scale_t, whole_above(top, t.scale_t));
      s_lb[n] = two ? log2f(sb) + fmaf(-top, kLog2e, whole_above(top, kLog2e)) : s_la[n];
    }
    __syncthreads();
  }
  const int rl = threadIdx.x >> 4, lane = threadIdx.x & 15;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 16 + rl, row = min(at, rows - 1);
  const int entries = t.entries();
  const float high = s_top[rl], la2 = s_la[rl], lb2 = s_lb[rl];
  float dot = 0.f;  // sum e ((t - max t) - (s - max s))
  const Soft s = soft_of<16, 4>(t, row, lane, [&](int k, bool there, int64_t, float d, float e) {
    const float z = picked[row * entries + k];
    if (there) dot = fmaf(e, d - (z - high), dot);
  });
  dot = lanes_sum<16>(dot);
  const bool some = s.sum != 0.f || s.bad;  // a present logit that is not a number too
  float value = 0.f, flag = some ? 1.f : 0.f;
  if (some) value = t.temperature * t.temperature * (dot / (s.sum * t.temperature) + kLn2 * (la2 - log2f(s.sum)));
  if (s.bad) value = flag = __builtin_nanf("");  // poisons its row; the host checks ids
  if (t.targets != nullptr) {
    const int64_t y = t.targets[row];
    const float ce = fmaf(kLn2, lb2, high - picked[row * entries + t.top]);
    if (y != t.ignore_index) value = y < 0 || y >= t.vocab ? __builtin_nanf("") : fmaf(t.weight, ce, value);
  }
  if (lane == 0 && at < rows) {
    loss[row] = value;
    stats[row] = high;
    stats[stats_ld + row] = la2;
    stats[2 * stats_ld + row] = lb2;
    stats[3 * stats_ld + row] = flag;
  }
}

// The gradients of a row's entries, over what lies there.  Entries of one token are one: the
// first writes, with the sum of their probabilities; the target's, where it is none of them.
// kept (nullable, dense): x with zeros in rows without any part, which may hold anything, for the
// table's gradient G^T x.
constexpr int padded4(int n) { return (n + 3) / 4 * 4; }
template <typename T>
__global__ __launch_bounds__(256) void distill_entries_kernel(Teacher t, int64_t rows, const float* __restrict__ stats,
                                                              int64_t stats_ld, const float* __restrict__ picked,
                                                              const float* __restrict__ grad, T* __restrict__ g,
                                                              int64_t ldg, const T* __restrict__ x, int64_t ldx,
                                                              int hidden, T* __restrict__ kept) {
  extern __shared__ __attribute__((aligned(16))) int s_entries[];  // [4][padded] ids, then exponentials
  typedef int int4_ __attribute__((ext_vector_type(4)));
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + wave;
  const int padded = padded4(t.top);
  int* ids = s_entries + wave * padded;
  float* es = reinterpret_cast<float*>(s_entries + 4 * padded) + wave * padded;
  if (row >= rows) return;  // (no barrier: a wavefront reads only what it wrote)
  const int entries = t.entries();
  const float high = stats[row], la2 = stats[stats_ld + row], lb2 = stats[2 * stats_ld + row];
  const float some = stats[3 * stats_ld + row], gr = grad[row];
  const int64_t y = t.targets != nullptr ? t.targets[row] : t.ignore_index;
  const int target = y != t.ignore_index && y >= 0 && y < t.vocab ? static_cast<int>(y) : -1;
  if (lane < padded - t.top) {
    ids[t.top + lane] = -1;
    es[t.top + lane] = 0.f;
  }
  const Soft s = soft_of<64, 1>(t, row, lane, [&](int k, bool there, int64_t id, float, float e) {
    ids[k] = there && id < t.vocab ? static_cast<int>(id) : -1;
    es[k] = e;
  });
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const Factors f = factors(gr, some, t.temperature, t.weight, y, t.ignore_index, t.vocab);
  const bool zeros = f.a == 0.f && f.b == 0.f;  // the row's gradient
  if (kept != nullptr) {
    constexpr int V = sizeof(T) == 2 ? 8 : 1;  // bf16: rows of whole, aligned 16 bytes
    typedef T vec __attribute__((ext_vector_type(V)));
    for (int c = V * lane; c < hidden; c += 64 * V) {
      vec v = *reinterpret_cast<const vec*>(x + row * ldx + c);
      if (zeros) v = vec(T(0));
      *reinterpret_cast<vec*>(kept + row * hidden + c) = v;
    }
  }
  if (zeros) return;
  auto write = [&](int at, float z, float p) {
    const float d = z - high;
    float v = f.a * (__builtin_amdgcn_exp2f(fmaf(d, t.scale_t, -la2)) - p);
    v = fmaf(f.b, __builtin_amdgcn_exp2f(fmaf(d, kLog2e, -lb2)) - (at == target ? 1.f : 0.f), v);
    g[row * ldg + at] = from_f32<T>(v);
  };
  bool found = false;
  for (int k = lane; k < t.top; k += 64) {
    const int at = ids[k];
    if (at < 0) continue;
    const float z = picked[row * entries + k];
    found = found || at == target;
    float e = 0.f;
    int first = k;
    for (int j = 0; j < padded; j += 4) {
      const int4_ id4 = *reinterpret_cast<const int4_*>(ids + j);
      const f32x4 e4 = *reinterpret_cast<const f32x4*>(es + j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool same = id4[i] == at;
        e += same ? e4[i] : 0.f;
        first = same ? min(first, j + i) : first;
      }
    }
    if (first == k) write(at, z, e / s.sum);
  }
  if (target >= 0 && !__any(found) && lane == 0) write(target, picked[row * entries + t.top], 0.f);
}

// ------------------------------------------------------------ fp32, by rows
// One workgroup per row: wide ones, whose threads have all their columns under way at once
// (512 x 8192, us with 256 threads and 1,024: forward 9.6 and 9.0, backward 10.2 and 9.1), and
// powers of two with the offsets of the bf16 head (forward 6.5, backward 7.6: 2.6 TB/s of the
// logits read, 4.4 of them read and written; short kernels of which a few us are their start).
constexpr int kRowThreads = 1024;
__device__ __forceinline__ float block_reduce(float v, float* sh, bool max) {
  v = max ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float all = sh[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) all = max ? fmaxf(all, sh[w]) : all + sh[w];
  return all;
}

// A row's maximum and sums, as one tile, and its entries' logits.  Eight columns of a thread at
// a time, as in head.hip.
constexpr int kRowCols = 8;
__global__ __launch_bounds__(kRowThreads) void distill_rows_fwd_kernel(
    const float* __restrict__ s, int64_t ld, int64_t rows, Teacher t, bool two, float* __restrict__ tile_max,
    float* __restrict__ tile_a, float* __restrict__ tile_b, float* __restrict__ picked) {
  __shared__ float sh[kRowThreads / 64];
  const int64_t row = blockIdx.x;
  const float* r = s + row * ld;
  const int entries = t.entries();
  const int64_t target = t.target(row);
  for (int k = threadIdx.x; k < entries; k += kRowThreads) {
    const int64_t id = k < t.top ? t.id(row, k) : target;
    picked[row * entries + k] = id >= 0 && id < t.vocab ? r[id] : 0.f;
  }
  float top = -__builtin_inff(), sa = 0.f, sb = 0.f;
  for (int64_t c0 = threadIdx.x; c0 < t.vocab; c0 += kRowThreads * kRowCols) {
    float y[kRowCols], most = top;
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      y[e] = c0 + kRowThreads * e < t.vocab ? r[c0 + kRowThreads * e] : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) most = fmaxf(most, y[e]);
    sa = moved(sa, top, most, t.scale_t);
    if (two) sb = moved(sb, top, most, kLog2e);
    top = most;
    const float oa = whole_above(top, t.scale_t), ob = whole_above(top, kLog2e);
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      sa += __builtin_amdgcn_exp2f(fmaf(y[e], t.scale_t, -oa));
      if (two) sb += __builtin_amdgcn_exp2f(fmaf(y[e], kLog2e, -ob));
    }
  }
  const float all = block_reduce(top, sh, true);
  sa = block_reduce(moved(sa, top, all, t.scale_t), sh, false);
  if (two) sb = block_reduce(moved(sb, top, all, kLog2e), sh, false);
  if (threadIdx.x != 0) return;
  tile_max[row] = all;
  tile_a[row] = sa;
  tile_b[row] = sb;
}

__global__ __launch_bounds__(kRowThreads) void distill_rows_bwd_kernel(
    float* __restrict__ s, int64_t ld, Teacher t, bool two, const float* __restrict__ stats, int64_t stats_ld,
    const float* __restrict__ grad) {
  const int64_t row = blockIdx.x;
  float* r = s + row * ld;
  const float top = stats[row];
  const Shift sa = shift_of(top, t.scale_t, stats[stats_ld + row]);
  const Shift sb = shift_of(top, kLog2e, stats[2 * stats_ld + row]);
  const int64_t target = t.targets != nullptr ? t.targets[row] : t.ignore_index;
  const Factors f = factors(grad[row], stats[3 * stats_ld + row], t.temperature, t.weight, target, t.ignore_index, t.vocab);
  const float fa = (two ? f.a : f.a + f.b) * sa.rest, fb = f.b * sb.rest;
  const bool any = !(f.a == 0.f && f.b == 0.f);
  for (int64_t c0 = threadIdx.x; c0 < t.vocab; c0 += kRowThreads * kRowCols) {
    float y[kRowCols];
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) y[e] = c0 + kRowThreads * e < t.vocab ? r[c0 + kRowThreads * e] : 0.f;
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      float g = fa * __builtin_amdgcn_exp2f(fmaf(y[e], t.scale_t, -sa.whole));
      if (two) g = fmaf(fb, __builtin_amdgcn_exp2f(fmaf(y[e], kLog2e, -sb.whole)), g);
      if (c0 + kRowThreads * e < t.vocab) r[c0 + kRowThreads * e] = any ? g : 0.f;
    }
  }
}

// ------------------------------------------------------------ sum and mean of the losses
// In 64 bits and one order.  (A library's sum of so many values may clear a semaphore in memory
// first, which a captured step does not take, and with the count it is eight launches: a step of
// 96 rows with its gradients 164 us, 102 with this.)  One workgroup for few rows (8,192 in 2.3
// us); for more, which it would take longer (70,000 17 us, a million 200), workgroups of
// kTotalRows rows or more write their sums and a second launch adds them up (a step of 70,000
// rows 233 -> 223 us, of a million 2,296 -> 2,110).
constexpr int kTotalRows = 8192, kTotalBlocks = 256;
struct Counted {
  double sum;
  int64_t count;
};
__device__ __forceinline__ Counted block_total(Counted v) {  // in thread 0
  __shared__ Counted s_part[16];
#pragma unroll
  for (int by = 32; by >= 1; by /= 2) {
    v.sum += __shfl_xor(v.sum, by);
    v.count += __shfl_xor(v.count, by);
  }
  if ((threadIdx.x & 63) == 0) s_part[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x != 0) return v;
  v = Counted{0., 0};
  for (int w = 0; w < static_cast<int>(blockDim.x >> 6); ++w) {
    v.sum += s_part[w].sum;
    v.count += s_part[w].count;
  }
  return v;
}
__device__ __forceinline__ void write_total(const Counted& v, bool mean, float* total, float* over) {
  const double by = mean && v.count > 0 ? static_cast<double>(v.count) : 1.;
  *total = static_cast<float>(v.sum / by);
  *over = static_cast<float>(by);
}

// parts: null for one workgroup, which writes the result
__global__ __launch_bounds__(1024) void distill_total_kernel(const float* __restrict__ loss,
                                                             const float* __restrict__ flags,
                                                             const int64_t* __restrict__ targets, int64_t ignore_index,
                                                             int64_t rows, bool mean, Counted* __restrict__ parts,
                                                             float* __restrict__ total, float* __restrict__ over) {
  constexpr int PER = 8;
  Counted t{0., 0};
  const int64_t step = static_cast<int64_t>(gridDim.x) * 1024;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * 1024 + threadIdx.x; r0 < rows; r0 += step * PER) {
    float v[PER], flag[PER];
    int64_t y[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int64_t r = min(r0 + step * j, rows - 1);
      v[j] = loss[r];
      flag[j] = flags[r];
      y[j] = ignore_index;
      if (targets != nullptr) y[j] = targets[r];
    }
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (r0 + step * j < rows) {
        t.sum += v[j];
        t.count += flag[j] != 0.f || y[j] != ignore_index;  // (a flag that is not a number counts)
      }
  }
  t = block_total(t);
  if (threadIdx.x != 0) return;
  if (parts != nullptr) parts[blockIdx.x] = t;
  else write_total(t, mean, total, over);
}

__global__ __launch_bounds__(kTotalBlocks) void distill_join_kernel(const Counted* __restrict__ parts, int n, bool mean,
                                                                    float* __restrict__ total,
                                                                    float* __restrict__ over) {
  Counted t{0., 0};
  if (static_cast<int>(threadIdx.x) < n) t = parts[threadIdx.x];
  t = block_total(t);
  if (threadIdx.x == 0) write_total(t, mean, total, over);
}

// ------------------------------------------------------------ host side
// Threads of a launch number fewer than 2^32: 64 a row and pass over its entries, or kRowThreads.
constexpr int64_t kMostWaves = int64_t{1} << 26, kMostRows = (int64_t{1} << 32) / kRowThreads;

int check_teacher(const nmb_teacher* t, int64_t rows, int64_t vocab) {
  NMB_REQUIRE(t != nullptr && (rows == 0 || (t->logits != nullptr && t->ids != nullptr)), "distill: null argument");
  NMB_REQUIRE(rows >= 0 && vocab > 0 && rows < (1 << 30) && vocab < (1 << 30), "distill: invalid shape");
  NMB_REQUIRE_SUPPORTED(t->top >= 1 && t->top <= kMostEntries, "distill: 1 to %lld teacher logits a row, got %lld",
                        (long long)kMostEntries, (long long)t->top);
  NMB_REQUIRE(t->ld >= 0 && t->ldi >= 0 && (t->id_bytes == 4 || t->id_bytes == 8) &&
                  (t->logits_dtype == NMB_F32 || t->logits_dtype == NMB_BF16),
              "distill: ids must be of 4 or 8 bytes, logits fp32 or bf16, strides not negative");
  NMB_REQUIRE(t->temperature >= 1e-2f && t->temperature <= 1e2f, "distill: the temperature must lie within 0.01 and 100");
  NMB_REQUIRE(isfinite(t->target_weight) && t->target_weight >= 0.f, "distill: the target's weight must be finite and >= 0");
  return NMB_OK;
}

int check_head(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t hidden) {
  NMB_REQUIRE(x != nullptr && w != nullptr, "distill: null argument");
  NMB_REQUIRE(hidden > 0 && hidden < (1 << 30) && ldx >= hidden && ldw >= hidden, "distill: invalid hidden size or leading dimension");
  NMB_REQUIRE_SUPPORTED(hidden % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0,
                        "distill: hidden and the leading dimensions must be multiples of 8");
  NMB_REQUIRE(aligned16(x) && aligned16(w), "distill: operands must be 16-byte aligned");
  NMB_REQUIRE_SUPPORTED(256 * ldx < (int64_t{1} << 30) && 256 * ldw < (int64_t{1} << 30),
                        "distill: an operand tile spans more than 2 GiB");
  return NMB_OK;
}

Teacher make_teacher(const nmb_teacher* t, int64_t vocab) {
  Teacher r{};
  r.logits = t->logits;
  r.ids = t->ids;
  r.ldt = t->ld;
  r.ldi = t->ldi;
  r.targets = t->targets;
  r.ignore_index = t->ignore_index;
  r.top = static_cast<int>(t->top);
  r.wide = t->id_bytes == 8;
  r.bf16 = t->logits_dtype == NMB_BF16;
  r.temperature = t->temperature;
  r.scale_t = static_cast<float>(1.4426950408889634074 / t->temperature);
  r.weight = t->target_weight;
  r.vocab = static_cast<int>(vocab);
  return r;
}

bool two_softmaxes(const nmb_teacher* t) { return t->targets != nullptr && t->temperature != 1.f; }

DistillArgs make_args(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab, int64_t hidden,
                      const Teacher& t) {
  DistillArgs a{};
  a.x = static_cast<const bf16*>(x);
  a.w = static_cast<const bf16*>(w);
  a.ldx = ldx;
  a.ldw = ldw;
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.hidden = static_cast<int>(hidden);
  a.scale_a = t.scale_t;
  a.scale_b = kLog2e;
  a.targets = t.targets;
  a.ignore_index = t.ignore_index;
  a.temperature = t.temperature;
  a.weight = t.weight;
  return a;
}

// Columns of the forward's 256 x 256 tiles that are better taken as 128 x 256 ones, in a launch of
// their own: those of the last round over the CUs, where the smaller tiles fit one round, which
// takes little more than half as long (the whole forward, us: 300 x 50304 x 768 60 -> 53, 709 x
// 50257 x 1024 102 -> 97, 900 x 50304 x 768 106 -> 101, 2048 x 50304 x 768 201 -> 196).  The
// gradient's 256 x 128 tiles, two a CU, lose less in theirs (the same, 59 -> 56, 95 -> 100, 103 ->
// 107, 196 -> 202).
int rest_columns(const DistillArgs& a) {
  const int64_t items = static_cast<int64_t>(a.tiles_m) * a.tiles_n, whole = items / 256 * 256;
  if (whole == 0 || whole == items) return 0;
  const int64_t rest = a.tiles_n - whole / a.tiles_m;
  return (a.rows + 127) / 128 * rest <= 256 ? static_cast<int>(rest) : 0;
}

// The entries' logits that a launch of 64 x 64 tiles forms beside its sums.
struct Picks {
  Teacher t;
  float* picked;
  int passes;
  unsigned items;
};

template <bool BACK, bool TWO>
int distill_launch(DistillArgs a, hipStream_t stream, const Picks* picks = nullptr) {
  const HeadPlan p = head_plan(a.rows, a.vocab, BACK);
  a.tiles_m = (a.rows + p.tbm - 1) / p.tbm;
  a.tiles_n = (a.vocab + p.tbn - 1) / p.tbn;
  const int rest = !BACK && p.tbm == 256 ? rest_columns(a) : 0;
  if (rest > 0) {
    a.tiles_n -= rest;
    DistillArgs b = a;
    b.first_n = a.tiles_n;
    b.tiles_m = (a.rows + 127) / 128;
    b.tiles_n = rest;
    b.per_xcd = (b.tiles_m * b.tiles_n + 7) / 8;
    hipLaunchKernelGGL((distill_sums_kernel<128, 256, 8, 64, TWO>), dim3(8u * b.per_xcd), dim3(512), 0, stream, b);
    NMB_CHECK_LAUNCH("distill");
  }
  const int64_t items = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  NMB_REQUIRE_SUPPORTED(items < (int64_t{1} << 23), "distill: too many tiles");  // of up to 512 threads
  a.per_xcd = static_cast<int>((items + 7) / 8);
  if constexpr (BACK) {
    const dim3 grid(static_cast<unsigned>(a.per_xcd) * 8u);
    if (p.tbm == 64) hipLaunchKernelGGL((distill_grad_kernel<64, 64, 4, 64, TWO>), grid, dim3(256), 0, stream, a);
    else if (p.tbm == 128) hipLaunchKernelGGL((distill_grad_kernel<128, 256, 8, 64, TWO>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((distill_grad_kernel<256, 128, 4, 32, TWO>), grid, dim3(256), 0, stream, a);
  } else {
    // as many workgroups as the CUs hold at a time: 32 an XCD, twice that of 64 x 64 tiles
    const dim3 grid(8u * std::min(a.per_xcd, p.tbm == 64 ? 64 : 32));
    if (picks != nullptr)
      hipLaunchKernelGGL(distill_few_kernel<TWO>, dim3(grid.x + picks->items), dim3(256), 0, stream, a, picks->t,
                         picks->picked, picks->passes, static_cast<int>(grid.x));
    else if (p.tbm == 64) hipLaunchKernelGGL((distill_sums_kernel<64, 64, 4, 64, TWO>), grid, dim3(256), 0, stream, a);
    else if (p.tbm == 128) hipLaunchKernelGGL((distill_sums_kernel<128, 256, 8, 64, TWO>), grid, dim3(512), 0, stream, a);
    else hipLaunchKernelGGL((distill_sums_kernel<256, 256, 8, 64, TWO>), grid, dim3(512), 0, stream, a);
  }
  NMB_CHECK_LAUNCH("distill");
  return NMB_OK;
}

int check_workspace(const void* workspace, int64_t bytes, int64_t need) {
  NMB_REQUIRE(workspace != nullptr && bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
              "distill: a 4-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need, (long long)bytes);
  return NMB_OK;
}

int merge(const float* ws, int tiles, int64_t rows, bool two, const Teacher& t, const float* picked, float* loss,
          float* stats, int64_t stats_ld, hipStream_t stream) {
  const float* sums = ws + rows * tiles;
  hipLaunchKernelGGL(distill_merge_kernel, dim3(static_cast<unsigned>((rows + 15) / 16)), dim3(256), 0, stream, ws, sums,
                     sums + rows * tiles, tiles, rows, two, t, picked, loss, stats, stats_ld);
  NMB_CHECK_LAUNCH("distill merge");
  return NMB_OK;
}

template <typename T>
int entries_launch(const Teacher& t, int64_t rows, const float* stats, int64_t stats_ld, const float* picked,
                   const float* grad, void* g, int64_t ldg, const void* x, int64_t ldx, int64_t hidden, void* kept,
                   hipStream_t stream) {
  hipLaunchKernelGGL(distill_entries_kernel<T>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256),
                     static_cast<size_t>(4) * padded4(t.top) * 8, stream, t, rows, stats, stats_ld, picked, grad,
                     static_cast<T*>(g), ldg, static_cast<const T*>(x), ldx, static_cast<int>(hidden),
                     static_cast<T*>(kept));
  NMB_CHECK_LAUNCH("distill entries");
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

extern "C" int nmb_distill_workspace_bytes(int64_t rows, int64_t vocab, int dtype, int64_t* bytes) {
  NMB_REQUIRE(bytes != nullptr && rows >= 0 && vocab > 0 && rows < (1 << 30) && vocab < (1 << 30),
              "distill_workspace_bytes: bad args");
  NMB_REQUIRE_SUPPORTED(dtype == NMB_BF16 || dtype == NMB_F32, "distill_workspace_bytes: unsupported dtype code %d", dtype);
  // a maximum and two sums per row and tile column (fp32: per row)
  *bytes = rows * 3 * (dtype == NMB_BF16 ? nmb::head_tiles_n(rows, vocab) : 1) * static_cast<int64_t>(sizeof(float));
  return NMB_OK;
}

extern "C" int nmb_distill_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab,
                               int64_t hidden, const nmb_teacher* teacher, float* loss, float* stats, int64_t stats_ld,
                               float* picked, void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  int st = nmb::check_teacher(teacher, rows, vocab);
  if (st != NMB_OK || rows == 0) return st;
  st = nmb::check_head(x, ldx, w, ldw, hidden);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(loss != nullptr && stats != nullptr && picked != nullptr && stats_ld >= rows, "distill_fwd: null output");
  int64_t need = 0;
  st = nmb_distill_workspace_bytes(rows, vocab, NMB_BF16, &need);
  if (st == NMB_OK) st = nmb::check_workspace(workspace, workspace_bytes, need);
  if (st != NMB_OK) return st;
  const nmb::Teacher t = nmb::make_teacher(teacher, vocab);
  const bool two = nmb::two_softmaxes(teacher);
  nmb::DistillArgs a = nmb::make_args(x, ldx, w, ldw, rows, vocab, hidden, t);
  const int tiles = static_cast<int>(nmb::head_tiles_n(rows, vocab));
  a.tile_max = static_cast<float*>(workspace);
  a.tile_a = a.tile_max + rows * tiles;
  a.tile_b = a.tile_a + rows * tiles;
  const int passes = (t.entries() + 31) / 32;
  NMB_REQUIRE_SUPPORTED(rows * passes < nmb::kMostWaves, "distill_fwd: too many rows and entries");
  const int64_t items = rows * passes;
  const nmb::Picks picks{t, picked, passes, static_cast<unsigned>(items)};
  const bool together = items <= nmb::kFewItems && nmb::head_plan(rows, vocab, false).tbm == 64;
  if (together) {}
  else if (items <= nmb::kFewItems)
    hipLaunchKernelGGL(nmb::distill_pick_kernel<true>, dim3(static_cast<unsigned>(items)), dim3(256), 0, stream, a, t, picked,
                       passes);
  else
    hipLaunchKernelGGL(nmb::distill_pick_kernel<false>, dim3(static_cast<unsigned>((items + 3) / 4)), dim3(256), 0, stream, a,
                       t, picked, passes);
  NMB_CHECK_LAUNCH("distill pick");
  const nmb::Picks* with = together ? &picks : nullptr;
  st = two ? nmb::distill_launch<false, true>(a, stream, with) : nmb::distill_launch<false, false>(a, stream, with);
  if (st != NMB_OK) return st;
  return nmb::merge(a.tile_max, tiles, rows, two, t, picked, loss, stats, stats_ld, stream);
}

extern "C" int nmb_distill_grad(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t rows, int64_t vocab,
                                int64_t hidden, const nmb_teacher* teacher, const float* stats, int64_t stats_ld,
                                const float* picked, const float* grad, void* g, int64_t ldg, void* kept,
                                hipStream_t stream) {
  int st = nmb::check_teacher(teacher, rows, vocab);
  if (st != NMB_OK || rows == 0) return st;
  st = nmb::check_head(x, ldx, w, ldw, hidden);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(stats != nullptr && picked != nullptr && grad != nullptr && g != nullptr && stats_ld >= rows,
              "distill_grad: null argument");
  NMB_REQUIRE(nmb::aligned16(g) && ldg % 8 == 0 && ldg >= (vocab + 7) / 8 * 8,
              "distill_grad: g must be 16-byte aligned with rows of whole 8 columns");
  NMB_REQUIRE(kept == nullptr || nmb::aligned16(kept), "distill_grad: kept must be 16-byte aligned");
  NMB_REQUIRE_SUPPORTED(rows < nmb::kMostWaves, "distill_grad: too many rows");
  const nmb::Teacher t = nmb::make_teacher(teacher, vocab);
  nmb::DistillArgs a = nmb::make_args(x, ldx, w, ldw, rows, vocab, hidden, t);
  a.stats = stats;
  a.stats_ld = stats_ld;
  a.grad = grad;
  a.g = static_cast<nmb::bf16*>(g);
  a.ldg = ldg;
  a.past_cache = rows * ldg * static_cast<int64_t>(sizeof(nmb::bf16)) > (int64_t{256} << 20);
  st = nmb::two_softmaxes(teacher) ? nmb::distill_launch<true, true>(a, stream) : nmb::distill_launch<true, false>(a, stream);
  if (st != NMB_OK) return st;
  return nmb::entries_launch<nmb::bf16>(t, rows, stats, stats_ld, picked, grad, g, ldg, x, ldx, hidden, kept, stream);
}

extern "C" int nmb_distill_rows_fwd(const float* s, int64_t ld, int64_t rows, int64_t vocab, const nmb_teacher* teacher,
                                    float* loss, float* stats, int64_t stats_ld, float* picked, void* workspace,
                                    int64_t workspace_bytes, hipStream_t stream) {
  int st = nmb::check_teacher(teacher, rows, vocab);
  if (st != NMB_OK || rows == 0) return st;
  NMB_REQUIRE(s != nullptr && ld >= vocab && loss != nullptr && stats != nullptr && picked != nullptr && stats_ld >= rows,
              "distill_rows_fwd: null argument or rows that overlap");
  NMB_REQUIRE_SUPPORTED(rows < nmb::kMostRows, "distill_rows_fwd: too many rows");
  int64_t need = 0;
  st = nmb_distill_workspace_bytes(rows, vocab, NMB_F32, &need);
  if (st == NMB_OK) st = nmb::check_workspace(workspace, workspace_bytes, need);
  if (st != NMB_OK) return st;
  const nmb::Teacher t = nmb::make_teacher(teacher, vocab);
  const bool two = nmb::two_softmaxes(teacher);
  float* ws = static_cast<float*>(workspace);
  hipLaunchKernelGGL(nmb::distill_rows_fwd_kernel, dim3(static_cast<unsigned>(rows)), dim3(nmb::kRowThreads), 0, stream,
                     s, ld, rows, t, two, ws, ws + rows, ws + 2 * rows, picked);
  NMB_CHECK_LAUNCH("distill rows");
  return nmb::merge(ws, 1, rows, two, t, picked, loss, stats, stats_ld, stream);
}

extern "C" int nmb_distill_rows_grad(float* s, int64_t ld, int64_t rows, int64_t vocab, const nmb_teacher* teacher,
                                     const float* stats, int64_t stats_ld, const float* picked, const float* grad,
                                     const float* x, int64_t ldx, int64_t hidden, float* kept, hipStream_t stream) {
  int st = nmb::check_teacher(teacher, rows, vocab);
  if (st != NMB_OK || rows == 0) return st;
  NMB_REQUIRE(s != nullptr && ld >= vocab && stats != nullptr && picked != nullptr && grad != nullptr && stats_ld >= rows,
              "distill_rows_grad: null argument or rows that overlap");
  NMB_REQUIRE(kept == nullptr || (x != nullptr && hidden > 0 && hidden < (1 << 30) && ldx >= hidden),
              "distill_rows_grad: kept needs x and its size");
  NMB_REQUIRE_SUPPORTED(rows < nmb::kMostRows, "distill_rows_grad: too many rows");
  const nmb::Teacher t = nmb::make_teacher(teacher, vocab);
  hipLaunchKernelGGL(nmb::distill_rows_bwd_kernel, dim3(static_cast<unsigned>(rows)), dim3(nmb::kRowThreads), 0, stream,
                     s, ld, t, nmb::two_softmaxes(teacher), stats, stats_ld, grad);
  NMB_CHECK_LAUNCH("distill rows grad");
  return nmb::entries_launch<float>(t, rows, stats, stats_ld, picked, grad, s, ld, x, ldx, hidden, kept, stream);
}

extern "C" int nmb_distill_total_workspace_bytes(int64_t rows, int64_t* bytes) {
  NMB_REQUIRE(rows >= 0 && rows < (1 << 30) && bytes != nullptr, "distill_total_workspace_bytes: bad args");
  *bytes = rows > nmb::kTotalRows ? static_cast<int64_t>(nmb::kTotalBlocks * sizeof(nmb::Counted)) : 0;
  return NMB_OK;
}

extern "C" int nmb_distill_total(const float* loss, const float* stats, int64_t stats_ld, const int64_t* targets,
                                 int64_t ignore_index, int64_t rows, int mean, float* total, float* over,
                                 void* workspace, int64_t workspace_bytes, hipStream_t stream) {
  NMB_REQUIRE(total != nullptr && over != nullptr, "distill_total: null output");
  int64_t need = 0;
  const int st = nmb_distill_total_workspace_bytes(rows, &need);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(rows == 0 || (loss != nullptr && stats != nullptr && stats_ld >= rows), "distill_total: null argument");
  NMB_REQUIRE(need == 0 || (workspace != nullptr && workspace_bytes >= need &&
                            (reinterpret_cast<uintptr_t>(workspace) & 7) == 0),
              "distill_total: an 8-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need,
              (long long)workspace_bytes);
  const bool one = need == 0;
  const int blocks =
      static_cast<int>(std::clamp<int64_t>((rows + nmb::kTotalRows - 1) / nmb::kTotalRows, 1, nmb::kTotalBlocks));
  auto* parts = one ? nullptr : static_cast<nmb::Counted*>(workspace);
  hipLaunchKernelGGL(nmb::distill_total_kernel, dim3(blocks), dim3(1024), 0, stream, loss,
                     rows == 0 ? nullptr : stats + 3 * stats_ld, rows == 0 ? nullptr : targets, ignore_index, rows,
                     mean != 0, parts, total, over);
  NMB_CHECK_LAUNCH("distill total");
  if (one) return NMB_OK;
  hipLaunchKernelGGL(nmb::distill_join_kernel, dim3(1), dim3(nmb::kTotalBlocks), 0, stream, parts, blocks, mean != 0,
                     total, over);
  NMB_CHECK_LAUNCH("distill total (join)");
  return NMB_OK;
}
