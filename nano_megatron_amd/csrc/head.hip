// The LM head with capped logits and its loss, for gfx950: no counterpart in the
// reference (its head and loss: tensor_parallel/layers.py:207-214,
// cross_entropy.py:30-86).
//
//   s = x w^T;  y = cap tanh(s / cap) (y = s without a cap);  lse = log sum exp y
//   loss = lse - y_t + z lse^2  (0 for an ignored target)
//   dL/ds = (exp(y - lse) (1 + 2 z lse) - [t]) (1 - tanh^2) grad
//
// bf16: the loss is the epilogue of the product's tiles: each takes the sum (and,
// where no cap bounds the logits, the maximum) of its columns' exponentials from
// the fp32 accumulators, so that logits are neither rounded nor written, and a
// second launch joins the tiles of a row.  The backward forms the tiles again and
// writes only the gradient, rounded to bf16 once (half a step, 2^-8) as the operand
// of the two products that follow it.  fp32: row kernels over stored logits.
// Measured, 8192 x 50304 x 768 with a cap: 638 us forward (0.99 PFLOP/s; the plain product
// that writes bf16 logits 766), 745 the gradient with its 824 MB; the matrix unit is busy 44
// and 40% of the time, the epilogues' three transcendentals a logit and the K loop's
// start (12 K tiles) are the rest.
#include <math.h>

#include <algorithm>

#include "gemm_core.h"
#include "head_plan.h"

namespace nmb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// Capped logits of at most this in base 2 need no running maximum: sums of 2^30 of
// their exponentials stay within fp32, at the same relative precision.
constexpr float kFixedMax = 80.f;

struct HeadArgs {
  const bf16* x;
  const bf16* w;
  int64_t ldx, ldw;
  int rows, vocab, hidden;
  const int64_t* targets;
  int64_t ignore_index;
  float cap_in, cap_out;  // 2 log2(e) / cap, cap log2(e); 0 without a cap
  float z;
  // forward
  float* tile_sum;  // [tiles_n][rows]
  float* tile_max;  // the same; not with a fixed maximum
  float* picked;    // [rows]: y_t in base 2
  // backward
  const float* lse2;  // [rows]
  const float* grad;  // [rows]
  bf16* g;            // [rows, ldg]; columns vocab .. round8(vocab) are zeros
  int64_t ldg;
  bool past_cache;  // g is larger than the last-level cache
  int tiles_m, tiles_n, per_xcd;
};

// 1 / (1 + e^(2 y)) for s = y cap: tanh = 1 - 2 t, 1 - tanh^2 = 4 t (1 - t)
__device__ __forceinline__ float cap_t(float s, float cap_in) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(s * cap_in));
}

template <bool CAP>
__device__ __forceinline__ float logit2(const HeadArgs& a, float s) {
  return CAP ? fmaf(-2.f * a.cap_out, cap_t(s, a.cap_in), a.cap_out) : s * kLog2e;
}

// MODE 0: forward, maximum fixed at 0; 1: forward with a maximum; 2: backward.
// Tiles of 8 waves have a CU to themselves, of those of 4 waves two share one.
template <int TBM, int TBN, int NW, int BKT, int MODE, bool CAP>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void head_kernel(HeadArgs a) {
  constexpr int WAVES_N = NW == 4 ? (TBN == 64 ? 1 : 2) : (TBN == 256 ? 4 : 2);
  constexpr int WAVES_M = NW / WAVES_N;
  constexpr int WM = TBM / WAVES_M, WN = TBN / WAVES_N, TM = WM / 16, TN = WN / 16;
  constexpr int S = Stages<TBM, TBN, NW, BKT>::S;
  __shared__ __attribute__((aligned(1024))) bf16 sA[S][TBM * BKT];
  __shared__ __attribute__((aligned(1024))) bf16 sB[S][TBN * BKT];

  const int L = static_cast<int>(blockIdx.x);
  const int item = (L % 8) * a.per_xcd + L / 8;
  if (item >= a.tiles_m * a.tiles_n) return;
  // 4 tile rows at a time, the rows fastest, as in gemm.hip
  constexpr int GM = 4;
  const int grp = item / (GM * a.tiles_n);
  const int gsize = min(a.tiles_m - grp * GM, GM);
  const int r = item - grp * GM * a.tiles_n;
  const int m0 = (grp * GM + r % gsize) * TBM, tile_n = r / gsize, n0 = tile_n * TBN;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = (wave / WAVES_N) * WM, wn = (wave % WAVES_N) * WN;
  const int l16 = lane & 15, q4 = lane >> 4;

  Loader<TBM, true, BKT, NW> la;
  Loader<TBN, true, BKT, NW> lb;
  const int va = min(TBM, a.rows - m0), vb = min(TBN, a.vocab - n0);
  la.init(a.x + static_cast<int64_t>(m0) * a.ldx, a.ldx, va,
          static_cast<uint32_t>(((va - 1) * a.ldx + a.hidden) * 2), wave, lane);
  lb.init(a.w + static_cast<int64_t>(n0) * a.ldw, a.ldw, vb,
          static_cast<uint32_t>(((vb - 1) * a.ldw + a.hidden) * 2), wave, lane);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  k_loop<TBM, TBN, NW, BKT, true, true, TM, TN>(la, lb, sA, sB, acc, wm, wn, 0, a.hidden, wave, lane);

  // acc[i][j][e] = s[m0 + wm + 16 i + l16][n0 + wn + 16 j + 4 q4 + e]
  const int col0 = n0 + wn + 4 * q4;
  const bool edge = n0 + TBN > a.vocab;
  // the target's place among this lane's columns: 16 j + e, or something else
  auto target_at = [&](int i) {
    const int m = min(m0 + wm + 16 * i + l16, a.rows - 1);
    const int64_t t = a.targets[m] - col0;
    return t >= 0 && t < WN && (t & 12) == 0 ? static_cast<int>(t) : -1;
  };
  if constexpr (MODE < 2) {
    float* red = reinterpret_cast<float*>(&sA[0][0]);            // [WAVES_N][TBM]: sums
    float* red_max = red + WAVES_N * TBM;
    static_assert(2 * WAVES_N * TBM * sizeof(float) <= sizeof(sA), "the reduction takes the operands' place");
    __syncthreads();  // every wave is done with the operand stages
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int lr = wm + 16 * i + l16, m = m0 + lr;
      const int hit = target_at(i);
      if (__any(hit >= 0)) {
        float y = 0.f;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) y = hit == 16 * j + e ? acc[i][j][e] : y;
        if (hit >= 0 && m < a.rows) a.picked[m] = logit2<CAP>(a, y);
      }
      float top = -__builtin_inff(), sum = 0.f;
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float y = logit2<CAP>(a, acc[i][j][e]);
          if (edge) y = col0 + 16 * j + e < a.vocab ? y : -__builtin_inff();
          if constexpr (MODE == 0) {
            sum += __builtin_amdgcn_exp2f(y);
          } else {
            acc[i][j][e] = y;
            top = fmaxf(top, y);
          }
        }
      if constexpr (MODE == 1) {
        top = xor32_max(xor16_max(top));
        const float off = top == -__builtin_inff() ? 0.f : top;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum += __builtin_amdgcn_exp2f(acc[i][j][e] - off);
      }
      sum = xor32_sum(xor16_sum(sum));
      if (q4 == 0) {
        red[(wave % WAVES_N) * TBM + lr] = sum;
        if constexpr (MODE == 1) red_max[(wave % WAVES_N) * TBM + lr] = top;
      }
    }
    __syncthreads();
    const int lr = static_cast<int>(threadIdx.x), m = m0 + lr;
    if (lr < TBM && m < a.rows) {
      float top = -__builtin_inff(), sum = 0.f;
      if constexpr (MODE == 1) {
#pragma unroll
        for (int w = 0; w < WAVES_N; ++w) top = fmaxf(top, red_max[w * TBM + lr]);
      }
#pragma unroll
      for (int w = 0; w < WAVES_N; ++w) {
        const float s = red[w * TBM + lr];
        if constexpr (MODE == 0) sum += s;
        else sum += red_max[w * TBM + lr] == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f(red_max[w * TBM + lr] - top);
      }
      const int64_t at = static_cast<int64_t>(tile_n) * a.rows + m;
      a.tile_sum[at] = sum;
      if constexpr (MODE == 1) a.tile_max[at] = top;
    }
  } else {
    constexpr int RPA = (S * TBM * BKT) / TBN;  // tile rows that fit in sA, the rest in sB
    static_assert(RPA + S * BKT >= TBM, "the bf16 tile fits in the operand stages");
    auto tile_at = [&](int row, int c) -> bf16* {  // element (row, c), c a multiple of 4
      bf16* rp = row < RPA ? &sA[0][0] + row * TBN : &sB[0][0] + (row - RPA) * TBN;
      return rp + 8 * ((c >> 3) ^ (row & (TBN == 64 ? 7 : 15))) + (c & 4);
    };
    __syncthreads();  // every wave is done with the operand stages
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int lr = wm + 16 * i + l16, m = min(m0 + lr, a.rows - 1);
      const bool used = a.targets[m] != a.ignore_index;
      const float l2 = a.lse2[m];
      const float gr = (CAP ? 4.f : 1.f) * a.grad[m];
      const float f = gr * (1.f + 2.f * a.z * l2 * kLn2);
      const float nl2 = a.cap_out - l2;
      const int hit = target_at(i);
      const bool any_hit = __any(hit >= 0);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        bf16x4 out;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s = acc[i][j][e];
          float u = 1.f, y;
          if constexpr (CAP) {
            const float t = cap_t(s, a.cap_in);
            u = fmaf(-t, t, t);
            y = fmaf(-2.f * a.cap_out, t, nl2);
          } else {
            y = fmaf(s, kLog2e, nl2);
          }
          float g = __builtin_amdgcn_exp2f(y) * f;
          if (any_hit) g = hit == 16 * j + e ? g - gr : g;
          if constexpr (CAP) g *= u;
          g = used ? g : 0.f;
          if (edge) g = col0 + 16 * j + e < a.vocab ? g : 0.f;
          out[e] = static_cast<bf16>(g);
        }
        *reinterpret_cast<bf16x4*>(tile_at(lr, wn + 16 * j + 4 * q4)) = out;
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
      const int m = m0 + row, n = n0 + 8 * sl;
      if (m >= a.rows || n >= a.vocab) continue;
      bf16x8* out = reinterpret_cast<bf16x8*>(a.g + m * a.ldg + n);
      // What the products that follow find in the cache anyway is written there; the rest
      // past it.  With both of them, g of 824 MB 2650 -> 2592 us, of 131 MB 420 -> 427.
      if (a.past_cache) {
        __builtin_nontemporal_store(v, out);
        asm volatile("");  // or the two stores become one, an ordinary one
      } else {
        *out = v;
      }
    }
  }
}

// The loss and the base-2 lse of 16 rows per workgroup: a row's tiles are joined by
// 16 threads, in an order that depends on their number alone.
template <bool MAX>
__global__ __launch_bounds__(256) void head_merge_kernel(HeadArgs a, float* __restrict__ loss,
                                                         float* __restrict__ lse2) {
  __shared__ float sSum[16][17], sMax[16][17];
  const int n = threadIdx.x & 15, part = threadIdx.x >> 4;  // row, share of its tiles
  const int64_t m = static_cast<int64_t>(blockIdx.x) * 16 + n;
  float top = MAX ? -__builtin_inff() : 0.f, sum = 0.f;
  if (m < a.rows) {
    if constexpr (MAX) {
#pragma unroll 4
      for (int t = part; t < a.tiles_n; t += 16) top = fmaxf(top, a.tile_max[static_cast<int64_t>(t) * a.rows + m]);
    }
#pragma unroll 4
    for (int t = part; t < a.tiles_n; t += 16) {
      const int64_t at = static_cast<int64_t>(t) * a.rows + m;
      const float s = a.tile_sum[at];
      if constexpr (MAX) sum += a.tile_max[at] == -__builtin_inff() ? s : s * __builtin_amdgcn_exp2f(a.tile_max[at] - top);
      else sum += s;
    }
  }
  sSum[part][n] = sum;
  sMax[part][n] = top;
  __syncthreads();
  if (part != 0 || m >= a.rows) return;
  float all = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) top = MAX ? fmaxf(top, sMax[k][n]) : 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k)
    all += !MAX || sMax[k][n] == -__builtin_inff() ? sSum[k][n] : sSum[k][n] * __builtin_amdgcn_exp2f(sMax[k][n] - top);
  const float l2 = top + log2f(all);
  lse2[m] = l2;
  const int64_t t = a.targets[m];
  const float lse = l2 * kLn2;
  // a target outside the vocabulary poisons its row; the host checks targets
  loss[m] = t == a.ignore_index ? 0.f
            : t < 0 || t >= a.vocab ? __builtin_nanf("")
                                    : fmaf(a.z * lse, lse, (l2 - a.picked[m]) * kLn2);
}

// ------------------------------------------------------------ fp32, by rows
struct RowArgs {
  float* s;  // [rows, ld]: the products; the backward writes their gradient over them
  int64_t ld, vocab;
  const int64_t* targets;
  int64_t ignore_index;
  float cap, inv, z;  // inv: 1 / cap
};

__device__ __forceinline__ float block_reduce(float v, float* sh, bool max) {
  v = max ? wave_max(v) : wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return max ? fmaxf(fmaxf(sh[0], sh[1]), fmaxf(sh[2], sh[3])) : (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__device__ __forceinline__ float bend(const RowArgs& a, float s) { return a.cap > 0.f ? a.cap * tanhf(s * a.inv) : s; }

// One workgroup per row; the running maximum and sum of each thread's columns in one pass,
// eight of them at a time: their loads and exponentials then do not wait for each other
// (512 x 8192: forward 16.7 -> 8.4 us, backward 17.3 -> 10.8 against one at a time and a division by the cap).
constexpr int kRowCols = 8;
__global__ __launch_bounds__(256) void head_rows_fwd_kernel(RowArgs a, float* __restrict__ loss,
                                                            float* __restrict__ lse2) {
  __shared__ float sh[4];
  const int64_t row = blockIdx.x;
  const float* s = a.s + row * a.ld;
  float top = -__builtin_inff(), sum = 0.f;
  for (int64_t c0 = threadIdx.x; c0 < a.vocab; c0 += 256 * kRowCols) {
    float y[kRowCols], most = top;
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      const int64_t c = c0 + 256 * e;
      y[e] = c < a.vocab ? s[c] : -__builtin_inff();
    }
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      if (c0 + 256 * e < a.vocab) y[e] = bend(a, y[e]);
      most = fmaxf(most, y[e]);
    }
    if (most > top) {
      sum *= expf(top - most);
      top = most;
    }
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) sum += top == -__builtin_inff() && y[e] == y[e] ? 0.f : expf(y[e] - top);
  }
  const float all = block_reduce(top, sh, true);
  sum = block_reduce(top == -__builtin_inff() ? sum : sum * expf(top - all), sh, false);
  if (threadIdx.x != 0) return;
  const float lse = all + logf(sum);
  lse2[row] = lse * kLog2e;
  const int64_t t = a.targets[row];
  loss[row] = t == a.ignore_index ? 0.f
              : t < 0 || t >= a.vocab ? __builtin_nanf("") : fmaf(a.z * lse, lse, logf(sum) - (bend(a, s[t]) - all));
}

__global__ __launch_bounds__(256) void head_rows_bwd_kernel(RowArgs a, const float* __restrict__ lse2,
                                                            const float* __restrict__ grad) {
  const int64_t row = blockIdx.x;
  float* s = a.s + row * a.ld;
  const int64_t t = a.targets[row];
  const float lse = lse2[row] * kLn2, gr = grad[row], f = gr * (1.f + 2.f * a.z * lse);
  for (int64_t c0 = threadIdx.x; c0 < a.vocab; c0 += 256 * kRowCols) {
    float x[kRowCols];
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) x[e] = c0 + 256 * e < a.vocab ? s[c0 + 256 * e] : 0.f;
#pragma unroll
    for (int e = 0; e < kRowCols; ++e) {
      const int64_t c = c0 + 256 * e;
      const float y = bend(a, x[e]);
      float g = expf(y - lse) * f;
      if (c == t) g -= gr;
      if (a.cap > 0.f) g *= 1.f - (y * a.inv) * (y * a.inv);
      if (c < a.vocab) s[c] = t == a.ignore_index ? 0.f : g;
    }
  }
}

// ------------------------------------------------------------ host side
// 0: none.  A capped logit is off by up to 2^-20 of the cap, which grows past use for large
// ones, and 2 log2(e) / cap overflows for the smallest.
bool cap_allowed(float cap) { return cap == 0.f || (cap >= 1e-3f && cap <= 1e4f); }
int check_head(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* targets, int64_t rows, int64_t vocab,
               int64_t hidden, float cap, float z) {
  NMB_REQUIRE(x != nullptr && w != nullptr && targets != nullptr, "head: null argument");
  NMB_REQUIRE(rows >= 0 && vocab > 0 && hidden > 0 && rows < (1 << 30) && vocab < (1 << 30) && hidden < (1 << 30),
              "head: invalid shape");
  NMB_REQUIRE(ldx >= hidden && ldw >= hidden, "head: leading dimension too small");
  NMB_REQUIRE(cap_allowed(cap) && isfinite(z) && z >= 0.f, "head: cap and z must be finite and >= 0, a cap within 1e-3 and 1e4");
  NMB_REQUIRE_SUPPORTED(hidden % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0,
                        "head: hidden and the leading dimensions must be multiples of 8");
  NMB_REQUIRE(aligned16(x) && aligned16(w), "head: operands must be 16-byte aligned");
  NMB_REQUIRE_SUPPORTED(256 * ldx < (int64_t{1} << 30) && 256 * ldw < (int64_t{1} << 30),
                        "head: an operand tile spans more than 2 GiB");
  return NMB_OK;
}

HeadArgs make_head(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* targets, int64_t rows,
                   int64_t vocab, int64_t hidden, int64_t ignore_index, float cap, float z) {
  HeadArgs a{};
  a.x = static_cast<const bf16*>(x);
  a.w = static_cast<const bf16*>(w);
  a.ldx = ldx;
  a.ldw = ldw;
  a.rows = static_cast<int>(rows);
  a.vocab = static_cast<int>(vocab);
  a.hidden = static_cast<int>(hidden);
  a.targets = targets;
  a.ignore_index = ignore_index;
  a.cap_in = cap > 0.f ? static_cast<float>(2.0 * 1.4426950408889634074 / cap) : 0.f;
  a.cap_out = cap > 0.f ? static_cast<float>(cap * 1.4426950408889634074) : 0.f;
  a.z = z;
  return a;
}

template <int MODE, bool CAP>
int head_launch(HeadArgs a, hipStream_t stream) {
  const HeadPlan p = head_plan(a.rows, a.vocab, MODE == 2);
  a.tiles_m = (a.rows + p.tbm - 1) / p.tbm;
  a.tiles_n = (a.vocab + p.tbn - 1) / p.tbn;
  const int64_t items = static_cast<int64_t>(a.tiles_m) * a.tiles_n;
  NMB_REQUIRE(items < (int64_t{1} << 28), "head: too many tiles");
  a.per_xcd = static_cast<int>((items + 7) / 8);
  const dim3 grid(static_cast<unsigned>(a.per_xcd) * 8u);
  if (p.tbm == 64) hipLaunchKernelGGL((head_kernel<64, 64, 4, 64, MODE, CAP>), grid, dim3(256), 0, stream, a);
  else if (p.tbm == 128) hipLaunchKernelGGL((head_kernel<128, 256, 8, 64, MODE, CAP>), grid, dim3(512), 0, stream, a);
  else if constexpr (MODE == 2) hipLaunchKernelGGL((head_kernel<256, 128, 4, 32, MODE, CAP>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((head_kernel<256, 256, 8, 64, MODE, CAP>), grid, dim3(512), 0, stream, a);
  NMB_CHECK_LAUNCH("head");
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

extern "C" int nmb_head_loss_workspace_bytes(int64_t rows, int64_t vocab, int64_t* bytes) {
  NMB_REQUIRE(bytes != nullptr && rows >= 0 && vocab > 0 && rows < (1 << 30) && vocab < (1 << 30),
              "head_loss_workspace_bytes: bad args");
  // a sum and a maximum per row and tile column, and the target's logit
  *bytes = rows * (2 * nmb::head_tiles_n(rows, vocab) + 1) * static_cast<int64_t>(sizeof(float));
  return NMB_OK;
}

extern "C" int nmb_head_loss_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* targets,
                                 int64_t rows, int64_t vocab, int64_t hidden, int64_t ignore_index, float cap, float z,
                                 float* loss, float* lse2, void* workspace, int64_t workspace_bytes,
                                 hipStream_t stream) {
  if (rows == 0) return NMB_OK;
  const int st = nmb::check_head(x, ldx, w, ldw, targets, rows, vocab, hidden, cap, z);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(loss != nullptr && lse2 != nullptr, "head_loss_fwd: null output");
  int64_t need = 0;
  const int sq = nmb_head_loss_workspace_bytes(rows, vocab, &need);
  if (sq != NMB_OK) return sq;
  NMB_REQUIRE(workspace != nullptr && workspace_bytes >= need && (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
              "head_loss_fwd: a 4-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need,
              (long long)workspace_bytes);
  nmb::HeadArgs a = nmb::make_head(x, ldx, w, ldw, targets, rows, vocab, hidden, ignore_index, cap, z);
  a.tiles_n = static_cast<int>(nmb::head_tiles_n(rows, vocab));
  a.tile_sum = static_cast<float*>(workspace);
  a.tile_max = a.tile_sum + rows * a.tiles_n;
  a.picked = a.tile_max + rows * a.tiles_n;
  const bool fixed = a.cap_out > 0.f && a.cap_out <= nmb::kFixedMax;
  const int lt = fixed                ? nmb::head_launch<0, true>(a, stream)
                 : a.cap_out > 0.f ? nmb::head_launch<1, true>(a, stream)
                                   : nmb::head_launch<1, false>(a, stream);
  if (lt != NMB_OK) return lt;
  const dim3 grid(static_cast<unsigned>((rows + 15) / 16));
  if (fixed) hipLaunchKernelGGL(nmb::head_merge_kernel<false>, grid, dim3(256), 0, stream, a, loss, lse2);
  else hipLaunchKernelGGL(nmb::head_merge_kernel<true>, grid, dim3(256), 0, stream, a, loss, lse2);
  NMB_CHECK_LAUNCH("head merge");
  return NMB_OK;
}

extern "C" int nmb_head_loss_grad(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* targets,
                                  int64_t rows, int64_t vocab, int64_t hidden, int64_t ignore_index, float cap, float z,
                                  const float* lse2, const float* grad, void* g, int64_t ldg, hipStream_t stream) {
  if (rows == 0) return NMB_OK;
  const int st = nmb::check_head(x, ldx, w, ldw, targets, rows, vocab, hidden, cap, z);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(lse2 != nullptr && grad != nullptr && g != nullptr, "head_loss_grad: null argument");
  NMB_REQUIRE(nmb::aligned16(g) && ldg % 8 == 0 && ldg >= (vocab + 7) / 8 * 8,
              "head_loss_grad: g must be 16-byte aligned with rows of whole 8 columns");
  nmb::HeadArgs a = nmb::make_head(x, ldx, w, ldw, targets, rows, vocab, hidden, ignore_index, cap, z);
  a.lse2 = lse2;
  a.grad = grad;
  a.g = static_cast<nmb::bf16*>(g);
  a.ldg = ldg;
  a.past_cache = rows * ldg * static_cast<int64_t>(sizeof(nmb::bf16)) > (int64_t{256} << 20);
  return cap > 0.f ? nmb::head_launch<2, true>(a, stream) : nmb::head_launch<2, false>(a, stream);
}

namespace nmb {
namespace {
int check_rows(const float* s, int64_t ld, const int64_t* targets, int64_t rows, int64_t vocab, float cap, float z) {
  NMB_REQUIRE(s != nullptr && targets != nullptr, "head_rows: null argument");
  NMB_REQUIRE(rows >= 0 && rows <= 0x7fffffff && vocab > 0 && ld >= vocab, "head_rows: invalid shape");
  NMB_REQUIRE(cap_allowed(cap) && isfinite(z) && z >= 0.f, "head_rows: cap and z must be finite and >= 0, a cap within 1e-3 and 1e4");
  return NMB_OK;
}
}  // namespace
}  // namespace nmb

extern "C" int nmb_head_rows_fwd(const float* s, int64_t ld, const int64_t* targets, int64_t rows, int64_t vocab,
                                 int64_t ignore_index, float cap, float z, float* loss, float* lse2,
                                 hipStream_t stream) {
  if (rows == 0) return NMB_OK;
  const int st = nmb::check_rows(s, ld, targets, rows, vocab, cap, z);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(loss != nullptr && lse2 != nullptr, "head_rows_fwd: null output");
  const nmb::RowArgs a{const_cast<float*>(s), ld, vocab, targets, ignore_index, cap, cap > 0.f ? 1.f / cap : 0.f, z};
  hipLaunchKernelGGL(nmb::head_rows_fwd_kernel, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, a, loss, lse2);
  NMB_CHECK_LAUNCH("head_rows_fwd");
  return NMB_OK;
}

extern "C" int nmb_head_rows_bwd(float* s, int64_t ld, const int64_t* targets, int64_t rows, int64_t vocab,
                                 int64_t ignore_index, float cap, float z, const float* lse2, const float* grad,
                                 hipStream_t stream) {
  if (rows == 0) return NMB_OK;
  const int st = nmb::check_rows(s, ld, targets, rows, vocab, cap, z);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(lse2 != nullptr && grad != nullptr, "head_rows_bwd: null argument");
  const nmb::RowArgs a{s, ld, vocab, targets, ignore_index, cap, cap > 0.f ? 1.f / cap : 0.f, z};
  hipLaunchKernelGGL(nmb::head_rows_bwd_kernel, dim3(static_cast<unsigned>(rows)), dim3(256), 0, stream, a, lse2, grad);
  NMB_CHECK_LAUNCH("head_rows_bwd");
  return NMB_OK;
}
