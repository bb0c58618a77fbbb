// Scored attention in fp32, on the fp32 matrix core, for any strides and head dim
// <= 128: the shape of attention_f32.h (a workgroup owns 16 rows of one side, its
// four waves take the 16-row tiles of the other side in turn, operands straight from
// global memory with the next tile's in flight, merged through LDS in wave order)
// with the scores and spans of attention_scored.h.  What bounds it at the lengths of
// the fp32 configuration is the chain of loads and products of a wave's few tiles (3 x 4 / 2
// heads of 64 x 333: forward 18 us, dQ 21, dK and dV 43 in 126 workgroups).
#include "attention_scored.h"

#include "attention_f32.h"

namespace nmb {
namespace {

template <int DM>
__global__ __launch_bounds__(256) void scored_f32_fwd_kernel(ScoredShape p, const float* __restrict__ q,
                                                             const float* __restrict__ k,
                                                             const float* __restrict__ v, float* __restrict__ o,
                                                             float* __restrict__ lse2, int vec) {
  constexpr int DT = DM / 16;
  __shared__ __attribute__((aligned(16))) WaveSums<DM> sums;
  __shared__ float sM[4][16], sL[4][16];
  __shared__ uint32_t bad;  // rows with a NaN
  if (threadIdx.x == 0) bad = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int q0 = 16 * (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x));  // the most keys first
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.Hq / p.Hkv);
  const int i = min(q0 + l16, p.Sq - 1);
  const RowView r = row_view(p, b);
  const float slope2 = slope2_of(p, h), pos = bias_pos(p, r, i);
  const Span seen = seen_keys(p, r, i);
  const int k_lo = __builtin_amdgcn_readlane(seen.lo, 0), k_hi = __builtin_amdgcn_readlane(seen.hi, 15);
  const float* kb = k + b * p.k_sb + hk * p.k_sh;
  const float* vb = v + b * p.v_sb + hk * p.v_sh;
  f32x4 qf[DT], kf[DT];
  float vf[4][DT];
  load_row<float, DM>(q + b * p.q_sb + i * p.q_ss + h * p.q_sh, true, p.D, g, vec, qf);
  float m = -__builtin_inff(), l = 0.f;
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int tiles = (k_hi - k_lo + 15) / 16;
  auto load = [&](int t) {
    const int key = k_lo + 16 * t + l16;
    load_row<float, DM>(kb + min(key, k_hi - 1) * p.k_ss, key < k_hi, p.D, g, vec, kf);
    load_cols<float, DM>(vb, p.v_ss, k_lo + 16 * t, k_hi, p.D, l16, g, vf);
  };
  if (wave < tiles) load(wave);
  for (int t = wave; t < tiles; t += 4) {
    const f32x4 s = row_product<DM>(kf, qf);
    float vc[4][DT];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) vc[e][dt] = vf[e][dt];
    if (t + 4 < tiles) load(t + 4);
    float x[4], top = -__builtin_inff(), w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = k_lo + 16 * t + 4 * g + e;
      float bent;
      const float full = score_exact(p, s[e], slope2, pos - static_cast<float>(key), bent);
      x[e] = key < seen.lo || key >= seen.hi ? -__builtin_inff() : full;
      top = fmaxf(top, x[e]);
    }
    top = xor32_max(xor16_max(top));
    if (__any(top > m)) {
      const float mn = fmaxf(m, top);
      const float alpha = m == -__builtin_inff() ? 0.f : exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
    }
    const float off = m == -__builtin_inff() ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      w[e] = exp2f(x[e] - off);
      l += w[e];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma_f32x4(vc[e][dt], w[e], acc[dt]);
    }
  }
  l = xor32_sum(xor16_sum(l));
  sums.put(wave, l16, g, acc);
  if (g == 0) {
    sM[wave][l16] = m;
    sL[wave][l16] = l;
  }
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * DM; x += 256) {
    const int n = x / DM, d = x % DM;
    if (q0 + n >= p.Sq) continue;
    const float top = fmaxf(fmaxf(sM[0][n], sM[1][n]), fmaxf(sM[2][n], sM[3][n]));
    float sum = 0.f, val = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = sM[w][n] == -__builtin_inff() ? 0.f : exp2f(sM[w][n] - top);
      sum = fmaf(f, sL[w][n], sum);
      val = fmaf(f, sums.v[w][n][d], val);
    }
    const bool lost = sum != sum;  // a visible score is not a number: no row to run again
    if (!lost && (!(fabsf(val) < __builtin_inff()) || !(sum < __builtin_inff()))) atomicOr(&bad, 1u << n);
    if (d < p.D) o[b * p.o_sb + (q0 + n) * p.o_ss + h * p.o_sh + d] = lost ? sum : sum > 0.f ? val / sum : 0.f;
    if (d == 0)
      lse2[(static_cast<int64_t>(b) * p.Hq + h) * p.Sq + q0 + n] =
          lost ? sum : sum > 0.f ? top + log2f(sum) : -__builtin_inff();
  }
  __syncthreads();
  for (uint32_t left = bad; left != 0; left &= left - 1) {
    const int n = __ffs(left) - 1;
    if ((n & 3) == wave) scored_row_fwd<float>(p, q, k, v, o, nullptr, lse2, b, h, q0 + n, lane);
  }
}

// ndelta = -rowsum(dO o), then dQ
template <int DM>
__global__ __launch_bounds__(256) void scored_f32_dq_kernel(ScoredShape p, const float* __restrict__ q,
                                                            const float* __restrict__ k, const float* __restrict__ v,
                                                            const float* __restrict__ o,
                                                            const float* __restrict__ dout,
                                                            const float* __restrict__ lse2,
                                                            float* __restrict__ ndelta, float* __restrict__ dq,
                                                            int vec) {
  constexpr int DT = DM / 16;
  __shared__ __attribute__((aligned(16))) WaveSums<DM> sums;
  __shared__ uint32_t bad;
  if (threadIdx.x == 0) bad = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int q0 = 16 * (static_cast<int>(gridDim.x) - 1 - static_cast<int>(blockIdx.x));
  const int h = blockIdx.y, b = blockIdx.z, hk = h / (p.Hq / p.Hkv);
  const int i = min(q0 + l16, p.Sq - 1);
  const int64_t at = b * p.o_sb + i * p.o_ss + h * p.o_sh;
  const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;
  const RowView r = row_view(p, b);
  const float slope2 = slope2_of(p, h), pos = bias_pos(p, r, i);
  const Span seen = seen_keys(p, r, i);
  const int k_lo = __builtin_amdgcn_readlane(seen.lo, 0), k_hi = __builtin_amdgcn_readlane(seen.hi, 15);
  const float* kb = k + b * p.k_sb + hk * p.k_sh;
  const float* vb = v + b * p.v_sb + hk * p.v_sh;
  f32x4 qf[DT], df[DT], kf[DT], vf[DT];
  float kcol[4][DT];
  load_row<float, DM>(q + b * p.q_sb + i * p.q_ss + h * p.q_sh, true, p.D, g, vec, qf);
  load_row<float, DM>(dout + at, true, p.D, g, vec, df);
  float nd = 0.f;
  {
    f32x4 of[DT];
    load_row<float, DM>(o + at, true, p.D, g, vec, of);
#pragma unroll
    for (int j = 0; j < DT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) nd = fmaf(-of[j][e], df[j][e], nd);
  }
  nd = xor32_sum(xor16_sum(nd));
  if (wave == 0 && g == 0 && q0 + l16 < p.Sq) ndelta[row + i] = nd;
  const float l2 = lse2[row + i] == -__builtin_inff() ? __builtin_inff() : lse2[row + i];
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int tiles = (k_hi - k_lo + 15) / 16;
  auto load = [&](int t) {
    const int key = k_lo + 16 * t + l16;
    load_row<float, DM>(kb + min(key, k_hi - 1) * p.k_ss, key < k_hi, p.D, g, vec, kf);
    load_row<float, DM>(vb + min(key, k_hi - 1) * p.v_ss, key < k_hi, p.D, g, vec, vf);
    load_cols<float, DM>(kb, p.k_ss, k_lo + 16 * t, k_hi, p.D, l16, g, kcol);
  };
  if (wave < tiles) load(wave);
  for (int t = wave; t < tiles; t += 4) {
    const f32x4 s = row_product<DM>(kf, qf), dp = row_product<DM>(vf, df);
    float kc[4][DT];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) kc[e][dt] = kcol[e][dt];
    if (t + 4 < tiles) load(t + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int key = k_lo + 16 * t + 4 * g + e;
      float bent;
      const float x = score_exact(p, s[e], slope2, pos - static_cast<float>(key), bent);
      const float full = exp2f(x - l2) * (dp[e] + nd) * bent;
      const float ds = key < seen.lo || key >= seen.hi ? 0.f : full;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma_f32x4(kc[e][dt], ds, acc[dt]);
    }
  }
  sums.put(wave, l16, g, acc);
  __syncthreads();
  for (int x = threadIdx.x; x < 16 * DM; x += 256) {
    const int n = x / DM, d = x % DM;
    if (q0 + n >= p.Sq || d >= p.D) continue;
    const float val = (sums.v[0][n][d] + sums.v[1][n][d]) + (sums.v[2][n][d] + sums.v[3][n][d]);
    if (!(fabsf(val) < __builtin_inff())) atomicOr(&bad, 1u << n);
    dq[b * p.o_sb + (q0 + n) * p.o_ss + h * p.o_sh + d] = val * p.scale;
  }
  __syncthreads();
  for (uint32_t left = bad; left != 0; left &= left - 1) {
    const int n = __ffs(left) - 1;
    const float row_nd = __shfl(nd, n, 64);
    if ((n & 3) == wave) scored_row_dq<float>(p, q, k, v, dout, lse2[row + q0 + n], row_nd, dq, b, h, q0 + n, lane);
  }
}

// dK and dV of 16 keys; the waves take the (query head, 16 queries) pairs in turn
template <int DM>
__global__ __launch_bounds__(256) void scored_f32_dkdv_kernel(ScoredShape p, const float* __restrict__ q,
                                                              const float* __restrict__ k,
                                                              const float* __restrict__ v,
                                                              const float* __restrict__ dout,
                                                              const float* __restrict__ lse2,
                                                              const float* __restrict__ ndelta,
                                                              float* __restrict__ dk, float* __restrict__ dv,
                                                              int vec) {
  constexpr int DT = DM / 16;
  __shared__ __attribute__((aligned(16))) WaveSums<DM> sums;
  __shared__ uint32_t bad;
  if (threadIdx.x == 0) bad = 0;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int j0 = 16 * static_cast<int>(blockIdx.x), hk = blockIdx.y, b = blockIdx.z;
  const int group = p.Hq / p.Hkv;
  const int key = min(j0 + l16, p.Sk - 1);
  const RowView r = row_view(p, b);
  const Span seen = seen_by(p, r, key);
  const int q_lo = __builtin_amdgcn_readlane(seen.lo, 0), q_hi = __builtin_amdgcn_readlane(seen.hi, 15);
  f32x4 kf[DT], vf[DT], qf[DT], df[DT], ka[DT], va[DT];
  load_row<float, DM>(k + b * p.k_sb + key * p.k_ss + hk * p.k_sh, true, p.D, g, vec, kf);
  load_row<float, DM>(v + b * p.v_sb + key * p.v_ss + hk * p.v_sh, true, p.D, g, vec, vf);
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) ka[dt] = va[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int per_head = (q_hi - q_lo + 15) / 16;
  float qcol[4][DT], dcol[4][DT], ls[4], ns[4];
  int h = 0, i0 = 0;  // of the tile loaded last
  auto load = [&](int t) {
    h = hk * group + t / per_head;
    i0 = q_lo + 16 * (t % per_head);
    const int64_t i = min(i0 + l16, q_hi - 1);
    const float* qb = q + b * p.q_sb + h * p.q_sh;
    const float* db = dout + b * p.o_sb + h * p.o_sh;
    load_row<float, DM>(qb + i * p.q_ss, i0 + l16 < q_hi, p.D, g, vec, qf);
    load_row<float, DM>(db + i * p.o_ss, i0 + l16 < q_hi, p.D, g, vec, df);
    load_cols<float, DM>(qb, p.q_ss, i0, q_hi, p.D, l16, g, qcol);
    load_cols<float, DM>(db, p.o_ss, i0, q_hi, p.D, l16, g, dcol);
    const int64_t row = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = min(i0 + 4 * g + e, q_hi - 1);
      ls[e] = lse2[row + n];
      ns[e] = ndelta[row + n];
    }
  };
  const int total = group * per_head;
  if (wave < total) load(wave);
  for (int t = wave; t < total; t += 4) {
    const f32x4 s = row_product<DM>(qf, kf), dp = row_product<DM>(df, vf);
    const float slope2 = slope2_of(p, h);
    const int ci = i0;
    float qc[4][DT], dc[4][DT], lc[4], nc[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lc[e] = ls[e];
      nc[e] = ns[e];
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        qc[e][dt] = qcol[e][dt];
        dc[e][dt] = dcol[e][dt];
      }
    }
    if (t + 4 < total) load(t + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = ci + 4 * g + e;
      float bent;
      const float x = score_exact(p, s[e], slope2, bias_pos(p, r, i) - static_cast<float>(key), bent);
      const bool hidden = i < seen.lo || i >= seen.hi || lc[e] == -__builtin_inff();
      const float w = exp2f(x - lc[e]);
      const float pv = hidden ? 0.f : w, ds = hidden ? 0.f : w * (dp[e] + nc[e]) * bent;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        va[dt] = mfma_f32x4(dc[e][dt], pv, va[dt]);
        ka[dt] = mfma_f32x4(qc[e][dt], ds, ka[dt]);
      }
    }
  }
  // dK, then dV through the same LDS rows
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    sums.put(wave, l16, g, w == 0 ? ka : va);
    __syncthreads();
    for (int x = threadIdx.x; x < 16 * DM; x += 256) {
      const int n = x / DM, d = x % DM;
      if (j0 + n >= p.Sk || d >= p.D) continue;
      const float val = (sums.v[0][n][d] + sums.v[1][n][d]) + (sums.v[2][n][d] + sums.v[3][n][d]);
      if (!(fabsf(val) < __builtin_inff())) atomicOr(&bad, 1u << n);
      (w == 0 ? dk : dv)[b * p.g_sb + (j0 + n) * p.g_ss + hk * p.g_sh + d] = w == 0 ? val * p.scale : val;
    }
    __syncthreads();
  }
  for (uint32_t left = bad; left != 0; left &= left - 1) {
    const int n = __ffs(left) - 1;
    if ((n & 3) == wave) scored_row_dkdv<float>(p, q, k, v, dout, lse2, ndelta, dk, dv, b, hk, j0 + n, lane);
  }
}

// 16-byte row loads: every row of every tensor starts at a multiple of 4 elements
int rows_vec(const ScoredShape& p, std::initializer_list<const void*> tensors) {
  if (p.D % 4 != 0) return 0;
  for (int64_t s : {p.q_sb, p.q_ss, p.q_sh, p.k_sb, p.k_ss, p.k_sh, p.v_sb, p.v_ss, p.v_sh, p.o_sb, p.o_ss, p.o_sh})
    if (s % 4 != 0) return 0;
  for (const void* t : tensors)
    if (!aligned16(t)) return 0;
  return 1;
}

}  // namespace

int scored_f32_fwd(const ScoredShape& p, const float* q, const float* k, const float* v, float* o, float* lse2,
                   hipStream_t stream) {
  const int vec = rows_vec(p, {q, k, v});
  const dim3 grid((p.Sq + 15) / 16, p.Hq, p.B);
  if (p.D <= 64)
    hipLaunchKernelGGL(scored_f32_fwd_kernel<64>, grid, dim3(256), 0, stream, p, q, k, v, o, lse2, vec);
  else
    hipLaunchKernelGGL(scored_f32_fwd_kernel<128>, grid, dim3(256), 0, stream, p, q, k, v, o, lse2, vec);
  NMB_CHECK_LAUNCH("attn_scored_fwd(f32)");
  return NMB_OK;
}

int scored_f32_bwd(const ScoredShape& p, const float* q, const float* k, const float* v, const float* o,
                   const float* dout, const float* lse2, float* ndelta, float* dq, float* dk, float* dv,
                   hipStream_t stream) {
  const int vec = rows_vec(p, {q, k, v, o, dout});
  if (p.Sq > 0) {
    const dim3 grid((p.Sq + 15) / 16, p.Hq, p.B);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, q, k, v, o, dout, lse2, ndelta, dq, vec);
    };
    if (p.D <= 64) go(scored_f32_dq_kernel<64>); else go(scored_f32_dq_kernel<128>);
    NMB_CHECK_LAUNCH("attn_scored_bwd(f32 dq)");
  }
  if (p.Sk > 0) {
    const dim3 grid((p.Sk + 15) / 16, p.Hkv, p.B);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, q, k, v, dout, lse2, ndelta, dk, dv, vec);
    };
    if (p.D <= 64) go(scored_f32_dkdv_kernel<64>); else go(scored_f32_dkdv_kernel<128>);
    NMB_CHECK_LAUNCH("attn_scored_bwd(f32 dkdv)");
  }
  return NMB_OK;
}

}  // namespace nmb
