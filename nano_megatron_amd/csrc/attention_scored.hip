// Attention with capped scores, a distance bias and interval masks (documents,
// prefix, window), forward and backward, for gfx950.  attention_scored.h holds
// the mathematics.
#include <algorithm>

#include "attention_scored_tiles.h"

namespace nmb {
namespace {

// ------------------------------------------------------------ documents
// {start, end} of the run of equal ids that each token lies in ({start, ~end}
// where the id is negative).  A workgroup per row: the start of a token's run
// is the largest start of a run at or before it, the end the smallest after
// it, each by a scan over the row, forwards then backwards, 1,024 threads of 8
// tokens at a time.
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

// ------------------------------------------------------------ row kernels
template <typename T>
__global__ __launch_bounds__(256) void scored_rows_fwd_kernel(ScoredShape p, const T* q, const T* k, const T* v, T* o,
                                                              float* lse2) {
  const int i = static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6);
  const int h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  if (i < p.Sq) scored_row_fwd(p, q, k, v, o, lse2, b, h, i, static_cast<int>(threadIdx.x & 63));
}

// delta = rowsum(dO o) and dQ
template <typename T>
__global__ __launch_bounds__(256) void scored_rows_dq_kernel(ScoredShape p, const T* q, const T* k, const T* v,
                                                             const T* o, const T* dout, const float* lse2,
                                                             float* delta, T* dq) {
  const int i = static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6);
  const int h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  if (i >= p.Sq) return;
  const int lane = static_cast<int>(threadIdx.x & 63);
  const int64_t row = b * p.o_sb + i * p.o_ss + h * p.o_sh;
  const int64_t stat = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq + i;
  const float dl = scored_dot(o + row, dout + row, p.D, lane);
  if (lane == 0) delta[stat] = dl;
  scored_row_dq(p, q, k, v, dout, lse2[stat], dl, dq, b, h, i, lane);
}

template <typename T>
__global__ __launch_bounds__(256) void scored_rows_dkdv_kernel(ScoredShape p, const T* q, const T* k, const T* v,
                                                               const T* dout, const float* lse2, const float* delta,
                                                               T* dk, T* dv) {
  const int j = static_cast<int>(blockIdx.x) * 4 + static_cast<int>(threadIdx.x >> 6);
  const int hk = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  if (j < p.Sk)
    scored_row_dkdv(p, q, k, v, dout, lse2, delta, dk, dv, b, hk, j, static_cast<int>(threadIdx.x & 63));
}

// ------------------------------------------------------------ forward
// bf16.  A workgroup owns 64 TQ queries of one head: column tile t of wave w is
// queries 64 t + 16 w .. + 15 of them, so that under a causal mask the waves
// have about the same work.  The key tiles that any of its queries sees stream
// through LDS.  S^T = K Q^T puts all scores of a query in the lanes l, l + 16,
// l + 32, l + 48, where the statistics are plain registers, and exp2 of them
// is, rounded to bf16, the operand of O^T += V^T P as it stands (the 32-deep
// index of that product runs over the keys in the order the scores hold them).
// The probabilities are rounded to bf16 (half a step, 2^-8) because they are an
// operand of the bf16 matrix instruction; sums, maxima and outputs stay fp32.
template <int D, int TQ, class M>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void scored_fwd_kernel(ScoredShape p, const bf16* __restrict__ q,
                                                                          const bf16* __restrict__ k,
                                                                          const bf16* __restrict__ v,
                                                                          bf16* __restrict__ o,
                                                                          float* __restrict__ lse2, int n_qt,
                                                                          int items, int per_xcd) {
  constexpr int BQ = 64 * TQ, KS = D / 32, DT = D / 16;
  constexpr int kStages = D == 64 ? 3 : 2;  // 48 KB, 64 KB
  using Tile = RowTile<D>;
  using Load = RowLoader<D, 4>;
  __shared__ __attribute__((aligned(1024))) bf16 sK[kStages][Tile::kElems];
  __shared__ __attribute__((aligned(1024))) bf16 sV[kStages][Tile::kElems];
  const int w = xcd_item(items, per_xcd);
  if (w < 0) return;
  const int bh = w / n_qt, q0 = (n_qt - 1 - w % n_qt) * BQ;  // the most keys first
  const int b = bh / p.Hq, h = bh % p.Hq, hk = h / (p.Hq / p.Hkv);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
  const int l16 = lane & 15, g = lane >> 4;
  const RowView r = row_view(p, b);
  const float slope2 = M::BIAS ? slope2_of(p, h) : 0.f;

  const bf16* qb = q + b * p.q_sb + h * p.q_sh;
  bf16x8 qf[TQ][KS];
  ColSpan span[TQ];
  float pos[TQ], m[TQ], l[TQ];
  f32x4 acc[TQ][DT];
#pragma unroll
  for (int t = 0; t < TQ; ++t) {
    const int i = min(q0 + 64 * t + 16 * wave + l16, p.Sq - 1);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      qf[t][ks] = row_frag(qb + static_cast<int64_t>(i) * p.q_ss, ks * 32 + g * 8, p.D, true);
    span[t] = col_span(seen_keys(p, r, i));
    pos[t] = M::BIAS ? bias_pos(p, r, i) : 0.f;
    m[t] = M::FIXED ? 0.f : -__builtin_inff();
    l[t] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[t][dt] = zero4();
  }
  const int k_lo = __builtin_amdgcn_readfirstlane(seen_keys(p, r, q0).lo);
  const int k_hi = __builtin_amdgcn_readfirstlane(seen_keys(p, r, min(q0 + BQ, p.Sq) - 1).hi);
  const int n_kt = (k_hi - k_lo + 63) / 64;
  // everything above has landed before the first tile is on its way: the
  // compiler counts only its own loads and would wait for all
  wait_vmcnt<0>();
  Load lk, lv;
  lk.init(p.k_ss, p.D, wave, lane);
  lv.init(p.v_ss, p.D, wave, lane);
  const bf16* kb = k + b * p.k_sb + hk * p.k_sh;
  const bf16* vb = v + b * p.v_sb + hk * p.v_sh;
  auto issue = [&](int kt) {  // past the last tile: zeros, so that the waits stay constant
    const int k0 = k_lo + 64 * kt, n = kt < n_kt ? k_hi - k0 : 0;
    lk.issue(kb + k0 * p.k_ss, sK[kt % kStages], 0, n, wave);
    lv.issue(vb + k0 * p.v_ss, sV[kt % kStages], 0, n, wave);
  };
#pragma unroll
  for (int st = 0; st < kStages - 1; ++st) issue(st);

  for (int kt = 0; kt < n_kt; ++kt) {
    // this wave's loads of tile kt have landed, after the barrier everyone's;
    // and nobody reads the stage of tile kt - 1 any more
    tile_barrier<(kStages - 2) * 2 * Load::P>();
    issue(kt + kStages - 1);
    const bf16* tk = sK[kt % kStages];
    const bf16* tv = sV[kt % kStages];
    const int k0 = k_lo + 64 * kt;
    bool live[TQ], mask[TQ];
    bool any = false;
#pragma unroll
    for (int t = 0; t < TQ; ++t) {
      live[t] = k0 < span[t].hi_max && k0 + 64 > span[t].lo_min && q0 + 64 * t + 16 * wave < p.Sq;
      mask[t] = k0 < span[t].lo_max || k0 + 64 > span[t].hi_min;
      any = any || live[t];
    }
    if (!any) continue;
    f32x4 s[TQ][4];
#pragma unroll
    for (int t = 0; t < TQ; ++t)
#pragma unroll
      for (int mk = 0; mk < 4; ++mk) s[t][mk] = zero4();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      bf16x8 kk[4];
#pragma unroll
      for (int mk = 0; mk < 4; ++mk) kk[mk] = Tile::row8(tk, mk * 16 + l16, ks * 32 + g * 8);
#pragma unroll
      for (int t = 0; t < TQ; ++t)
        if (live[t]) {
#pragma unroll
          for (int mk = 0; mk < 4; ++mk) s[t][mk] = mfma16(kk[mk], qf[t][ks], s[t][mk]);
        }
    }
    bf16x8 pf[TQ][2];
#pragma unroll
    for (int t = 0; t < TQ; ++t) {
      if (!live[t]) continue;
      // lane: key k0 + 16 mk + 4 g + e of its query
      if constexpr (M::CAP || M::BIAS) {
        const float dist = pos[t] - static_cast<float>(k0 + 4 * g);
#pragma unroll
        for (int mk = 0; mk < 4; ++mk)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = M::CAP ? fmaf(-2.f * p.cap_out, cap_t(p, s[t][mk][e]), p.cap_out) : s[t][mk][e] * p.c;
            if constexpr (M::BIAS) x = fmaf(-slope2, fabsf(dist - static_cast<float>(16 * mk + e)), x);
            s[t][mk][e] = x;
          }
      }
      if (mask[t]) {
        const int lo = span[t].mine.lo - k0 - 4 * g, hi = span[t].mine.hi - k0 - 4 * g;
#pragma unroll
        for (int mk = 0; mk < 4; ++mk)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = s[t][mk][e];
            s[t][mk][e] = 16 * mk + e < lo || 16 * mk + e >= hi ? -__builtin_inff() : x;
          }
      }
      if constexpr (!M::FIXED) {
        // the raw products are ordered as their scores (c > 0) where nothing bends them
        constexpr bool RAW = !M::CAP && !M::BIAS;
        const float unit = RAW ? p.c : 1.f;
        float top = -__builtin_inff();
#pragma unroll
        for (int mk = 0; mk < 4; ++mk)
#pragma unroll
          for (int e = 0; e < 4; ++e) top = fmaxf(top, s[t][mk][e]);
        top = xor32_max(xor16_max(top));
        // the running maximum moves only when a tile's exceeds it by 2^8: until
        // then the probabilities are at most that, which fp32 sums can hold
        const bool grow = top > m[t] && (m[t] == -__builtin_inff() || (top - m[t]) * unit > 8.f);
        if (__any(grow)) {
          const float alpha = grow ? fast_exp2((m[t] - top) * unit) : 1.f;
          m[t] = grow ? top : m[t];
          l[t] *= alpha;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) acc[t][dt] *= alpha;
        }
        const float off = m[t] == -__builtin_inff() ? 0.f : -m[t] * unit;
#pragma unroll
        for (int mk = 0; mk < 4; ++mk)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[t][mk][e] = RAW ? fmaf(s[t][mk][e], p.c, off) : s[t][mk][e] + off;
      }
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = fast_exp2(s[t][2 * s2 + (e >> 2)][e & 3]);
          l[t] += x;
          pf[t][s2][e] = static_cast<bf16>(x);
        }
    }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      bf16x8 vv[2];
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) vv[s2] = Tile::col8(tv, 32 * s2, dt * 16, l16, g);
#pragma unroll
      for (int t = 0; t < TQ; ++t)
        if (live[t]) {
#pragma unroll
          for (int s2 = 0; s2 < 2; ++s2) acc[t][dt] = mfma16(vv[s2], pf[t][s2], acc[t][dt]);
        }
    }
  }
  wait_vmcnt<0>();  // no load may still write this workgroup's LDS when it ends
#pragma unroll
  for (int t = 0; t < TQ; ++t) {
    const int i = q0 + 64 * t + 16 * wave + l16;
    const float sum = xor32_sum(xor16_sum(l[t]));
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    const float unit = M::CAP || M::BIAS ? 1.f : p.c;
    bool fine = sum < __builtin_inff();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) fine = fine && fabsf(acc[t][dt][e]) < __builtin_inff();
    const uint32_t bad = rows_of(__ballot(!fine && i < p.Sq));
    if (i < p.Sq && (bad >> l16 & 1) == 0) {
      bf16* ob = o + b * p.o_sb + static_cast<int64_t>(i) * p.o_ss + h * p.o_sh;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = static_cast<bf16>(acc[t][dt][e] * inv);
        if (dt * 16 + g * 4 < p.D) *reinterpret_cast<bf16x4*>(ob + dt * 16 + g * 4) = x;
      }
      if (g == 0)
        lse2[(static_cast<int64_t>(b) * p.Hq + h) * p.Sq + i] = sum > 0.f ? fmaf(m[t], unit, log2f(sum)) : -__builtin_inff();
    }
    for (uint32_t left = bad; left != 0; left &= left - 1)  // not finite: on the visible keys alone
      scored_row_fwd(p, q, k, v, o, lse2, b, h, q0 + 64 * t + 16 * wave + __ffs(left) - 1, lane);
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
  NMB_REQUIRE(isfinite(sc->scale) && isfinite(sc->cap) && sc->cap >= 0.f,
              "scored attention: scale and cap must be finite, cap >= 0");
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
  p->window = sc->window;
  p->q_offset = sc->q_offset;
  p->slopes = sc->slopes;
  p->offsets = sc->offsets;
  p->prefix = sc->prefix;
  p->runs = reinterpret_cast<const int2*>(sc->runs);
  return NMB_OK;
}

template <typename T>
void rows_fwd_launch(const ScoredShape& p, const void* q, const void* k, const void* v, void* o, float* lse2,
                     hipStream_t stream) {
  hipLaunchKernelGGL((scored_rows_fwd_kernel<T>), dim3((p.Sq + 3) / 4, p.Hq, p.B), dim3(256), 0, stream, p,
                     static_cast<const T*>(q), static_cast<const T*>(k), static_cast<const T*>(v),
                     static_cast<T*>(o), lse2);
}

template <typename T>
int rows_bwd_launch(const ScoredShape& p, const void* q, const void* k, const void* v, const void* o, const void* dout,
                    const float* lse2, float* delta, void* dq, void* dk, void* dv, hipStream_t stream) {
  const T *qt = static_cast<const T*>(q), *kt = static_cast<const T*>(k), *vt = static_cast<const T*>(v),
          *dt = static_cast<const T*>(dout);
  if (p.Sq > 0)
    hipLaunchKernelGGL((scored_rows_dq_kernel<T>), dim3((p.Sq + 3) / 4, p.Hq, p.B), dim3(256), 0, stream, p, qt, kt,
                       vt, static_cast<const T*>(o), dt, lse2, delta, static_cast<T*>(dq));
  NMB_CHECK_LAUNCH("attn_scored_bwd(dq)");
  if (p.Sk > 0)
    hipLaunchKernelGGL((scored_rows_dkdv_kernel<T>), dim3((p.Sk + 3) / 4, p.Hkv, p.B), dim3(256), 0, stream, p, qt, kt,
                       vt, dt, lse2, delta, static_cast<T*>(dk), static_cast<T*>(dv));
  NMB_CHECK_LAUNCH("attn_scored_bwd(dkdv)");
  return NMB_OK;
}

// f(Mode): the compiled way of forming scores for p
template <class F>
void with_mode(const ScoredShape& p, F&& f) {
  const bool cap = p.cap_out > 0.f;
  // a cap too large for a fixed maximum runs as one with a bias of slope 0
  const bool bias = p.slopes != nullptr || p.cap_out > kFixedMax;
  if (cap && bias) f(Mode<true, true>{});
  else if (cap) f(Mode<true, false>{});
  else if (bias) f(Mode<false, true>{});
  else f(Mode<false, false>{});
}

void grid_of(int64_t items, int* per_xcd, dim3* grid) {
  *per_xcd = static_cast<int>((items + 7) / 8);
  *grid = dim3(static_cast<unsigned>(*per_xcd) * 8u);
}

int tiles_fwd_launch(const ScoredShape& p, const bf16* q, const bf16* k, const bf16* v, bf16* o, float* lse2,
                     hipStream_t stream) {
  // 128 queries per workgroup; 64 where those all run at once (3 workgroups per CU at D 64, 2 at 128)
  const int64_t heads = static_cast<int64_t>(p.Hq) * p.B;
  const bool small = (p.Sq + 63) / 64 * heads <= (p.D <= 64 ? 768 : 512);
  const int bq = small ? 64 : 128;
  const int n_qt = (p.Sq + bq - 1) / bq;
  NMB_REQUIRE(n_qt * heads < (int64_t{1} << 30), "attn_scored_fwd: problem too large for one launch");
  const int items = static_cast<int>(n_qt * heads);
  int per;
  dim3 grid;
  grid_of(items, &per, &grid);
  with_mode(p, [&](auto mode) {
    using M = decltype(mode);
    auto go = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, grid, dim3(256), 0, stream, p, q, k, v, o, lse2, n_qt, items, per);
    };
    if (p.D <= 64) {
      if (small) go(scored_fwd_kernel<64, 1, M>); else go(scored_fwd_kernel<64, 2, M>);
    } else {
      if (small) go(scored_fwd_kernel<128, 1, M>); else go(scored_fwd_kernel<128, 2, M>);
    }
  });
  NMB_CHECK_LAUNCH("attn_scored_fwd");
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
  if (forward != nullptr) *forward = 0;
  if (backward != nullptr) *backward = static_cast<size_t>(batch) * q_heads * seq_q * sizeof(float);
  return NMB_OK;
}

extern "C" int nmb_attn_scored_fwd(const void* q, const void* k, const void* v, void* o, float* lse2, int64_t batch,
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
  if (dtype == NMB_BF16)
    return nmb::tiles_fwd_launch(p, static_cast<const nmb::bf16*>(q), static_cast<const nmb::bf16*>(k),
                                 static_cast<const nmb::bf16*>(v), static_cast<nmb::bf16*>(o), lse2, stream);
  nmb::rows_fwd_launch<float>(p, q, k, v, o, lse2, stream);
  NMB_CHECK_LAUNCH("attn_scored_fwd");
  return NMB_OK;
}

extern "C" int nmb_attn_scored_bwd(const void* q, const void* k, const void* v, const void* o, const void* dout,
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
  size_t need = 0;
  nmb_attn_scored_workspace_bytes(batch, q_heads, kv_heads, seq_q, seq_k, head_dim, dtype, nullptr, &need);
  NMB_REQUIRE(workspace_bytes >= need && (need == 0 || workspace != nullptr),
              "attn_scored_bwd: workspace of %zu bytes is smaller than the %zu required", workspace_bytes, need);
  float* delta = static_cast<float*>(workspace);
  if (dtype == NMB_BF16) return nmb::rows_bwd_launch<nmb::bf16>(p, q, k, v, o, dout, lse2, delta, dq, dk, dv, stream);
  return nmb::rows_bwd_launch<float>(p, q, k, v, o, dout, lse2, delta, dq, dk, dv, stream);
}
