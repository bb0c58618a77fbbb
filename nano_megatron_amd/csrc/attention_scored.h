// Scored attention: which keys a query sees, how a score is formed, and the
// attention of one row at a time.
//
//   x = scale q.k;  x <- cap tanh(x / cap);  x <- x - slope_h |pos_q - pos_k|;
//   P = softmax of x over the visible keys;  o = P v
//
// Key j has position j, query i of row b position offset_b + i.  A key is
// visible if the two positions lie in one document (a run of equal,
// non-negative ids), if pos_k <= pos_q or pos_k < prefix_b (causal), and if
// |pos_q - pos_k| < window.  Each of these leaves a query an interval of keys
// and a key an interval of queries, whose ends do not decrease from one query
// (key) to the next.  So a tile of rows needs the ends of its first and last
// row only to know which tiles of the other side it meets and which of those
// are visible throughout, and no mask is ever stored.
#pragma once

#include <math.h>

#include "common.h"

namespace nmb {

struct ScoredShape {
  int B, Hq, Hkv, Sq, Sk, D;
  int64_t q_sb, q_ss, q_sh;  // element strides of (batch, token, head)
  int64_t k_sb, k_ss, k_sh;
  int64_t v_sb, v_ss, v_sh;
  int64_t o_sb, o_ss, o_sh;  // o, dO and dQ
  int64_t g_sb, g_ss, g_sh;  // dK and dV
  float scale;
  float c;           // scale log2(e)
  float cap_in;      // 2 log2(e) scale / cap: exp2(cap_in s) = e^(2 x / cap)
  float cap_out;     // cap log2(e)
  int causal;
  int64_t window;    // 0: none
  int64_t q_offset;
  const float* slopes;     // [Hq] or null
  const int32_t* offsets;  // [B] or null
  const int32_t* prefix;   // [B] or null
  const int2* runs;        // [B][Sk] {first token, one past the last} of each token's
                           // document, or null; no document: {first token of the run, ~end}
};

// the fp32 kernels (attention_scored_f32.hip)
int scored_f32_fwd(const ScoredShape& p, const float* q, const float* k, const float* v, float* o, float* lse2,
                   hipStream_t stream);
int scored_f32_bwd(const ScoredShape& p, const float* q, const float* k, const float* v, const float* o,
                   const float* dout, const float* lse2, float* ndelta, float* dq, float* dk, float* dv,
                   hipStream_t stream);

namespace {

constexpr float kToLog2 = 1.4426950408889634f;  // log2(e)

// What a row of the batch adds to the shape.
struct RowView {
  int64_t offset;  // position of query 0
  int prefix;
  const int2* runs;
};

__device__ __forceinline__ RowView row_view(const ScoredShape& p, int b) {
  RowView r;
  r.offset = p.offsets != nullptr ? p.offsets[b] : p.q_offset;
  r.prefix = p.prefix != nullptr ? p.prefix[b] : 0;
  r.runs = p.runs != nullptr ? p.runs + static_cast<int64_t>(b) * p.Sk : nullptr;
  return r;
}

struct Span {
  int lo, hi;  // [lo, hi), empty if hi <= lo
};

// The keys that query i sees, within [0, Sk].  Both ends are non-decreasing in i.
__device__ __forceinline__ Span seen_keys(const ScoredShape& p, const RowView& r, int i) {
  const int64_t pos = r.offset + i;
  int64_t lo = 0, hi = p.Sk;
  if (r.runs != nullptr) {
    if (pos < 0) return Span{0, 0};
    if (pos >= p.Sk) return Span{p.Sk, p.Sk};
    const int2 run = r.runs[pos];
    if (run.y < 0) {
      const int at = run.x < 0 ? 0 : (run.x < p.Sk ? run.x : p.Sk);
      return Span{at, at};
    }
    lo = run.x > 0 ? run.x : 0;  // (inside the row whatever a caller's runs hold)
    hi = run.y < p.Sk ? run.y : p.Sk;
  }
  if (p.causal) {
    const int64_t c = pos + 1 > r.prefix ? pos + 1 : r.prefix;
    hi = c < hi ? c : hi;
  }
  if (p.window > 0) {
    lo = pos - p.window + 1 > lo ? pos - p.window + 1 : lo;
    hi = pos + p.window < hi ? pos + p.window : hi;
  }
  lo = lo < p.Sk ? lo : p.Sk;
  hi = hi > lo ? hi : lo;
  return Span{static_cast<int>(lo), static_cast<int>(hi)};
}

// The queries that see key j, within [0, Sq].  Both ends are non-decreasing in j.
__device__ __forceinline__ Span seen_by(const ScoredShape& p, const RowView& r, int j) {
  int64_t lo = r.offset, hi = r.offset + p.Sq;  // positions
  bool none = false;
  if (r.runs != nullptr) {
    const int2 run = r.runs[j];
    none = run.y < 0;
    lo = run.x > lo ? run.x : lo;
    const int64_t end = none ? run.x : run.y;
    hi = end < hi ? end : hi;
  }
  if (!none) {
    if (p.causal && j >= r.prefix) lo = j > lo ? j : lo;
    if (p.window > 0) {
      lo = j - p.window + 1 > lo ? j - p.window + 1 : lo;
      hi = j + p.window < hi ? j + p.window : hi;
    }
  }
  lo -= r.offset;
  hi -= r.offset;
  lo = lo < p.Sq ? lo : p.Sq;
  hi = hi > 0 ? hi : 0;
  hi = hi > lo ? hi : lo;
  return Span{static_cast<int>(lo), static_cast<int>(hi)};
}

// The position that the distance bias of query i counts from.  Left of the
// first or right of the last key the distance to every key grows alike, which
// the softmax does not see, so it counts from that key: the bias, and with it
// the rounding of the score it is added to, stays as small as it can be.
__device__ __forceinline__ float bias_pos(const ScoredShape& p, const RowView& r, int i) {
  int64_t pos = r.offset + i;
  pos = pos < 0 ? 0 : (pos >= p.Sk ? p.Sk - 1 : pos);
  return static_cast<float>(pos);
}

// cap log2(e) tanh(scale s / cap), and the derivative 1 - tanh^2 of the cap there
__device__ __forceinline__ float bend_exact(const ScoredShape& p, float s, float& bent) {
  const float t = tanhf(s * p.scale * (kToLog2 / p.cap_out));
  bent = 1.f - t * t;
  return p.cap_out * t;
}

// The score in base 2 of raw product s, and the derivative of the cap there.
__device__ __forceinline__ float score_exact(const ScoredShape& p, float s, float slope2, float dist, float& bent) {
  bent = 1.f;
  const float x = p.cap_out > 0.f ? bend_exact(p, s, bent) : s * p.c;
  return fmaf(-slope2, fabsf(dist), x);
}

__device__ __forceinline__ float slope2_of(const ScoredShape& p, int h) {
  return p.slopes != nullptr ? p.slopes[h] * kToLog2 : 0.f;
}

// ------------------------------------------------------------ row by row
// A wavefront per query row (dK / dV: per key), lane l holding head-dim
// elements l and l + 64.  Only visible keys and queries are read.  These are
// the rows that the tiled kernels run again where a result is NaN: their
// matrix products multiply hidden rows of a tile by zero, and 0 x NaN (or
// infinity) is NaN, so a document may not be spoilt by its neighbour's.
// A key takes a wave about 1 us here (two sums over the wave and the score's
// functions, one key after the other): right, not fast.  Rows that are NaN
// themselves end at once; 24 tokens of NaN padding in the middle of rows, whose
// neighbours in the same tiles come here, take 16 x 16 heads x 512 in documents of
// 200 from 31 to 750 us forward and 71 to 3,600 backward, and 16 heads of 128 x 8192 in
// documents of 3000 from 140 to 1,090 and 370 to 50,000.  Padding at the end of rows costs
// nothing (58 and 109 us against 57 and 112): no tile reaches past its last visible row.
template <typename T>
__device__ __forceinline__ float scored_dot(const T* a, const T* b, int D, int lane) {
  float s = 0.f;
  for (int d = lane; d < D; d += 64) s = fmaf(to_f32(a[d]), to_f32(b[d]), s);
  return wave_sum(s);
}

template <typename T>
__device__ __forceinline__ void scored_store(T* row, const float (&v)[2], float f, int D, int lane) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const int d = lane + 64 * c;
    if (d < D) row[d] = from_f32<T>(v[c] * f);
  }
}

// the rows (bits 0 .. 15) that a lane of any of the wave's four 16-lane groups names
__device__ __forceinline__ uint32_t named_rows(uint64_t lanes) {
  const uint32_t x = static_cast<uint32_t>(lanes) | static_cast<uint32_t>(lanes >> 32);
  return (x | x >> 16) & 0xffffu;
}

// o (o_low: what its rounding cut off, nullable) and the base-2 log-sum-exp of query
// i of head h of row b
template <typename T>
__device__ void scored_row_fwd(const ScoredShape& p, const T* q, const T* k, const T* v, T* o, T* o_low, float* lse2,
                               int b, int h, int i, int lane) {
  const RowView r = row_view(p, b);
  const Span seen = seen_keys(p, r, i);
  const int hk = h / (p.Hq / p.Hkv);
  const T* qr = q + b * p.q_sb + i * p.q_ss + h * p.q_sh;
  const T* kb = k + b * p.k_sb + hk * p.k_sh;
  const T* vb = v + b * p.v_sb + hk * p.v_sh;
  const float slope2 = slope2_of(p, h), pos = bias_pos(p, r, i);
  float m = -__builtin_inff(), l = 0.f, acc[2] = {0.f, 0.f};
  for (int j = seen.lo; j < seen.hi; ++j) {
    float bent;
    const float x = score_exact(p, scored_dot(qr, kb + j * p.k_ss, p.D, lane), slope2, pos - j, bent);
    const float mn = fmaxf(m, x);
    // no score above -inf yet: weight 0
    const float alpha = mn == -__builtin_inff() ? 1.f : exp2f(m - mn);
    const float w = mn == -__builtin_inff() && x == x ? 0.f : exp2f(x - mn);
    m = mn;
    l = fmaf(l, alpha, w);
    const T* vr = vb + j * p.v_ss;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int d = lane + 64 * c;
      if (d < p.D) acc[c] = fmaf(acc[c], alpha, w * to_f32(vr[d]));
    }
    if (l != l) break;  // NaN: sum and outputs stay so
  }
  if (l != l) acc[0] = acc[1] = l;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int64_t at = b * p.o_sb + i * p.o_ss + h * p.o_sh;
  scored_store(o + at, acc, inv, p.D, lane);
  if (o_low != nullptr) {
#pragma unroll
    for (int c = 0; c < 2; ++c) acc[c] = acc[c] * inv - round_as<T>(acc[c] * inv);
    scored_store(o_low + at, acc, 1.f, p.D, lane);
  }
  if (lane == 0) lse2[(static_cast<int64_t>(b) * p.Hq + h) * p.Sq + i] = l == 0.f ? -__builtin_inff() : m + log2f(l);
}

// dQ of query i from its lse2 and ndelta = -rowsum(dO o)
template <typename T>
__device__ void scored_row_dq(const ScoredShape& p, const T* q, const T* k, const T* v, const T* dout, float lse2,
                              float ndelta, T* dq, int b, int h, int i, int lane) {
  const RowView r = row_view(p, b);
  const Span seen = seen_keys(p, r, i);
  const int hk = h / (p.Hq / p.Hkv);
  const T* qr = q + b * p.q_sb + i * p.q_ss + h * p.q_sh;
  const int64_t row = b * p.o_sb + i * p.o_ss + h * p.o_sh;
  const T* kb = k + b * p.k_sb + hk * p.k_sh;
  const T* vb = v + b * p.v_sb + hk * p.v_sh;
  const float slope2 = slope2_of(p, h), pos = bias_pos(p, r, i);
  float acc[2] = {0.f, 0.f};
  if (lse2 != -__builtin_inff()) {
    for (int j = seen.lo; j < seen.hi; ++j) {
      const T* kr = kb + j * p.k_ss;
      float bent;
      const float x = score_exact(p, scored_dot(qr, kr, p.D, lane), slope2, pos - j, bent);
      const float ds = exp2f(x - lse2) * (scored_dot(dout + row, vb + j * p.v_ss, p.D, lane) + ndelta) * bent;
      if (ds != ds) {  // so are all sums, whatever follows
        acc[0] = acc[1] = ds;
        break;
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = lane + 64 * c;
        if (d < p.D) acc[c] = fmaf(ds, to_f32(kr[d]), acc[c]);
      }
    }
  }
  scored_store(dq + row, acc, p.scale, p.D, lane);
}

// Whether one of the queries `seen` of the group's heads makes dK and dV NaN throughout:
// its log-sum-exp is NaN, or its whole row of dO (and so its ndelta).  64 queries at a
// time, so that a NaN far into a long row is not walked to one query after the other.
template <typename T>
__device__ bool scored_lost(const ScoredShape& p, const T* dout, const float* lse2, const float* ndelta, int b, int h0,
                            int group, const Span& seen, int lane) {
  for (int h = h0; h < h0 + group; ++h) {
    const int64_t stat = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;
    for (int i0 = seen.lo; i0 < seen.hi; i0 += 64) {
      const int i = i0 + lane;
      const float l2 = i < seen.hi ? lse2[stat + i] : 0.f, nd = i < seen.hi ? ndelta[stat + i] : 0.f;
      if (__any(l2 != l2)) return true;
      const uint64_t rows = __ballot(nd != nd && l2 != -__builtin_inff());
      if (rows == 0) continue;
      const T* dr = dout + b * p.o_sb + (i0 + __ffsll(static_cast<unsigned long long>(rows)) - 1) * p.o_ss + h * p.o_sh;
      bool all = true;
      for (int d = lane; d < p.D; d += 64) all = all && to_f32(dr[d]) != to_f32(dr[d]);
      if (__all(all)) return true;
    }
  }
  return false;
}

// dK and dV of key j of KV head hk
template <typename T>
__device__ void scored_row_dkdv(const ScoredShape& p, const T* q, const T* k, const T* v, const T* dout,
                                const float* lse2, const float* ndelta, T* dk, T* dv, int b, int hk, int j, int lane) {
  const RowView r = row_view(p, b);
  const Span seen = seen_by(p, r, j);
  const T* kr = k + b * p.k_sb + j * p.k_ss + hk * p.k_sh;
  const T* vr = v + b * p.v_sb + j * p.v_ss + hk * p.v_sh;
  const int group = p.Hq / p.Hkv;
  float ka[2] = {0.f, 0.f}, va[2] = {0.f, 0.f};
  bool lost = scored_lost(p, dout, lse2, ndelta, b, hk * group, group, seen, lane);
  if (lost) ka[0] = ka[1] = va[0] = va[1] = __builtin_nanf("");
  for (int h = hk * group; h < (hk + 1) * group && !lost; ++h) {
    const float slope2 = slope2_of(p, h);
    const int64_t stat = (static_cast<int64_t>(b) * p.Hq + h) * p.Sq;
    for (int i = seen.lo; i < seen.hi; ++i) {
      const float l2 = lse2[stat + i];
      if (l2 == -__builtin_inff()) continue;
      const T* qr = q + b * p.q_sb + i * p.q_ss + h * p.q_sh;
      const T* dr = dout + b * p.o_sb + i * p.o_ss + h * p.o_sh;
      float bent;
      const float x = score_exact(p, scored_dot(qr, kr, p.D, lane), slope2, bias_pos(p, r, i) - j, bent);
      const float w = exp2f(x - l2);
      const float ds = w * (scored_dot(dr, vr, p.D, lane) + ndelta[stat + i]) * bent;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = lane + 64 * c;
        if (d < p.D) {
          ka[c] = fmaf(ds, to_f32(qr[d]), ka[c]);
          va[c] = fmaf(w, to_f32(dr[d]), va[c]);
        }
      }
      if (ds != ds) {  // dK is NaN throughout; done where dV is too
        bool all = true;
#pragma unroll
        for (int c = 0; c < 2; ++c) all = all && (lane + 64 * c >= p.D || va[c] != va[c]);
        lost = __all(all);
        if (lost) break;
      }
    }
  }
  const int64_t out = b * p.g_sb + j * p.g_ss + hk * p.g_sh;
  scored_store(dk + out, ka, p.scale, p.D, lane);
  scored_store(dv + out, va, 1.f, p.D, lane);
}

}  // namespace
}  // namespace nmb
