// Rotary positions for gfx950: both layouts, a part of the head, any frequencies, queries and
// keys in one launch (rope.hip is the reference's form: the half layout over the whole head,
// from tables of fp32 angles, rounded after every operation).
//
//   pair j of a token at position p: c = m cos(p f_j), s = m sin(p f_j)
//   (a, b) -> (a c - b s, b c + a s);  backward: the same with -s
//
// Half layout: a = x[j], b = x[j + R / 2]; interleaved: a = x[2 j], b = x[2 j + 1]; elements
// from R on are copied.  Formed in fp32, rounded once.
//
// Angles need no table and no bound on positions: p f_j / 2 pi is formed in 64 bits and only its
// fraction kept, in units of 2^-32 turns (so an angle is off by three roundings, 3 x 2^-53 of its
// size, 5e-11 turns at position a million for f = 1, and by 2^-33), then sine and cosine are
// their Taylor sums on an eighth of a turn to either side (the rest 2e-9 and 1e-10).
//
// A wavefront takes one token: lane u of each head's `units` reads two 16-byte vectors, adjacent
// lanes adjacent memory, and keeps its sines and cosines for all of its heads of q and k.
// What bounds it: HBM (32768 tokens of 32 + 8 heads of 128 in 118 us, 5.7 TB/s, where a large
// copy reaches 5.1; 8192 of 16 + 16 heads of 64, which the last-level cache holds, in 13.9).
#include "common.h"
#include "vec.h"

namespace nmb {
namespace {

struct RotaryArgs {
  const void* x[2];
  void* y[2];
  int64_t xs[2][3], ys[2][3];  // batch, token, head strides
  int heads[2];
  const double* freq;
  const void* positions;  // int32 or int64, or null
  int64_t pos_b, pos_s;
  const int32_t* offsets;  // [batch], or null
  int64_t offset;
  int dim, rot;
  float magnitude, sign;
  int pair_units, units, lanes, heads_at_once, slices;
  bool wide_positions;
  uint32_t waves;
  FastDiv by_slices, by_seq, by_lanes;
};

template <typename T, int V> struct Chunk { T e[V]; };

template <typename T, int V>
__device__ __forceinline__ Chunk<T, V> ld_chunk(const T* p) {  // any alignment
  Chunk<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void st_chunk(T* p, const Chunk<T, V>& r) {
  __builtin_memcpy(p, &r, sizeof(r));
}

// cos and sin of 2 pi times the fraction of `turns`
__device__ __forceinline__ void cos_sin(double turns, float& c, float& s) {
  const double fraction = __builtin_amdgcn_fract(turns);
  // the nearest of 2^32 parts of a turn, where 2^52 puts the last bit; a whole turn is none
  const double parts = fma(fraction, 4294967296.0, 4503599627370496.0);
  const uint32_t at = static_cast<uint32_t>(__builtin_bit_cast(uint64_t, parts));
  const uint32_t quarter = (at + 0x20000000u) >> 30;
  const float x = static_cast<float>(static_cast<int32_t>(at - (quarter << 30))) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float sn = fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  sn = fmaf(z, sn, 8.33333333e-3f);
  sn = fmaf(z, sn, -1.66666667e-1f);
  sn = fmaf(x * z, sn, x);
  float cs = fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  cs = fmaf(z, cs, -1.38888889e-3f);
  cs = fmaf(z, cs, 4.16666667e-2f);
  cs = fmaf(z, cs, -0.5f);
  cs = fmaf(z, cs, 1.f);
  const bool swap = quarter & 1;
  c = swap ? sn : cs;
  s = swap ? cs : sn;
  if ((quarter + 1) & 2) c = -c;
  if (quarter & 2) s = -s;
  if (!(fraction == fraction)) c = s = __builtin_nanf("");
}

// G heads' vectors of a lane are loaded before any is used.
template <typename T, int VP, bool INTERLEAVED, int G>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  const uint32_t wave = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (wave >= a.waves) return;
  const uint32_t lane = threadIdx.x & 63;
  const uint32_t token = fast_div(wave, a.by_slices);
  const int slice = static_cast<int>(wave - token * a.by_slices.d);
  const uint32_t b = fast_div(token, a.by_seq);
  const int64_t s = token - b * a.by_seq.d;
  const int hl = static_cast<int>(fast_div(lane, a.by_lanes));
  if (hl >= a.heads_at_once) return;
  int64_t pos;
  if (a.positions != nullptr) {
    const int64_t at = b * a.pos_b + s * a.pos_s;
    pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
  } else {
    pos = (a.offsets != nullptr ? a.offsets[b] : a.offset) + s;
  }
  const int all = a.heads[0] + a.heads[1], half = a.rot / 2, tail = a.dim - a.rot;
  for (int u = static_cast<int>(lane) - hl * a.lanes; u < a.units; u += a.lanes) {
    const bool turn = u < a.pair_units;
    int p0, p1;
    int j0 = 0;
    if (turn) {
      // the last unit is moved back to end with the pairs: pairs of two units get the same bits twice
      j0 = min(u * VP, half - VP);
      p0 = INTERLEAVED ? 2 * j0 : j0;
      p1 = INTERLEAVED ? 2 * j0 + VP : half + j0;
    } else {
      p0 = min(a.rot + (u - a.pair_units) * 2 * VP, a.dim - 2 * VP);
      p1 = p0 + VP;
    }
    if (!turn && tail < 2 * VP) {  // fewer elements than a unit
      for (int g = 0; g < G; ++g) {
        const int i = (slice * G + g) * a.heads_at_once + hl;
        if (i >= all) break;
        const int k = i >= a.heads[0];
        const int h = k ? i - a.heads[0] : i;
        const T* x = static_cast<const T*>(a.x[k]) + b * a.xs[k][0] + s * a.xs[k][1] + h * a.xs[k][2];
        T* y = static_cast<T*>(a.y[k]) + b * a.ys[k][0] + s * a.ys[k][1] + h * a.ys[k][2];
        for (int e = a.rot; e < a.dim; ++e) y[e] = x[e];
      }
      continue;
    }
    Chunk<T, VP> lo[G], hi[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int i = min((slice * G + g) * a.heads_at_once + hl, all - 1);
      const int k = i >= a.heads[0];
      const int h = k ? i - a.heads[0] : i;
      const T* x = static_cast<const T*>(k ? a.x[1] : a.x[0]) + b * (k ? a.xs[1][0] : a.xs[0][0]) +
                   s * (k ? a.xs[1][1] : a.xs[0][1]) + h * (k ? a.xs[1][2] : a.xs[0][2]);
      lo[g] = ld_chunk<T, VP>(x + p0);
      hi[g] = ld_chunk<T, VP>(x + p1);
    }
    float c[VP], sn[VP];
    if (turn) {
#pragma unroll
      for (int e = 0; e < VP; ++e) {
        cos_sin(static_cast<double>(pos) * (a.freq[j0 + e] * 0.15915494309189533577), c[e], sn[e]);
        c[e] *= a.magnitude;
        sn[e] *= a.magnitude * a.sign;
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int i = (slice * G + g) * a.heads_at_once + hl;
      if (i >= all) break;
      const int k = i >= a.heads[0];
      const int h = k ? i - a.heads[0] : i;
      T* y = static_cast<T*>(k ? a.y[1] : a.y[0]) + b * (k ? a.ys[1][0] : a.ys[0][0]) +
             s * (k ? a.ys[1][1] : a.ys[0][1]) + h * (k ? a.ys[1][2] : a.ys[0][2]);
      if (turn) {
        float v0[VP], v1[VP];
#pragma unroll
        for (int e = 0; e < VP; ++e) {
          v0[e] = to_f32(lo[g].e[e]);
          v1[e] = to_f32(hi[g].e[e]);
        }
#pragma unroll
        for (int e = 0; e < VP; ++e) {
          if constexpr (INTERLEAVED) {
            // elements 2 e and 2 e + 1 of the 2 VP
            float& p = 2 * e < VP ? v0[2 * e % VP] : v1[2 * e % VP];
            float& q = 2 * e + 1 < VP ? v0[(2 * e + 1) % VP] : v1[(2 * e + 1) % VP];
            const float x0 = p, x1 = q;
            p = fmaf(x0, c[e], -(x1 * sn[e]));
            q = fmaf(x1, c[e], x0 * sn[e]);
          } else {
            const float x0 = v0[e], x1 = v1[e];
            v0[e] = fmaf(x0, c[e], -(x1 * sn[e]));
            v1[e] = fmaf(x1, c[e], x0 * sn[e]);
          }
        }
#pragma unroll
        for (int e = 0; e < VP; ++e) {
          lo[g].e[e] = from_f32<T>(v0[e]);
          hi[g].e[e] = from_f32<T>(v1[e]);
        }
      }
      st_chunk<T, VP>(y + p0, lo[g]);
      st_chunk<T, VP>(y + p1, hi[g]);
    }
  }
}

template <typename T, int VP>
void rotary_launch(const RotaryArgs& a, bool interleaved, int g, dim3 grid, hipStream_t stream) {
#define NMB_LAUNCH(I, G) hipLaunchKernelGGL((rotary_kernel<T, VP, I, G>), grid, dim3(256), 0, stream, a)
  if (interleaved) {
    if (g == 4) NMB_LAUNCH(true, 4);
    else if (g == 2) NMB_LAUNCH(true, 2);
    else NMB_LAUNCH(true, 1);
  } else {
    if (g == 4) NMB_LAUNCH(false, 4);
    else if (g == 2) NMB_LAUNCH(false, 2);
    else NMB_LAUNCH(false, 1);
  }
#undef NMB_LAUNCH
}

template <typename T>
int rotary_impl(RotaryArgs a, int64_t batch, int64_t seq, bool interleaved, hipStream_t stream) {
  const int half = a.rot / 2, tail = a.dim - a.rot;
  int vp = VecTraits<T>::N;  // pairs of a unit: 16-byte vectors, or as many as there are
  while (vp > half) vp /= 2;
  a.pair_units = (half + vp - 1) / vp;
  a.units = a.pair_units + (tail + 2 * vp - 1) / (2 * vp);
  a.lanes = a.units < 64 ? a.units : 64;
  a.heads_at_once = 64 / a.lanes;
  const int64_t tokens = batch * seq;
  const int rounds = (a.heads[0] + a.heads[1] + a.heads_at_once - 1) / a.heads_at_once;
  // Up to four heads a lane, while that leaves every SIMD four wavefronts: fewer sines, more loads
  // under way (us, four, two and one: 32768 tokens of 32 + 8 heads of 128 118, 119 and 132, 8192 of
  // them 34, 35 and 37; 8192 of 16 + 16 heads of 64, which are two a lane, 13.9 and, one, 16.0).
  int g = 4;
  while (g > 1 && (g > rounds || tokens * ((rounds + g - 1) / g) < 4096)) g /= 2;
  a.slices = (rounds + g - 1) / g;
  // (fewer than 2^32 threads a launch)
  NMB_REQUIRE_SUPPORTED(tokens < (int64_t{1} << 26) / a.slices, "rotary: too many tokens and heads");
  a.waves = static_cast<uint32_t>(tokens * a.slices);
  a.by_slices = make_fastdiv(static_cast<uint32_t>(a.slices));
  a.by_seq = make_fastdiv(static_cast<uint32_t>(seq));
  a.by_lanes = make_fastdiv(static_cast<uint32_t>(a.lanes));
  const dim3 grid((a.waves + 3) / 4);
  if (vp == 8) {
    if constexpr (VecTraits<T>::N == 8) rotary_launch<T, 8>(a, interleaved, g, grid, stream);
  } else if (vp == 4) {
    rotary_launch<T, 4>(a, interleaved, g, grid, stream);
  } else if (vp == 2) {
    rotary_launch<T, 2>(a, interleaved, g, grid, stream);
  } else {
    rotary_launch<T, 1>(a, interleaved, g, grid, stream);
  }
  NMB_CHECK_LAUNCH("rotary");
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

extern "C" int nmb_rotary(const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides,
                          int64_t q_heads, const void* k, const int64_t* k_strides, void* k_out,
                          const int64_t* k_out_strides, int64_t k_heads, const double* frequencies, int64_t rotary_dim,
                          const void* positions, int position_bytes, int64_t pos_batch_stride, int64_t pos_stride,
                          const int32_t* offsets, int64_t offset, int64_t batch, int64_t seq, int64_t head_dim,
                          int interleaved, int inverse, float magnitude, int dtype, hipStream_t stream) {
  constexpr int64_t kMost = int64_t{1} << 20;
  NMB_REQUIRE(batch >= 0 && seq >= 0 && q_heads >= 0 && k_heads >= 0 && q_heads <= kMost && k_heads <= kMost &&
                  batch < (int64_t{1} << 31) && seq < (int64_t{1} << 31),
              "rotary: invalid shape");
  NMB_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim && head_dim <= kMost,
              "rotary: rotary_dim must be even, at least 2 and at most the head dim %lld, got %lld", (long long)head_dim,
              (long long)rotary_dim);
  NMB_REQUIRE_SUPPORTED(dtype == NMB_BF16 || dtype == NMB_F32, "rotary: unsupported dtype code %d", dtype);
  if (batch == 0 || seq == 0 || q_heads + k_heads == 0) return NMB_OK;
  NMB_REQUIRE((q_heads == 0 || (q != nullptr && q_out != nullptr && q_strides != nullptr && q_out_strides != nullptr)) &&
                  (k_heads == 0 || (k != nullptr && k_out != nullptr && k_strides != nullptr && k_out_strides != nullptr)) &&
                  frequencies != nullptr,
              "rotary: null argument");
  NMB_REQUIRE(positions == nullptr || position_bytes == 4 || position_bytes == 8,
              "rotary: positions must be of 4 or 8 bytes, got %d", position_bytes);
  NMB_REQUIRE(positions == nullptr || offsets == nullptr, "rotary: positions and offsets exclude each other");
  nmb::RotaryArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.y[0] = q_out;
  a.y[1] = k_out;
  for (int i = 0; i < 3; ++i) {
    a.xs[0][i] = q_heads ? q_strides[i] : 0;
    a.ys[0][i] = q_heads ? q_out_strides[i] : 0;
    a.xs[1][i] = k_heads ? k_strides[i] : 0;
    a.ys[1][i] = k_heads ? k_out_strides[i] : 0;
  }
  a.heads[0] = static_cast<int>(q_heads);
  a.heads[1] = static_cast<int>(k_heads);
  a.freq = frequencies;
  a.positions = positions;
  a.wide_positions = position_bytes == 8;
  a.pos_b = pos_batch_stride;
  a.pos_s = pos_stride;
  a.offsets = offsets;
  a.offset = offset;
  a.dim = static_cast<int>(head_dim);
  a.rot = static_cast<int>(rotary_dim);
  a.magnitude = magnitude;
  a.sign = inverse ? -1.f : 1.f;
  return dtype == NMB_BF16 ? nmb::rotary_impl<nmb::bf16>(a, batch, seq, interleaved != 0, stream)
                           : nmb::rotary_impl<float>(a, batch, seq, interleaved != 0, stream);
}
