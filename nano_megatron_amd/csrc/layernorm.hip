// Layer norm forward/backward for gfx950, with the residual addition before it
// (RMSNorm, the reference's norm, is in rmsnorm.hip; this one has no counterpart there).
//
//   h = round(x + r) (or x);  mu = mean(h);  s = 1 / sqrt(mean((h - mu)^2) + eps)
//   n = (h - mu) s;  y = n w + b
//   g = dy w;  dx = s (g - mean(g) - n mean(g n)) + dh;  dw = sum_rows dy n;  db = sum_rows dy
//
// Everything is formed in fp32 and rounded once where it is stored.  The mean is taken off before
// the squares are summed, and what the rounding of its sum left is taken off the differences, so
// the forward loses nothing on a row far from zero (fp32 rows around 1000, or 10^6, of spread 1 and 3:
// y off by 5e-7, by 1.2e-4 and 0.029 with the mean of one sum; rows of 1234.567 throughout 0 and
// 0.039).  The backward's mean is that one rounded, off by up to 2^-24 of itself.
//
// A row is held in the registers of a group of LANES lanes, ITERS vectors of 16 bytes each, so
// that every tensor crosses HBM once: groups of 8 to 64 lanes lie in one wavefront and reduce
// by DPP, groups of 256 and 1024 through LDS.  Rows need no alignment (a vector may start at
// any element), and the last vector of a row is moved back to end with it: its first
// elements are the vector's before, left out of the sums and stored twice with the same bits.
//
// dw and db: each group adds up its rows in registers, the groups of a workgroup are joined
// in LDS, and a second launch adds up the workgroups' rows, all in a fixed order.
#include "common.h"
#include "vec.h"

namespace nmb {
namespace {

struct NormArgs {
  const void* x;    // forward: x; backward: h
  const void* res;  // forward: the residual; backward: dh
  const void* w;
  const void* b;
  const void* dy;
  void* y;  // forward: y; backward: dx
  void* h;
  float2* stats;   // [rows]: mu, s
  float* partial;  // [blocks][2][cols]
  int64_t ldx, ldres, lddy, rows;
  int cols;
  float eps;
};

template <typename T, int V> struct Vec { T e[V]; };

// V elements from an address of any alignment: one load
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> ld_any(const T* p) {
  Vec<T, V> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <typename T, int V>
__device__ __forceinline__ void st_any(T* p, const float (&v)[V]) {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.e[i] = from_f32<T>(v[i]);
  __builtin_memcpy(p, &r, sizeof(r));
}

// The sum over a group of LANES lanes, the same bits in each of them.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v += dpp<0xB1>(v);
  v += dpp<0x4E>(v);
  v += dpp<0x141>(v);
  if constexpr (LANES >= 16) v += dpp<0x140>(v);
  if constexpr (LANES >= 32) v = xor16_sum(v);
  if constexpr (LANES >= 64) v = xor32_sum(v);
  return v;
}

// K sums over the group at once; groups of several wavefronts join them in sh, which
// alternates between two places so that one barrier a call is enough.
template <int LANES, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* sh, int& flip) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = lanes_sum<LANES < 64 ? LANES : 64>(v[k]);
  if constexpr (LANES > 64) {
    constexpr int W = LANES / 64;
    const int wave = static_cast<int>(threadIdx.x) >> 6;
    float* at = sh + flip * 16 * 2;
    flip ^= 1;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) at[wave * 2 + k] = v[k];
    }
    __syncthreads();
    const int w0 = wave / W * W;
    if constexpr (W == 16) {
      // a lane reads one wavefront's: all of them, two sums at a time, would take more registers
      // than two workgroups a CU leave (2048 x 16384 22.5 us and 35)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = lanes_sum<16>(at[(threadIdx.x & 15) * 2 + k]);
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) t += at[(w0 + j) * 2 + k];
        v[k] = t;
      }
    }
  }
}

constexpr int fwd_threads(int lanes) { return lanes > 256 ? lanes : 256; }
constexpr int bwd_threads(int lanes) { return lanes > 512 ? lanes : 512; }

// Where vector `it` of a lane starts, and how many of its first elements are another's.
struct Place {
  int at, skip;
};
template <int V, int LANES>
__device__ __forceinline__ Place place(int it, int lane, int cols) {
  const int c = (it * LANES + lane) * V;
  const int at = min(c, cols - V);
  return Place{at, c - at};
}

template <typename T, int V, int LANES, int ITERS, bool RES>
__global__ __launch_bounds__(fwd_threads(LANES)) void layernorm_fwd_kernel(NormArgs a) {
  constexpr int GROUPS = fwd_threads(LANES) / LANES;
  __shared__ float sh[64];
  int flip = 0;
  const int lane = static_cast<int>(threadIdx.x) % LANES;
  const int64_t at_row = static_cast<int64_t>(blockIdx.x) * GROUPS + static_cast<int>(threadIdx.x) / LANES;
  const bool there = at_row < a.rows;
  const int64_t row = there ? at_row : a.rows - 1;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* res = static_cast<const T*>(a.res) + row * a.ldres;
  Vec<T, V> xr[ITERS], rr[ITERS], wr[ITERS], br[ITERS];
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
    xr[it] = ld_any<T, V>(x + p.at);
    if constexpr (RES) rr[it] = ld_any<T, V>(res + p.at);
  }
  const T* bias = static_cast<const T*>(a.b != nullptr ? a.b : a.w);
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
    wr[it] = ld_any<T, V>(static_cast<const T*>(a.w) + p.at);
    br[it] = ld_any<T, V>(bias + p.at);
  }
  float v[ITERS][V], sum[1] = {0.f};
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      v[it][i] = to_f32(xr[it].e[i]);
      if constexpr (RES) v[it][i] = round_as<T>(v[it][i] + to_f32(rr[it].e[i]));
      sum[0] += i >= p.skip ? v[it][i] : 0.f;
    }
  }
  group_sum<LANES>(sum, sh, flip);
  const float count = static_cast<float>(a.cols);  // divided by: a row of one value has its mean
  const float mu = sum[0] / count;
  // what the rounding of that sum left in the differences: their own mean, as exact as they are
  float off[2] = {0.f, 0.f};
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float d = i >= p.skip ? v[it][i] - mu : 0.f;
      off[0] += d;
      off[1] = fmaf(d, d, off[1]);
    }
  }
  group_sum<LANES>(off, sh, flip);
  const float c = off[0] / count;
  const float s = 1.f / sqrtf(fmaxf(fmaf(-c, c, off[1] / count), 0.f) + a.eps);
  if (!there) return;
  T* y = static_cast<T*>(a.y) + row * a.cols;
  T* h = static_cast<T*>(a.h) + row * a.cols;
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const float n = fmaf(v[it][i] - mu, s, -c * s);
      o[i] = fmaf(n, to_f32(wr[it].e[i]), a.b != nullptr ? to_f32(br[it].e[i]) : 0.f);
    }
    if (p.skip < V) {
      st_any<T, V>(y + p.at, o);
      if constexpr (RES) st_any<T, V>(h + p.at, v[it]);
    }
  }
  if (a.stats != nullptr && lane == 0) a.stats[row] = float2{mu + c, s};
}

template <typename T, int V, int LANES, int ITERS, bool DH>
__global__ __launch_bounds__(bwd_threads(LANES)) void layernorm_bwd_kernel(NormArgs a) {
  constexpr int THREADS = bwd_threads(LANES), GROUPS = THREADS / LANES;
  constexpr int SLOTS = LANES >= 64 ? GROUPS : THREADS / 64;  // sums that LDS joins
  __shared__ float s_sum[SLOTS > 1 ? SLOTS / 2 * ITERS * V * LANES : 1];
  __shared__ float sh[64];
  int flip = 0;
  const int lane = static_cast<int>(threadIdx.x) % LANES;
  const int group = static_cast<int>(threadIdx.x) / LANES;
  float w[ITERS][V], dw[ITERS][V], db[ITERS][V];
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const Place p = place<V, LANES>(it, lane, a.cols);
    const Vec<T, V> r = ld_any<T, V>(static_cast<const T*>(a.w) + p.at);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      w[it][i] = to_f32(r.e[i]);
      dw[it][i] = db[it][i] = 0.f;
    }
  }
  const float inv = 1.f / static_cast<float>(a.cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * GROUPS;
  struct Loaded {
    Vec<T, V> x[ITERS], dy[ITERS], dh[DH ? ITERS : 1];
    float2 stats;
  };
  // every group walks the same number of rows: those past the end repeat the last, unstored
  auto load = [&](Loaded& l, int64_t r0) {
    const int64_t row = min(r0 + group, a.rows - 1);
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* dy = static_cast<const T*>(a.dy) + row * a.lddy;
    const T* dh = static_cast<const T*>(a.res) + row * a.ldres;
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      const Place p = place<V, LANES>(it, lane, a.cols);
      l.x[it] = ld_any<T, V>(x + p.at);
      l.dy[it] = ld_any<T, V>(dy + p.at);
      if constexpr (DH) l.dh[it] = ld_any<T, V>(dh + p.at);
    }
    l.stats = a.stats[row];
  };
  // with one vector a lane there are registers for the next row's, loaded under this one's sums
  // (4000 x 5000 44.6 -> 35.8 us, 4096 x 2736 28.4 -> 21.5, 8192 x 768 17.1 -> 16.4)
  constexpr bool AHEAD = ITERS == 1;
  Loaded now, next;
  if constexpr (AHEAD) load(next, static_cast<int64_t>(blockIdx.x) * GROUPS);
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * GROUPS; r0 < a.rows; r0 += step) {
    const bool there = r0 + group < a.rows;
    const int64_t row = there ? r0 + group : a.rows - 1;
    if constexpr (AHEAD) {
      now = next;
      load(next, r0 + step);
    } else {
      load(now, r0);
    }
    const float2 st = now.stats;
    float n[ITERS][V], g[ITERS][V], sums[2] = {0.f, 0.f};
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      const Place p = place<V, LANES>(it, lane, a.cols);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = to_f32(now.dy[it].e[i]);
        n[it][i] = (to_f32(now.x[it].e[i]) - st.x) * st.y;
        g[it][i] = d * w[it][i];
        if (there) {
          dw[it][i] = fmaf(d, n[it][i], dw[it][i]);
          db[it][i] += d;
        }
        if (i >= p.skip) {
          sums[0] += g[it][i];
          sums[1] = fmaf(g[it][i], n[it][i], sums[1]);
        }
      }
    }
    group_sum<LANES>(sums, sh, flip);
    const float m1 = sums[0] * inv, m2 = sums[1] * inv;
    if (there) {
      T* dx = static_cast<T*>(a.y) + row * a.cols;
#pragma unroll
      for (int it = 0; it < ITERS; ++it) {
        const Place p = place<V, LANES>(it, lane, a.cols);
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          o[i] = st.y * (g[it][i] - m1 - n[it][i] * m2);
          if constexpr (DH) o[i] += to_f32(now.dh[it].e[i]);
        }
        if (p.skip < V) st_any<T, V>(dx + p.at, o);
      }
    }
  }
  if (a.partial == nullptr) return;
  if constexpr (LANES < 64) {  // the groups of a wavefront hold the same columns
#pragma unroll
    for (int it = 0; it < ITERS; ++it)
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if constexpr (LANES == 8) {
          dw[it][i] += __shfl_xor(dw[it][i], 8);
          db[it][i] += __shfl_xor(db[it][i], 8);
        }
        if constexpr (LANES <= 16) {
          dw[it][i] = xor16_sum(dw[it][i]);
          db[it][i] = xor16_sum(db[it][i]);
        }
        dw[it][i] = xor32_sum(dw[it][i]);
        db[it][i] = xor32_sum(db[it][i]);
      }
  }
  const int slot = LANES >= 64 ? group : static_cast<int>(threadIdx.x) >> 6;
  float* out = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * a.cols;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&acc)[ITERS][V] = which == 0 ? dw : db;
#pragma unroll
    for (int half = SLOTS / 2; half >= 1; half /= 2) {
      // every slot's lanes hold the same columns: lane after lane, element by element
      __syncthreads();
      if (slot >= half && slot < 2 * half) {
#pragma unroll
        for (int k = 0; k < ITERS * V; ++k) s_sum[((slot - half) * ITERS * V + k) * LANES + lane] = acc[k / V][k % V];
      }
      __syncthreads();
      if (slot < half) {
#pragma unroll
        for (int k = 0; k < ITERS * V; ++k) acc[k / V][k % V] += s_sum[(slot * ITERS * V + k) * LANES + lane];
      }
    }
    if (slot == 0) {
#pragma unroll
      for (int it = 0; it < ITERS; ++it) {
        const Place p = place<V, LANES>(it, lane, a.cols);
        if (p.skip < V) st_any<float, V>(out + which * a.cols + p.at, acc[it]);
      }
    }
  }
}

// dw[c], db[c]: the workgroups' sums, 16 columns of `2 cols` a workgroup, each added up by 64
// threads in a fixed order.
constexpr int kMostBlocks = 512;
template <typename T>
__global__ __launch_bounds__(1024) void layernorm_columns_kernel(const float* __restrict__ partial, int blocks,
                                                                 int cols, T* __restrict__ dw, T* __restrict__ db) {
  __shared__ float s[64][17];
  const int cl = threadIdx.x & 15, part = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + cl;
  float t = 0.f;
  if (c < 2 * cols) {
    float v[kMostBlocks / 64];
#pragma unroll
    for (int j = 0; j < kMostBlocks / 64; ++j) {
      const int b = part + 64 * j;
      v[j] = b < blocks ? partial[static_cast<int64_t>(b) * 2 * cols + c] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kMostBlocks / 64; ++j) t += v[j];
  }
  s[part][cl] = t;
  __syncthreads();
  if (part < 8) {
    float u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) u += s[part + 8 * k][cl];
    s[part][cl] = u;
  }
  __syncthreads();
  if (part == 0 && c < 2 * cols) {
    float u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) u += s[k][cl];
    if (c < cols) {
      if (dw != nullptr) dw[c] = from_f32<T>(u);
    } else if (db != nullptr) {
      db[c - cols] = from_f32<T>(u);
    }
  }
}

// ------------------------------------------------------------ host side
constexpr int64_t kMostCols = 16384;

// The group that holds a row of `nv` vectors, and how many each lane holds of it.  The forward
// takes the fewest lanes, up to four vectors a lane: fewer steps of its two sums, and enough
// loads in flight either way (us, these first, then one vector a lane: 8192 x 768 10.2 and 10.7,
// 8192 x 1024 11.6 and 12.4, 4000 x 5000 30.2 and 34.1, 16384 x 2048 43.8 and 43.2).  The
// backward takes one vector a lane as far as 1,024 lanes go: it holds three tensors, the weight
// and two sums of each, and more wavefronts hide more than fewer steps save (with the sums over rows,
// 16384 x 2048 53 and, with the forward's groups, 83; 8192 x 768 15 and 35; 4099 x 1001 in fp32
// 16 and 27).
struct NormPlan {
  int lanes, iters;
};
template <int N>
NormPlan first_that_holds(const NormPlan (&plans)[N], int nv) {
  for (const NormPlan& p : plans)
    if (nv <= p.lanes * p.iters) return p;
  return NormPlan{0, 0};
}
template <typename T>
NormPlan norm_plan(int cols, bool backward) {
  constexpr int V = VecTraits<T>::N;
  static const NormPlan fwd[] = {{8, 1},  {16, 1},  {32, 1},  {32, 2},  {32, 3},   {64, 2},  {64, 3},
                                 {64, 4}, {256, 2}, {256, 3}, {256, 4}, {1024, 2}, {1024, 4}};
  static const NormPlan bwd[] = {{8, 1},   {16, 1},  {32, 1},   {64, 1},   {128, 1},
                                 {256, 1}, {512, 1}, {1024, 1}, {1024, 2}, {1024, 4}};
  if (cols < V) return NormPlan{8, 1};  // vectors of one element
  const int nv = (cols + V - 1) / V;
  return backward ? first_that_holds(bwd, nv) : first_that_holds(fwd, nv);
}

int bwd_blocks(int64_t rows, int lanes) {
  const int64_t groups = bwd_threads(lanes) / lanes;
  const int64_t most = lanes > 256 ? kMostBlocks / 2 : kMostBlocks;
  const int64_t b = (rows + groups - 1) / groups;
  return static_cast<int>(b < 1 ? 1 : b < most ? b : most);
}

int check_norm(int64_t rows, int64_t cols, const void* x, int64_t ldx, const void* res, int64_t ldres, const void* w) {
  NMB_REQUIRE(rows >= 0 && rows < (int64_t{1} << 31) && cols > 0, "layernorm: invalid shape rows=%lld cols=%lld",
              (long long)rows, (long long)cols);
  NMB_REQUIRE_SUPPORTED(cols <= kMostCols, "layernorm: hidden size %lld exceeds the supported maximum %lld",
                        (long long)cols, (long long)kMostCols);
  NMB_REQUIRE(rows == 0 || (x != nullptr && w != nullptr), "layernorm: null tensor");
  NMB_REQUIRE(ldx >= 0 && (res == nullptr || ldres >= 0), "layernorm: row strides must not be negative");
  return NMB_OK;
}

// LAUNCH(V, LANES, ITERS) of a plan
#define NMB_FWD_PLANS(T, p, LAUNCH)                                                     \
  switch ((p).lanes * 16 + (p).iters) {                                                 \
    case 8 * 16 + 1: LAUNCH(VecTraits<T>::N, 8, 1); break;                              \
    case 16 * 16 + 1: LAUNCH(VecTraits<T>::N, 16, 1); break;                            \
    case 32 * 16 + 1: LAUNCH(VecTraits<T>::N, 32, 1); break;                            \
    case 32 * 16 + 2: LAUNCH(VecTraits<T>::N, 32, 2); break;                            \
    case 32 * 16 + 3: LAUNCH(VecTraits<T>::N, 32, 3); break;                            \
    case 64 * 16 + 2: LAUNCH(VecTraits<T>::N, 64, 2); break;                            \
    case 64 * 16 + 3: LAUNCH(VecTraits<T>::N, 64, 3); break;                            \
    case 64 * 16 + 4: LAUNCH(VecTraits<T>::N, 64, 4); break;                            \
    case 256 * 16 + 2: LAUNCH(VecTraits<T>::N, 256, 2); break;                          \
    case 256 * 16 + 3: LAUNCH(VecTraits<T>::N, 256, 3); break;                          \
    case 256 * 16 + 4: LAUNCH(VecTraits<T>::N, 256, 4); break;                          \
    case 1024 * 16 + 2: LAUNCH(VecTraits<T>::N, 1024, 2); break;                        \
    case 1024 * 16 + 4:                                                                 \
      if constexpr (sizeof(T) == 4) LAUNCH(VecTraits<T>::N, 1024, 4);                   \
      break;                                                                            \
    default: break;                                                                     \
  }
#define NMB_BWD_PLANS(T, p, LAUNCH)                                                     \
  switch ((p).lanes * 16 + (p).iters) {                                                 \
    case 8 * 16 + 1: LAUNCH(VecTraits<T>::N, 8, 1); break;                              \
    case 16 * 16 + 1: LAUNCH(VecTraits<T>::N, 16, 1); break;                            \
    case 32 * 16 + 1: LAUNCH(VecTraits<T>::N, 32, 1); break;                            \
    case 64 * 16 + 1: LAUNCH(VecTraits<T>::N, 64, 1); break;                            \
    case 128 * 16 + 1: LAUNCH(VecTraits<T>::N, 128, 1); break;                          \
    case 256 * 16 + 1: LAUNCH(VecTraits<T>::N, 256, 1); break;                          \
    case 512 * 16 + 1: LAUNCH(VecTraits<T>::N, 512, 1); break;                          \
    case 1024 * 16 + 1: LAUNCH(VecTraits<T>::N, 1024, 1); break;                        \
    case 1024 * 16 + 2: LAUNCH(VecTraits<T>::N, 1024, 2); break;                        \
    case 1024 * 16 + 4:                                                                 \
      if constexpr (sizeof(T) == 4) LAUNCH(VecTraits<T>::N, 1024, 4);                   \
      break;                                                                            \
    default: break;                                                                     \
  }

template <typename T>
int fwd_impl(const NormArgs& a, hipStream_t stream) {
  const NormPlan p = norm_plan<T>(a.cols, false);
  NMB_REQUIRE_SUPPORTED(a.rows * p.lanes < (int64_t{1} << 32) - 1024, "layernorm_fwd: %lld rows are too many for a launch",
                        (long long)a.rows);
#define NMB_LAUNCH(V, L, I)                                                                                       \
  do {                                                                                                            \
    constexpr int kGroups = fwd_threads(L) / L;                                                                   \
    const dim3 grid(static_cast<unsigned>((a.rows + kGroups - 1) / kGroups));                                     \
    if (a.res != nullptr)                                                                                         \
      hipLaunchKernelGGL((layernorm_fwd_kernel<T, V, L, I, true>), grid, dim3(fwd_threads(L)), 0, stream, a);     \
    else                                                                                                          \
      hipLaunchKernelGGL((layernorm_fwd_kernel<T, V, L, I, false>), grid, dim3(fwd_threads(L)), 0, stream, a);    \
  } while (0)
  if (a.cols < VecTraits<T>::N) NMB_LAUNCH(1, 8, 1);  // rows shorter than a vector
  else NMB_FWD_PLANS(T, p, NMB_LAUNCH)
#undef NMB_LAUNCH
  NMB_CHECK_LAUNCH("layernorm_fwd");
  return NMB_OK;
}

template <typename T>
int bwd_impl(const NormArgs& a, void* dw, void* db, hipStream_t stream) {
  const NormPlan p = norm_plan<T>(a.cols, true);
  const int blocks = a.rows == 0 ? 0 : bwd_blocks(a.rows, p.lanes);  // without rows the sums are of nothing
#define NMB_LAUNCH(V, L, I)                                                                                        \
  do {                                                                                                             \
    if (a.res != nullptr)                                                                                          \
      hipLaunchKernelGGL((layernorm_bwd_kernel<T, V, L, I, true>), dim3(blocks), dim3(bwd_threads(L)), 0, stream, a);  \
    else                                                                                                           \
      hipLaunchKernelGGL((layernorm_bwd_kernel<T, V, L, I, false>), dim3(blocks), dim3(bwd_threads(L)), 0, stream, a); \
  } while (0)
  if (blocks == 0) {}
  else if (a.cols < VecTraits<T>::N) NMB_LAUNCH(1, 8, 1);
  else NMB_BWD_PLANS(T, p, NMB_LAUNCH)
#undef NMB_LAUNCH
  NMB_CHECK_LAUNCH("layernorm_bwd");
  if (a.partial == nullptr) return NMB_OK;
  hipLaunchKernelGGL(layernorm_columns_kernel<T>, dim3((2 * a.cols + 15) / 16), dim3(1024), 0, stream, a.partial, blocks,
                     a.cols, static_cast<T*>(dw), static_cast<T*>(db));
  NMB_CHECK_LAUNCH("layernorm_bwd(dw, db)");
  return NMB_OK;
}

int dtype_known(int dtype) {
  NMB_REQUIRE_SUPPORTED(dtype == NMB_BF16 || dtype == NMB_F32, "layernorm: unsupported dtype code %d", dtype);
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

extern "C" int nmb_layernorm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldres, const void* w,
                                 const void* b, void* y, void* h, float* stats, int64_t rows, int64_t cols, float eps,
                                 int dtype, hipStream_t stream) {
  NMB_REQUIRE(eps > 0.f, "layernorm_fwd: eps must be positive, got %g", (double)eps);
  int st = nmb::dtype_known(dtype);
  if (st == NMB_OK) st = nmb::check_norm(rows, cols, x, ldx, residual, ldres, w);
  if (st != NMB_OK) return st;
  if (rows == 0) return NMB_OK;
  NMB_REQUIRE(y != nullptr && (residual == nullptr) == (h == nullptr),
              "layernorm_fwd: an output is missing, or the sum's without a residual");
  nmb::NormArgs a{};
  a.x = x;
  a.res = residual;
  a.w = w;
  a.b = b;
  a.y = y;
  a.h = h;
  a.stats = reinterpret_cast<float2*>(stats);
  a.ldx = ldx;
  a.ldres = ldres;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  a.eps = eps;
  return dtype == NMB_BF16 ? nmb::fwd_impl<nmb::bf16>(a, stream) : nmb::fwd_impl<float>(a, stream);
}

extern "C" int nmb_layernorm_bwd_workspace_bytes(int64_t rows, int64_t cols, int dtype, size_t* bytes) {
  NMB_REQUIRE(bytes != nullptr, "layernorm_bwd_workspace_bytes: null argument");
  int st = nmb::dtype_known(dtype);
  if (st == NMB_OK) st = nmb::check_norm(rows, cols, bytes, 0, nullptr, 0, bytes);
  if (st != NMB_OK) return st;
  const int lanes = (dtype == NMB_BF16 ? nmb::norm_plan<nmb::bf16>(static_cast<int>(cols), true)
                                       : nmb::norm_plan<float>(static_cast<int>(cols), true)).lanes;
  *bytes = static_cast<size_t>(nmb::bwd_blocks(rows, lanes)) * 2 * static_cast<size_t>(cols) * sizeof(float);
  return NMB_OK;
}

extern "C" int nmb_layernorm_bwd(const void* h, int64_t ldh, const float* stats, const void* w, const void* dy,
                                 int64_t lddy, const void* dh, int64_t lddh, void* dx, void* dw, void* db,
                                 void* workspace, size_t workspace_bytes, int64_t rows, int64_t cols, int dtype,
                                 hipStream_t stream) {
  int st = nmb::dtype_known(dtype);
  if (st == NMB_OK) st = nmb::check_norm(rows, cols, h, ldh, dh, lddh, w);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(rows == 0 || (stats != nullptr && dy != nullptr && dx != nullptr && lddy >= 0),
              "layernorm_bwd: null tensor or negative row stride");
  const bool sums = dw != nullptr || db != nullptr;
  size_t need = 0;
  st = nmb_layernorm_bwd_workspace_bytes(rows, cols, dtype, &need);
  if (st != NMB_OK) return st;
  NMB_REQUIRE(!sums || (workspace != nullptr && workspace_bytes >= need &&
                        (reinterpret_cast<uintptr_t>(workspace) & 3) == 0),
              "layernorm_bwd: a 4-byte aligned workspace of %zu bytes is needed, got %zu", need, workspace_bytes);
  if (rows == 0 && !sums) return NMB_OK;
  nmb::NormArgs a{};
  a.x = h;
  a.res = dh;
  a.w = w;
  a.dy = dy;
  a.y = dx;
  a.stats = reinterpret_cast<float2*>(const_cast<float*>(stats));
  a.partial = sums ? static_cast<float*>(workspace) : nullptr;
  a.ldx = ldh;
  a.ldres = lddh;
  a.lddy = lddy;
  a.rows = rows;
  a.cols = static_cast<int>(cols);
  if (dtype == NMB_BF16) return nmb::bwd_impl<nmb::bf16>(a, dw, db, stream);
  return nmb::bwd_impl<float>(a, dw, db, stream);
}
