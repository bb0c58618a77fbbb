// fp32 GEMM on the fp32 MFMA (v_mfma_f32_16x16x4_f32) for gfx950.
//
// The dense projections of the fp32 parity configuration (reference
// nn.Linear / F.linear at nn/kernels/torch_backend.py:19-20 and
// tensor_parallel/layers.py:214, and their autograd products, in fp32):
//   D[M, N] = alpha * op(A)[M, K] * op(B)[K, N] + beta * C[M, N]   (row-major)
// with the operand layouts of nmb_gemm_bf16 (A [M, K] or [K, M]; B [N, K] or
// [K, N]), any shape, leading dimension and alignment.  Every product is an
// exact fp32 product accumulated in fp32 by the matrix core, so results agree
// with an fp32 reference GEMM to the rounding of the summation order.
//
// Workgroup tile 64 x 64, four wavefronts of 32 x 32 (2 x 2 MFMA tiles), K
// tiles of 32 double-buffered in LDS, the next two tiles' global loads in flight
// in registers during the current one's 32 MFMAs per wave.  A lane's fragments
// are of four consecutive k: lane group q supplies k = 16 j + 4 q + e to the e-th
// MFMA of step j for A and B alike, which sums the same products in a fixed
// order.  An operand lies in LDS as it is stored, so that both ways are 16-byte
// writes: along k as rows of 32 (36 floats apart, so the rows of a fragment read
// spread over the banks), along M or N as 32 rows of 64 (72 apart), of which a
// lane reads two neighbours at a time, one for each of its two fragments.  Rows
// past the matrix repeat its last one: no lane's condition holds up a load.  Each
// MFMA computes a D^T tile (B fragment as the A operand), so a lane holds four
// consecutive columns of one row of D.
//
// Measured with the same bits, us: transposed on the way into LDS, one tile
// ahead, conditions at edges / as stored / two tiles ahead / rows repeated:
// 8192 x 256 x 512 from [K, M] and [K, N] 34.8, 25.2, 23.4, 23.1; 512 x 256 x 8192
// from [M, K] and [K, N] 35.9, 30.2, 29.3, 29.5; 512 x 8192 x 256 25.6, 25.2, 24.0,
// 23.8; 600 x 768 x 8192 119, 104, 96, 81; 4096^3 1187, 1173, 1070, 1075 (128
// TFLOP/s of the 154 that a large product of a library reaches).
//
// What bounds it: the smoke configuration's products (512 tokens, K 256 to
// 8192) are a few tens of tiles of 64 x 64, so launch and memory latency and
// idle CUs, not the 256 FLOP per clock and CU of the fp32 matrix core.  The K
// range is therefore split over workgroups until about two per CU run, with
// the partial products (caller's workspace) summed in split order by a second
// launch.  Over the 64 products of one smoke-configuration step (4 x 128
// tokens, forward and backward): 0.58 ms and 0.27 ms of sums, against 4.95 ms
// with 16-deep single-buffered tiles of element loads and no split (512 x 256
// x 8192 alone 1.4 ms on its 32 workgroups).
#include <algorithm>

#include "common.h"

namespace nmb {
namespace {

constexpr int kTile = 64;
constexpr int kKT = 32;
constexpr int kRow = kKT + 4;    // floats between rows in LDS
constexpr int kCol = kTile + 8;  // and between the k of an operand that is stored along its rows

struct GemmF32Args {
  const float* a;
  const float* b;
  const float* c;
  float* d;
  float* partial;  // split K: [splits][M][N]
  int64_t lda, ldb, ldc, ldd;
  int M, N, K;
  float alpha, beta;
  int kps;               // K range of a split (a multiple of kKT, or K)
  int vec_a, vec_b;      // 16-byte loads allowed (base and leading dimension)
  int vec_c, vec_d;      // the same for C and D (and the partial rows: vec_p)
  int vec_p;
};

__device__ __forceinline__ f32x4 mfma_f32(float a, float b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}

// One thread's 2 x 4 consecutive elements of a 64 x 32 operand tile: rows r0
// .. (valid up to rows), k range [k0, k_end).  KC: stored [row][k], each group
// of 4 along k; else stored [k][row], along the row dimension.  Elements
// outside read as zeros or, with whole (every k of the tile is there, and 16-byte
// groups of rows are or are not), rows outside as the last ones.
template <bool KC>
struct TileLoad {
  f32x4 v[2];
  __device__ __forceinline__ void load(const float* p, int64_t ld, int r0, int rows, int k0, int k_end, bool vec,
                                       bool whole) {
    if (whole) {
      // loads that no lane's condition holds up (where such branches join, the wave waits for
      // their data, and the tile in flight is no longer under the MFMAs)
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int idx = static_cast<int>(threadIdx.x) + 256 * j;
        const int64_t at =
            KC ? static_cast<int64_t>(min(r0 + idx / (kKT / 4), rows - 1)) * ld + k0 + 4 * (idx % (kKT / 4))
               : static_cast<int64_t>(k0 + idx / (kTile / 4)) * ld + min(r0 + 4 * (idx % (kTile / 4)), rows - 4);
        v[j] = *reinterpret_cast<const f32x4*>(p + at);
      }
      return;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int idx = static_cast<int>(threadIdx.x) + 256 * j;
      if (KC) {
        const int r = r0 + idx / (kKT / 4), k = k0 + 4 * (idx % (kKT / 4));
        v[j] = group(p + static_cast<int64_t>(r) * ld + k, r < rows ? k_end - k : 0, vec);
      } else {
        const int k = k0 + idx / (kTile / 4), r = r0 + 4 * (idx % (kTile / 4));
        v[j] = group(p + static_cast<int64_t>(k) * ld + r, k < k_end ? rows - r : 0, vec);
      }
    }
  }
  // p[0..3], the first n of them (n may be negative or above 4)
  __device__ static f32x4 group(const float* p, int n, bool vec) {
    if (vec && n >= 4) return *reinterpret_cast<const f32x4*>(p);
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) o[e] = p[e];
    return o;
  }
  __device__ __forceinline__ void store(float* s) const {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int idx = static_cast<int>(threadIdx.x) + 256 * j;
      if (KC) {
        *reinterpret_cast<f32x4*>(s + idx / (kKT / 4) * kRow + 4 * (idx % (kKT / 4))) = v[j];
      } else {
        *reinterpret_cast<f32x4*>(s + idx / (kTile / 4) * kCol + 4 * (idx % (kTile / 4))) = v[j];
      }
    }
  }
};

// A wave's two fragments of a tile in LDS, k from k0 + 4 q on, and which row of the tile lane l
// of fragment i is: 16 i + l or, of a tile that keeps its rows together, 2 l + i, so that a read
// holds both fragments' element.
template <bool KC>
__device__ __forceinline__ void fragments(const float* s, int row0, int l16, int k0, f32x4 (&f)[2]) {
  if constexpr (KC) {
#pragma unroll
    for (int i = 0; i < 2; ++i) f[i] = *reinterpret_cast<const f32x4*>(s + (row0 + 16 * i + l16) * kRow + k0);
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x2 v = *reinterpret_cast<const f32x2*>(s + (k0 + e) * kCol + row0 + 2 * l16);
      f[0][e] = v[0];
      f[1][e] = v[1];
    }
  }
}

// row[n .. n + 3] = v (+ beta * c[..]), the columns below N
__device__ __forceinline__ void store_row(float* row, const float* crow, float beta, f32x4 v, int n, int N, bool vec,
                                          bool vec_c) {
  if (n >= N) return;
  if (n + 3 < N && vec && (crow == nullptr || vec_c)) {
    if (crow != nullptr) {
      const f32x4 c = *reinterpret_cast<const f32x4*>(crow + n);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += beta * c[e];
    }
    *reinterpret_cast<f32x4*>(row + n) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < N) row[n + e] = crow != nullptr ? v[e] + beta * crow[n + e] : v[e];
}

// A_KC: A stored [M, K] (K contiguous), else [K, M].  B_KC: B stored [N, K],
// else [K, N].  blockIdx: (column tile, row tile, split).
template <bool A_KC, bool B_KC>
__global__ __launch_bounds__(256) void gemm_f32_kernel(GemmF32Args g) {
  static_assert(kKT * kCol == kTile * kRow, "both forms of a tile take as much");
  __shared__ __attribute__((aligned(16))) float sA[2][kTile * kRow];
  __shared__ __attribute__((aligned(16))) float sB[2][kTile * kRow];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int l16 = lane & 15, q = lane >> 4;
  const int m0 = static_cast<int>(blockIdx.y) * kTile;
  const int n0 = static_cast<int>(blockIdx.x) * kTile;
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32;
  const int k_begin = static_cast<int>(blockIdx.z) * g.kps;
  const int k_end = min(g.K, k_begin + g.kps);

  f32x4 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  int buf = 0, k0 = k_begin;
  const auto multiply = [&] {
#pragma unroll
    for (int j16 = 0; j16 < kKT; j16 += 16) {
      f32x4 fa[2], fb[2];
      fragments<A_KC>(sA[buf], wm, l16, j16 + 4 * q, fa);
      fragments<B_KC>(sB[buf], wn, l16, j16 + 4 * q, fb);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = mfma_f32(fb[j][e], fa[i][e], acc[i][j]);
    }
    buf ^= 1;
    k0 += kKT;
  };
  struct Loads {
    TileLoad<A_KC> a;
    TileLoad<B_KC> b;
  };
  const auto load = [&](Loads& l, int k, bool whole) {
    l.a.load(g.a, g.lda, m0, g.M, k, k_end, g.vec_a, whole);
    l.b.load(g.b, g.ldb, n0, g.N, k, k_end, g.vec_b, whole);
  };
  // the buffer last read two tiles ago: every wave has passed the barrier since
  const auto store = [&](const Loads& l) {
    l.a.store(sA[buf]);
    l.b.store(sB[buf]);
    __syncthreads();
  };
  // l0 holds the next tile and l1 the one after; without conditions in the loop, the wait for
  // the one leaves the other's loads under way
  Loads l0, l1;
  const int n = (k_end - k_begin) / kKT;  // whole tiles
  const bool inside = g.vec_a && g.vec_b && (A_KC || g.M % 4 == 0) && (B_KC || g.N % 4 == 0);
  if (inside && n >= 2) {
    load(l0, k0, true);
    load(l1, k0 + kKT, true);
    int left = n;
    for (; left > 3; left -= 2) {
      store(l0);
      load(l0, k0 + 2 * kKT, true);
      multiply();
      store(l1);
      load(l1, k0 + 2 * kKT, true);
      multiply();
    }
    store(l0);
    if (left == 3) load(l0, k0 + 2 * kKT, true);
    multiply();
    store(l1);
    multiply();
    if (left == 3) {
      store(l0);
      multiply();
    }
  }
  if (k0 < k_end) load(l0, k0, inside && k0 + kKT <= k_end);
  while (k0 < k_end) {
    store(l0);
    if (k0 + kKT < k_end) load(l0, k0 + kKT, false);
    multiply();
  }

  // acc[i][j][e] is of row l16 of A's fragment i and row 4 q + e of B's fragment j
  if constexpr (!B_KC) {  // columns 8 q + 2 e + j: to four consecutive ones a vector
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 lo = acc[i][0], hi = acc[i][1];
      acc[i][0] = f32x4{lo[0], hi[0], lo[1], hi[1]};
      acc[i][1] = f32x4{lo[2], hi[2], lo[3], hi[3]};
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int m = m0 + wm + (A_KC ? 16 * i + l16 : 2 * l16 + i);
    if (m >= g.M) continue;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int n = n0 + wn + (B_KC ? 16 * j + 4 * q : 8 * q + 4 * j);
      if (g.partial != nullptr) {
        float* row = g.partial + (static_cast<int64_t>(blockIdx.z) * g.M + m) * g.N;
        store_row(row, nullptr, 0.f, acc[i][j], n, g.N, g.vec_p, false);
      } else {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = g.alpha * acc[i][j][e];
        const float* crow = g.beta != 0.f ? g.c + static_cast<int64_t>(m) * g.ldc : nullptr;
        store_row(g.d + static_cast<int64_t>(m) * g.ldd, crow, g.beta, v, n, g.N, g.vec_d, g.vec_c);
      }
    }
  }
}

// D = alpha * (sum of the splits' partials, in order) + beta * C; a thread
// takes four columns.
__global__ __launch_bounds__(256) void gemm_f32_reduce_kernel(GemmF32Args g, int splits) {
  const int groups = (g.N + 3) / 4;
  const int64_t idx = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (idx >= static_cast<int64_t>(g.M) * groups) return;
  const int m = static_cast<int>(idx / groups), n = 4 * static_cast<int>(idx % groups);
  const int cnt = min(4, g.N - n);
  f32x4 v = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < splits; ++s) {
    const float* p = g.partial + (static_cast<int64_t>(s) * g.M + m) * g.N + n;
    const f32x4 t = TileLoad<true>::group(p, cnt, g.vec_p);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= g.alpha;
  const float* crow = g.beta != 0.f ? g.c + static_cast<int64_t>(m) * g.ldc : nullptr;
  store_row(g.d + static_cast<int64_t>(m) * g.ldd, crow, g.beta, v, n, g.N, g.vec_d, g.vec_c);
}

// K range of a split: with fewer than 512 tiles (two workgroups per CU) as
// many splits as bring the launch near that, each of 64 k at least (two K
// tiles: shorter ones spend more on the partials than the idle CUs cost) and
// 32 at most (the reduction reads one partial per split one after the other).
int split_k(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = ((m + kTile - 1) / kTile) * ((n + kTile - 1) / kTile);
  int64_t want = tiles > 0 ? std::min<int64_t>(512 / tiles, 32) : 1;
  want = std::min(want, k / 64);
  if (want <= 1) return static_cast<int>(k);
  const int64_t kps = ((k + want - 1) / want + kKT - 1) / kKT * kKT;
  return static_cast<int>(kps);
}

bool vec_ok(const float* p, int64_t ld) { return aligned16(p) && ld % 4 == 0; }

int gemm_f32(int a_layout, int b_layout, int64_t m, int64_t n, int64_t k, float alpha, const float* a, int64_t lda,
             const float* b, int64_t ldb, float beta, const float* c, int64_t ldc, float* d, int64_t ldd,
             float* workspace, int64_t workspace_bytes, hipStream_t stream) {
  NMB_REQUIRE(a_layout == 0 || a_layout == 1, "gemm_f32: a_layout must be 0 ([M,K]) or 1 ([K,M])");
  NMB_REQUIRE(b_layout == 0 || b_layout == 1, "gemm_f32: b_layout must be 0 ([N,K]) or 1 ([K,N])");
  NMB_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m < (1 << 30) && n < (1 << 30) && k < (1 << 30),
              "gemm_f32: invalid shape %lld x %lld x %lld", (long long)m, (long long)n, (long long)k);
  NMB_REQUIRE(d != nullptr && (k == 0 || (a != nullptr && b != nullptr)), "gemm_f32: null operand");
  NMB_REQUIRE(beta == 0.f || c != nullptr, "gemm_f32: beta != 0 needs C");
  const bool a_kc = a_layout == 0, b_kc = b_layout == 0;
  NMB_REQUIRE(lda >= (a_kc ? k : m) && ldb >= (b_kc ? k : n) && ldd >= n && (beta == 0.f || ldc >= n),
              "gemm_f32: leading dimension too small");
  if (m == 0 || n == 0) return NMB_OK;
  const int64_t gy = (m + kTile - 1) / kTile, gx = (n + kTile - 1) / kTile;
  NMB_REQUIRE(gy <= 65535 && gx < (int64_t{1} << 31), "gemm_f32: problem too large for one launch");
  GemmF32Args g{};
  g.a = a;
  g.b = b;
  g.c = c;
  g.d = d;
  g.lda = lda;
  g.ldb = ldb;
  g.ldc = ldc;
  g.ldd = ldd;
  g.M = static_cast<int>(m);
  g.N = static_cast<int>(n);
  g.K = static_cast<int>(k);
  g.alpha = alpha;
  g.beta = beta;
  g.kps = workspace != nullptr ? split_k(m, n, k) : static_cast<int>(k);
  const int splits = g.kps > 0 ? static_cast<int>((k + g.kps - 1) / g.kps) : 1;
  if (splits > 1) {
    NMB_REQUIRE(workspace_bytes >= static_cast<int64_t>(splits) * m * n * 4 && aligned16(workspace),
                "gemm_f32: workspace of %lld bytes is too small or not 16-byte aligned", (long long)workspace_bytes);
    g.partial = workspace;
  }
  g.vec_a = vec_ok(a, lda);
  g.vec_b = vec_ok(b, ldb);
  g.vec_c = vec_ok(c, ldc);
  g.vec_d = vec_ok(d, ldd);
  g.vec_p = n % 4 == 0;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy), static_cast<unsigned>(splits));
  if (a_kc && b_kc) hipLaunchKernelGGL((gemm_f32_kernel<true, true>), grid, dim3(256), 0, stream, g);
  else if (a_kc) hipLaunchKernelGGL((gemm_f32_kernel<true, false>), grid, dim3(256), 0, stream, g);
  else if (b_kc) hipLaunchKernelGGL((gemm_f32_kernel<false, true>), grid, dim3(256), 0, stream, g);
  else hipLaunchKernelGGL((gemm_f32_kernel<false, false>), grid, dim3(256), 0, stream, g);
  if (splits > 1) {
    const int64_t blocks = (m * ((n + 3) / 4) + 255) / 256;
    hipLaunchKernelGGL(gemm_f32_reduce_kernel, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, g, splits);
  }
  NMB_CHECK_LAUNCH("gemm_f32");
  return NMB_OK;
}

}  // namespace
}  // namespace nmb

extern "C" int nmb_gemm_f32(int a_layout, int b_layout, int64_t m, int64_t n, int64_t k, float alpha,
                            const float* a, int64_t lda, const float* b, int64_t ldb, float beta,
                            const float* c, int64_t ldc, float* d, int64_t ldd, hipStream_t stream) {
  return nmb::gemm_f32(a_layout, b_layout, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc, d, ldd, nullptr, 0, stream);
}

extern "C" int nmb_gemm_f32_workspace_bytes(int64_t m, int64_t n, int64_t k, int64_t* bytes) {
  NMB_REQUIRE(bytes != nullptr, "gemm_f32_workspace_bytes: null output");
  NMB_REQUIRE(m >= 0 && n >= 0 && k >= 0 && m < (1 << 30) && n < (1 << 30) && k < (1 << 30),
              "gemm_f32: invalid shape %lld x %lld x %lld", (long long)m, (long long)n, (long long)k);
  const int64_t kps = nmb::split_k(m, n, k);
  const int64_t splits = kps > 0 ? (k + kps - 1) / kps : 1;
  *bytes = splits > 1 ? splits * m * n * 4 : 0;
  return NMB_OK;
}

extern "C" int nmb_gemm_f32_split(int a_layout, int b_layout, int64_t m, int64_t n, int64_t k, float alpha,
                                  const float* a, int64_t lda, const float* b, int64_t ldb, float beta,
                                  const float* c, int64_t ldc, float* d, int64_t ldd, void* workspace,
                                  int64_t workspace_bytes, hipStream_t stream) {
  return nmb::gemm_f32(a_layout, b_layout, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc, d, ldd,
                       static_cast<float*>(workspace), workspace_bytes, stream);
}
