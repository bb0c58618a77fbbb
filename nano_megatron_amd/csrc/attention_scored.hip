// Attention with capped scores, a distance bias and interval masks (documents,
// prefix, window), forward and backward, for gfx950.  attention_scored.h holds
// the mathematics.
#include <algorithm>

#include "attention_scored.h"

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

// ------------------------------------------------------------ host side
int fill_scored(ScoredShape* p, const nmb_scores* sc, int64_t B, int64_t Hq, int64_t Hkv, int64_t Sq, int64_t Sk,
                int64_t D, const int64_t* qs, const int64_t* ks, const int64_t* vs, const int64_t* os,
                const int64_t* gs, int dtype) {
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
                                  v_strides, o_strides, nullptr, dtype);
  if (st != NMB_OK) return st;
  if (batch == 0 || seq_q == 0) return NMB_OK;
  NMB_REQUIRE(q != nullptr && o != nullptr && lse2 != nullptr && (seq_k == 0 || (k != nullptr && v != nullptr)),
              "attn_scored_fwd: null tensor");
  if (dtype == NMB_BF16) nmb::rows_fwd_launch<nmb::bf16>(p, q, k, v, o, lse2, stream);
  else nmb::rows_fwd_launch<float>(p, q, k, v, o, lse2, stream);
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
                                  v_strides, o_strides, dkv_strides, dtype);
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
