// Log-probability of one token a row of float32 logits:  out[i] = (x[t_i] - m) - log sum_j exp(x[j] - m),  m = max_j x[j],
// by which finished continuations are ranked and given tokens scored.  One pass over the row with a running maximum and sum (float32), each thread its
// own; threads, warps and the blocks of a cluster that share a row are joined in a fixed order.
//
// Bound: the bytes of the logits.  Measured, rows of 152,064: 2,000 177 us (6.9 TB/s, a part of them in L2), 61 9.4 us (3.9 TB/s: a cluster's
// placement and meeting, and one round of loads a block), one 3.7 us, of which the launch and the cluster are most.
//
// As of the formula: a row with a NaN or with +inf, and a row of nothing but -inf, have no log-probabilities (NaN); a token of logit -inf has
// -inf in any other row.  A token id outside the vocabulary gives NaN.
#include "common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 512;
constexpr int WARP_ROWS = 8, WARP_VOCAB = 1024;        // rows of at most so many logits are a warp's each, eight a block

struct MaxSum { float m, s; };

// (m, s) and (m2, s2), each s a sum of exp(x - m), joined.  s = 0 with m = -inf: nothing seen, or nothing but -inf.
__device__ __forceinline__ MaxSum joined(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  return {m, a.s * exp2f((a.m - ref) * LOG2E) + b.s * exp2f((b.m - ref) * LOG2E)};
}

// N more values (-inf where there is none): one step of the running maximum for all of them.
template <int N>
__device__ __forceinline__ void take(MaxSum& r, const float (&v)[N]) {
  float m = r.m;
#pragma unroll
  for (int u = 0; u < N; u++) m = fmaxf(m, v[u]);
  const float ref = m == -INFINITY ? 0.f : m;
  float s[4] = {r.s * exp2f((r.m - ref) * LOG2E), 0.f, 0.f, 0.f};
#pragma unroll
  for (int u = 0; u < N; u++) s[u & 3] += exp2f((v[u] - ref) * LOG2E);
  r = {m, (s[0] + s[1]) + (s[2] + s[3])};
}

__device__ __forceinline__ float finished(MaxSum r, float x, bool known) { return known ? (x - r.m) - logf(r.s) : __int_as_float(0x7fc00000); }

__device__ __forceinline__ float4 ld_stream(const float* p) {        // a row is read once
  float4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// The blocks of a cluster (1 to 16) share a row, which is read once.  A thread has four vectors of 16 bytes on their way.
__global__ void __launch_bounds__(THREADS)
k_token_logprobs(const float* __restrict__ logits, int V, const int* __restrict__ tokens, float* __restrict__ out) {
  cima_pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ MaxSum part[THREADS / 32], mine;
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), row = blockIdx.y;
  const float* x = logits + (size_t)row * V;
  int t = -1;
  float xt = 0.f;
  if (c == 0 && threadIdx.x == 0) {                    // on its way while the row is read
    t = tokens[row];
    if (t >= 0 && t < V) xt = x[t];
  }
  const int per = (V + C - 1) / C, lo = min(V, c * per), hi = min(V, lo + per);
  MaxSum r{-INFINITY, 0.f};
  const int head = min(hi, lo + (int)((16 - ((uintptr_t)(x + lo) & 15)) >> 2 & 3));      // up to the first aligned vector
  const int vectors = (hi - head) >> 2, tail = head + 4 * vectors;
  {
    const int i = threadIdx.x;                         // what lies beside the vectors: 3 values at either end at most
    const float v[1] = {i < head - lo ? x[lo + i] : i >= 4 && i - 4 < hi - tail ? x[tail + i - 4] : -INFINITY};
    if (i < 8) take(r, v);
  }
  const float* base = x + head;
  for (int i = threadIdx.x; i < vectors; i += 4 * THREADS) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int k = i + u * THREADS;
      const float4 q = k < vectors ? ld_stream(base + 4 * k) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      v[4 * u] = q.x, v[4 * u + 1] = q.y, v[4 * u + 2] = q.z, v[4 * u + 3] = q.w;
    }
    take(r, v);
  }
  for (int o = 16; o > 0; o >>= 1) r = joined(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
  __syncthreads();
  if (threadIdx.x < 32) {
    r = threadIdx.x < THREADS / 32 ? part[threadIdx.x] : MaxSum{-INFINITY, 0.f};
    for (int o = THREADS / 64; o > 0; o >>= 1) r = joined(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
    if (threadIdx.x == 0) mine = r;
  }
  if (C == 1) {
    if (threadIdx.x == 0) out[row] = finished(r, xt, t >= 0 && t < V);
    return;
  }
  cluster.sync();
  if (c == 0 && threadIdx.x < 32) {
    r = threadIdx.x < C ? *cluster.map_shared_rank(&mine, threadIdx.x) : MaxSum{-INFINITY, 0.f};
    for (int o = 8; o > 0; o >>= 1) r = joined(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
    if (threadIdx.x == 0) out[row] = finished(r, xt, t >= 0 && t < V);
  }
  cluster.sync();                                      // a block's shared memory outlives the first one's reads
}

__global__ void __launch_bounds__(32 * WARP_ROWS)
k_token_logprobs_short(const float* __restrict__ logits, int n, int V, const int* __restrict__ tokens, float* __restrict__ out) {
  cima_pdl_wait();
  const int lane = threadIdx.x & 31, row = blockIdx.x * WARP_ROWS + (threadIdx.x >> 5);
  if (row >= n) return;
  const float* x = logits + (size_t)row * V;
  const int t = tokens[row];
  const bool known = t >= 0 && t < V;
  const float xt = known ? x[t] : 0.f;
  MaxSum r{-INFINITY, 0.f};
  for (int i = lane; i < V; i += 16 * 32) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; u++) v[u] = i + 32 * u < V ? x[i + 32 * u] : -INFINITY;
    take(r, v);
  }
  for (int o = 16; o > 0; o >>= 1) r = joined(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if (lane == 0) out[row] = finished(r, xt, known);
}

// Clusters of 16 are more than every device has to offer: asked for once a device.
bool wide_clusters() {
  static signed char can[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return false;
  if (can[dev] == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(16);
    cfg.blockDim = dim3(THREADS);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 16;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    const bool ok = cudaFuncSetAttribute(k_token_logprobs, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess &&
                    cudaOccupancyMaxActiveClusters(&n, k_token_logprobs, &cfg) == cudaSuccess && n > 0;
    if (!ok) cudaGetLastError();
    can[dev] = ok ? 1 : -1;
  }
  return can[dev] > 0;
}

}  // namespace

extern "C" int cima_token_logprobs(const float* logits, int n, int V, const int* tokens, float* out, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (V <= 0) return cima_fail(CIMA_E_SIZE, "token_logprobs: vocabulary %d must be positive", V);
  if (V <= WARP_VOCAB) {
    const int rc = cima_launch(k_token_logprobs_short, dim3((n - 1) / WARP_ROWS + 1), dim3(32 * WARP_ROWS), (size_t)0, stream, 1, logits, n, V, tokens, out);
    return rc ? rc : cima_launch_result();
  }
  // Blocks a row.  A cluster costs about a microsecond to place and to meet in, and its blocks must be placed together: many of them wait.
  // Measured (us by blocks a row; V = 152,064): 1 row 10.9 / 7.6 / 5.3 / 4.3 / 3.7 for 1 / 2 / 4 / 8 / 16; 8 rows 11.3 / 7.9 / 5.6 / 4.6 / 4.7; 61 rows
  // 17.3 / 11.9 / 9.5 / 10.9 / 14.8; 150 rows 22.3 / 19.0 / 20.7 / 22.6; 300 rows 32.0 / 37.1 / 35.1; 1,200 rows 113 / 113 / 115 / 149.  V = 32,003: 1 row
  // 3.9 / 3.8 / 3.3 / 3.3, 100 rows 4.3 / 5.3 / 5.6 / 8.9; V = 5,001: 1 row 2.3 / 3.3.  A block has one round of loads at least.
  int C = 16;
  for (; C > 1; C /= 2)
    if (V / C >= (n <= 64 ? 7500 : 16384) && (long long)n * C <= (C == 16 ? 64 : C == 8 ? 128 : C == 4 ? 400 : 300)) break;
  if (C == 16 && !wide_clusters()) C = 8;
  for (int i = 0; i < n; i += 65535) {
    const int m = n - i < 65535 ? n - i : 65535;
    const int rc = cima_launch(k_token_logprobs, dim3(C, m), dim3(THREADS), (size_t)0, stream, C, logits + (size_t)i * V, V, tokens + i, out + i);
    if (rc) return rc;
  }
  return cima_launch_result();
}
