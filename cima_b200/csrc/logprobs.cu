// Log-probability of one token a row of float32 logits:  out[i] = (x[t_i] - m) - log sum_j exp(x[j] - m),  m = max_j x[j],
// by which finished continuations are ranked and given tokens scored.  One pass over the row with a running maximum and sum (float32); the
// blocks of a thread-block cluster share a row and the first of them joins their (m, s) in the order of their ranks.
//
// As of the formula: a row with a NaN or with +inf, and a row of nothing but -inf, have no log-probabilities (NaN); a token of logit -inf has
// -inf in any other row.  A token id outside the vocabulary gives NaN.
#include "common.cuh"
#include <cooperative_groups.h>
namespace cg = cooperative_groups;

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int THREADS = 512, BLOCKS = 8;

struct MaxSum { float m, s; };

// (m, s) and (m2, s2), each s a sum of exp(x - m), joined.  s = 0 with m = -inf: nothing seen, or nothing but -inf.
__device__ __forceinline__ MaxSum joined(MaxSum a, MaxSum b) {
  const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
  return {m, a.s * exp2f((a.m - ref) * LOG2E) + b.s * exp2f((b.m - ref) * LOG2E)};
}

__global__ void __launch_bounds__(THREADS)
k_token_logprobs(const float* __restrict__ logits, int V, const int* __restrict__ tokens, float* __restrict__ out) {
  cima_pdl_wait();
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ MaxSum part[THREADS / 32], mine;
  const int C = (int)cluster.num_blocks(), c = (int)cluster.block_rank(), row = blockIdx.y;
  const float* x = logits + (size_t)row * V;
  const int per = (V + C - 1) / C, lo = min(V, c * per), hi = min(V, lo + per);
  MaxSum r{-INFINITY, 0.f};
  for (int i = lo + threadIdx.x; i < hi; i += 4 * THREADS) {
    float v[4];
#pragma unroll
    for (int u = 0; u < 4; u++) v[u] = i + u * THREADS < hi ? x[i + u * THREADS] : -INFINITY;
    const float m = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), r.m), ref = m == -INFINITY ? 0.f : m;
    r.s *= exp2f((r.m - ref) * LOG2E);
#pragma unroll
    for (int u = 0; u < 4; u++) r.s += exp2f((v[u] - ref) * LOG2E);
    r.m = m;
  }
  for (int o = 16; o > 0; o >>= 1) r = joined(r, {__shfl_xor_sync(0xffffffffu, r.m, o), __shfl_xor_sync(0xffffffffu, r.s, o)});
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = r;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < THREADS / 32; w++) r = joined(r, part[w]);
    mine = r;
  }
  cluster.sync();
  if (c == 0 && threadIdx.x == 0) {
    for (int k = 1; k < C; k++) r = joined(r, *cluster.map_shared_rank(&mine, k));
    const int t = tokens[row];
    out[row] = t >= 0 && t < V ? (x[t] - r.m) - logf(r.s) : __int_as_float(0x7fc00000);
  }
  cluster.sync();                                      // a block's shared memory outlives the first one's reads
}

}  // namespace

extern "C" int cima_token_logprobs(const float* logits, int n, int V, const int* tokens, float* out, cudaStream_t stream) {
  if (n <= 0) return 0;
  if (V <= 0) return cima_fail(CIMA_E_SIZE, "token_logprobs: vocabulary %d must be positive", V);
  for (int i = 0; i < n; i += 65535) {
    const int m = n - i < 65535 ? n - i : 65535;
    const int rc = cima_launch(k_token_logprobs, dim3(BLOCKS, m), dim3(THREADS), (size_t)0, stream, BLOCKS, logits + (size_t)i * V, V, tokens + i, out + i);
    if (rc) return rc;
  }
  return cima_launch_result();
}
