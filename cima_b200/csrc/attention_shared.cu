// Decoding attention of a batch in which groups of sequences hold the same pages for a prefix: one new query a sequence,
// grouped-query, keys from the paged cache.
//
// With the keys of a sequence in two parts, the group's prefix P and its own rest R, a softmax over both is
//   m = max(m_P, m_R),  o = (2^(m_P - m) o_P + 2^(m_R - m) o_R) / (2^(m_P - m) l_P + 2^(m_R - m) l_R)
// with each part's maximum m (base 2), sum l of 2^(s - m) and accumulator o of 2^(s - m) v.  The prefix part of all of a group's sequences
// is one product: count * G query rows a kv head against keys that are read once, not once a sequence.
//
// One launch has two sorts of blocks, the sequences' own pages and the groups' prefixes; both split their pages further where there are few
// of them.  A block of a prefix walks its pages through shared memory with cp.async, a tile of 16 rows belonging to one warp (64 rows: four
// tiles; 32: two, whose warps share a page's 64 keys).  Up to 16 rows, and a sequence's own pages, whose rows are the heads of its kv head, take
// keys and values straight to registers (head sizes 64 and 128).  The parts go to scratch and k_shared_combine joins them in a fixed order.
//
// Bound: for the few rows that come here the chain of one block, plan, table, pages, merge.  Measured: 2 sequences over 320 positions, 14 heads on 2 of
// 64 dims, 6.6 us with the merge; 24 over 2,560, 8 heads on 2 of 96, 11.7; in float32 4 over 960 12.0 us, 54 over 7,360 72 us (its 1.4 GFLOP of multiply-adds would take
// 20 at 72 TFLOP/s; a page is loaded, then multiplied).
//
// Scores, maxima, exponentials and sums are float32, base 2; probabilities are rounded to bfloat16 only as operand of P V.
#include "attention_shared.cuh"

namespace {

// Rows of a block's prefix: RW tiles of 16 through shared memory, a sequence's own rows one such tile; or, with PRE > 0, 8 PRE rows of either
// straight to registers.
template <int HD, int PLANES, int RW, int PRE>
__global__ void __launch_bounds__(WARPS * 32)
k_attention_shared(const __grid_constant__ SharedArgs a) {
  if (!a.early) wait_then_let_next();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Task t;
  if (!find_task(a, PRE > 0 ? 8 * PRE : 16 * RW, t)) return;
  if constexpr (PRE > 0) {
    walk_near<HD, PLANES, PRE, WARPS>(a, t, smem_raw);
  } else {
    if (RW > 1 && t.prefix) walk<HD, PLANES, RW>(a, t, smem_raw);
    else walk<HD, PLANES, 1>(a, t, smem_raw);
  }
}

// The same in float32, sums and all, by multiply-adds: a block takes 16 RT rows, a page's keys and values lie in shared memory, a thread has RT rows x 8
// keys of the scores and RT rows x HDP / 8 values of the result, so that what it reads of a page serves RT rows at once.  hd is a multiple of 4.
constexpr int F_THREADS = 128, F_ROWS = 32;
template <int HDP> struct F32Smem {
  static constexpr int PITCH = HDP + 4, PP = PS + 4;
  static constexpr size_t floats = (size_t)F_ROWS * PITCH + 2 * PS * PITCH + F_ROWS * PP;
};

template <int HDP, int RT>
__device__ __forceinline__ void walk_f32(const SharedArgs& a, const Task& tk, int hd, float* sf) {
  constexpr int PITCH = F32Smem<HDP>::PITCH, PP = F32Smem<HDP>::PP, ND = HDP / 8;
  float *sq = sf, *sk = sq + F_ROWS * PITCH, *sv = sk + PS * PITCH, *sp = sv + PS * PITCH;
  const float* cache = (const float*)a.cache;
  const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7, len = tk.len, h4 = hd / 4;
  for (int i = tid; i < 16 * RT * (HDP / 4); i += F_THREADS) {
    const int r = i / (HDP / 4), c = i % (HDP / 4);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r < tk.rows && c < h4) {
      int seq, head;
      row_of(a, tk, r, seq, head);
      const float* qp = (const float*)a.qkv + (size_t)seq * a.ld + (size_t)head * hd + 4 * c;
      v = make_float4(qp[0], qp[1], qp[2], qp[3]);
    }
    *reinterpret_cast<float4*>(sq + r * PITCH + 4 * c) = v;
  }
  float acc[RT][ND], m[RT], l[RT], slope[RT];
  int last_key[RT];
#pragma unroll
  for (int r = 0; r < RT; r++) {
    m[r] = -INFINITY, l[r] = 0.f, slope[r] = 0.f, last_key[r] = 0;
    if (a.slopes && ty + 16 * r < tk.rows) {
      int seq, head;
      row_of(a, tk, ty + 16 * r, seq, head);
      last_key[r] = a.seq_len[seq] - 1;
      slope[r] = a.slopes[head];
    }
#pragma unroll
    for (int d = 0; d < ND; d++) acc[r][d] = 0.f;
  }
  const int* table = a.pg.table + (size_t)tk.slot * a.pg.width;
  for (int p = tk.first; p < tk.last; p++) {
    const float* ksrc = cache + ((size_t)table[p] * a.pg.planes * a.nkv + tk.kvh) * (size_t)(PS * hd);
    const float* vsrc = ksrc + a.pg.value_offset();
    const int n = min(PS, len - p * PS);                // positions behind the sequence's end count as zeros
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < PS * (HDP / 4); i += F_THREADS) {
      const int r = i / (HDP / 4), c = i % (HDP / 4);
      float4 kv = make_float4(0.f, 0.f, 0.f, 0.f), vv = kv;
      if (r < n && c < h4) {
        kv = *reinterpret_cast<const float4*>(ksrc + (size_t)r * hd + 4 * c);
        vv = *reinterpret_cast<const float4*>(vsrc + (size_t)r * hd + 4 * c);
      }
      *reinterpret_cast<float4*>(sk + r * PITCH + 4 * c) = kv;
      *reinterpret_cast<float4*>(sv + r * PITCH + 4 * c) = vv;
    }
    __syncthreads();
    float s[RT][8];
#pragma unroll
    for (int r = 0; r < RT; r++)
#pragma unroll
      for (int j = 0; j < 8; j++) s[r][j] = 0.f;
    for (int c = 0; c < h4; c++) {
      float4 q[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) q[r] = *reinterpret_cast<const float4*>(sq + (ty + 16 * r) * PITCH + 4 * c);
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float4 kv = *reinterpret_cast<const float4*>(sk + (tx + 8 * j) * PITCH + 4 * c);
#pragma unroll
        for (int r = 0; r < RT; r++) s[r][j] = fmaf(q[r].x, kv.x, fmaf(q[r].y, kv.y, fmaf(q[r].z, kv.z, fmaf(q[r].w, kv.w, s[r][j]))));
      }
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int key = tx + 8 * j;
        s[r][j] = key < n ? fmaf(slope[r], (float)(p * PS + key - last_key[r]), s[r][j] * a.scale) : -INFINITY;
        mx = fmaxf(mx, s[r][j]);
      }
#pragma unroll
      for (int x = 1; x < 8; x *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[r], mx), ref = mn == -INFINITY ? 0.f : mn, corr = expf(m[r] - ref);
      m[r] = mn;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        s[r][j] = expf(s[r][j] - ref);
        ps += s[r][j];
        sp[(ty + 16 * r) * PP + tx + 8 * j] = s[r][j];
      }
      l[r] = fmaf(l[r], corr, ps);
#pragma unroll
      for (int d = 0; d < ND; d++) acc[r][d] *= corr;
    }
    __syncwarp();                                      // a row's 8 threads are of one warp
#pragma unroll 4
    for (int k = 0; k < PS; k++) {
      float w[RT];
#pragma unroll
      for (int r = 0; r < RT; r++) w[r] = sp[(ty + 16 * r) * PP + k];
#pragma unroll
      for (int d = 0; d < ND; d += 4) {
        const float4 vv = *reinterpret_cast<const float4*>(sv + k * PITCH + 4 * tx + 8 * d);
#pragma unroll
        for (int r = 0; r < RT; r++) {
          acc[r][d] = fmaf(w[r], vv.x, acc[r][d]);
          acc[r][d + 1] = fmaf(w[r], vv.y, acc[r][d + 1]);
          acc[r][d + 2] = fmaf(w[r], vv.z, acc[r][d + 2]);
          acc[r][d + 3] = fmaf(w[r], vv.w, acc[r][d + 3]);
        }
      }
    }
  }
  const int parts = a.prefix_splits + a.own_splits;
#pragma unroll
  for (int r = 0; r < RT; r++) {
    float lt = l[r];
#pragma unroll
    for (int x = 1; x < 8; x *= 2) lt += __shfl_xor_sync(0xffffffffu, lt, x);
    if (ty + 16 * r >= tk.rows) continue;
    int seq, head;
    row_of(a, tk, ty + 16 * r, seq, head);
    const size_t pi = ((size_t)seq * a.nh + head) * parts + tk.part;
#pragma unroll
    for (int d = 0; d < ND; d += 4) {
      const int at = 4 * tx + 8 * d;
      if (at < hd) *reinterpret_cast<float4*>(a.part_o + pi * hd + at) = make_float4(acc[r][d], acc[r][d + 1], acc[r][d + 2], acc[r][d + 3]);
    }
    if (tx == 0) { a.part_ml[pi * 2] = m[r] * LOG2E; a.part_ml[pi * 2 + 1] = lt; }
  }
}

template <int HDP>
__global__ void __launch_bounds__(F_THREADS)
k_attention_shared_f32(const __grid_constant__ SharedArgs a, int hd) {
  wait_then_let_next();
  extern __shared__ __align__(16) float sf[];
  Task tk;
  if (!find_task(a, F_ROWS, tk)) return;
  if (tk.rows > 16) walk_f32<HDP, 2>(a, tk, hd, sf);
  else walk_f32<HDP, 1>(a, tk, hd, sf);
}

template <int HD, int PLANES, int RW, int PRE>
int launch_shared_rows(SharedArgs a, int most, cudaStream_t stream) {
  const int G = a.nh / a.nkv, rows = PRE > 0 ? 8 * PRE : 16 * RW;
  a.prefix_tiles = (most * G + rows - 1) / rows;
  a.own_rows = PRE > 0 ? rows : 16;
  a.own_tiles = (G + a.own_rows - 1) / a.own_rows;
  a.least = PRE > 0 ? 1 : 2;
  a.own_least = own_least_of(a);
  constexpr size_t smem = PRE > 0 ? near_smem<HD, PRE, WARPS>() : walk_smem<HD, PLANES>();
  if (const int rc = prepare_kernel<k_attention_shared<HD, PLANES, RW, PRE>>(smem)) return rc;
  if (const int rc = cima_launch(k_attention_shared<HD, PLANES, RW, PRE>, dim3(blocks_of(a)), dim3(WARPS * 32), smem, stream, 1, a)) return rc;
  return launch_combine<__nv_bfloat16>(a, HD, stream);
}

// (Sixteen rows straight to registers are too many at head size 128, 255 registers and 112 bytes of spills: two blocks of eight there.)
template <int HD, int PLANES>
int launch_shared(const SharedArgs& a, int most, cudaStream_t stream) {
  const int rows = most * (a.nh / a.nkv);
  if constexpr (HD == 64 || HD == 128) {
    if (rows <= 16 && a.ld % 4 == 0 && ((uintptr_t)a.qkv & 7) == 0)
      return rows <= 8 || HD == 128 ? launch_shared_rows<HD, PLANES, 1, 1>(a, most, stream) : launch_shared_rows<HD, PLANES, 1, HD == 64 ? 2 : 1>(a, most, stream);
  }
  if (rows <= 16) return launch_shared_rows<HD, PLANES, 1, 0>(a, most, stream);
  return rows <= 32 ? launch_shared_rows<HD, PLANES, 2, 0>(a, most, stream) : launch_shared_rows<HD, PLANES, 4, 0>(a, most, stream);
}

template <int HDP>
int launch_shared_f32(SharedArgs a, int hd, int most, cudaStream_t stream) {
  const int G = a.nh / a.nkv;
  a.prefix_tiles = (most * G + F_ROWS - 1) / F_ROWS;
  a.own_rows = 16;
  a.own_tiles = (G + 15) / 16;
  const size_t smem = F32Smem<HDP>::floats * 4;
  if (const int rc = prepare_kernel<k_attention_shared_f32<HDP>>(smem)) return rc;
  if (const int rc = cima_launch(k_attention_shared_f32<HDP>, dim3(blocks_of(a)), dim3(F_THREADS), smem, stream, 1, a, hd)) return rc;
  return launch_combine<float>(a, hd, stream);
}

}  // namespace

// Row b of qkv is sequence b's new position, which the cache holds already (as position seq_len[b] - 1).  order [B], own_page [B],
// groups [n_groups, 3]: see SharedArgs; a group's pages are the same in all its sequences' tables and lie below their newest
// positions; `most`: sequences of the largest group.  part_o / part_ml: scratch of B * nh * (prefix_splits + own_splits) * (hd, 2) floats.
// early: as cima_attention_decode's (its lowest bit).
extern "C" int cima_attention_shared(const void* qkv, int dtype, int ld, const void* cache, const int* table, int table_width, int page_size,
                                     int planes, const int* seq_slot, const int* seq_len, const int* order, const int* own_page, const int* groups,
                                     int n_groups, int most, float* part_o, float* part_ml, int prefix_splits, int own_splits, void* out, int ldo,
                                     int B, int nh, int nkv, int hd, float scale, float sink, const float* head_sink, int gate_col,
                                     const float* slopes, int early, cudaStream_t stream) {
  if (B <= 0) return 0;
  const CimaPaged pg{table, table_width, 0, page_size, nkv, hd, planes};
  const SharedArgs a{qkv, cache, pg, seq_slot, seq_len, order, own_page, groups, head_sink, slopes, part_o, part_ml, out,
                     ld, ldo, B, nh, nkv, n_groups, 0, prefix_splits, 0, own_splits, gate_col, early & 1, scale, sink, 1, 16, 0};
  if (const int rc = check_shared("attention_shared", a, most)) return rc;
  if (dtype == CIMA_F32) {
    if (hd % 4 || hd < 4 || hd > 128) return cima_fail(CIMA_E_SIZE, "attention_shared: head_dim %d; in float32 this kernel takes multiples of 4 up to 128", hd);
    return hd <= 64 ? launch_shared_f32<64>(a, hd, most, stream) : launch_shared_f32<128>(a, hd, most, stream);
  }
  if (dtype != CIMA_BF16) return cima_fail(CIMA_E_DTYPE, "attention_shared: dtype code %d is neither float32 nor bfloat16", dtype);
  if (hd % 16 || hd < 16 || hd > 128) return cima_fail(CIMA_E_SIZE, "attention_shared: head_dim %d; this kernel takes multiples of 16 up to 128", hd);
  if (ld % 2 || ((uintptr_t)qkv & 3)) return cima_fail(CIMA_E_ARG, "attention_shared: qkv rows must be 4-byte aligned");
#define CASE(H) case H: return planes == 2 ? launch_shared<H, 2>(a, most, stream) : launch_shared<H, 1>(a, most, stream)
  switch (hd) {
    CASE(16); CASE(32); CASE(48); CASE(64); CASE(80); CASE(96); CASE(112); CASE(128);
  }
#undef CASE
  return cima_fail(CIMA_E_SIZE, "attention_shared: head_dim %d is not instantiated", hd);
}
