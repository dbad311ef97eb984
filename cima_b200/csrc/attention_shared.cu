// Decoding attention of a batch in which groups of sequences hold the same pages for a prefix: one new query a sequence,
// grouped-query, keys from the paged cache.
//
// With the keys of a sequence in two parts, the group's prefix P and its own rest R, a softmax over both is
//   m = max(m_P, m_R),  o = (2^(m_P - m) o_P + 2^(m_R - m) o_R) / (2^(m_P - m) l_P + 2^(m_R - m) l_R)
// with each part's maximum m (base 2), sum l of 2^(s - m) and accumulator o of 2^(s - m) v.  The prefix part of all of a group's sequences
// is one product: count * G query rows a kv head against keys that are read once, not once a sequence.
//
// One launch has two sorts of blocks, the groups' prefixes (first: they are the longer ones) and the sequences' own pages; both split
// their pages further where there are few of them.  A block walks its pages through shared memory with cp.async, and a tile of 16 rows
// belongs to one warp (prefixes of 64 rows: four tiles; fewer rows: the warps share the page's 64 keys, as for a sequence's own pages, whose rows
// are the heads of its kv head).  The parts go to scratch and k_shared_combine joins them in a fixed order.
//
// Scores, maxima, exponentials and sums are float32, base 2; probabilities are rounded to bfloat16 only as operand of P V.
#include "common.cuh"

namespace {

constexpr int PS = 64;             // keys per page
constexpr int WARPS = 4;
constexpr int MAX_PARTS = 128;     // parts of a row that the merge takes
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ void cp_async16(void* smem, const void* gmem) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(s), "l"(gmem));
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], const void* smem) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], const void* smem) {
  const unsigned s = (unsigned)__cvta_generic_to_shared(smem);
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {          // 2^x, float32, about 2 ulp; 2^(-inf) = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

struct SharedArgs {
  const void* qkv;                // [B, ld]: queries (and, from gate_col on, gates) of each sequence's new position
  const void* cache;              // a layer's pages [pages, planes, kv heads, 64, head_dim]
  CimaPaged pg;
  const int *seq_slot, *seq_len;  // [B]
  const int *order, *own_page;    // [B]: sequences group by group; page of sequence b at which its own keys begin
  const int* groups;              // [n_groups, 3]: place of the first sequence in `order`, sequences, pages
  const float *head_sink, *slopes;
  float *part_o, *part_ml;        // [B, nh, prefix_splits + own_splits, hd] and [.., 2]
  void* out;
  int ld, ldo, B, nh, nkv, n_groups, prefix_tiles, prefix_splits, own_tiles, own_splits, gate_col, early;
  float scale, sink;
};

// The part of `pages` pages that split s of at most n takes: pages [first, last).  Splits beyond the pages get none.
struct Share { int first, last; };
__device__ __forceinline__ int live_splits(int pages, int n) { return min(n, max(0, pages)); }
__device__ __forceinline__ Share share_of(int pages, int s, int n) {
  const int S = live_splits(pages, n);
  if (s >= S) return {0, 0};
  return {(int)((long long)s * pages / S), (int)((long long)(s + 1) * pages / S)};
}
__device__ __forceinline__ int pages_of(int len) { return (len + PS - 1) / PS; }

// What a block works on: rows (sequence, head) 0 .. rows - 1 against pages [first, last) of sequence `table_of`'s table, into part `part`.
struct Task {
  int kvh, rows, row0, G, group_first, seq, slot, first, last, part;
  bool prefix;
};

__device__ __forceinline__ bool find_task(const SharedArgs& a, int prefix_rows, Task& t) {
  t.G = a.nh / a.nkv;
  int i = blockIdx.x;
  const int prefix_blocks = a.n_groups * a.prefix_tiles * a.nkv * a.prefix_splits;
  t.prefix = i < prefix_blocks;
  if (t.prefix) {
    const int split = i % a.prefix_splits;
    i /= a.prefix_splits;
    t.kvh = i % a.nkv;
    i /= a.nkv;
    const int* g = a.groups + 3 * (i / a.prefix_tiles);
    t.row0 = (i % a.prefix_tiles) * prefix_rows;
    t.group_first = g[0];
    t.rows = min(prefix_rows, g[1] * t.G - t.row0);
    const Share s = share_of(g[2], split, a.prefix_splits);
    t.first = s.first, t.last = s.last, t.part = split;
    if (t.rows <= 0 || s.first >= s.last) return false;
    t.seq = a.order[t.group_first];                    // the group's pages are in any of its sequences' tables
  } else {
    i -= prefix_blocks;
    const int split = i % a.own_splits;
    i /= a.own_splits;
    const int tile = i % a.own_tiles;
    i /= a.own_tiles;
    t.kvh = i % a.nkv;
    t.seq = i / a.nkv;
    t.row0 = tile * 16;
    t.rows = min(16, t.G - t.row0);
    t.group_first = 0;
    const int from = a.own_page[t.seq];
    const Share s = share_of(pages_of(a.seq_len[t.seq]) - from, split, a.own_splits);
    t.first = from + s.first, t.last = from + s.last, t.part = a.prefix_splits + split;
    if (s.first >= s.last) return false;
  }
  t.slot = a.seq_slot[t.seq];
  return true;
}

// Row r of a task: its sequence and head.
__device__ __forceinline__ void row_of(const SharedArgs& a, const Task& t, int r, int& seq, int& head) {
  const int at = t.row0 + r;
  if (t.prefix) {
    seq = a.order[t.group_first + at / t.G];
    head = t.kvh * t.G + at % t.G;
  } else {
    seq = t.seq;
    head = t.kvh * t.G + at;
  }
}

__host__ __device__ constexpr int shared_stages(int hd, int planes) {
  const int n = (104 * 1024) / (planes * PS * (hd + 8) * 2);
  return n < 3 ? 3 : (n > 8 * (3 - planes) ? 8 * (3 - planes) : n);
}

// RW tiles of 16 rows, one a warp, 4 / RW warps share a page's keys.
template <int HD, int PLANES, int RW>
__device__ __forceinline__ void walk(const SharedArgs& a, const Task& tk, unsigned char* smem_raw) {
  constexpr int ROW = HD + 8, TILE = PS * ROW, KSTEPS = HD / 16, NTILES = HD / 8, STAGES = shared_stages(HD, PLANES);
  constexpr int KEYS = PS / (WARPS / RW), NJ = KEYS / 8;       // keys of a page that a warp takes, in tiles of 8
  const __nv_bfloat16* cache = (const __nv_bfloat16*)a.cache;
  const __nv_bfloat16* qkv = (const __nv_bfloat16*)a.qkv;
  __nv_bfloat16* tiles = reinterpret_cast<__nv_bfloat16*>(smem_raw);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int rt = warp % RW, kw = warp / RW * KEYS;
  const int p0 = tk.first, p1 = tk.last, len = a.seq_len[tk.seq];

  auto page_of = [&](int p) { return a.pg.table[(size_t)tk.slot * a.pg.width + p]; };
  auto issue = [&](int page, int stage) {
    const __nv_bfloat16* src = cache + (((size_t)page * PLANES) * a.nkv + tk.kvh) * (size_t)(PS * HD);
    const __nv_bfloat16* vsrc = src + (size_t)a.nkv * (PS * HD);
    __nv_bfloat16* dst = tiles + (size_t)stage * PLANES * TILE;
    constexpr int CPR = HD / 8;
    for (int c = threadIdx.x; c < PS * CPR; c += WARPS * 32) {
      const int r = c / CPR, cc = c % CPR;
      cp_async16(dst + r * ROW + cc * 8, src + r * HD + cc * 8);
      if (PLANES == 2) cp_async16(dst + TILE + r * ROW + cc * 8, vsrc + r * HD + cc * 8);
    }
  };
  // pages below the one of the newest position are older than the kernel before this one, which may still be running
  int ahead = 0;
  if (a.early) {
    while (ahead < STAGES - 1 && p0 + ahead < p1 && (tk.prefix || p0 + ahead < (len - 1) / PS)) {
      issue(page_of(p0 + ahead), ahead);
      cp_async_commit();
      ahead++;
    }
    cima_pdl_wait();
  }
  for (; ahead < STAGES - 1; ahead++) {
    if (p0 + ahead < p1) issue(page_of(p0 + ahead), ahead);
    cp_async_commit();
  }
  int page_next = p0 + STAGES - 1 < p1 ? page_of(p0 + STAGES - 1) : 0;

  // this warp's rows g and g + 8: their queries as A fragments, slopes and lengths
  uint32_t q[KSTEPS][4];
  float sl2[2] = {0.f, 0.f};
  int last_key[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 2; e++) {
    const int r = rt * 16 + g + 8 * e;
    const __nv_bfloat16* qp = nullptr;
    if (r < tk.rows) {
      int seq, head;
      row_of(a, tk, r, seq, head);
      qp = qkv + (size_t)seq * a.ld + (size_t)head * HD;
      last_key[e] = a.seq_len[seq] - 1;
      if (a.slopes) sl2[e] = a.slopes[head] * LOG2E;
    }
#pragma unroll
    for (int kk = 0; kk < KSTEPS; kk++) {
      q[kk][e] = qp ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 2 * t) : 0u;
      q[kk][2 + e] = qp ? *reinterpret_cast<const uint32_t*>(qp + kk * 16 + 2 * t + 8) : 0u;
    }
  }
  const float sc2 = a.scale * LOG2E;
  float o[NTILES][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NTILES; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  for (int p = p0; p < p1; p++) {
    const int stage = (p - p0) % STAGES;
    cp_async_wait<STAGES - 2>();
    __syncthreads();
    if (p + STAGES - 1 < p1) issue(page_next, (p - p0 + STAGES - 1) % STAGES);
    cp_async_commit();
    if (p + STAGES < p1) page_next = page_of(p + STAGES);
    const __nv_bfloat16* Kt = tiles + (size_t)stage * PLANES * TILE;
    __nv_bfloat16* Vt = PLANES == 2 ? const_cast<__nv_bfloat16*>(Kt) + TILE : const_cast<__nv_bfloat16*>(Kt);
    const bool ends = !tk.prefix && p * PS + PS > len;          // positions behind the sequence's end may hold anything
    if (ends) {                                        // a weight of 0 times infinity would be NaN: their values (and keys) are taken as 0
      for (int i = threadIdx.x; i < (p * PS + PS - len) * (HD / 8); i += WARPS * 32) {
        const int at = (len - p * PS + i / (HD / 8)) * ROW + i % (HD / 8) * 8;
        *reinterpret_cast<uint4*>(Vt + at) = make_uint4(0u, 0u, 0u, 0u);
      }
      __syncthreads();
    }
    if (rt * 16 >= tk.rows) continue;                  // a tile without rows (its warp still moved its part of the page)
    float s[NJ][4];
#pragma unroll
    for (int j = 0; j < NJ; j++) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; kk++)
#pragma unroll
      for (int j = 0; j < NJ; j += 2) {
        uint32_t kb[4];
        ldmatrix_x4(kb, Kt + (kw + j * 8 + (lane & 7) + 8 * (lane >> 4)) * ROW + kk * 16 + 8 * ((lane >> 3) & 1));
        mma_bf16(s[j], q[kk], kb[0], kb[1]);
        mma_bf16(s[j + 1], q[kk], kb[2], kb[3]);
      }
    float mx[2] = {-INFINITY, -INFINITY};
    const int key0 = p * PS + kw;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int key = key0 + j * 8 + 2 * t + (e & 1);
        float v = s[j][e] * sc2;
        if (a.slopes) v = fmaf(sl2[e >> 1], (float)(key - last_key[e >> 1]), v);
        if (ends && key >= len) v = -INFINITY;
        s[j][e] = v;
        mx[e >> 1] = fmaxf(mx[e >> 1], v);
      }
    float corr[2], ref[2], psum[2] = {0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 2; r++) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      const float mn = fmaxf(m_run[r], mx[r]);
      ref[r] = mn == -INFINITY ? 0.f : mn;
      corr[r] = ex2(m_run[r] - ref[r]);
      m_run[r] = mn;
    }
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[j][e] = ex2(s[j][e] - ref[e >> 1]);
        psum[e >> 1] += s[j][e];
      }
#pragma unroll
    for (int r = 0; r < 2; r++) l_run[r] = fmaf(l_run[r], corr[r], psum[r]);         // this thread's keys; the quad is summed at the end
#pragma unroll
    for (int j = 0; j < NTILES; j++) {
      o[j][0] *= corr[0]; o[j][1] *= corr[0];
      o[j][2] *= corr[1]; o[j][3] *= corr[1];
    }
#pragma unroll
    for (int k = 0; k < KEYS / 16; k++) {
      const uint32_t pa[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]),
                              pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]), pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
      for (int j = 0; j < NTILES; j += 2) {
        uint32_t vb[4];
        ldmatrix_x4_trans(vb, Vt + (kw + k * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * ROW + j * 8 + 8 * (lane >> 4));
        mma_bf16(o[j], pa, vb[0], vb[1]);
        mma_bf16(o[j + 1], pa, vb[2], vb[3]);
      }
    }
  }
  cp_async_wait<0>();
  __syncthreads();
  cima_pdl_trigger();
#pragma unroll
  for (int r = 0; r < 2; r++) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
  }
  const int parts = a.prefix_splits + a.own_splits;
  if (RW == WARPS) {                                   // a warp has its rows to itself
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = rt * 16 + g + 8 * e;
      if (r >= tk.rows) continue;
      int seq, head;
      row_of(a, tk, r, seq, head);
      const size_t pi = ((size_t)seq * a.nh + head) * parts + tk.part;
#pragma unroll
      for (int j = 0; j < NTILES; j++) *reinterpret_cast<float2*>(a.part_o + pi * HD + j * 8 + 2 * t) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
      if (t == 0) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(m_run[e], l_run[e]);
    }
    return;
  }
  // the warps that share a tile of rows, joined in their order through shared memory (in the pages' place)
  float* so = reinterpret_cast<float*>(smem_raw);      // [WARPS][16][HD]
  float* sml = so + WARPS * 16 * HD;                   // [WARPS][16][2]
#pragma unroll
  for (int j = 0; j < NTILES; j++) {
    float* base = so + ((size_t)warp * 16 + g) * HD + j * 8 + 2 * t;
    base[0] = o[j][0]; base[1] = o[j][1];
    base[8 * HD] = o[j][2]; base[8 * HD + 1] = o[j][3];
  }
  if (t == 0) {
    sml[(warp * 16 + g) * 2] = m_run[0]; sml[(warp * 16 + g) * 2 + 1] = l_run[0];
    sml[(warp * 16 + g + 8) * 2] = m_run[1]; sml[(warp * 16 + g + 8) * 2 + 1] = l_run[1];
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < tk.rows * HD; idx += WARPS * 32) {
    const int r = idx / HD, d = idx - r * HD, w0 = r / 16, rr = r % 16;
    float M = -INFINITY;
#pragma unroll
    for (int w = w0; w < WARPS; w += RW) M = fmaxf(M, sml[(w * 16 + rr) * 2]);
    const float ref = M == -INFINITY ? 0.f : M;
    float acc = 0.f, l = 0.f;
#pragma unroll
    for (int w = w0; w < WARPS; w += RW) {
      const float f = ex2(sml[(w * 16 + rr) * 2] - ref);
      acc += f * so[((size_t)w * 16 + rr) * HD + d];
      l += f * sml[(w * 16 + rr) * 2 + 1];
    }
    int seq, head;
    row_of(a, tk, r, seq, head);
    const size_t pi = ((size_t)seq * a.nh + head) * parts + tk.part;
    a.part_o[pi * HD + d] = acc;
    if (d == 0) { a.part_ml[pi * 2] = M; a.part_ml[pi * 2 + 1] = l; }
  }
}

// PREFIX_RW: tiles of 16 rows in a block of a group's prefix.
template <int HD, int PLANES, int PREFIX_RW>
__global__ void __launch_bounds__(WARPS * 32)
k_attention_shared(const __grid_constant__ SharedArgs a) {
  if (!a.early) cima_pdl_wait();
  extern __shared__ __align__(16) unsigned char smem_raw[];
  Task t;
  if (!find_task(a, 16 * PREFIX_RW, t)) return;
  if (PREFIX_RW > 1 && t.prefix) walk<HD, PLANES, PREFIX_RW>(a, t, smem_raw);
  else walk<HD, PLANES, 1>(a, t, smem_raw);
}

// The same in float32, sums and all, by multiply-adds: a block takes ROWS rows, a page's keys lie in shared memory, a thread has RT rows x 8 keys of
// the scores and RT rows x HDP / 8 values of the result.  hd is a multiple of 4.
constexpr int F_THREADS = 128, F_ROWS = 32;
template <int HDP> struct F32Smem {
  static constexpr int PITCH = HDP + 4, PP = PS + 4;
  static constexpr size_t floats = (size_t)F_ROWS * PITCH + 2 * PS * PITCH + F_ROWS * PP;
};

template <int HDP>
__global__ void __launch_bounds__(F_THREADS)
k_attention_shared_f32(const __grid_constant__ SharedArgs a, int hd) {
  cima_pdl_wait();
  extern __shared__ __align__(16) float sf[];
  constexpr int PITCH = F32Smem<HDP>::PITCH, PP = F32Smem<HDP>::PP, RT = F_ROWS / 16, ND = HDP / 8;
  float *sq = sf, *sk = sq + F_ROWS * PITCH, *sv = sk + PS * PITCH, *sp = sv + PS * PITCH;
  Task tk;
  if (!find_task(a, F_ROWS, tk)) return;
  const float* cache = (const float*)a.cache;
  const int tid = threadIdx.x, ty = tid >> 3, tx = tid & 7, len = a.seq_len[tk.seq], h4 = hd / 4;
  for (int i = tid; i < F_ROWS * (HDP / 4); i += F_THREADS) {
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
    if (ty + 16 * r < tk.rows) {
      int seq, head;
      row_of(a, tk, ty + 16 * r, seq, head);
      last_key[r] = a.seq_len[seq] - 1;
      if (a.slopes) slope[r] = a.slopes[head];
    }
#pragma unroll
    for (int d = 0; d < ND; d++) acc[r][d] = 0.f;
  }
  const int live_rt = (tk.rows + 15) / 16;
  for (int p = tk.first; p < tk.last; p++) {
    const int page = a.pg.table[(size_t)tk.slot * a.pg.width + p];
    const float* ksrc = cache + ((size_t)page * a.pg.planes * a.nkv + tk.kvh) * (size_t)(PS * hd);
    const float* vsrc = ksrc + a.pg.value_offset();
    const int n = tk.prefix ? PS : min(PS, len - p * PS);       // positions behind the sequence's end count as zeros
    __syncthreads();
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
#pragma unroll
    for (int rr = 0; rr < RT; rr++) {
      if (rr >= live_rt) break;
      const int row = ty + 16 * rr;
      float s[8];
#pragma unroll
      for (int j = 0; j < 8; j++) s[j] = 0.f;
      for (int c = 0; c < h4; c++) {
        const float4 qv = *reinterpret_cast<const float4*>(sq + row * PITCH + 4 * c);
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const float4 kv = *reinterpret_cast<const float4*>(sk + (tx + 8 * j) * PITCH + 4 * c);
          s[j] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[j]))));
        }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int key = tx + 8 * j;
        s[j] = key < n ? fmaf(slope[rr], (float)(p * PS + key - last_key[rr]), s[j] * a.scale) : -INFINITY;
        mx = fmaxf(mx, s[j]);
      }
#pragma unroll
      for (int x = 1; x < 8; x *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
      const float mn = fmaxf(m[rr], mx), ref = mn == -INFINITY ? 0.f : mn, corr = expf(m[rr] - ref);
      m[rr] = mn;
      float ps = 0.f;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        s[j] = expf(s[j] - ref);
        ps += s[j];
        sp[row * PP + tx + 8 * j] = s[j];
      }
      l[rr] = fmaf(l[rr], corr, ps);
#pragma unroll
      for (int d = 0; d < ND; d++) acc[rr][d] *= corr;
      __syncwarp();                                    // a row's 8 threads are of one warp
      for (int k = 0; k < PS; k++) {
        const float w = sp[row * PP + k];
#pragma unroll
        for (int d = 0; d < ND; d += 4) {
          const float4 vv = *reinterpret_cast<const float4*>(sv + k * PITCH + 4 * tx + 8 * d);
          acc[rr][d] = fmaf(w, vv.x, acc[rr][d]);
          acc[rr][d + 1] = fmaf(w, vv.y, acc[rr][d + 1]);
          acc[rr][d + 2] = fmaf(w, vv.z, acc[rr][d + 2]);
          acc[rr][d + 3] = fmaf(w, vv.w, acc[rr][d + 3]);
        }
      }
      __syncwarp();
    }
  }
  cima_pdl_trigger();
  const int parts = a.prefix_splits + a.own_splits;
#pragma unroll
  for (int rr = 0; rr < RT; rr++) {
    float lt = l[rr];
#pragma unroll
    for (int x = 1; x < 8; x *= 2) lt += __shfl_xor_sync(0xffffffffu, lt, x);
    if (ty + 16 * rr >= tk.rows) continue;
    int seq, head;
    row_of(a, tk, ty + 16 * rr, seq, head);
    const size_t pi = ((size_t)seq * a.nh + head) * parts + tk.part;
#pragma unroll
    for (int d = 0; d < ND; d++) {
      const int at = 4 * tx + 8 * (d & ~3) + (d & 3);
      if (at < hd) a.part_o[pi * hd + at] = acc[rr][d];
    }
    if (tx == 0) { a.part_ml[pi * 2] = m[rr] * LOG2E; a.part_ml[pi * 2 + 1] = lt; }
  }
}

// The row's parts joined: first the prefix's splits, then its own pages'.
template <typename T>
__global__ void __launch_bounds__(128)
k_shared_combine(const __grid_constant__ SharedArgs a, int hd) {
  cima_pdl_wait();
  __shared__ float w[MAX_PARTS];
  __shared__ float s_inv;
  const int b = blockIdx.y, h = blockIdx.x, parts = a.prefix_splits + a.own_splits, own = a.own_page[b];
  const size_t base = ((size_t)b * a.nh + h) * parts;
  const int np = live_splits(own, a.prefix_splits), nr = live_splits(pages_of(a.seq_len[b]) - own, a.own_splits), n = np + nr;
  auto place = [&](int i) { return i < np ? i : a.prefix_splits + i - np; };
  if (threadIdx.x < 32) {
    float m[MAX_PARTS / 32], l[MAX_PARTS / 32], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < MAX_PARTS / 32; i++) {
      const int s = threadIdx.x + 32 * i;
      const float2 ml = s < n ? *reinterpret_cast<const float2*>(a.part_ml + (base + place(s)) * 2) : make_float2(-INFINITY, 0.f);
      m[i] = ml.x, l[i] = ml.y;
      M = fmaxf(M, m[i]);
    }
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < MAX_PARTS / 32; i++) {
      const int s = threadIdx.x + 32 * i;
      const float f = exp2f(m[i] - ref);
      if (s < n) w[s] = f;
      L += f * l[i];
    }
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
    const float extra = a.head_sink ? expf(a.head_sink[h]) : a.sink;
    if (extra != 0.f) L += extra * exp2f(-ref);
    if (threadIdx.x == 0) s_inv = L > 0.f ? 1.0f / L : 0.f;
  }
  __syncthreads();
  const T* qkv = (const T*)a.qkv;
  for (int d = threadIdx.x; d < hd; d += blockDim.x) {
    float acc = 0.f;
    for (int s = 0; s < n; s++) acc += w[s] * a.part_o[(base + place(s)) * hd + d];
    acc *= s_inv;
    if (a.gate_col > 0) acc *= cima_sigmoid(cima_to_f32<T>(qkv[(size_t)b * a.ld + a.gate_col + (size_t)h * hd + d]));
    ((T*)a.out)[(size_t)b * a.ldo + (size_t)h * hd + d] = cima_from_f32<T>(acc);
  }
}

int blocks_of(const SharedArgs& a) { return a.n_groups * a.prefix_tiles * a.nkv * a.prefix_splits + a.B * a.nkv * a.own_tiles * a.own_splits; }

template <typename K>
int raise_smem(K kern, size_t smem) {
  const cudaError_t e = smem > 48 * 1024 ? cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) : cudaSuccess;
  return e == cudaSuccess ? 0 : cima_fail((int)e, "attention_shared: cannot raise shared memory to %zu bytes: %s", smem, cudaGetErrorString(e));
}

template <int HD, int PLANES, int RW>
int launch_shared_rows(SharedArgs a, int most, cudaStream_t stream) {
  const int G = a.nh / a.nkv;
  a.prefix_tiles = (most * G + 16 * RW - 1) / (16 * RW);
  a.own_tiles = (G + 15) / 16;
  const size_t tiles = (size_t)shared_stages(HD, PLANES) * PLANES * PS * (HD + 8) * 2, merge = (size_t)WARPS * 16 * (HD + 2) * 4;
  const size_t smem = tiles > merge ? tiles : merge;
  auto kern = k_attention_shared<HD, PLANES, RW>;
  if (const int rc = raise_smem(kern, smem)) return rc;
  if (const int rc = cima_launch(kern, dim3(blocks_of(a)), dim3(WARPS * 32), smem, stream, 1, a)) return rc;
  const int rc = cima_launch(k_shared_combine<__nv_bfloat16>, dim3(a.nh, a.B), dim3(128), (size_t)0, stream, 1, a, HD);
  return rc ? rc : cima_launch_result();
}

template <int HD, int PLANES>
int launch_shared(const SharedArgs& a, int most, cudaStream_t stream) {
  const int rows = most * (a.nh / a.nkv);
  if (rows <= 16) return launch_shared_rows<HD, PLANES, 1>(a, most, stream);
  if (rows <= 32) return launch_shared_rows<HD, PLANES, 2>(a, most, stream);
  return launch_shared_rows<HD, PLANES, 4>(a, most, stream);
}

template <int HDP>
int launch_shared_f32(SharedArgs a, int hd, int most, cudaStream_t stream) {
  const int G = a.nh / a.nkv;
  a.prefix_tiles = (most * G + F_ROWS - 1) / F_ROWS;
  a.own_tiles = (G + 15) / 16;
  const size_t smem = F32Smem<HDP>::floats * 4;
  if (const int rc = raise_smem(k_attention_shared_f32<HDP>, smem)) return rc;
  if (const int rc = cima_launch(k_attention_shared_f32<HDP>, dim3(blocks_of(a)), dim3(F_THREADS), smem, stream, 1, a, hd)) return rc;
  const int rc = cima_launch(k_shared_combine<float>, dim3(a.nh, a.B), dim3(128), (size_t)0, stream, 1, a, hd);
  return rc ? rc : cima_launch_result();
}

}  // namespace

// Row b of qkv is sequence b's new position, which the cache holds already (as position seq_len[b] - 1).  order [B], own_page [B],
// groups [n_groups, 3]: see SharedArgs; a group's pages are the same in all its sequences' tables and lie below their newest
// positions; `most`: sequences of the largest group.  part_o / part_ml: scratch of B * nh * (prefix_splits + own_splits) * (hd, 2) floats.
// early: as cima_attention_decode's.
extern "C" int cima_attention_shared(const void* qkv, int dtype, int ld, const void* cache, const int* table, int table_width, int page_size,
                                     int planes, const int* seq_slot, const int* seq_len, const int* order, const int* own_page, const int* groups,
                                     int n_groups, int most, float* part_o, float* part_ml, int prefix_splits, int own_splits, void* out, int ldo,
                                     int B, int nh, int nkv, int hd, float scale, float sink, const float* head_sink, int gate_col,
                                     const float* slopes, int early, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (planes != 1 && planes != 2) return cima_fail(CIMA_E_ARG, "attention_shared: %d planes; pages hold keys | values (2) or one shared vector (1)", planes);
  if (page_size != PS) return cima_fail(CIMA_E_SIZE, "attention_shared: page size %d; this kernel takes 64", page_size);
  if (nh <= 0 || nkv <= 0 || nh % nkv || nh > 65535) return cima_fail(CIMA_E_SIZE, "attention_shared: %d heads are not a multiple of %d kv heads", nh, nkv);
  if (n_groups < 0 || most < 0 || n_groups > B || most > B || (n_groups > 0 && (!groups || most < 1))) return cima_fail(CIMA_E_ARG, "attention_shared: %d groups of at most %d sequences in a batch of %d", n_groups, most, B);
  if (prefix_splits < 1 || own_splits < 1 || prefix_splits + own_splits > MAX_PARTS || B > 65535)
    return cima_fail(CIMA_E_SIZE, "attention_shared: %d and %d splits / %d sequences exceed one launch", prefix_splits, own_splits, B);
  if (!part_o || !part_ml || !order || !own_page || !table || !cache) return cima_fail(CIMA_E_ARG, "attention_shared: the cache, its block table, the order of the sequences and scratch are needed");
  if (gate_col < 0 || (gate_col > 0 && gate_col + nh * hd > ld)) return cima_fail(CIMA_E_ARG, "attention_shared: %d gate values from column %d on exceed the rows of %d", nh * hd, gate_col, ld);
  if ((uintptr_t)cache & 15) return cima_fail(CIMA_E_ARG, "attention_shared: the cache must be 16-byte aligned");
  const long long G = nh / nkv, blocks = ((long long)n_groups * ((most * G + 15) / 16) * prefix_splits + (long long)B * ((G + 15) / 16) * own_splits) * nkv;
  if (blocks > 0x7fffffffll) return cima_fail(CIMA_E_SIZE, "attention_shared: %lld blocks exceed one launch", blocks);
  const CimaPaged pg{table, table_width, 0, page_size, nkv, hd, planes};
  const SharedArgs a{qkv, cache, pg, seq_slot, seq_len, order, own_page, groups, head_sink, slopes, part_o, part_ml, out,
                     ld, ldo, B, nh, nkv, n_groups, 0, prefix_splits, 0, own_splits, gate_col, early, scale, sink};
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
