// What the kernels of the attention over shared prefixes have in common: a step's arguments, a block's task, the walk of a block of
// mma.sync tiles through its pages, the merge of a row's parts.  (attention_shared.cu says what they compute.)
#pragma once
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

// The 128 threads that walk (a block may have more warps, which have no part in it).
__device__ __forceinline__ void block_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// The wait on the kernel before this one, and from then on the one behind may be placed beside this one's blocks, where it waits in turn.  (Not before:
// a kernel that begins may take it that all but the one just before it are complete.)
__device__ __forceinline__ void wait_then_let_next() {
  cima_pdl_wait();
  cima_pdl_trigger();
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
  int least;                      // pages of a split
  int own_rows;                   // rows of a block of a sequence's own pages
  int prefix_first;               // order of the two sorts of blocks (is_prefix)
  int own_least = 1;              // pages of a split of a sequence's own (own_least_of)
};

// The splits of `pages` pages, n at most and of at least `least` pages each (a split costs its results' way through memory and a place in the
// merge; a recorded step is launched for longer contexts than it may find), and the pages [first, last) of split s: splits beyond those get none.
struct Share { int first, last; };
__device__ __forceinline__ int live_splits(int pages, int n, int least) { return min(n, max(0, (pages + least - 1) / least)); }
__device__ __forceinline__ Share share_of(int pages, int s, int n, int least) {
  const int S = live_splits(pages, n, least);
  if (s >= S) return {0, 0};
  return {(int)((long long)s * pages / S), (int)((long long)(s + 1) * pages / S)};
}
__device__ __forceinline__ int pages_of(int len) { return (len + PS - 1) / PS; }

// What a block works on: rows (sequence, head) 0 .. rows - 1 against pages [first, last) of sequence `table_of`'s table, into part `part`.
struct Task {
  int kvh, rows, row0, G, group_first, seq, slot, first, last, part, len;
  bool prefix;
};

// Where there are blocks enough, a split of own pages only for 8 of them: a part more costs its way through memory and the merge, and most sequences have few.
inline int own_least_of(const SharedArgs& a) { return (long long)a.B * a.nkv * a.own_tiles * a.own_splits > 64 ? 8 : a.least; }

__host__ __device__ __forceinline__ int own_blocks_of(const SharedArgs& a) { return a.B * a.nkv * a.own_tiles * a.own_splits; }
__host__ __device__ __forceinline__ int prefix_blocks_of(const SharedArgs& a) { return a.n_groups * a.prefix_tiles * a.nkv * a.prefix_splits; }

// Which sort of blocks comes first; the other's take their places as they end.  On tcgen05 the prefixes where every sequence is in a group (a
// prefix's block has the longer chain), else the sequences' own pages, as one that shares nothing has the longest blocks.  Measured, prefixes first
// against own pages first: 48 sequences over 1,664 positions, 40 heads on 8, 20.3 / 24.4 us; 8 groups of 22 over 256, 28 on 4, 27.1 / 32.4; 64 over 16,384
// with up to 500 of their own 43.0 / 51.0; 28 over 3,520 with up to 760 20.3 / 19.5; with sequences alone 36 and 2 over 11,584 44.9 / 40.9, 24 and 7 over
// 1,536 19.6 / 19.1; over 50 drawn cases the other order is 3 % longer.  (In turn, one of each sort on an SM, was 4 us longer for 64 over 16,384 when a page
// was one product of P V: a prefix's block walks no faster beside one that waits for memory than beside its like.)  i: the block's index, then its index among its sort.
__device__ __forceinline__ bool is_prefix(const SharedArgs& a, int& i) {
  const int first = a.prefix_first ? prefix_blocks_of(a) : own_blocks_of(a);
  if (i < first) return a.prefix_first;
  i -= first;
  return !a.prefix_first;
}

__device__ __forceinline__ bool find_task(const SharedArgs& a, int prefix_rows, Task& t) {
  t.G = a.nh / a.nkv;
  int i = blockIdx.x;
  t.prefix = is_prefix(a, i);
  if (t.prefix) {
    const int split = i % a.prefix_splits;
    i /= a.prefix_splits;
    t.kvh = i % a.nkv;
    i /= a.nkv;
    const int* g = a.groups + 3 * (i / a.prefix_tiles);
    t.row0 = (i % a.prefix_tiles) * prefix_rows;
    t.group_first = g[0];
    t.rows = min(prefix_rows, g[1] * t.G - t.row0);
    const Share s = share_of(g[2], split, a.prefix_splits, a.least);
    t.first = s.first, t.last = s.last, t.part = split;
    if (t.rows <= 0 || s.first >= s.last) return false;
    t.seq = a.order[t.group_first];                    // the group's pages are in any of its sequences' tables
    t.len = t.last * PS;                               // every key of them is visible
  } else {
    const int split = i % a.own_splits;
    i /= a.own_splits;
    const int tile = i % a.own_tiles;
    i /= a.own_tiles;
    t.kvh = i % a.nkv;
    t.seq = i / a.nkv;
    t.row0 = tile * a.own_rows;
    t.rows = min(a.own_rows, t.G - t.row0);
    t.group_first = 0;
    const int from = a.own_page[t.seq];
    t.len = a.seq_len[t.seq];
    const Share s = share_of(pages_of(t.len) - from, split, a.own_splits, a.own_least);
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
  const int p0 = tk.first, p1 = tk.last, len = tk.len;

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
    wait_then_let_next();
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
    block_sync();
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
      block_sync();
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
    // Probabilities against the maximum of their own 16 keys, whose key's is 1 and so has no rounding to bfloat16, the 16 keys' sums from 0, brought to
    // the running maximum by float32 multiply-adds: against the running maximum the result was the further from 64 bits the more pages a block walks
    // (24 sequences over 2,560 positions, 8 heads on 2 of 96 dims: 2.1e-3, the ordinary kernel 1.96e-3).
    constexpr int STEPS = KEYS / 16;
    float mx[STEPS][2], f[STEPS][2], corr[2];
    const int key0 = p * PS + kw;
#pragma unroll
    for (int k = 0; k < STEPS; k++) mx[k][0] = mx[k][1] = -INFINITY;
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int key = key0 + j * 8 + 2 * t + (e & 1);
        float v = s[j][e] * sc2;
        if (a.slopes) v = fmaf(sl2[e >> 1], (float)(key - last_key[e >> 1]), v);
        if (ends && key >= len) v = -INFINITY;
        s[j][e] = v;
        mx[j / 2][e >> 1] = fmaxf(mx[j / 2][e >> 1], v);
      }
#pragma unroll
    for (int r = 0; r < 2; r++) {
      float mn = m_run[r];
#pragma unroll
      for (int k = 0; k < STEPS; k++) {
        mx[k][r] = fmaxf(mx[k][r], __shfl_xor_sync(0xffffffffu, mx[k][r], 1));
        mx[k][r] = fmaxf(mx[k][r], __shfl_xor_sync(0xffffffffu, mx[k][r], 2));
        mn = fmaxf(mn, mx[k][r]);
      }
      const float ref = mn == -INFINITY ? 0.f : mn;
      corr[r] = ex2(m_run[r] - ref);
      m_run[r] = mn;
      l_run[r] *= corr[r];                               // this thread's keys; the quad is summed at the end
#pragma unroll
      for (int k = 0; k < STEPS; k++) {
        const float own = mx[k][r] == -INFINITY ? 0.f : mx[k][r];
        f[k][r] = ex2(mx[k][r] - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 2 * k; j < 2 * k + 2; j++)
#pragma unroll
          for (int e = 2 * r; e < 2 * r + 2; e++) sum += s[j][e] = ex2(s[j][e] - own);
        l_run[r] = fmaf(sum, f[k][r], l_run[r]);
      }
    }
#pragma unroll
    for (int j = 0; j < NTILES; j++) {
      o[j][0] *= corr[0]; o[j][1] *= corr[0];
      o[j][2] *= corr[1]; o[j][3] *= corr[1];
    }
#pragma unroll
    for (int k = 0; k < STEPS; k++) {
      const uint32_t pa[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]),
                              pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]), pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
      for (int j = 0; j < NTILES; j += 2) {
        uint32_t vb[4];
        float s16[2][4] = {};
        ldmatrix_x4_trans(vb, Vt + (kw + k * 16 + (lane & 7) + 8 * ((lane >> 3) & 1)) * ROW + j * 8 + 8 * (lane >> 4));
        mma_bf16(s16[0], pa, vb[0], vb[1]);
        mma_bf16(s16[1], pa, vb[2], vb[3]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          o[j][e] = fmaf(s16[0][e], f[k][e >> 1], o[j][e]);
          o[j + 1][e] = fmaf(s16[1][e], f[k][e >> 1], o[j + 1][e]);
        }
      }
    }
  }
  cp_async_wait<0>();
  block_sync();
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
  block_sync();
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

__device__ __forceinline__ uint4 ld_once16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void mma_ab(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// A block's warps joined: each left the maxima (mr), sums (lr, of the lane's keys) and accumulators of 8 NB rows, tile (d, e) of o holding dims
// 32 d + 8 (g / 2) + g % 2 + 4 e (rows g) and those + 2 (rows g + 8); first all of them side by side in shared memory, then a warp a row.
template <int HD, int NB, int NW>
__device__ __forceinline__ void join_warps(const SharedArgs& a, const Task& tk, const float (&o)[NB][HD / 16][4], const float (&mr)[NB][2], const float (&lr)[NB][2],
                                           unsigned char* smem_raw) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  constexpr int R = 8 * NB, PITCH = HD + 1;
  float* so = reinterpret_cast<float*>(smem_raw);              // [NW][R][PITCH]
  float2* sml = reinterpret_cast<float2*>(so + NW * R * PITCH + (NW * R * PITCH & 1));      // [NW][R]
#pragma unroll
  for (int n = 0; n < NB; n++)
#pragma unroll
    for (int j = 0; j < 2; j++) {
      float l = lr[n][j];
#pragma unroll
      for (int x = 4; x < 32; x *= 2) l += __shfl_xor_sync(0xffffffffu, l, x);
      float* row = so + (warp * R + 8 * n + 2 * t + j) * PITCH + 8 * (g >> 1) + (g & 1);
#pragma unroll
      for (int i = 0; i < HD / 16; i++) {
        row[32 * (i >> 1) + 4 * (i & 1)] = o[n][i][j];
        row[32 * (i >> 1) + 4 * (i & 1) + 2] = o[n][i][j + 2];
      }
      if (g == 0) sml[warp * R + 8 * n + 2 * t + j] = make_float2(mr[n][j], l);
    }
  asm volatile("bar.sync 1, %0;" ::"n"(32 * NW) : "memory");
  const int parts = a.prefix_splits + a.own_splits;
#pragma unroll 1
  for (int r = warp; r < tk.rows; r += NW) {
    const float2 w = lane < NW ? sml[lane * R + r] : make_float2(-INFINITY, 0.f);
    float M = w.x;
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, x));
    M = __shfl_sync(0xffffffffu, M, 0);
    const float f = ex2(w.x - (M == -INFINITY ? 0.f : M));
    float l = f * w.y;
#pragma unroll
    for (int x = 4; x > 0; x >>= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
    float mine[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; i++) mine[i] = 0.f;
#pragma unroll
    for (int k = 0; k < NW; k++) {
      const float fw = __shfl_sync(0xffffffffu, f, k);
#pragma unroll
      for (int i = 0; i < HD / 32; i++) mine[i] = fmaf(fw, so[(k * R + r) * PITCH + lane + 32 * i], mine[i]);
    }
    int seq, head;
    row_of(a, tk, r, seq, head);
    const size_t pi = ((size_t)seq * a.nh + head) * parts + tk.part;
#pragma unroll
    for (int i = 0; i < HD / 32; i++) a.part_o[pi * HD + lane + 32 * i] = mine[i];
    if (lane == 0) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(M, l);
  }
}

// Up to 8 NB rows against the block's pages, keys and values straight to registers (as attention_decode_near.cu does): a warp takes 16 keys at a
// time, S = K Q^T with the keys as its 16 rows and the rows of the task as its columns, O = V^T P^T.  For few rows this chain of a page's
// way is half as long as through shared memory.  NW warps; smem: NW * 8 NB * (HD + 3) floats.
template <int HD, int PLANES, int NB, int NW>
__device__ __forceinline__ void walk_near(const SharedArgs& a, const Task& tk, unsigned char* smem_raw) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int len = tk.len, first = tk.first * (PS / 16), end = min(tk.last * (PS / 16), (len + 15) / 16);       // pieces of 16 keys
  const __nv_bfloat16* kbase = (const __nv_bfloat16*)a.cache + (size_t)tk.kvh * (PS * HD) + 8 * t;
  const size_t v_off = PLANES == 2 ? (size_t)a.nkv * (PS * HD) : 0;
  const int* table = a.pg.table + (size_t)tk.slot * a.pg.width;
  auto place = [&](int c) { return kbase + (size_t)table[c / (PS / 16)] * PLANES * a.nkv * (PS * HD) + (c % (PS / 16)) * 16 * HD; };
  // rows that are not loaded: keys keep what the registers hold (their scores are masked), values are cleared (a weight of 0 times an
  // earlier key's infinity would be NaN)
  uint4 kf[HD / 32][2] = {}, vf[HD / 32][2] = {};
  auto load = [&](uint4 (&r)[HD / 32][2], const __nv_bfloat16* src, int c, int from, int to, bool clear) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int key = c * 16 + g + 8 * h;
      if (key >= from && key < to) {
#pragma unroll
        for (int d = 0; d < HD / 32; d++) r[d][h] = ld_once16(src + (g + 8 * h) * HD + 32 * d);
      } else if (clear) {
#pragma unroll
        for (int d = 0; d < HD / 32; d++) r[d][h] = make_uint4(0u, 0u, 0u, 0u);
      }
    }
  };
  int c = first + warp;
  const bool busy = c < end;
  const int newest = a.early && !tk.prefix ? len - 1 : len;           // (the kernel before this one may still be writing that position)
  const __nv_bfloat16* src = nullptr;
  if (busy) {
    src = place(c);
    load(kf, src, c, 0, newest, false);
    load(vf, src + v_off, c, 0, newest, false);
  }
  if (a.early) wait_then_let_next();
  float o[NB][HD / 16][4], mr[NB][2], lr[NB][2];
#pragma unroll
  for (int n = 0; n < NB; n++) {
#pragma unroll
    for (int j = 0; j < HD / 16; j++) o[n][j][0] = o[n][j][1] = o[n][j][2] = o[n][j][3] = 0.f;
    mr[n][0] = mr[n][1] = -INFINITY;
    lr[n][0] = lr[n][1] = 0.f;
  }
  if (busy) {
    if (newest < len && c * 16 + 16 >= len) {
      load(kf, src, c, newest, len, false);
      load(vf, src + v_off, c, newest, len, false);
    }
    uint4 q[NB][HD / 32] = {};
    float sl2[NB][2] = {};
    int last_key[NB][2] = {};
#pragma unroll
    for (int n = 0; n < NB; n++) {
      if (8 * n + g < tk.rows) {
        int seq, head;
        row_of(a, tk, 8 * n + g, seq, head);
        const __nv_bfloat16* qp = (const __nv_bfloat16*)a.qkv + (size_t)seq * a.ld + (size_t)head * HD + 8 * t;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) {
          const uint2 lo = *reinterpret_cast<const uint2*>(qp + 32 * d), hi = *reinterpret_cast<const uint2*>(qp + 32 * d + 4);
          q[n][d] = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
      }
      if (a.slopes) {
#pragma unroll
        for (int j = 0; j < 2; j++)
          if (8 * n + 2 * t + j < tk.rows) {
            int seq, head;
            row_of(a, tk, 8 * n + 2 * t + j, seq, head);
            sl2[n][j] = a.slopes[head] * LOG2E;
            last_key[n][j] = a.seq_len[seq] - 1;
          }
      }
    }
    const float sc2 = a.scale * LOG2E;
#pragma unroll 1
    for (; c < end; c += NW) {
      const bool more = c + NW < end;
      if (more) src = place(c + NW);
      float sa[NB][4], sb[NB][4];
#pragma unroll
      for (int n = 0; n < NB; n++) {
#pragma unroll
        for (int e = 0; e < 4; e++) sa[n][e] = sb[n][e] = 0.f;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) {
          mma_ab(sa[n], kf[d][0].x, kf[d][1].x, kf[d][0].y, kf[d][1].y, q[n][d].x, q[n][d].y);
          mma_ab(sb[n], kf[d][0].z, kf[d][1].z, kf[d][0].w, kf[d][1].w, q[n][d].z, q[n][d].w);
        }
      }
      if (more) load(kf, src, c + NW, 0, len, false);
      const int key = c * 16 + g;
      uint32_t b0[NB], b1[NB];
      float corr[NB][2], f[NB][2];
      // probabilities against the 16 keys' own maximum, their sums brought to the running one in float32
#pragma unroll
      for (int n = 0; n < NB; n++) {
        float p[4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float v0 = (sa[n][j] + sb[n][j]) * sc2, v1 = (sa[n][j + 2] + sb[n][j + 2]) * sc2;
          if (a.slopes) {
            v0 = fmaf(sl2[n][j], (float)(key - last_key[n][j]), v0);
            v1 = fmaf(sl2[n][j], (float)(key + 8 - last_key[n][j]), v1);
          }
          if (key >= len) v0 = -INFINITY;
          if (key + 8 >= len) v1 = -INFINITY;
          float mx = fmaxf(v0, v1);
#pragma unroll
          for (int x = 4; x < 32; x *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, x));
          const float own = mx == -INFINITY ? 0.f : mx, mn = fmaxf(mr[n][j], mx), ms = mn == -INFINITY ? 0.f : mn;
          p[j] = ex2(v0 - own);
          p[j + 2] = ex2(v1 - own);
          corr[n][j] = ex2(mr[n][j] - ms);
          f[n][j] = ex2(mx - ms);
          mr[n][j] = mn;
          lr[n][j] = fmaf(lr[n][j], corr[n][j], (p[j] + p[j + 2]) * f[n][j]);
        }
        b0[n] = transposed(pack_bf16(p[0], p[1]));
        b1[n] = transposed(pack_bf16(p[2], p[3]));
      }
#pragma unroll
      for (int d = 0; d < HD / 32; d++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t a0 = transposed(e ? vf[d][0].z : vf[d][0].x), a1 = transposed(e ? vf[d][0].w : vf[d][0].y),
                         a2 = transposed(e ? vf[d][1].z : vf[d][1].x), a3 = transposed(e ? vf[d][1].w : vf[d][1].y);
#pragma unroll
          for (int n = 0; n < NB; n++) {
            float s16[4] = {0.f, 0.f, 0.f, 0.f};
            mma_ab(s16, a0, a1, a2, a3, b0[n], b1[n]);
#pragma unroll
            for (int i = 0; i < 4; i++) o[n][2 * d + e][i] = fmaf(o[n][2 * d + e][i], corr[n][i & 1], s16[i] * f[n][i & 1]);
          }
        }
      if (more) load(vf, src + v_off, c + NW, 0, len, true);
    }
  }
  join_warps<HD, NB, NW>(a, tk, o, mr, lr, smem_raw);
}

// The row's parts joined, first the prefix's splits, then its own pages': four warps a row (sequence, head), a lane has 4 neighbouring dims of every
// fourth part's accumulator, four parts' loads on their way at a time; then the warps in their order.  (One warp a row was 2 us slower with 56 parts.)
// What it reads of the step's plan is older than the kernel before it where that is so for that kernel, and is read before the wait then.
constexpr int COMBINE_WARPS = 4;

template <typename T>
__global__ void __launch_bounds__(32 * COMBINE_WARPS)
k_shared_combine(const __grid_constant__ SharedArgs a, int hd) {
  __shared__ float4 sums[COMBINE_WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, row = blockIdx.x;
  const int b = row / a.nh, h = row - b * a.nh, parts = a.prefix_splits + a.own_splits;
  const size_t base = (size_t)row * parts;
  if (!a.early) wait_then_let_next();
  const int own = a.own_page[b];
  const int np = live_splits(own, a.prefix_splits, a.least), nr = live_splits(pages_of(a.seq_len[b]) - own, a.own_splits, a.own_least);
  // the entry without a value, as one more part: its score (base 2; a stored one of +inf stands for the largest number, against which all else is nothing)
  // and how many of it there are.  (exp of the sink and of the maximum apart pass float32's range where their difference does not.)
  const float sink_m = a.head_sink ? a.head_sink[h] * LOG2E : 0.f, extra_m = sink_m > 3e38f ? 3e38f : sink_m, extra_n = a.head_sink ? 1.f : a.sink;
  if (a.early) wait_then_let_next();
  float w[MAX_PARTS / 32], l[MAX_PARTS / 32], M = -INFINITY, L = 0.f;
#pragma unroll
  for (int i = 0; i < MAX_PARTS / 32; i++) {
    const int s = lane + 32 * i;
    const bool live = s < np || (s >= a.prefix_splits && s < a.prefix_splits + nr);
    const float2 ml = live ? *reinterpret_cast<const float2*>(a.part_ml + (base + s) * 2) : make_float2(-INFINITY, 0.f);
    w[i] = ml.x, l[i] = ml.y;
    M = fmaxf(M, ml.x);
  }
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
  if (extra_n != 0.f) M = fmaxf(M, extra_m);
  const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
  for (int i = 0; i < MAX_PARTS / 32; i++) {
    w[i] = exp2f(w[i] - ref);                          // 0 for a place without a part
    L += w[i] * l[i];
  }
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
  if (extra_n != 0.f) L += extra_n * exp2f(extra_m - ref);
  const float inv = L == 0.f ? 0.f : 1.0f / L;
  const int n = np + nr, d = 4 * lane;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = warp; s0 < n; s0 += 4 * COMBINE_WARPS) {
    float4 o[4];
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int s = s0 + COMBINE_WARPS * u, at = s < np ? s : a.prefix_splits + s - np;
      o[u] = s < n && d < hd ? *reinterpret_cast<const float4*>(a.part_o + (base + at) * hd + d) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int u = 0; u < 4; u++) {
      const int s = s0 + COMBINE_WARPS * u, at = min(s < np ? s : a.prefix_splits + s - np, MAX_PARTS - 1);
      float f = 0.f;
#pragma unroll
      for (int i = 0; i < MAX_PARTS / 32; i++) {
        const float v = __shfl_sync(0xffffffffu, w[i], at & 31);
        if (at >> 5 == i) f = v;
      }
      if (s < n) {
        acc.x = fmaf(f, o[u].x, acc.x);
        acc.y = fmaf(f, o[u].y, acc.y);
        acc.z = fmaf(f, o[u].z, acc.z);
        acc.w = fmaf(f, o[u].w, acc.w);
      }
    }
  }
  sums[warp][lane] = acc;
  __syncthreads();
  const T *qkv = (const T*)a.qkv;
  for (int e = threadIdx.x; e < hd; e += 32 * COMBINE_WARPS) {
    float r = 0.f;
#pragma unroll
    for (int k = 0; k < COMBINE_WARPS; k++) r += reinterpret_cast<const float*>(sums[k])[e];
    r *= inv;
    if (a.gate_col > 0) r *= cima_sigmoid(cima_to_f32<T>(qkv[(size_t)b * a.ld + a.gate_col + (size_t)h * hd + e]));
    ((T*)a.out)[(size_t)b * a.ldo + (size_t)h * hd + e] = cima_from_f32<T>(r);
  }
}

inline int blocks_of(const SharedArgs& a) { return prefix_blocks_of(a) + own_blocks_of(a); }

template <int HD, int NB, int NW> __host__ __device__ constexpr size_t near_smem() { return (size_t)NW * 8 * NB * (HD + 3) * 4 + 8; }

template <int HD, int PLANES> __host__ __device__ constexpr size_t walk_smem() {
  const size_t tiles = (size_t)shared_stages(HD, PLANES) * PLANES * PS * (HD + 8) * 2, merge = (size_t)WARPS * 16 * (HD + 2) * 4;
  return tiles > merge ? tiles : merge;
}

// Once a kernel and device (as cudaFuncSetAttribute is).
template <auto KERN>
int prepare_kernel(size_t smem) {
  static bool done[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && dev >= 0 && dev < 64 && done[dev]) return 0;
  if (e == cudaSuccess && smem > 48 * 1024) e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return cima_fail((int)e, "attention_shared: cannot raise shared memory to %zu bytes: %s", smem, cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) done[dev] = true;
  return 0;
}

template <typename T>
int launch_combine(const SharedArgs& a, int hd, cudaStream_t stream) {
  const int rc = cima_launch(k_shared_combine<T>, dim3(a.B * a.nh), dim3(32 * COMBINE_WARPS), (size_t)0, stream, 1, a, hd);
  return rc ? rc : cima_launch_result();
}

// What holds of every call; `who` names the entry.
inline int check_shared(const char* who, const SharedArgs& a, int most) {
  const int planes = a.pg.planes;
  if (planes != 1 && planes != 2) return cima_fail(CIMA_E_ARG, "%s: %d planes; pages hold keys | values (2) or one shared vector (1)", who, planes);
  if (a.pg.page_size != PS) return cima_fail(CIMA_E_SIZE, "%s: page size %d; this kernel takes 64", who, a.pg.page_size);
  if (a.nh <= 0 || a.nkv <= 0 || a.nh % a.nkv || a.nh > 65535) return cima_fail(CIMA_E_SIZE, "%s: %d heads are not a multiple of %d kv heads", who, a.nh, a.nkv);
  if (a.n_groups < 0 || most < 0 || a.n_groups > a.B || most > a.B || (a.n_groups > 0 && (!a.groups || most < 1)))
    return cima_fail(CIMA_E_ARG, "%s: %d groups of at most %d sequences in a batch of %d", who, a.n_groups, most, a.B);
  if (a.prefix_splits < 1 || a.own_splits < 1 || a.prefix_splits + a.own_splits > MAX_PARTS || a.B > 65535)
    return cima_fail(CIMA_E_SIZE, "%s: %d and %d splits / %d sequences exceed one launch", who, a.prefix_splits, a.own_splits, a.B);
  if (!a.part_o || !a.part_ml || !a.order || !a.own_page || !a.pg.table || !a.cache)
    return cima_fail(CIMA_E_ARG, "%s: the cache, its block table, the order of the sequences and scratch are needed", who);
  if (a.gate_col < 0 || (a.gate_col > 0 && a.gate_col + a.nh * a.pg.head_dim > a.ld))
    return cima_fail(CIMA_E_ARG, "%s: %d gate values from column %d on exceed the rows of %d", who, a.nh * a.pg.head_dim, a.gate_col, a.ld);
  if ((uintptr_t)a.cache & 15) return cima_fail(CIMA_E_ARG, "%s: the cache must be 16-byte aligned", who);
  const long long G = a.nh / a.nkv, blocks = ((long long)a.n_groups * ((most * G + 7) / 8) * a.prefix_splits + (long long)a.B * ((G + 7) / 8) * a.own_splits) * a.nkv;
  if (blocks > 0x7fffffffll || (long long)a.B * a.nh > 0x7fffffffll) return cima_fail(CIMA_E_SIZE, "%s: %lld blocks, or %d rows of %d heads, exceed one launch", who, blocks, a.B, a.nh);
  return 0;
}

}  // namespace
