// Attention over shared prefixes (attention_shared.cu) with the prefixes' products on the fifth-generation tensor cores: for groups of more
// query rows a kv head than the mma.sync tiles carry, head_dim 64 or 128.
//
// A block of a prefix has 128 rows (sequence, head) of one kv head, TMEM's lanes, against a share of the group's pages: S = Q K^T of a page
// (128 x 64) and O += P V as tcgen05.mma with their results in tensor memory, P written over S as the A operand.  Warps 0 .. 3: a row a
// thread (rows are gathered into the swizzled Q tile by them, then softmax); warp 4: TMA of K and V through the block table; warp 5: TMEM and the
// MMAs.  S has two buffers, so S of the next page is computed while this one's probabilities are.  The K and V rings are two pages deep each.  Every key of a whole page is visible: no
// mask.  The reference point of the exponentials moves when a row's maximum has grown by more than 2^8, which spares O most rescalings and
// leaves probabilities below 2^8.  A probability goes into its product in two parts, its upper 16 bits and the next 8 of what they leave (2^-14 of it at most
// is lost), over the two halves of its S: rounded to bfloat16 once, a row stood 2.2 to 2.35e-3 from 64 bits where the ordinary kernel, whose probabilities
// are rounded against their own 16 keys' maximum, stands at 1.95e-3; in two parts 1.69e-3, the result's own rounding (the reference point at the maximum
// and the rounded ones summed: 2.15e-3).  The second product costs 64 sequences over 16,384 positions 37.4 -> 42.8 us, 4 groups of 6 over 4,032 18.5 -> 20.1, 8 over
// 2,048 10.6 -> 11.7; the parts are cut off and not rounded, as two conversions a pair took 6 us more.  (An infinite value makes its column NaN.)  The sequences' own pages are blocks of mma.sync as there, in the same launch: they are bound by bytes while the
// prefixes are bound by the tensor cores.
//
// Measured, 28 heads on 4 of 128 dims, 64 sequences over 16,384 positions and up to 500 of their own (15 GFLOP, 67 MB): 42.8 us with the merge.  A
// prefix's block: 4.8 until its first product, 21 pages at some 2,500 cycles (two blocks an SM; 1,875 with one product of P V a page), 2 to leave; own pages beside them; the merge 4.  8 sequences over 2,048 11.7 us, a chain of latencies.  (A kernel of the own pages alone
// beside one of the prefixes, a third launch, was no shorter, and 5 us longer where a few sequences share nothing.)
//
// Every wait on an mbarrier is bounded (2 s); one that runs out sets *error_flag, and all roles leave their loops, free the tensor memory and
// return.
#include "attention_shared.cuh"
#include "tcgen05.cuh"

namespace {

using namespace cima_tc;

constexpr int TC_ROWS = 128, TC_THREADS = 192, UMMA_K = 16;
constexpr int Q_BLOCK = TC_ROWS * 64 * 2, KV_BLOCK = PS * 64 * 2;      // 128 rows or 64 keys of 64 dims: 128-byte rows, swizzled

constexpr int FEW_ROWS = 8;
constexpr size_t ONE_AN_SM = 120 * 1024;                       // more than half of what an SM offers
constexpr int OWN_STAGES = 3;                                  // pages of a sequence's own on their way
constexpr int TMEM_PREFIX = 256, TMEM_OWN = 32;               // columns of tensor memory: two buffers of S and O; the fewest there are
// Shared memory: a prefix's Q tile, two stages of K and V, barriers and where its rows' queries lie, which is more than a sequence's own three
// pages and barriers; the last 16 bytes hold the address of the block's tensor memory, whatever its role.
template <int HD> __host__ __device__ constexpr size_t tc_smem() { return (HD / 64) * (size_t)(Q_BLOCK + 4 * KV_BLOCK) + 16 * 8 + TC_ROWS * 8 + 16; }

template <int HD, int PLANES>
__device__ __forceinline__ void prefix_tc(const CUtensorMap* map, const SharedArgs& a, const Task& tk, unsigned char* smem, const unsigned* tmem_slot, int* error_flag) {
  constexpr int NH = HD / 64;
  unsigned char* sq = smem;                                    // NH blocks (dims 0 .. 63, 64 .. 127) of 128 rows
  unsigned char* sk = sq + NH * Q_BLOCK;                       // [2 stages][NH][64 keys]
  unsigned char* sv = sk + 2 * NH * KV_BLOCK;
  unsigned long long* bars = (unsigned long long*)(sv + 2 * NH * KV_BLOCK);
  unsigned long long *q_full = bars, *k_full = bars + 1, *k_empty = bars + 3, *v_full = bars + 5, *v_empty = bars + 7, *s_full = bars + 9, *p_full = bars + 11,
                     *pv_done = bars + 13, *all_done = bars + 14;
  volatile int* abort_flag = (volatile int*)(bars + 15);
  long long* row_at = (long long*)(bars + 16);                 // [rows] where a row's query begins, -1: no row
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = tk.last - tk.first;

  if (threadIdx.x == 0) {
    if (smem_u32(smem) & 1023u) atomicExch(error_flag, 2);     // never seen; the tiles would be misread
    mbar_init(q_full, 4);
    for (int s = 0; s < 2; s++) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1);
      mbar_init(&s_full[s], 1); mbar_init(&p_full[s], 4);
    }
    mbar_init(pv_done, 1);
    mbar_init(all_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  const int r = threadIdx.x;                                   // the row of a thread of the first four warps
  const bool live = r < tk.rows;
  int seq = 0, head = 0;
  if (warp < 4) {
    if (live) row_of(a, tk, r, seq, head);
    row_at[r] = live ? (long long)seq * a.ld + head * HD : -1;
  }
  const int* table = a.pg.table + (size_t)tk.slot * a.pg.width + tk.first;
  const int first_page = warp == 4 ? table[0] : 0;
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const unsigned tmem_base = *tmem_slot;
  const unsigned tm_s[2] = {tmem_base, tmem_base + 64u};
  const unsigned tm_o = tmem_base + 128u;

  if (warp == 4) {
    // ---------------------------------------------------------------- TMA: lane 0 K, lane 1 V (pages are older than the kernel before this one)
    // (the two lanes' loops are apart: K's place is free a page's softmax before V's, and K must not wait for it)
    auto fetch = [&](unsigned char* dst, unsigned long long* full, unsigned long long* empty, int plane) {
      int page = first_page;
      for (int j = 0; j < n; j++) {
        const int s = j & 1, next = j + 1 < n ? table[j + 1] : 0;
        if (j >= 2 && !mbar_wait(&empty[s], ((j >> 1) - 1) & 1, error_flag, abort_flag)) break;
        mbar_expect_tx(&full[s], NH * KV_BLOCK);
        const int y = ((page * PLANES + plane) * a.nkv + tk.kvh) * PS;
#pragma unroll
        for (int kb = 0; kb < NH; kb++) tma_load_2d(dst + (size_t)(NH * s + kb) * KV_BLOCK, map, 64 * kb, y, &full[s]);
        page = next;
      }
    };
    if (lane == 0) fetch(sk, k_full, k_empty, 0);
    else if (lane == 1) fetch(sv, v_full, v_empty, PLANES - 1);
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA issue (one thread)
    if (lane == 0) {
      const unsigned idesc_s = umma_idesc(TC_ROWS, PS), idesc_o = umma_idesc(TC_ROWS, HD) | (1u << 16);      // B of P V is MN-major
      auto issue_s = [&](int j) {
        const int s = j & 1;
#pragma unroll
        for (int kb = 0; kb < NH; kb++) {
          const unsigned long long qd = umma_smem_desc(smem_u32(sq + (size_t)kb * Q_BLOCK));
          const unsigned long long kd = umma_smem_desc(smem_u32(sk + (size_t)(NH * s + kb) * KV_BLOCK));
#pragma unroll
          for (int k = 0; k < 64 / UMMA_K; k++)
            umma_bf16(tm_s[s], qd + (unsigned long long)(k * 2), kd + (unsigned long long)(k * 2), idesc_s, (kb | k) ? 1u : 0u);
        }
        umma_commit(&s_full[s]);
        umma_commit(&k_empty[s]);
      };
      bool ok = mbar_wait(q_full, 0, error_flag, abort_flag) && mbar_wait(&k_full[0], 0, error_flag, abort_flag);
      if (ok) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        issue_s(0);
      }
      for (int j = 0; j < n && ok; j++) {
        if (j + 1 < n) {
          const int s1 = (j + 1) & 1;
          ok = mbar_wait(&k_full[s1], ((j + 1) >> 1) & 1, error_flag, abort_flag);
          // buffer s1 held S of page j - 1 and then its P: free once P V of page j - 1 is complete
          if (ok && j >= 1) ok = mbar_wait(pv_done, (j - 1) & 1, error_flag, abort_flag);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          issue_s(j + 1);
        }
        const int s = j & 1;
        ok = mbar_wait(&v_full[s], (j >> 1) & 1, error_flag, abort_flag) && mbar_wait(&p_full[s], (j >> 1) & 1, error_flag, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const unsigned long long vd = umma_smem_desc_mn(smem_u32(sv + (size_t)NH * s * KV_BLOCK), KV_BLOCK);
#pragma unroll
        for (int k = 0; k < 2 * (PS / UMMA_K); k++)             // P in two parts, both against the same values
          umma_bf16_ts(tm_o, tm_s[s] + (unsigned)(k * (UMMA_K / 2)), vd + (unsigned long long)(k % (PS / UMMA_K) * (UMMA_K * 128 >> 4)), idesc_o, (j | k) ? 1u : 0u);
        umma_commit(&v_empty[s]);
        umma_commit(pv_done);
      }
      if (ok) umma_commit(all_done);
    }
  } else {
    // ---------------------------------------------------------------- the rows
    if (a.early) wait_then_let_next();
    const __nv_bfloat16* qkv = (const __nv_bfloat16*)a.qkv;
    {                                                          // Q: chunk c of 16 bytes of a 128-byte row lies at place c ^ (row & 7); all loads at once
      constexpr int CPR = HD / 8;
      uint4 v[CPR];
#pragma unroll
      for (int i = 0; i < CPR; i++) {
        const int at = threadIdx.x + 128 * i;
        const long long from = row_at[at / CPR];
        v[i] = from >= 0 ? *reinterpret_cast<const uint4*>(qkv + from + 8 * (at % CPR)) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int i = 0; i < CPR; i++) {
        const int at = threadIdx.x + 128 * i, row = at / CPR, c = at % CPR;
        *reinterpret_cast<uint4*>(sq + (c / 8) * Q_BLOCK + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = v[i];
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    const unsigned lane_off = (unsigned)(warp * 32) << 16;
    const float sc_in = a.scale * LOG2E;
    const float sl2 = a.slopes && live ? a.slopes[head] * LOG2E : 0.f;
    const int last_key = a.slopes && live ? a.seq_len[seq] - 1 : 0;
    const float sc2 = a.slopes ? 1.0f : sc_in;                 // with a distance bias the scores are scaled where it is added
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    for (int j = 0; j < n && ok; j++) {
      const int s = j & 1;
      ok = mbar_wait(&s_full[s], (j >> 1) & 1, error_flag, abort_flag);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      unsigned raw[2][32];
      tmem_ld32_issue(tm_s[s] + lane_off, raw[0]);
      tmem_ld32_issue(tm_s[s] + lane_off + 32u, raw[1]);
      tmem_ld_wait();
      if (a.slopes) {
        const float far = sl2 * (float)((tk.first + j) * PS - last_key);
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int e = 0; e < 32; e++) raw[c][e] = __float_as_uint(fmaf(__uint_as_float(raw[c][e]), sc_in, fmaf(sl2, (float)(c * 32 + e), far)));
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 32; e++) mx4[e & 3] = fmaxf(mx4[e & 3], __uint_as_float(raw[c][e]));
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sc2;
      float alpha = 1.0f;
      if (mx > m_run + 8.0f) {                                 // also the first page (m_run = -inf)
        alpha = ex2(m_run - mx);
        m_run = mx;
      }
      const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
      l_run *= alpha;
      float ps4[4] = {0.f, 0.f, 0.f, 0.f};
      unsigned pk[32], rest[32];
#pragma unroll
      for (int c = 0; c < 2; c++)
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float p0 = ex2(fmaf(__uint_as_float(raw[c][e]), sc2, neg_m));
          const float p1 = ex2(fmaf(__uint_as_float(raw[c][e + 1]), sc2, neg_m));
          const unsigned u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
          pk[c * 16 + (e >> 1)] = __byte_perm(u0, u1, 0x7632);
          rest[c * 16 + (e >> 1)] = __byte_perm(__float_as_uint(p0 - __uint_as_float(u0 & 0xffff0000u)), __float_as_uint(p1 - __uint_as_float(u1 & 0xffff0000u)), 0x7632);
          ps4[(e >> 1) & 3] += p0 + p1;
        }
      l_run += (ps4[0] + ps4[1]) + (ps4[2] + ps4[3]);
      if (j > 0 && __any_sync(0xffffffffu, alpha != 1.0f)) {    // O may be touched once the page before's P V is complete
        ok = mbar_wait(pv_done, (j - 1) & 1, error_flag, abort_flag);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll 1
        for (int c = 0; c < HD / 32; c++) {
          float o[32];
          tmem_ld32(tm_o + lane_off + (unsigned)(c * 32), o);
#pragma unroll
          for (int e = 0; e < 32; e++) o[e] *= alpha;
          tmem_st32(tm_o + lane_off + (unsigned)(c * 32), o);
        }
      }
      tmem_st32_words(tm_s[s] + lane_off, pk);                 // P over the first 32 columns of its S, what its rounding left over the others
      tmem_st32_words(tm_s[s] + lane_off + 32u, rest);
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[s]);                  // (one barrier a buffer: no waiter can be a phase behind)
    }
    // The last P V has a barrier of its own: pv_done, asked by parity, would answer for page n - 3 while page n - 2 is not complete, and not
    // at all for page n - 2 once page n - 1 is (a warp held up between its last announcement and here waited two seconds).
    if (ok) ok = mbar_wait(all_done, 0, error_flag, abort_flag);
    if (ok) {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      // a warp's 32 rows through shared memory (in the tiles' place: every MMA that read them is complete), so that a row leaves as one piece
      const size_t pi = live ? ((size_t)seq * a.nh + head) * (a.prefix_splits + a.own_splits) + tk.part : 0;
      constexpr int PITCH = HD + 4;
      float* rows = reinterpret_cast<float*>(smem) + warp * 32 * PITCH;
#pragma unroll 1
      for (int c = 0; c < HD / 32; c++) {
        float o[32];
        tmem_ld32(tm_o + lane_off + (unsigned)(c * 32), o);
#pragma unroll
        for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(rows + lane * PITCH + c * 32 + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
      }
      if (live) *reinterpret_cast<float2*>(a.part_ml + pi * 2) = make_float2(m_run, l_run);
      __syncwarp();
      constexpr int LPR = HD / 4;                              // lanes of a row
      const int here = min(32, tk.rows - warp * 32);
#pragma unroll 4
      for (int i = lane / LPR; i < 32; i += 32 / LPR) {
        const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)pi, i);
        if (i < here) *reinterpret_cast<float4*>(a.part_o + to * HD + 4 * (lane % LPR)) = *reinterpret_cast<const float4*>(rows + i * PITCH + 4 * (lane % LPR));
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
}

// A sequence's own pages (8 NB rows at most): three pages on their way by TMA, 16 keys of a page to each of the first four warps, mma.sync as
// walk_near (which had one round of loads on its way a warp: four to five thousand cycles a round, 23,000 a block of 250 positions in a launch of 256).
template <int HD, int PLANES, int NB>
__device__ __forceinline__ void own_tma(const CUtensorMap* map, const SharedArgs& a, const Task& tk, unsigned char* smem, int* error_flag) {
  constexpr int NH = HD / 64, STAGE = PLANES * NH * KV_BLOCK;
  unsigned long long *full = (unsigned long long*)(smem + OWN_STAGES * 2 * NH * KV_BLOCK), *empty = full + OWN_STAGES;
  volatile int* abort_flag = (volatile int*)(empty + OWN_STAGES);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n = tk.last - tk.first, len = tk.len;
  if (threadIdx.x == 0) {
    for (int s = 0; s < OWN_STAGES; s++) { mbar_init(&full[s], 1); mbar_init(&empty[s], 4); }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  const int* table = a.pg.table + (size_t)tk.slot * a.pg.width + tk.first;
  int page = warp == 4 ? table[0] : 0;
  __syncthreads();
  if (warp == 4) {
    if (lane == 0) {
      bool waited = !a.early;
      for (int j = 0; j < n; j++) {
        const int s = j % OWN_STAGES, next = j + 1 < n ? table[j + 1] : 0;
        if (!waited && (tk.first + j) * PS + PS >= len) {      // the page of the newest position, which the kernel before this one may be writing
          cima_pdl_wait();
          asm volatile("fence.proxy.async;" ::: "memory");
          waited = true;
        }
        if (j >= OWN_STAGES && !mbar_wait(&empty[s], (j / OWN_STAGES - 1) & 1, error_flag, abort_flag)) break;
        mbar_expect_tx(&full[s], STAGE);
#pragma unroll
        for (int pl = 0; pl < PLANES; pl++)
#pragma unroll
          for (int kb = 0; kb < NH; kb++)
            tma_load_2d(smem + s * STAGE + (pl * NH + kb) * KV_BLOCK, map, 64 * kb, ((page * PLANES + pl) * a.nkv + tk.kvh) * PS, &full[s]);
        page = next;
      }
    }
  } else if (warp < 4) {
    if (a.early) wait_then_let_next();
    uint4 q[NB][HD / 32] = {};
    float sl2[NB][2] = {};
    int last_key[NB][2] = {};
#pragma unroll
    for (int i = 0; i < NB; i++) {
      if (8 * i + g < tk.rows) {
        int seq, head;
        row_of(a, tk, 8 * i + g, seq, head);
        const __nv_bfloat16* qp = (const __nv_bfloat16*)a.qkv + (size_t)seq * a.ld + (size_t)head * HD + 8 * t;
#pragma unroll
        for (int d = 0; d < HD / 32; d++) q[i][d] = *reinterpret_cast<const uint4*>(qp + 32 * d);
      }
      if (a.slopes) {
#pragma unroll
        for (int j = 0; j < 2; j++)
          if (8 * i + 2 * t + j < tk.rows) {
            int seq, head;
            row_of(a, tk, 8 * i + 2 * t + j, seq, head);
            sl2[i][j] = a.slopes[head] * LOG2E;
            last_key[i][j] = a.seq_len[seq] - 1;
          }
      }
    }
    float o[NB][HD / 16][4], mr[NB][2], lr[NB][2];
#pragma unroll
    for (int i = 0; i < NB; i++) {
#pragma unroll
      for (int j = 0; j < HD / 16; j++) o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.f;
      mr[i][0] = mr[i][1] = -INFINITY;
      lr[i][0] = lr[i][1] = 0.f;
    }
    const float sc2 = a.scale * LOG2E;
    bool ok = true;
#pragma unroll 1
    for (int j = 0; j < n; j++) {
      const int s = j % OWN_STAGES, key = (tk.first + j) * PS + 16 * warp + g;
      ok = mbar_wait(&full[s], (j / OWN_STAGES) & 1, error_flag, abort_flag);
      if (!ok) break;
      // dims 32 d + 8 t .. + 7 of keys g and g + 8 of the warp's 16: chunk 4 (d & 1) + t of a 128-byte row lies at place chunk ^ (row & 7)
      const unsigned char* row = smem + s * STAGE + (16 * warp + g) * 128;
      auto chunk = [&](int plane, int d, int h) -> uint4 {
        return *reinterpret_cast<const uint4*>(row + (plane * NH + d / 2) * KV_BLOCK + h * 1024 + (((4 * (d & 1) + t) ^ g) << 4));
      };
      float sa[NB][4], sb[NB][4];
#pragma unroll
      for (int i = 0; i < NB; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) sa[i][e] = sb[i][e] = 0.f;
#pragma unroll
      for (int d = 0; d < HD / 32; d++) {
        const uint4 k0 = chunk(0, d, 0), k1 = chunk(0, d, 1);
#pragma unroll
        for (int i = 0; i < NB; i++) {
          mma_ab(sa[i], k0.x, k1.x, k0.y, k1.y, q[i][d].x, q[i][d].y);
          mma_ab(sb[i], k0.z, k1.z, k0.w, k1.w, q[i][d].z, q[i][d].w);
        }
      }
      uint32_t b0[NB], b1[NB];
      float corr[NB][2], f[NB][2];
#pragma unroll
      for (int i = 0; i < NB; i++) {
        float p[4];
#pragma unroll
        for (int x = 0; x < 2; x++) {
          float v0 = (sa[i][x] + sb[i][x]) * sc2, v1 = (sa[i][x + 2] + sb[i][x + 2]) * sc2;
          if (a.slopes) {
            v0 = fmaf(sl2[i][x], (float)(key - last_key[i][x]), v0);
            v1 = fmaf(sl2[i][x], (float)(key + 8 - last_key[i][x]), v1);
          }
          if (key >= len) v0 = -INFINITY;
          if (key + 8 >= len) v1 = -INFINITY;
          float mx = fmaxf(v0, v1);
#pragma unroll
          for (int y = 4; y < 32; y *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, y));
          const float own = mx == -INFINITY ? 0.f : mx, mn = fmaxf(mr[i][x], mx), ms = mn == -INFINITY ? 0.f : mn;
          p[x] = ex2(v0 - own);
          p[x + 2] = ex2(v1 - own);
          corr[i][x] = ex2(mr[i][x] - ms);
          f[i][x] = ex2(mx - ms);
          mr[i][x] = mn;
          lr[i][x] = fmaf(lr[i][x], corr[i][x], (p[x] + p[x + 2]) * f[i][x]);
        }
        b0[i] = transposed(pack_bf16(p[0], p[1]));
        b1[i] = transposed(pack_bf16(p[2], p[3]));
      }
#pragma unroll
      for (int d = 0; d < HD / 32; d++) {
        uint4 v0 = chunk(PLANES - 1, d, 0), v1 = chunk(PLANES - 1, d, 1);
        if (key >= len) v0 = make_uint4(0u, 0u, 0u, 0u);       // positions behind the end may hold anything: 0 times infinity would be NaN
        if (key + 8 >= len) v1 = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const uint32_t a0 = transposed(e ? v0.z : v0.x), a1 = transposed(e ? v0.w : v0.y), a2 = transposed(e ? v1.z : v1.x), a3 = transposed(e ? v1.w : v1.y);
#pragma unroll
          for (int i = 0; i < NB; i++) {
            float s16[4] = {0.f, 0.f, 0.f, 0.f};
            mma_ab(s16, a0, a1, a2, a3, b0[i], b1[i]);
#pragma unroll
            for (int y = 0; y < 4; y++) o[i][2 * d + e][y] = fmaf(o[i][2 * d + e][y], corr[i][y & 1], s16[y] * f[i][y & 1]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[s]);
    }
    block_sync();                                              // every page has been read: the warps' results take their place
    if (ok) join_warps<HD, NB, 4>(a, tk, o, mr, lr, smem);
    else block_sync();                                         // (join_warps' own)
  }
}

template <int HD, int PLANES, int OWN>
__global__ void __launch_bounds__(TC_THREADS, 2)
k_attention_shared_tc(const __grid_constant__ CUtensorMap map, const __grid_constant__ SharedArgs a, int* error_flag) {
  if (!a.early) wait_then_let_next();
  extern __shared__ __align__(1024) unsigned char smem[];
  // An SM takes no second block of a kernel that allocates tensor memory until the first one has given up its permit to do so: so every block with
  // work does that early, those of the sequences' own pages too (without, they ran one an SM, and a prefix's second block came 1.9 us late).
  constexpr size_t SMEM = tc_smem<HD>();
  unsigned* tmem_slot = (unsigned*)(smem + SMEM - 16);
  int index = blockIdx.x;
  const int warp = threadIdx.x >> 5, columns = is_prefix(a, index) ? TMEM_PREFIX : TMEM_OWN;
  Task t;
  if (columns == TMEM_OWN && !find_task(a, TC_ROWS, t)) return;        // (a place for a longer context's splits)
  if (warp == 5) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(columns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (columns == TMEM_OWN) own_tma<HD, PLANES, OWN>(&map, a, t, smem, error_flag);
  else if (find_task(a, TC_ROWS, t)) prefix_tc<HD, PLANES>(&map, a, t, smem, tmem_slot, error_flag);
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  if (warp == 5) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(columns) : "memory");
  }
}

template <int HD, int PLANES>
int launch_shared_tc(SharedArgs a, long long n_pages, int most, int* error_flag, cudaStream_t stream) {
  CUtensorMap map;
  if (const int rc = make_map(&map, a.cache, n_pages * PLANES * a.nkv * PS, HD, HD, PS)) return rc;
  const int G = a.nh / a.nkv;
  a.prefix_tiles = (most * G + TC_ROWS - 1) / TC_ROWS;
  constexpr int WIDE = HD == 64 ? 2 : 1;                        // (16 rows are too many for the registers at head size 128: two blocks of 8)
  a.own_rows = 8 * (G <= 8 ? 1 : WIDE);
  a.own_tiles = (G + a.own_rows - 1) / a.own_rows;
  a.own_least = own_least_of(a);
  constexpr size_t smem = tc_smem<HD>();
  static_assert(smem <= ONE_AN_SM && smem >= near_smem<HD, WIDE, 4>() && smem >= OWN_STAGES * 2 * (HD / 64) * KV_BLOCK + 16 * OWN_STAGES + 32, "a sequence's own pages and their merge fit");
  const dim3 grid(blocks_of(a));
  // Steps of few rows: one block an SM.  Two set the SM up for nearly all of its memory as shared memory, which it keeps while kernels follow without a
  // pause; the products of few rows, which read their rows through L1 again and again, are 1.3 to 2 times slower then (8 sequences of the 7B shape,
  // 2,048 / 8,192 positions in common, us a layer in the step: 50 more).  Beyond them the products are the library's, and two blocks an SM are better
  // (48 sequences, 2,048 positions: 6 us).
  const size_t room = a.B <= FEW_ROWS ? ONE_AN_SM : smem;
  auto go = [&](auto kern, int rc) { return rc ? rc : cima_launch(kern, grid, dim3(TC_THREADS), room, stream, 1, map, a, error_flag); };
  const int rc = G <= 8 ? go(k_attention_shared_tc<HD, PLANES, 1>, prepare_kernel<k_attention_shared_tc<HD, PLANES, 1>>(ONE_AN_SM))
                        : go(k_attention_shared_tc<HD, PLANES, WIDE>, prepare_kernel<k_attention_shared_tc<HD, PLANES, WIDE>>(ONE_AN_SM));
  if (rc) return rc;
  return launch_combine<__nv_bfloat16>(a, HD, stream);
}

}  // namespace

// cima_attention_shared for bfloat16 and head sizes 64 and 128, blocks of 128 rows of a prefix on tcgen05.  early: 2 more where some sequence is in no
// group (which sort of blocks comes first, is_prefix).  n_pages: of the storage;
// error_flag: device int that a wait that ran out sets to 1 (never cleared here).
extern "C" int cima_attention_shared_tc(const void* qkv, int ld, const void* cache, long long n_pages, const int* table, int table_width, int page_size,
                                        int planes, const int* seq_slot, const int* seq_len, const int* order, const int* own_page, const int* groups,
                                        int n_groups, int most, float* part_o, float* part_ml, int prefix_splits, int own_splits, void* out, int ldo,
                                        int B, int nh, int nkv, int hd, float scale, float sink, const float* head_sink, int gate_col,
                                        const float* slopes, int early, int* error_flag, cudaStream_t stream) {
  if (B <= 0) return 0;
  if (hd != 64 && hd != 128) return cima_fail(CIMA_E_SIZE, "attention_shared_tc: head_dim %d; this kernel takes 64 or 128", hd);
  if (!error_flag) return cima_fail(CIMA_E_ARG, "attention_shared_tc: an error flag on the device is needed");
  if (!(scale >= 0.f)) return cima_fail(CIMA_E_ARG, "attention_shared_tc: a scale of %g; this kernel takes the maxima of the unscaled scores and no negative one", scale);
  if (ld % 8 || ((uintptr_t)qkv & 15)) return cima_fail(CIMA_E_ARG, "attention_shared_tc: qkv rows must be 16-byte aligned");
  const CimaPaged pg{table, table_width, 0, page_size, nkv, hd, planes};
  const SharedArgs a{qkv, cache, pg, seq_slot, seq_len, order, own_page, groups, head_sink, slopes, part_o, part_ml, out,
                     ld, ldo, B, nh, nkv, n_groups, 0, prefix_splits, 0, own_splits, gate_col, early & 1, scale, sink, 2, 16, !(early & 2)};
  if (const int rc = check_shared("attention_shared_tc", a, most)) return rc;
  if (n_pages <= 0 || n_pages * planes * nkv * PS >= (1ll << 31)) return cima_fail(CIMA_E_SIZE, "attention_shared_tc: %lld pages exceed a tensor map's 32-bit row coordinate", n_pages);
  if (hd == 64) return planes == 2 ? launch_shared_tc<64, 2>(a, n_pages, most, error_flag, stream) : launch_shared_tc<64, 1>(a, n_pages, most, error_flag, stream);
  return planes == 2 ? launch_shared_tc<128, 2>(a, n_pages, most, error_flag, stream) : launch_shared_tc<128, 1>(a, n_pages, most, error_flag, stream);
}
