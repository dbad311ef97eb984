// Pages of the cache copied inside their storage, for every layer in one launch:
//   storage[l, to, s, t, :] = storage[l, from, s, t, :],  t < positions,
// for each (from, to, positions) of a plan, all layers l and segments s (a segment is the positions of one plane and head:
// planes * heads of them make a page).  Bits are moved, so any element type will do.  Per-slot state goes the same way: a tensor
// [slots, values] is pages of one segment and one position.
//
// The plan lies on the host, where the cache's bookkeeping makes it, and travels as a kernel parameter: no copy to the device, no
// wait for one, and it can be checked before anything runs (ids inside the storage, no page written twice, none both read and
// written: the copies of a plan have no order among them).
//
// Bound: bytes.  A thread moves four vectors of 16 bytes (narrower ones where a position's bytes or the storage are not so aligned), all
// four on their way before the first is written.  Measured: 333 pages of 28 layers (1.22 GB read and written) 186 us, 6.6 TB/s; 66 pages of 24 layers
// (208 MB) 33 us, 6.3 TB/s; a page of 21 positions 1.5 us, 7 of 37 positions in 28 layers 3.9 us, which is the launch and latency of one load and store.
#include "common.cuh"
#include <stdlib.h>
#include <string.h>

namespace {

struct CopyPage { int from, to, positions; };
template <int N> struct CopyPlan { CopyPage page[N]; };
constexpr int THREADS = 256, UNROLL = 4;
constexpr int PLAN_FEW = 16, PLAN_MANY = 320;      // pages of a launch: 192 or 3,840 bytes of parameters

// row: vectors of a position; seg: of a segment; page: of a page; layer: of a layer.
template <typename V, int N>
__global__ void __launch_bounds__(THREADS)
k_copy_pages(V* __restrict__ storage, const __grid_constant__ CopyPlan<N> plan, int segments, unsigned row, unsigned seg, unsigned long long layer) {
  cima_pdl_wait();
  const CopyPage c = plan.page[blockIdx.y];
  const unsigned fill = row * (unsigned)c.positions, all = fill * (unsigned)segments;
  const unsigned long long page = (unsigned long long)seg * segments, base = blockIdx.z * layer;
  const V* src = storage + base + page * (unsigned)c.from;
  V* dst = storage + base + page * (unsigned)c.to;
  const bool whole = fill == seg;
  for (unsigned v0 = blockIdx.x * THREADS * UNROLL + threadIdx.x; v0 < all; v0 += gridDim.x * THREADS * UNROLL) {
    V got[UNROLL];
    unsigned at[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; u++) {
      const unsigned v = v0 + u * THREADS;
      at[u] = whole ? v : v / fill * seg + v % fill;
      if (v < all) got[u] = src[at[u]];
    }
#pragma unroll
    for (int u = 0; u < UNROLL; u++)
      if (v0 + u * THREADS < all) dst[at[u]] = got[u];
  }
}

template <typename V>
int launch(void* storage, int layers, long long pages, int segments, int page_size, long long row_bytes, const CopyPage* plan, int n, cudaStream_t stream) {
  const unsigned row = (unsigned)(row_bytes / sizeof(V)), seg = row * (unsigned)page_size;
  const unsigned long long layer = (unsigned long long)pages * segments * seg;
  for (int i = 0; i < n;) {
    const int m = n - i <= PLAN_FEW ? n - i : (n - i < PLAN_MANY ? n - i : PLAN_MANY);
    int most = 0;
    for (int k = 0; k < m; k++) most = plan[i + k].positions > most ? plan[i + k].positions : most;
    const unsigned long long vectors = (unsigned long long)row * most * segments;
    const unsigned per = THREADS * UNROLL;
    const unsigned blocks = (unsigned)((vectors + per - 1) / per);
    int rc = 0;
    if (blocks) {
      const dim3 grid(blocks, m, layers);
      if (m <= PLAN_FEW) {
        CopyPlan<PLAN_FEW> p = {};
        memcpy(p.page, plan + i, sizeof(CopyPage) * m);
        rc = cima_launch(k_copy_pages<V, PLAN_FEW>, grid, dim3(THREADS), (size_t)0, stream, 1, (V*)storage, p, segments, row, seg, layer);
      } else {
        CopyPlan<PLAN_MANY> p = {};
        memcpy(p.page, plan + i, sizeof(CopyPage) * m);
        rc = cima_launch(k_copy_pages<V, PLAN_MANY>, grid, dim3(THREADS), (size_t)0, stream, 1, (V*)storage, p, segments, row, seg, layer);
      }
    }
    if (rc) return rc;
    i += m;
  }
  return cima_launch_result();
}

}  // namespace

// storage [layers, pages, segments, page_size, row_bytes]; plan: n triples (from, to, positions) on the host, copied before this returns.
extern "C" int cima_copy_pages(void* storage, int layers, long long pages, int segments, int page_size, long long row_bytes, const int* plan, int n,
                               cudaStream_t stream) {
  if (n <= 0) return 0;
  if (layers <= 0 || layers > 65535 || pages <= 0 || pages > 0x7fffffffll || segments <= 0 || page_size <= 0 || row_bytes <= 0)
    return cima_fail(CIMA_E_SIZE, "copy_pages: storage of %d layers, %lld pages, %d segments of %d positions of %lld bytes", layers, pages, segments, page_size, row_bytes);
  if (row_bytes >= (1ll << 30) || row_bytes * page_size >= (1ll << 30) || row_bytes * page_size * segments >= (1ll << 30))
    return cima_fail(CIMA_E_SIZE, "copy_pages: pages of %d segments of %d positions of %lld bytes; below 2^30 bytes a page are possible", segments, page_size, row_bytes);
  const int width = (int)((unsigned long long)row_bytes | (unsigned long long)(uintptr_t)storage) & 15;
  const CopyPage* pg = reinterpret_cast<const CopyPage*>(plan);
  unsigned char* seen = (unsigned char*)calloc((size_t)pages, 1);       // 1: read, 2: written
  if (!seen) return cima_fail(CIMA_E_ARG, "copy_pages: no host memory to check a plan over %lld pages", pages);
  int bad = -1;
  const char* why = "";
  for (int i = 0; i < n && bad < 0; i++) {
    const CopyPage& c = pg[i];
    if (c.from < 0 || c.from >= pages || c.to < 0 || c.to >= pages) { bad = i; why = "a page outside the storage"; }
    else if (c.positions < 0 || c.positions > page_size) { bad = i; why = "more positions than a page has, or fewer than none"; }
    else if (seen[c.to]) { bad = i; why = "writes a page that the plan reads or writes elsewhere"; }
    else if (c.from == c.to || (seen[c.from] & 2)) { bad = i; why = "reads a page that the plan writes"; }
    else { seen[c.to] |= 2; seen[c.from] |= 1; }
  }
  free(seen);
  if (bad >= 0) return cima_fail(CIMA_E_ARG, "copy_pages: entry %d (%d -> %d, %d positions): %s", bad, pg[bad].from, pg[bad].to, pg[bad].positions, why);
  if (width == 0) return launch<uint4>(storage, layers, pages, segments, page_size, row_bytes, pg, n, stream);
  if (width == 8) return launch<uint2>(storage, layers, pages, segments, page_size, row_bytes, pg, n, stream);
  if ((width & 3) == 0) return launch<unsigned>(storage, layers, pages, segments, page_size, row_bytes, pg, n, stream);
  if ((width & 1) == 0) return launch<unsigned short>(storage, layers, pages, segments, page_size, row_bytes, pg, n, stream);
  return launch<unsigned char>(storage, layers, pages, segments, page_size, row_bytes, pg, n, stream);
}
