// Paged cache: tables, argument checks, and what moves whole pages or rows (extend, fork, free, compact, copy).
#include <atomic>
#include <cmath>
#include <cstring>
#include <mutex>

#include "mz_paged.cuh"

namespace {
__device__ __align__(16) uint8_t g_book[MZP_BOOKS * MZP_LEVELS];
__device__ __align__(16) uint8_t g_nearest[MZP_BOOKS * MZP_NEAR_ROW];
std::mutex g_mu;
struct Tables { const uint8_t *book, *nearest; } g_tables[256];     // by device; NULL until they are in place

// Levels of book z: z' = round(15 z / 127) codes lie below the zero level and 15 - z' above it, spaced by the law (3^t - 1) / 2.  No entry
// is near a rounding boundary (the closest by 0.001), so any correctly working pow gives the same table.
void fill_books(uint8_t* book, uint8_t* nearest) {
  for (int z = 0; z < MZP_BOOKS; ++z) {
    const int zc = (int)std::lround(15.0 * z / 127.0);
    for (int e = 0; e < MZP_LEVELS; ++e) {
      const double t = e >= zc ? (double)(e - zc) / (zc < 15 ? 15 - zc : 1) : (double)(zc - e) / zc;
      const double grown = (std::pow(3.0, t) - 1.0) / 2.0;
      book[z * MZP_LEVELS + e] = (uint8_t)(e >= zc ? z + std::lround((127 - z) * grown) : z - std::lround(z * grown));
    }
    for (int r = 0; r < 128; ++r) {
      int best = 0;
      for (int e = 1; e < MZP_LEVELS; ++e)
        if (std::abs(book[z * MZP_LEVELS + e] - r) < std::abs(book[z * MZP_LEVELS + best] - r)) best = e;
      nearest[z * 128 + r] = (uint8_t)best;
    }
  }
}
}  // namespace

extern "C" int mz_paged_books(unsigned char* book, unsigned char* nearest) {
  MZ_REQUIRE(book != nullptr && nearest != nullptr, "a table is NULL");
  fill_books(book, nearest);
  return MZ_OK;
}

int mz_paged_sms(int* sms) {
  static std::atomic<int> known[256];
  int dev = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  MZ_REQUIRE(dev >= 0 && dev < 256, "device %d", dev);
  *sms = known[dev].load(std::memory_order_relaxed);
  if (*sms == 0) {
    MZ_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
    known[dev].store(*sms, std::memory_order_relaxed);
  }
  return MZ_OK;
}

int mz_paged_tables(const uint8_t** book, const uint8_t** nearest) {
  int dev = 0;
  MZ_CUDA(cudaGetDevice(&dev));
  MZ_REQUIRE(dev >= 0 && dev < 256, "device %d", dev);
  std::lock_guard<std::mutex> lk(g_mu);
  Tables& t = g_tables[dev];
  if (t.nearest == nullptr) {
    uint8_t b[sizeof(g_book)], n[MZP_BOOKS * 128], padded[sizeof(g_nearest)] = {};
    fill_books(b, n);
    for (int z = 0; z < MZP_BOOKS; ++z)
      for (int r = -1; r <= 128; ++r) padded[z * MZP_NEAR_ROW + r + 1] = n[z * 128 + (r < 0 ? 0 : r > 127 ? 127 : r)];
    MZ_CUDA(cudaMemcpyToSymbol(g_book, b, sizeof(b)));
    MZ_CUDA(cudaMemcpyToSymbol(g_nearest, padded, sizeof(padded)));
    // the copies may still be on their way from their staging memory, and a non-blocking stream does not wait for the legacy one
    MZ_CUDA(cudaStreamSynchronize(cudaStreamLegacy));
    void *book_at = nullptr, *nearest_at = nullptr;
    MZ_CUDA(cudaGetSymbolAddress(&book_at, g_book));
    MZ_CUDA(cudaGetSymbolAddress(&nearest_at, g_nearest));
    t.book = (const uint8_t*)book_at;
    t.nearest = (const uint8_t*)nearest_at;
  }
  if (book) *book = t.book;
  if (nearest) *nearest = t.nearest;
  return MZ_OK;
}

extern "C" int mz_paged_prepare(void) { return mz_paged_tables(nullptr, nullptr); }

int mz_paged_check(const mz_paged_cache* c) {
  MZ_REQUIRE(c != nullptr, "cache is NULL");
  MZ_REQUIRE(c->head_dim == 64 || c->head_dim == 128, "head_dim %d (64 or 128)", c->head_dim);
  MZ_REQUIRE(c->kv_dtype == MZ_F16 || c->kv_dtype == MZ_BF16, "kv_dtype must be fp16 or bf16");
  MZ_REQUIRE(c->layers > 0 && c->rows > 0 && c->pages > 0 && c->width > 0 && c->kv_heads > 0 && c->kv_heads <= 1024,
             "sizes must be positive (layers %d, rows %d, pages %d, width %d, kv_heads %d)", c->layers, c->rows, c->pages, c->width, c->kv_heads);
  MZ_REQUIRE(c->width <= (1 << 24), "a table row has %d entries, more than 2^24", c->width);
  MZ_REQUIRE(c->residual >= 0 && c->residual % MZP_PAGE == 0, "residual %d is not a multiple of %d", c->residual, MZP_PAGE);
  MZ_REQUIRE(c->ring >= c->residual + MZP_PAGE && c->ring <= (1 << 20), "ring %d: at least residual + %d", c->ring, MZP_PAGE);
  MZ_REQUIRE(c->store && c->tail && c->block_table && c->lengths && c->page_refs && c->status, "a cache pointer is NULL");
  // attention reads the 32 bytes of a row of codes with one load (a page's size and the places of its rows are multiples of 32)
  MZ_REQUIRE((uintptr_t)c->store % 32 == 0 && (uintptr_t)c->tail % 16 == 0, "store must be 32-byte aligned and tail 16-byte");
  MZ_REQUIRE(c->store_stride_page % 32 == 0 && c->store_stride_layer % 32 == 0 &&
                 c->store_stride_page >= (long long)c->kv_heads * mzp_page_bytes(c->head_dim),
             "page stride %lld bytes, layer stride %lld: multiples of 32, and a page's bytes at least", c->store_stride_page, c->store_stride_layer);
  MZ_REQUIRE(c->tail_stride_row % 8 == 0 && c->tail_stride_layer % 8 == 0 &&
                 c->tail_stride_row >= 2ll * c->kv_heads * c->ring * c->head_dim,
             "ring stride %lld elements", c->tail_stride_row);
  return MZ_OK;
}

namespace {
constexpr int kMaxBatch = 4096;

__device__ __forceinline__ int block_scan_exclusive(int v, int* total, int* s_warp) {      // 1024 threads
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const int y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
  __syncthreads();
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  int before = 0, all = 0;
  for (int w = 0; w < 32; ++w) { const int t = s_warp[w]; if (w < warp) before += t; all += t; }
  *total = all;
  return before + x - v;
}

// One CTA: the list's pages are counted and checked first, then the free ones are dealt out in ascending order.  Bound by its launch and barriers: 64 rows of one token that
// fill no page, which end after the first pass over the list, 8 us; that fill 64 pages 10 us.  The counts are looked through twice from the pool's first page, a barrier per 1024 of
// them: 14 us where the free pages come after 3968 taken ones, 127 us after 65408.
__global__ void __launch_bounds__(1024) extend_kernel(const mz_paged_cache c, const int* __restrict__ rows, const int* __restrict__ offsets, int batch) {
  __shared__ int s_warp[32], s_bad;
  __shared__ int s_first[kMaxBatch + 1];        // pages needed by the entries before
  if (threadIdx.x == 0) s_bad = 0;
  __syncthreads();
  int need_all = 0, bad = 0;
  for (int i0 = 0; i0 < batch; i0 += 1024) {
    const int i = i0 + threadIdx.x;
    int need = 0;
    if (i < batch) {
      const int row = rows ? rows[i] : i;
      if (row < 0 || row >= c.rows) bad |= MZ_PAGED_BAD_INDEX;
      else {
        const int n = offsets ? offsets[i + 1] - offsets[i] : 1;
        const long long len = c.lengths[row], after = len + n;
        if (n < 0) bad |= MZ_PAGED_BAD_INDEX;
        else if (after > 0x7fffffff - 4096 || mzp_packed((int)after, c.residual) / MZP_PAGE > c.width) bad |= MZ_PAGED_TOO_LONG;
        else need = (mzp_packed((int)after, c.residual) - mzp_packed((int)len, c.residual)) / MZP_PAGE;
      }
    }
    int total;
    const int at = block_scan_exclusive(need, &total, s_warp);
    if (i < batch) s_first[i] = need_all + at;
    need_all += total;
    __syncthreads();
  }
  if (bad) atomicOr(&s_bad, bad);
  if (threadIdx.x == 0) s_first[batch] = need_all;
  __syncthreads();
  if (s_bad) { if (threadIdx.x == 0) atomicOr(c.status, s_bad | MZ_PAGED_REFUSED); return; }
  if (need_all > 0) {
    // are there enough?
    int found = 0;
    for (int p0 = 0; p0 < c.pages && found < need_all; p0 += 1024) {
      const int p = p0 + threadIdx.x;
      found += __syncthreads_count(p < c.pages && c.page_refs[p] == 0);
    }
    if (found < need_all) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_NO_PAGES | MZ_PAGED_REFUSED); return; }
    int dealt = 0;
    for (int p0 = 0; p0 < c.pages && dealt < need_all; p0 += 1024) {      // (ends whatever another stream does to the counts meanwhile)
      const int p = p0 + threadIdx.x;
      const bool free_page = p < c.pages && c.page_refs[p] == 0;
      int total;
      const int k = dealt + block_scan_exclusive(free_page, &total, s_warp);
      if (free_page && k < need_all) {
        int lo = 0, hi = batch;                 // the entry that the k-th page goes to: s_first[lo] <= k < s_first[lo + 1]
        while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (s_first[mid] <= k) lo = mid; else hi = mid; }
        const int row = rows ? rows[lo] : lo;
        const int place = mzp_packed(c.lengths[row], c.residual) / MZP_PAGE + k - s_first[lo];
        c.block_table[(long long)row * c.width + place] = p;
        c.page_refs[p] = 1;
      }
      dealt += total;
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < batch; i += 1024) c.lengths[rows ? rows[i] : i] += offsets ? offsets[i + 1] - offsets[i] : 1;
  if (threadIdx.x == 0) atomicAnd(c.status, ~MZ_PAGED_REFUSED);       // what is appended next has been announced
}

__device__ __forceinline__ void release(const mz_paged_cache& c, int page) {
  if (page >= 0 && page < c.pages) atomicSub(c.page_refs + page, 1);
}

// Moves no page: 48 targets x 4 layers x 8 kv heads with 128 to 191 live tokens take 31 us for the 126 MB read and 126 MB written, the copy rate of the memory.
// CTAs 0 .. n-1 renew a target's table row (counts are integers: the order of the additions does not matter), the others copy the live part of one
// ring of one (target, layer, side, kv head) each: at most two runs of tokens, 16 bytes per thread and step
__global__ void __launch_bounds__(256) fork_kernel(const mz_paged_cache c, const int* __restrict__ source, const int* __restrict__ target, int n) {
  const int rings = c.layers * 2 * c.kv_heads;
  const int i = (int)blockIdx.x < n ? blockIdx.x : ((int)blockIdx.x - n) / rings;
  const int src = source[i], dst = target[i];
  bool ok = src >= 0 && src < c.rows && dst >= 0 && dst < c.rows;
  for (int j = threadIdx.x; j < n; j += blockDim.x) ok = ok && target[j] != src;
  if (!__syncthreads_and(ok)) {
    if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX);
    return;
  }
  const int len = c.lengths[src], packed = mzp_packed(len, c.residual);
  if ((int)blockIdx.x < n) {
    const int used = packed / MZP_PAGE;
    for (int k = threadIdx.x; k < c.width; k += blockDim.x) {
      const int page = k < used ? c.block_table[(long long)src * c.width + k] : -1;
      const int old = atomicExch(c.block_table + (long long)dst * c.width + k, page);
      release(c, old);
      if (page >= 0 && page < c.pages) atomicAdd(c.page_refs + page, 1);
    }
    if (threadIdx.x == 0) c.lengths[dst] = len;
    return;
  }
  const int ring = ((int)blockIdx.x - n) % rings, layer = ring / (2 * c.kv_heads), side_head = ring % (2 * c.kv_heads);
  const int per_token = c.head_dim / 8;         // 16-byte pieces
  const long long at = (long long)layer * c.tail_stride_layer + (long long)side_head * c.ring * c.head_dim;
  const uint4* from = (const uint4*)((const uint16_t*)c.tail + at + (long long)src * c.tail_stride_row);
  uint4* to = (uint4*)((uint16_t*)c.tail + at + (long long)dst * c.tail_stride_row);
  const int first = packed % c.ring * per_token, all = c.ring * per_token, count = (len - packed) * per_token;
  int k = threadIdx.x;
  for (; k + 3 * 256 < count; k += 4 * 256) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) { int x = first + k + u * 256; if (x >= all) x -= all; v[u] = from[x]; }
#pragma unroll
    for (int u = 0; u < 4; ++u) { int x = first + k + u * 256; if (x >= all) x -= all; to[x] = v[u]; }
  }
  for (; k < count; k += 256) { int x = first + k; if (x >= all) x -= all; to[x] = from[x]; }
}

__global__ void __launch_bounds__(256) free_kernel(const mz_paged_cache c, const int* __restrict__ rows) {
  const int row = rows[blockIdx.x];
  if (row < 0 || row >= c.rows) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); return; }
  // the exchange makes a row that is listed twice be released once
  for (int k = threadIdx.x; k < c.width; k += blockDim.x) release(c, atomicExch(c.block_table + (long long)row * c.width + k, -1));
  if (threadIdx.x == 0) c.lengths[row] = 0;
}

// workspace of a compaction: {pages to move, pad, pad, pad}, map[pages], from[pages], to[pages].  One CTA, four neighbouring pages per thread: the places
// in both lists come from one scan of two 16-bit counts.  7.4 us for 1786 pages (6.4 for a few: launch and
// barriers; with one page per thread the whole retirement of 16 rows of 48 took 66 us instead of 63).
__global__ void __launch_bounds__(1024) compact_plan_kernel(const mz_paged_cache c, int* __restrict__ ws) {
  __shared__ int s_warp[32];
  int *map = ws + 4, *from = map + c.pages, *to = from + c.pages;
  int live = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4096) {
    int mine = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) { const int p = p0 + 4 * (int)threadIdx.x + j; mine += p < c.pages && c.page_refs[p] > 0; }
    block_scan_exclusive(mine, &total, s_warp);
    live += total;
  }
  int movers = 0, holes = 0;
  for (int p0 = 0; p0 < c.pages; p0 += 4096) {
    bool mover[4], hole[4];
    int mine = 0, total;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + 4 * (int)threadIdx.x + j;
      const bool in = p < c.pages, used = in && c.page_refs[p] > 0;
      mover[j] = used && p >= live;
      hole[j] = in && !used && p < live;
      mine += (int)mover[j] | (int)hole[j] << 16;
      if (in) map[p] = p;
    }
    const int both = block_scan_exclusive(mine, &total, s_warp);       // at most 4096 of each
    int m = movers + (both & 0xffff), h = holes + (both >> 16);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = p0 + 4 * (int)threadIdx.x + j;
      if (mover[j]) from[m++] = p;
      if (hole[j]) to[h++] = p;
    }
    movers += total & 0xffff;
    holes += total >> 16;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < movers; k += 1024) {
    const int a = from[k], b = to[k];
    map[a] = b;
    c.page_refs[b] = c.page_refs[a];
    c.page_refs[a] = 0;
  }
  if (threadIdx.x == 0) ws[0] = movers;
}

// moves pages (list from -> to) in all layers, a kv head of a page at a time; with a map the table's entries are rewritten as well.
// A CTA has three 16-byte pieces per thread in flight, eight CTAs to an SM: 36 us for the compaction of 16 ended rows of 48 of up to 4224 tokens in 4 layers, the copy
// rate of the memory.
__global__ void __launch_bounds__(256) move_pages_kernel(const mz_paged_cache c, const int* __restrict__ from, const int* __restrict__ to,
                                                         const int* __restrict__ count, int n, const int* __restrict__ map) {
  const int moves = count ? *count : n;
  const int pieces = mzp_page_bytes(c.head_dim) / 16;        // 576 or 288
  const long long units = (long long)moves * c.layers * c.kv_heads;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int head = (int)(u % c.kv_heads);
    const long long v = u / c.kv_heads;
    const int layer = (int)(v % c.layers), k = (int)(v / c.layers);
    const int a = from[k], b = to[k];
    if (a < 0 || a >= c.pages || b < 0 || b >= c.pages) { if (threadIdx.x == 0) atomicOr(c.status, MZ_PAGED_BAD_INDEX); continue; }
    const long long at = (long long)layer * c.store_stride_layer + (long long)head * mzp_page_bytes(c.head_dim);
    const uint4* src = (const uint4*)((const uint8_t*)c.store + at + (long long)a * c.store_stride_page);
    uint4* dst = (uint4*)((uint8_t*)c.store + at + (long long)b * c.store_stride_page);
    uint4 x[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) if ((int)threadIdx.x + j * 256 < pieces) x[j] = src[threadIdx.x + j * 256];
#pragma unroll
    for (int j = 0; j < 3; ++j) if ((int)threadIdx.x + j * 256 < pieces) dst[threadIdx.x + j * 256] = x[j];
  }
  if (map) {
    const long long entries = (long long)c.rows * c.width;
    for (long long e = (long long)blockIdx.x * blockDim.x + threadIdx.x; e < entries; e += (long long)gridDim.x * blockDim.x) {
      const int page = c.block_table[e];
      if (page >= 0 && page < c.pages) c.block_table[e] = map[page];
    }
  }
}

}  // namespace

extern "C" int mz_paged_extend(const mz_paged_cache* cache, const int* rows, const int* offsets, int batch, void* stream) {
  MZ_RANGE("mz_paged_extend");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(batch >= 0 && batch <= kMaxBatch, "batch %d (at most %d)", batch, kMaxBatch);
  MZ_REQUIRE(rows != nullptr || batch <= cache->rows, "batch %d of %d rows", batch, cache->rows);
  if (batch == 0) return MZ_OK;
  extend_kernel<<<1, 1024, 0, (cudaStream_t)stream>>>(*cache, rows, offsets, batch);
  MZ_LAUNCH_CHECK("extend");
  return MZ_OK;
}

extern "C" int mz_paged_fork(const mz_paged_cache* cache, const int* source, const int* target, int n, void* stream) {
  MZ_RANGE("mz_paged_fork");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(n >= 0 && n <= cache->rows, "%d targets of %d rows", n, cache->rows);
  if (n == 0) return MZ_OK;
  MZ_REQUIRE(source != nullptr && target != nullptr, "a list is NULL");
  const long long ctas = (long long)n * (1 + (long long)cache->layers * 2 * cache->kv_heads);
  MZ_REQUIRE(ctas < (1ll << 31), "too many rings for one call");
  fork_kernel<<<(unsigned)ctas, 256, 0, (cudaStream_t)stream>>>(*cache, source, target, n);
  MZ_LAUNCH_CHECK("fork");
  return MZ_OK;
}

extern "C" int mz_paged_free(const mz_paged_cache* cache, const int* rows, int n, void* stream) {
  MZ_RANGE("mz_paged_free");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(n >= 0 && n < (1 << 30), "%d rows", n);
  if (n == 0) return MZ_OK;
  MZ_REQUIRE(rows != nullptr, "the list is NULL");
  free_kernel<<<n, 256, 0, (cudaStream_t)stream>>>(*cache, rows);
  MZ_LAUNCH_CHECK("free");
  return MZ_OK;
}

extern "C" size_t mz_paged_compact_workspace_bytes(const mz_paged_cache* cache) {
  return mz_paged_check(cache) == MZ_OK ? (4 + 3 * (size_t)cache->pages) * sizeof(int) : 0;
}

extern "C" int mz_paged_compact(const mz_paged_cache* cache, void* workspace, size_t workspace_bytes, void* stream) {
  MZ_RANGE("mz_paged_compact");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  if (!workspace || (uintptr_t)workspace % 16 != 0 || workspace_bytes < mz_paged_compact_workspace_bytes(cache))
    return mz_fail(MZ_ERR_WORKSPACE, "workspace of %zu bytes, %zu needed", workspace_bytes, mz_paged_compact_workspace_bytes(cache));
  int sms = 0;
  if ((rc = mz_paged_sms(&sms)) != MZ_OK) return rc;
  int* ws = (int*)workspace;
  compact_plan_kernel<<<1, 1024, 0, (cudaStream_t)stream>>>(*cache, ws);
  MZ_LAUNCH_CHECK("compact_plan");
  move_pages_kernel<<<sms * 8, 256, 0, (cudaStream_t)stream>>>(*cache, ws + 4 + cache->pages, ws + 4 + 2 * cache->pages, ws, 0, ws + 4);
  MZ_LAUNCH_CHECK("move_pages");
  return MZ_OK;
}

extern "C" int mz_paged_copy_pages(const mz_paged_cache* cache, const int* source, const int* target, int n, void* stream) {
  MZ_RANGE("mz_paged_copy_pages");
  int rc = mz_paged_check(cache);
  if (rc != MZ_OK) return rc;
  MZ_REQUIRE(n >= 0 && n <= cache->pages, "%d of %d pages", n, cache->pages);
  if (n == 0) return MZ_OK;
  MZ_REQUIRE(source != nullptr && target != nullptr, "a list is NULL");
  int sms = 0;
  if ((rc = mz_paged_sms(&sms)) != MZ_OK) return rc;
  const long long units = (long long)n * cache->layers * cache->kv_heads;
  move_pages_kernel<<<(unsigned)(units < sms * 8 ? units : sms * 8), 256, 0, (cudaStream_t)stream>>>(*cache, source, target, nullptr, n, nullptr);
  MZ_LAUNCH_CHECK("move_pages");
  return MZ_OK;
}
