// cache.cu - operations on the pages of a key/value cache.
//
// The cache's k and v are [layers, pages, kv_heads, page, head_dim] (any strides whose rows
// stay 16-byte aligned), shared by all sequences; row b of `tables` lists the pages of
// slot b in order of position (-1: none), lens[b] counts its cached positions and refs[p]
// counts the table entries that name page p (0: free). All of it lives on the device: no
// call reads it on the host, so the operations queue like any kernel and can be captured.
// Tables, lengths and counts come out as new arrays and only the pages' contents change in
// place, so a call repeated on the same inputs gives the same result.
//
//   append   rows of new tokens (all of them, or an accepted path's) -> pages
//   reserve  pages for `extra` more positions of each slot, from the free ones
//   fork     a slot's full pages shared with another one, its last, partly filled page copied
//   free     a slot's pages given back
//   compact  live pages moved to the lowest indices
//
// Allocation takes free pages in ascending order, so every result is a function of the
// inputs alone. The copies read each byte once and write it once; what bounds them is HBM.
// A cache in 8 bits has powers of two besides (rotary.cu); a copied page's go with it.
#include <algorithm>

#include <atomic>

#include "common.cuh"
#include "sm100.cuh"

namespace nkl {
namespace {

__device__ unsigned int g_cache_dev_error = 0;

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over a block of THREADS of two counts at once, one in each half of v;
// `total` gets the sums. `scratch` is shared, 33 values.
typedef unsigned long long u64;
template <int THREADS>
__device__ __forceinline__ u64 block_scan(u64 v, u64* scratch, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  u64 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();  // the scratch may still be read from the call before
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const u64 w = lane < THREADS / 32 ? scratch[lane] : 0ull;
    u64 wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 x = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += x;
    }
    scratch[lane] = wi - w;
    if (lane == 31) scratch[32] = wi;
  }
  __syncthreads();
  total = scratch[32];
  return scratch[warp] + inc - v;
}

// The plans below run over the pages in rounds of four consecutive ones for each thread.
constexpr int kPerThread = 4;

// Calls take(rank, page) for the first `wanted` free pages, in ascending order, if there are so
// many; `each(page, refs)` for every page first. Returns how many are free.
template <int THREADS, typename Each, typename Take>
__device__ __forceinline__ int free_pages(const int* refs, int pages, int wanted, u64* scratch, Each each, Take take) {
  int mine = 0;
  for (int p0 = 0; p0 < pages; p0 += kPerThread * THREADS)
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int p = p0 + (int)threadIdx.x * kPerThread + k;
      if (p >= pages) continue;
      const int n = refs[p];
      each(p, n);
      mine += n == 0;
    }
  u64 total;
  block_scan<THREADS>((u64)mine, scratch, total);
  const int all = (int)total;
  int seen = 0;
  for (int p0 = 0; all >= wanted && p0 < pages && seen < wanted; p0 += kPerThread * THREADS) {
    bool open[kPerThread];
    int count = 0;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int p = p0 + (int)threadIdx.x * kPerThread + k;
      open[k] = p < pages && refs[p] == 0;
      count += open[k];
    }
    int r = seen + (int)block_scan<THREADS>((u64)count, scratch, total);
#pragma unroll
    for (int k = 0; k < kPerThread; ++k)
      if (open[k] && r < wanted) take(r++, p0 + (int)threadIdx.x * kPerThread + k);
    seen += (int)total;
  }
  return all;
}

// Which pages a compaction moves: on_page(page, refs, kind, rank) for every page, kind 1 for
// the rank-th hole below `live`, 2 for the rank-th page in use from `live` on, else 0.
template <int THREADS, typename OnPage>
__device__ __forceinline__ void compact_plan(const int* refs, int pages, u64* scratch, int& live, int& movers, OnPage on_page) {
  int mine = 0;
  for (int p0 = 0; p0 < pages; p0 += kPerThread * THREADS)
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int p = p0 + (int)threadIdx.x * kPerThread + k;
      mine += p < pages && refs[p] > 0;
    }
  u64 total, seen = 0;
  block_scan<THREADS>((u64)mine, scratch, total);
  live = (int)total;
  for (int p0 = 0; p0 < pages; p0 += kPerThread * THREADS) {
    int n[kPerThread];
    u64 both = 0;  // holes in the upper half, movers in the lower one
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int p = p0 + (int)threadIdx.x * kPerThread + k;
      n[k] = p < pages ? refs[p] : 0;
      both += p < live ? (n[k] <= 0 ? 1ull << 32 : 0ull) : (n[k] > 0 ? 1ull : 0ull);
    }
    u64 at = seen + block_scan<THREADS>(both, scratch, total);
    seen += total;
#pragma unroll
    for (int k = 0; k < kPerThread; ++k) {
      const int p = p0 + (int)threadIdx.x * kPerThread + k;
      if (p >= pages) continue;
      const int kind = p < live ? (n[k] <= 0 ? 1 : 0) : (n[k] > 0 ? 2 : 0);
      on_page(p, n[k], kind, kind == 1 ? (int)(at >> 32) : (int)(uint32_t)at);
      at += kind == 1 ? 1ull << 32 : kind == 2 ? 1ull : 0ull;
    }
  }
  movers = (int)(uint32_t)seen;
}

// Strides of the cache in 16-byte vectors.
struct CacheLayout {
  int64_t layer, page, head, slot;
};

struct CacheDims {
  int layers, pages, heads, page, vecs;  // vecs: 16-byte vectors per row
};

// ------------------------------------------------------------------ append

struct AppendArgs {
  const uint4 *k, *v;
  uint4 *kc, *vc;
  const int *tables, *lens, *path, *count;
  int* lens_out;
  int64_t n_layer, n_batch, n_token, n_head;  // strides of k and v, in vectors
  CacheLayout c;
  CacheDims d;
  int batch, tokens, max_pages;
  uint32_t vecs_magic;  // ceil(2^32 / vecs): exact quotients for the vectors of a row
};

constexpr int kCopyThreads = 256;
constexpr int kCopyBlocks = 2;  // of an SM, for the copies of pages
constexpr int kCopyAhead = 4;  // vectors of k and of v that a lane has on their way

// One warp per row (layer, sequence, token): its place is looked up once, then all heads' k
// and v are copied, kCopyAhead vectors of each at a time. blockIdx.y: sequence, z: layer.
// Measured: prompts of 4 x 4096 tokens, 32 heads of 128, bf16 (537 MB read and written)
// 88.6 us, 6.06 TB/s; a thread per vector, each with the lookup, 105 us. A few accepted tokens
// (2.4 us) are one chain lens -> table -> row.
__global__ void __launch_bounds__(kCopyThreads) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_enter();
  const int lane = threadIdx.x & 31, b = blockIdx.y, l = blockIdx.z;
  const int j = blockIdx.x * (kCopyThreads / 32) + (threadIdx.x >> 5);
  const int len = max(a.lens[b], 0), n = a.count ? min(max(a.count[b], 0), a.tokens) : a.tokens;
  if (j == 0 && l == 0 && lane == 0) a.lens_out[b] = len + n;
  if (j >= n) return;
  const int src = a.path ? a.path[(int64_t)b * a.tokens + j] : j;
  const uint32_t pos = (uint32_t)len + j;
  const int p = (int)(pos / (uint32_t)a.d.page);
  if (src < 0 || src >= a.tokens || p >= a.max_pages) return;
  const int at = a.tables[(int64_t)b * a.max_pages + p];
  if (at < 0 || at >= a.d.pages) return;
  const int64_t from = l * a.n_layer + b * a.n_batch + src * a.n_token;
  const int64_t to = l * a.c.layer + at * a.c.page + (pos - p * a.d.page) * a.c.slot;
  const int row_vecs = a.d.heads * a.d.vecs;
  for (int x0 = lane; x0 < row_vecs; x0 += 32 * kCopyAhead) {
    uint4 kx[kCopyAhead], vx[kCopyAhead];
    int64_t go[kCopyAhead];
#pragma unroll
    for (int i = 0; i < kCopyAhead; ++i) {
      const int x = x0 + 32 * i;
      const int h = a.vecs_magic ? (int)__umulhi((uint32_t)x, a.vecs_magic) : x, e = x - h * a.d.vecs;
      go[i] = to + h * a.c.head + e;
      if (x < row_vecs) {
        kx[i] = ld_stream(a.k + from + h * a.n_head + e);
        vx[i] = ld_stream(a.v + from + h * a.n_head + e);
      }
    }
#pragma unroll
    for (int i = 0; i < kCopyAhead; ++i)
      if (x0 + 32 * i < row_vecs) {
        a.kc[go[i]] = kx[i];
        a.vc[go[i]] = vx[i];
      }
  }
}

// ------------------------------------------------------------------ page copies

// Runs of memory go through shared memory by bulk copies that one thread issues: kRing
// chunks of up to kChunk bytes in a ring, kRingAhead loads on their way before the first of them is
// stored. Two blocks of an SM have 64 KB of loads on their way. Measured against loads and stores
// by threads (four to eight 16-byte vectors each, 2 to 8 blocks an SM): 64 forks of 16 layers' last
// pages (272 MB read and written) 45 against 61 us, 6.0 TB/s; compaction after every second
// of 128 slots has left (1.01 GB) 174 against 195 us, 5.8 TB/s.
constexpr int kRing = 8, kRingAhead = 4, kChunk = 8192;
struct BulkRing {
  uint64_t full[kRing];
  void* to[kRing];
  uint32_t bytes[kRing];
  int abort;
};

struct BulkCopy {
  BulkRing& r;
  uint8_t* const ring;  // kRing * kChunk bytes
  uint32_t n = 0;       // chunks begun
  bool ok = true;

  __device__ void init() {
    for (int i = 0; i < kRing; ++i) sm100::mbar_init(&r.full[i], 1);
    r.abort = 0;
    sm100::fence_barrier_init();
    sm100::fence_proxy_async_smem();
  }
  __device__ void store(uint32_t i) {  // chunk i, once it has arrived
    const uint32_t at = i % kRing;
    if (!ok || !(ok = sm100::mbar_wait(&r.full[at], (i / kRing) & 1u, &r.abort, &g_cache_dev_error, 1))) return;
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(r.to[at]),
                 "r"(sm100::smem_u32(ring + at * kChunk)), "r"(r.bytes[at])
                 : "memory");
    sm100::tma_store_commit();
  }
  __device__ void push(const uint8_t* from, uint8_t* to, uint32_t bytes) {
    const uint32_t at = n % kRing;
    // the store that this place had last was the (kRing - kRingAhead)-th before the latest one
    asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kRing - kRingAhead - 1) : "memory");
    r.to[at] = to;
    r.bytes[at] = bytes;
    sm100::mbar_arrive_expect_tx(&r.full[at], bytes);
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     sm100::smem_u32(ring + at * kChunk)),
                 "l"(from), "r"(bytes), "r"(sm100::smem_u32(&r.full[at]))
                 : "memory");
    if (++n > kRingAhead) store(n - 1 - kRingAhead);
  }
  __device__ void run(const uint4* from, uint4* to, int64_t vecs) {
    const uint8_t* f = reinterpret_cast<const uint8_t*>(from);
    uint8_t* t = reinterpret_cast<uint8_t*>(to);
    for (int64_t left = vecs * 16; ok && left > 0; left -= kChunk, f += kChunk, t += kChunk)
      push(f, t, (uint32_t)min(left, (int64_t)kChunk));
  }
  __device__ void finish() {
    for (uint32_t i = n > kRingAhead ? n - kRingAhead : 0; i < n; ++i) store(i);
    sm100::tma_store_wait_all();
    if (!ok) {  // let the copies that were begun land before shared memory is released
      const uint64_t begin = sm100::globaltimer();
      for (uint32_t i = n > kRing ? n - kRing : 0; i < n; ++i)
        while (!sm100::mbar_try_wait(&r.full[i % kRing], (i / kRing) & 1u) &&
               sm100::globaltimer() - begin < sm100::kWaitTimeoutNs) {}
    }
  }
};

// The first `rows` rows of every head of page `from` to page `to` in one layer of k or v, where
// a head's rows are one run (and a page, where its heads follow one another).
__device__ __forceinline__ void bulk_page(BulkCopy& bulk, uint4* c, int from, int to, int rows, const CacheLayout& s,
                                          const CacheDims& d) {
  const uint4* const src = c + from * s.page;
  uint4* const dst = c + to * s.page;
  if (rows == d.page && s.head == (int64_t)d.page * d.vecs) {
    bulk.run(src, dst, (int64_t)d.heads * d.page * d.vecs);
  } else {
    for (int h = 0; h < d.heads; ++h) bulk.run(src + h * s.head, dst + h * s.head, (int64_t)rows * d.vecs);
  }
}

// The same by all threads of a block, where rows are apart.
__device__ __forceinline__ void copy_page(uint4* c, int from, int to, int rows, const CacheLayout& s,
                                          const CacheDims& d) {
  const uint4* const src = c + from * s.page;
  uint4* const dst = c + to * s.page;
  constexpr int kAhead = 4;
  const uint32_t per_row = (uint32_t)(d.heads * d.vecs), n = per_row * (uint32_t)rows;  // heads of a row follow one another in one such layout
  for (uint32_t x0 = threadIdx.x; x0 < n; x0 += kAhead * blockDim.x) {
    uint4 v[kAhead];
    int64_t at[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const uint32_t x = x0 + i * blockDim.x, r = x / per_row, y = x - r * per_row, h = y / (uint32_t)d.vecs;
      at[i] = h * s.head + r * s.slot + (y - h * (uint32_t)d.vecs);
      if (x < n) v[i] = src[at[i]];
    }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (x0 + i * blockDim.x < n) dst[at[i]] = v[i];
  }
}

// Copies of pages, dealt out to the blocks: unit u of n_units * layers * 2 is a layer's k or v of
// one copy; pages(i, from, to, rows) says which. All threads call it, the block's first warp
// when rows are runs; the others may go on with something else.
template <typename Pages>
__device__ __forceinline__ void copy_pages(uint4* kc, uint4* vc, const CacheLayout& s, const CacheDims& d, int64_t copies,
                                           int first, uint8_t* ring, BulkRing& r, Pages pages) {
  const int64_t units = copies * d.layers * 2;
  const bool runs = s.slot == d.vecs || d.page == 1;
  if (runs && threadIdx.x != 0) return;
  BulkCopy bulk{r, ring};
  if (runs) bulk.init();
  for (int64_t u = first; u < units; u += gridDim.x) {
    const int i = (int)(u / (d.layers * 2)), x = (int)(u - (int64_t)i * (d.layers * 2));
    int from, to, rows;
    if (!pages(i, from, to, rows)) continue;
    uint4* const c = ((x & 1) ? vc : kc) + (x >> 1) * s.layer;
    if (runs) bulk_page(bulk, c, from, to, rows, s, d);
    else copy_page(c, from, to, rows, s, d);
  }
  if (runs) bulk.finish();
}

// The powers of two of a cache in 8 bits (C8): dense, `bytes` to a layer's page.
struct PageScales {
  uint8_t *k, *v;
  int bytes;
};

// Where pages are copied to, their powers of two go too, by the warps that the copies of runs leave free.
template <typename Pages>
__device__ __forceinline__ void copy_scales(const PageScales& s, const CacheDims& d, int64_t copies, int first, Pages pages) {
  constexpr int kOthers = kCopyThreads / 32 - 1;
  const int warp = (int)(threadIdx.x >> 5) - 1, lane = threadIdx.x & 31;
  if (warp < 0) return;
  const bool vec = s.bytes % 16 == 0 && (reinterpret_cast<uintptr_t>(s.k) | reinterpret_cast<uintptr_t>(s.v)) % 16 == 0;
  const int64_t units = copies * d.layers * 2;
  for (int64_t u = (int64_t)first * kOthers + warp; u < units; u += (int64_t)gridDim.x * kOthers) {
    const int i = (int)(u / (d.layers * 2)), x = (int)(u - (int64_t)i * (d.layers * 2));
    int from, to, rows;
    if (!pages(i, from, to, rows)) continue;
    uint8_t* const c = ((x & 1) ? s.v : s.k) + (int64_t)(x >> 1) * d.pages * s.bytes;
    const uint8_t* const src = c + (int64_t)from * s.bytes;
    uint8_t* const dst = c + (int64_t)to * s.bytes;
    if (vec)
      for (int e = 16 * lane; e < s.bytes; e += 512) *reinterpret_cast<uint4*>(dst + e) = *reinterpret_cast<const uint4*>(src + e);
    else
      for (int e = lane; e < s.bytes; e += 32) dst[e] = src[e];
  }
}

// ------------------------------------------------------------------ reserve

struct ReserveArgs {
  const int *tables, *lens, *refs, *extra;
  int *tables_out, *refs_out, *missing;
  int *need, *first, *have;  // workspace [batch]: pages wanted, the rank of the first, pages held
  int batch, max_pages, pages, page;
};

// One block. Measured, calls in a row: 64 slots of 64 entries, 4096 pages 7.8 us; 256 of 64, 16384 pages
// 14.8; 1024 of 128, 65536 pages 48: it reads and writes all tables and counts.
__global__ void __launch_bounds__(kPlanThreads) cache_reserve_kernel(const __grid_constant__ ReserveArgs a) {
  __shared__ u64 scratch[33];
  __shared__ int over;
  pdl_enter();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) over = 0;
  // the pages that each slot has (a row's entries; a warp a row) and the ones it wants
  for (int b = warp; b < a.batch; b += kPlanThreads / 32) {
    const int* const row = a.tables + (int64_t)b * a.max_pages;
    int have = 0;
    for (int i0 = 0; i0 < a.max_pages; i0 += 32) {
      const int p = i0 + lane < a.max_pages ? row[i0 + lane] : -1;
      if (i0 + lane < a.max_pages) a.tables_out[(int64_t)b * a.max_pages + i0 + lane] = p;
      have += __popc(__ballot_sync(0xffffffffu, p >= 0));
    }
    if (lane == 0) a.have[b] = have;
  }
  __syncthreads();
  const int per = (a.batch + kPlanThreads - 1) / kPlanThreads;  // sequences of a thread, in a row
  const int b0 = min((int)threadIdx.x * per, a.batch), b1 = min(b0 + per, a.batch);
  int mine = 0, beyond = 0;
  for (int b = b0; b < b1; ++b) {
    const int64_t want = ((int64_t)max(a.lens[b], 0) + max(a.extra[b], 0) + a.page - 1) / a.page;
    const int n = max((int)(min(want, (int64_t)0x3fffffff) - a.have[b]), 0);
    a.need[b] = n;
    beyond = min(beyond + max(n + a.have[b] - a.max_pages, 0), 0x3fffffff);
    mine = min(mine + n, 0x3fffffff);
  }
  u64 total64;
  u64 at = block_scan<kPlanThreads>((u64)mine, scratch, total64);
  for (int b = b0; b < b1; ++b) {
    a.first[b] = (int)min(at, (u64)0x3fffffff);
    at += a.need[b];
  }
  if (beyond) atomicAdd(&over, min(beyond, 0x3fffffff / kPlanThreads));
  __syncthreads();
  const int wanted = (int)min(total64, (u64)0x3fffffff);
  const bool fits = over == 0;  // rows that would not fit their table cannot be served
  const int free_total = free_pages<kPlanThreads>(a.refs, a.pages, fits ? wanted : 0, scratch,
                                                  [&](int p, int n) { a.refs_out[p] = n; }, [&](int r, int p) {
    int lo = 0, hi = a.batch - 1;  // the last slot whose first rank is <= r: it has a need
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.first[mid] <= r) lo = mid; else hi = mid - 1;
    }
    a.tables_out[(int64_t)lo * a.max_pages + a.have[lo] + r - a.first[lo]] = p;
    a.refs_out[p] = 1;
  });
  if (threadIdx.x == 0) a.missing[0] = max(max(wanted - free_total, over), 0);
}

// ------------------------------------------------------------------ fork

struct ForkArgs {
  const int *tables, *lens, *refs, *src, *dst;
  int *tables_out, *lens_out, *refs_out, *missing;
  int *owner, *fresh, *page_of;  // workspace: fork of each slot [batch]; page of each fork, and of each rank [forks]
  uint4 *kc, *vc;
  CacheLayout c;
  CacheDims d;
  int batch, forks, max_pages;
  PageScales scales;
};

constexpr int kNoFork = 0x7fffffff;

__device__ __forceinline__ bool fork_valid(const ForkArgs& a, int s, int t) {
  return s >= 0 && s < a.batch && t >= 0 && t < a.batch && s != t;
}

// Which forks are valid and the pages they get: owner[slot] (or kNoFork), fresh[fork] (-1: no
// page). `each` as in free_pages. Returns how many pages lack; then there is no fork.
template <int THREADS, typename Each>
__device__ __forceinline__ int fork_plan(const ForkArgs& a, int* owner, int* fresh, int* page_of, u64* scratch, Each each) {
  const int tid = threadIdx.x;
  for (int b = tid; b < a.batch; b += THREADS) owner[b] = kNoFork;
  __syncthreads();
  // the first valid fork into a slot is the one that counts
  for (int f = tid; f < a.forks; f += THREADS) {
    const int s = a.src[f], t = a.dst[f];
    if (fork_valid(a, s, t)) atomicMin(&owner[t], f);
  }
  __syncthreads();
  int wanted = 0;
  for (int f0 = 0; f0 < a.forks; f0 += THREADS) {
    const int f = f0 + tid;
    bool need = false;
    if (f < a.forks) {
      const int s = a.src[f], t = a.dst[f];
      if (fork_valid(a, s, t) && owner[t] == f) {
        const int n = max(a.lens[s], 0);
        need = n % a.d.page != 0 && n / a.d.page < a.max_pages;
      }
    }
    u64 total;
    const int r = wanted + (int)block_scan<THREADS>((u64)need, scratch, total);
    if (f < a.forks) fresh[f] = need ? r : -1;  // the rank of its page
    wanted += (int)total;
  }
  const int lacking = wanted - free_pages<THREADS>(a.refs, a.d.pages, wanted, scratch, each,
                                                   [&](int rank, int p) { page_of[rank] = p; });
  __syncthreads();
  for (int f = tid; f < a.forks; f += THREADS) fresh[f] = lacking > 0 || fresh[f] < 0 ? -1 : page_of[fresh[f]];
  if (lacking > 0)
    for (int b = tid; b < a.batch; b += THREADS) owner[b] = kNoFork;
  __syncthreads();
  return max(lacking, 0);
}

// Row `b` of the tables and its length, by the threads of a warp; count(page, by) changes refs.
template <typename Count>
__device__ __forceinline__ void fork_row(const ForkArgs& a, int b, int f, int fresh, bool write, Count count) {
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)b * a.max_pages;
  const int s = f == kNoFork ? b : a.src[f], n = max(a.lens[s], 0), full = n / a.d.page;
  for (int i = lane; i < a.max_pages; i += 32) {
    const int old = a.tables[row + i];
    int now = old;
    if (f != kNoFork) {
      now = i < full ? a.tables[(int64_t)s * a.max_pages + i] : i == full ? fresh : -1;
      if (old >= 0 && old < a.d.pages) count(old, -1);
      if (now >= 0 && now < a.d.pages) count(now, 1);
    }
    if (write) a.tables_out[row + i] = now;
  }
  if (write && lane == 0) a.lens_out[b] = f == kNoFork ? a.lens[b] : a.lens[s];
}

// The used rows of the forks' last pages, and these pages' powers of two.
template <bool C8>
__device__ __forceinline__ void fork_copies(const ForkArgs& a, const int* fresh, int first, uint8_t* ring, BulkRing& r) {
  auto pages = [&](int f, int& from, int& to, int& rows) {
    to = fresh[f];
    if (to < 0) return false;
    const int s = a.src[f], n = max(a.lens[s], 0), full = n / a.d.page;
    from = a.tables[(int64_t)s * a.max_pages + full];
    rows = n - full * a.d.page;
    return from >= 0 && from < a.d.pages;
  };
  if constexpr (C8) copy_scales(a.scales, a.d, a.forks, first, pages);
  copy_pages(a.kc, a.vc, a.c, a.d, a.forks, first, ring, r, pages);
}

// Small caches: every block makes the whole plan for itself, in shared memory, which costs
// less than a launch of its own; block 0 counts the refs, the rows and copies are dealt out.
// Measured against a plan by one block and a second launch that applies it, forks of pages of
// 16: 256 pages 6.3 against 8.5 us, 4096 9.5 against 10.2, 8192 14.2 against 11.3 (one plan by 1024
// threads). Compaction: 256 pages 3.8 against 7.4 us, 8192 15.6 against 20.7; its plan's place in
// shared memory ends there.
constexpr int kSmallForkPages = 4096, kSmallSlots = 512, kSmallForks = 256, kSmallEntries = 8192;
constexpr int kSmallPages = 8192;

template <bool C8>
__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) cache_fork_small_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ u64 scratch[33];
  __shared__ int owner[kSmallSlots], fresh[kSmallForks], page_of[kSmallForks];
  __shared__ BulkRing bulk;
  extern __shared__ __align__(128) uint8_t ring[];
  int* const refs = reinterpret_cast<int*>(ring + kRing * kChunk);  // block 0: the counts
  pdl_enter();
  const bool counts = blockIdx.x == 0;
  const int lacking = fork_plan<kCopyThreads>(a, owner, fresh, page_of, scratch, [&](int p, int n) {
    if (counts) refs[p] = n;
  });
  constexpr int kWarps = kCopyThreads / 32;
  const int warp = threadIdx.x >> 5;
  auto row = [&](int b, bool write, auto count) {
    const int f = owner[b];
    fork_row(a, b, f, f == kNoFork ? -1 : fresh[f], write, count);
  };
  if (counts) {
    for (int b = warp; b < a.batch; b += kWarps)
      if (owner[b] != kNoFork) row(b, false, [&](int p, int by) { atomicAdd(&refs[p], by); });
    if (threadIdx.x == 0) a.missing[0] = lacking;
    __syncthreads();
    for (int p = threadIdx.x; p < a.d.pages; p += kCopyThreads) a.refs_out[p] = refs[p];
  }
  for (int b = (int)blockIdx.x * kWarps + warp; b < a.batch; b += (int)gridDim.x * kWarps) row(b, true, [](int, int) {});
  // block 0 comes last: it has had the counts to do
  fork_copies<C8>(a, fresh, (int)((blockIdx.x + gridDim.x - 1) % gridDim.x), ring, bulk);
}

__global__ void __launch_bounds__(kPlanThreads) cache_fork_plan_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ u64 scratch[33];
  pdl_enter();
  const int lacking = fork_plan<kPlanThreads>(a, a.owner, a.fresh, a.page_of, scratch, [&](int p, int n) { a.refs_out[p] = n; });
  if (threadIdx.x == 0) a.missing[0] = lacking;
}

template <bool C8>
__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) cache_fork_apply_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ BulkRing bulk;
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_enter();
  constexpr int kWarps = kCopyThreads / 32;
  for (int b = (int)blockIdx.x * kWarps + (threadIdx.x >> 5); b < a.batch; b += (int)gridDim.x * kWarps) {
    const int f = a.owner[b];
    fork_row(a, b, f, f == kNoFork ? -1 : a.fresh[f], true, [&](int p, int by) { atomicAdd(&a.refs_out[p], by); });
  }
  fork_copies<C8>(a, a.fresh, (int)blockIdx.x, ring, bulk);
}

// ------------------------------------------------------------------ free

struct FreeArgs {
  const int *tables, *lens, *refs, *slots;
  int *tables_out, *lens_out, *refs_out;
  int batch, n_slots, max_pages, pages;
};

// A cluster of blocks (one for small tables): counts copied, slots marked, then a warp a row.
__global__ void __launch_bounds__(kPlanThreads) cache_free_kernel(const __grid_constant__ FreeArgs a) {
  pdl_enter();
  const int threads = gridDim.x * kPlanThreads, id = blockIdx.x * kPlanThreads + threadIdx.x;
  for (int p = id; p < a.pages; p += threads) a.refs_out[p] = a.refs[p];
  for (int b = id; b < a.batch; b += threads) a.lens_out[b] = max(a.lens[b], 0);
  if (gridDim.x > 1) cluster_sync(); else __syncthreads();
  for (int i = id; i < a.n_slots; i += threads) {
    const int b = a.slots[i];
    if (b >= 0 && b < a.batch) a.lens_out[b] = -1;  // marks the slot until the end
  }
  if (gridDim.x > 1) cluster_sync(); else __syncthreads();
  const int lane = threadIdx.x & 31;
  for (int b = id >> 5; b < a.batch; b += threads >> 5) {
    const bool gone = __ldcg(a.lens_out + b) == -1;
    const int64_t row = (int64_t)b * a.max_pages;
    for (int i = lane; i < a.max_pages; i += 32) {
      const int p = a.tables[row + i];
      if (gone && p >= 0 && p < a.pages) atomicSub(&a.refs_out[p], 1);
      a.tables_out[row + i] = gone ? -1 : p;
    }
    __syncwarp();
    if (gone && lane == 0) a.lens_out[b] = 0;
  }
}

// ------------------------------------------------------------------ compact

struct CompactArgs {
  const int *tables, *refs;
  int *tables_out, *refs_out;
  int *place, *come, *go, *moves;  // workspace: new index of each page, the moves' ends, their number
  uint4 *kc, *vc;
  CacheLayout c;
  CacheDims d;
  int64_t entries;
  PageScales scales;
};

__global__ void __launch_bounds__(kPlanThreads) cache_compact_plan_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ u64 scratch[33];
  pdl_enter();
  int live, movers;
  compact_plan<kPlanThreads>(a.refs, a.d.pages, scratch, live, movers, [&](int p, int n, int kind, int rank) {
    if (kind == 1) a.go[rank] = p;
    if (kind == 2) a.come[rank] = p;
    a.place[p] = p;
    a.refs_out[p] = p < live && n > 0 ? n : 0;
  });
  __syncthreads();
  if (threadIdx.x == 0) a.moves[0] = movers;
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
    const int from = a.come[i], to = a.go[i];
    a.place[from] = to;
    a.refs_out[to] = a.refs[from];
  }
}

// Whole pages; `come` and `go` are indices, of 32 or 16 bits.
template <bool C8, typename I>
__device__ __forceinline__ void compact_copies(const CompactArgs& a, const I* come, const I* go, int moves, uint8_t* ring,
                                               BulkRing& r) {
  auto pages = [&](int i, int& from, int& to, int& rows) {
    from = come[i];
    to = go[i];
    rows = a.d.page;
    return true;
  };
  if constexpr (C8) copy_scales(a.scales, a.d, moves, (int)blockIdx.x, pages);
  copy_pages(a.kc, a.vc, a.c, a.d, moves, (int)blockIdx.x, ring, r, pages);
}

template <bool C8>
__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) cache_compact_apply_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ BulkRing bulk;
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * blockDim.x) {
    const int p = a.tables[i];
    a.tables_out[i] = p >= 0 && p < a.d.pages ? a.place[p] : p;
  }
  compact_copies<C8>(a, a.come, a.go, a.moves[0], ring, bulk);
}

// As cache_fork_small_kernel: every block plans for itself. There are at most as many moves as
// half of the pages, rounded down.
template <bool C8>
__global__ void __launch_bounds__(kCopyThreads, kCopyBlocks) cache_compact_small_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ u64 scratch[33];
  __shared__ uint16_t come[kSmallPages / 2], go[kSmallPages / 2], rank_of[kSmallPages];
  __shared__ BulkRing bulk;
  extern __shared__ __align__(128) uint8_t ring[];
  pdl_enter();
  int live, movers;
  compact_plan<kCopyThreads>(a.refs, a.d.pages, scratch, live, movers, [&](int p, int n, int kind, int rank) {
    if (kind == 1) go[rank] = (uint16_t)p;
    if (kind == 2) come[rank] = (uint16_t)p;
    rank_of[p] = (uint16_t)rank;
  });
  __syncthreads();
  const int id = (int)blockIdx.x * kCopyThreads + threadIdx.x, threads = (int)gridDim.x * kCopyThreads;
  for (int p = id; p < a.d.pages; p += threads) {
    const int n = a.refs[p];
    a.refs_out[p] = p >= live ? 0 : n > 0 ? n : a.refs[come[rank_of[p]]];
  }
  for (int64_t i = id; i < a.entries; i += threads) {
    const int p = a.tables[i];
    // a page in use from `live` on moves; a table entry for one that is not in use stays
    a.tables_out[i] = p >= live && p < a.d.pages && a.refs[p] > 0 ? go[rank_of[p]] : p;
  }
  compact_copies<C8>(a, come, go, movers, ring, bulk);
}

// ------------------------------------------------------------------ host

constexpr int64_t kMaxInt = 0x7fffffffLL;

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

constexpr int kBytes = -1;  // beside the dtypes: a cache in 8 bits

// Checks and converts the cache's description; strides (elements) are layer, page, head, slot.
int cache_dims(const char* op, const void* kc, const void* vc, const int64_t* strides, int64_t layers, int64_t pages,
               int64_t kv_heads, int64_t page_size, int64_t head_dim, int dtype, CacheDims* d, CacheLayout* c) {
  if (dtype != kBytes && !valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (layers < 1 || pages < 1 || kv_heads < 1 || page_size < 1 || head_dim < 1)
    return fail(NKL_ERR_SHAPE, "%s: layers, pages, heads, page size and head_dim must be positive", op);
  const int64_t per = dtype == kBytes ? 16 : 16 / (int64_t)dtype_size(dtype);
  if (head_dim % per)
    return fail(NKL_ERR_SHAPE, "%s: a row must be a multiple of 16 bytes (head_dim %lld)", op, (long long)head_dim);
  if (layers > 65535 || pages > kMaxInt / 4 || kv_heads > 65535 || page_size > 65536 || head_dim > 65536 ||
      kv_heads * page_size * (head_dim / per) > kMaxInt)
    return fail(NKL_ERR_SHAPE, "%s: size out of range", op);
  if (!kc || !vc) return fail(NKL_ERR_ARG, "%s: NULL cache", op);
  if (!is_aligned(kc, 16) || !is_aligned(vc, 16)) return fail(NKL_ERR_ALIGN, "%s: cache not 16-byte aligned", op);
  int64_t s[4];
  if (strides) {
    for (int i = 0; i < 4; ++i) s[i] = strides[i];
  } else {
    s[3] = head_dim;
    s[2] = page_size * s[3];
    s[1] = kv_heads * s[2];
    s[0] = pages * s[1];
  }
  const int64_t dims[4] = {layers, pages, kv_heads, page_size};
  for (int i = 0; i < 4; ++i)
    if (dims[i] > 1 && (s[i] < head_dim || s[i] % per))
      return fail(NKL_ERR_ALIGN, "%s: cache stride %lld is not a multiple of 16 bytes of at least a row", op,
                  (long long)s[i]);
  *d = {(int)layers, (int)pages, (int)kv_heads, (int)page_size, (int)(head_dim / per)};
  *c = {s[0] / per, s[1] / per, s[2] / per, s[3] / per};
  return NKL_OK;
}

// The powers of two of a cache in 8 bits, given its checked dimensions.
int page_scales(const char* op, void* k_scales, void* v_scales, int64_t block, const CacheDims& d, PageScales* s) {
  if (block < 1 || d.page % block)
    return fail(NKL_ERR_SHAPE, "%s: blocks of %lld positions do not divide pages of %d", op, (long long)block, d.page);
  if (!k_scales || !v_scales) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  const int64_t bytes = d.heads * (d.page / block);
  if (bytes > kMaxInt) return fail(NKL_ERR_SHAPE, "%s: size out of range", op);
  *s = {static_cast<uint8_t*>(k_scales), static_cast<uint8_t*>(v_scales), (int)bytes};
  return NKL_OK;
}

int check_table(const char* op, int64_t batch, int64_t max_pages) {
  if (batch < 0 || max_pages < 1) return fail(NKL_ERR_SHAPE, "%s: batch must not be negative, tables need a column", op);
  if (batch > kMaxInt / 4 || max_pages > kMaxInt / 4 || batch * max_pages > kMaxInt)
    return fail(NKL_ERR_SHAPE, "%s: tables too large", op);
  return NKL_OK;
}

unsigned grid_for(int64_t blocks, int per_sm) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)sm_count() * per_sm));
}

// Allows the kernels that copy pages their ring, once per device.
template <bool C8>
int allow_ring(const char* op) {
  static std::atomic<bool> set[64] = {};  // idempotent
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && set[dev].load(std::memory_order_acquire)) return NKL_OK;
  cudaError_t e = cudaSuccess;
  auto allow = [&](const void* kernel, int bytes) {
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  };
  allow((const void*)cache_fork_small_kernel<C8>, kRing * kChunk + kSmallForkPages * 4);
  allow((const void*)cache_fork_apply_kernel<C8>, kRing * kChunk);
  allow((const void*)cache_compact_small_kernel<C8>, kRing * kChunk);
  allow((const void*)cache_compact_apply_kernel<C8>, kRing * kChunk);
  if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  return NKL_OK;
}

}  // namespace

int cache_read_and_clear_device_error() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_cache_dev_error, sizeof(v)) != cudaSuccess) return -1;
  if (v && cudaMemcpyToSymbol(g_cache_dev_error, &zero, sizeof(zero)) != cudaSuccess) return -1;
  return (int)v;
}

}  // namespace nkl

using namespace nkl;

extern "C" int nkl_cache_append(const void* k, const void* v, const int64_t* kv_strides, void* k_cache, void* v_cache,
                                const int64_t* cache_strides, const int32_t* tables, const int32_t* lens,
                                const int32_t* path, const int32_t* count, int32_t* lens_out, int64_t layers,
                                int64_t batch, int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                int64_t page_size, int64_t max_pages, int dtype, void* stream) {
  const char* op = "nkl_cache_append";
  AppendArgs a = {};
  int rc = cache_dims(op, k_cache, v_cache, cache_strides, layers, pages, kv_heads, page_size, head_dim, dtype, &a.d,
                      &a.c);
  if (rc) return rc;
  rc = check_table(op, batch, max_pages);
  if (rc) return rc;
  if (tokens < 0 || tokens > kMaxInt / 4) return fail(NKL_ERR_SHAPE, "%s: bad number of tokens", op);
  if (batch == 0) return NKL_OK;
  if (!tables || !lens || !lens_out || (tokens && (!k || !v))) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (tokens && (!is_aligned(k, 16) || !is_aligned(v, 16))) return fail(NKL_ERR_ALIGN, "%s: k and v need 16-byte alignment", op);
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  int64_t s[4] = {batch * tokens * kv_heads * head_dim, tokens * kv_heads * head_dim, kv_heads * head_dim, head_dim};
  const int64_t dims[4] = {layers, batch, tokens, kv_heads};
  for (int i = 0; i < 4; ++i) {
    if (kv_strides) s[i] = kv_strides[i];
    if (dims[i] > 1 && (s[i] < 0 || s[i] % per))
      return fail(NKL_ERR_ALIGN, "%s: stride %lld of k and v is not a multiple of 16 bytes", op, (long long)s[i]);
  }
  a.k = static_cast<const uint4*>(k);
  a.v = static_cast<const uint4*>(v);
  a.kc = static_cast<uint4*>(k_cache);
  a.vc = static_cast<uint4*>(v_cache);
  a.tables = tables;
  a.lens = lens;
  a.path = path;
  a.count = count;
  a.lens_out = lens_out;
  a.n_layer = s[0] / per;
  a.n_batch = s[1] / per;
  a.n_token = s[2] / per;
  a.n_head = s[3] / per;
  a.batch = (int)batch;
  a.tokens = (int)tokens;
  a.max_pages = (int)max_pages;
  a.vecs_magic = a.d.vecs > 1 ? (uint32_t)(((1ull << 32) + a.d.vecs - 1) / a.d.vecs) : 0u;
  if (batch > 65535 || kv_heads * a.d.vecs > 65535)  // the magic's range, and the grid's
    return fail(NKL_ERR_SHAPE, "%s: more than 65535 sequences, or rows longer than 1 MB", op);
  const int64_t warps = kCopyThreads / 32;
  return launch_pdl(cache_append_kernel,
                    dim3((unsigned)std::max<int64_t>(1, (tokens + warps - 1) / warps), (unsigned)batch, (unsigned)layers),
                    dim3(kCopyThreads), 0, static_cast<cudaStream_t>(stream), op, a);
}

extern "C" size_t nkl_cache_reserve_workspace_size(int64_t batch) {
  return batch > 0 ? round256((size_t)batch * 12) : 0;
}

extern "C" int nkl_cache_reserve(const int32_t* tables, const int32_t* lens, const int32_t* refs, const int32_t* extra,
                                 int32_t* tables_out, int32_t* refs_out, int32_t* missing, void* workspace,
                                 size_t workspace_bytes, int64_t batch, int64_t pages, int64_t page_size,
                                 int64_t max_pages, void* stream) {
  const char* op = "nkl_cache_reserve";
  int rc = check_table(op, batch, max_pages);
  if (rc) return rc;
  if (pages < 1 || pages > kMaxInt / 4 || page_size < 1 || page_size > 65536)
    return fail(NKL_ERR_SHAPE, "%s: bad number or size of pages", op);
  if (!refs || !refs_out || !missing || (batch && (!tables || !lens || !extra || !tables_out)))
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (workspace_bytes < nkl_cache_reserve_workspace_size(batch) || (batch && !workspace))
    return fail(NKL_ERR_ARG, "%s: workspace too small", op);
  int* const ws = static_cast<int*>(workspace);
  ReserveArgs a = {tables, lens,       refs,           extra,      tables_out,     refs_out,   missing,       ws,
                   ws + batch, ws + 2 * batch, (int)batch, (int)max_pages, (int)pages, (int)page_size};
  return launch_pdl(cache_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), op, a);
}

extern "C" size_t nkl_cache_fork_workspace_size(int64_t batch, int64_t forks) {
  return batch > 0 && forks >= 0 ? round256(((size_t)batch + 2 * (size_t)forks) * 4) : 0;
}

namespace {

// Both entry points; C8: with scales, of dtype kBytes.
template <bool C8>
int fork(const char* op, void* k_cache, void* v_cache, const int64_t* cache_strides, void* k_scales, void* v_scales,
         const int32_t* tables, const int32_t* lens, const int32_t* refs, const int32_t* src, const int32_t* dst,
         int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* missing, void* workspace,
         size_t workspace_bytes, int64_t forks, int64_t layers, int64_t batch, int64_t kv_heads, int64_t head_dim,
         int64_t pages, int64_t page_size, int64_t max_pages, int64_t block, int dtype, void* stream) {
  ForkArgs a = {};
  int rc = cache_dims(op, k_cache, v_cache, cache_strides, layers, pages, kv_heads, page_size, head_dim, dtype, &a.d,
                      &a.c);
  if (rc) return rc;
  if (C8 && (rc = page_scales(op, k_scales, v_scales, block, a.d, &a.scales))) return rc;
  rc = check_table(op, batch, max_pages);
  if (rc) return rc;
  if (forks < 0 || forks > kMaxInt / 4) return fail(NKL_ERR_SHAPE, "%s: bad number of forks", op);
  if (batch < 1) return fail(NKL_ERR_SHAPE, "%s: no slots", op);
  if (!tables || !lens || !refs || !tables_out || !lens_out || !refs_out || !missing || (forks && (!src || !dst)))
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (!workspace || workspace_bytes < nkl_cache_fork_workspace_size(batch, forks))
    return fail(NKL_ERR_ARG, "%s: workspace too small", op);
  a.tables = tables;
  a.lens = lens;
  a.refs = refs;
  a.src = src;
  a.dst = dst;
  a.tables_out = tables_out;
  a.lens_out = lens_out;
  a.refs_out = refs_out;
  a.missing = missing;
  a.owner = static_cast<int*>(workspace);
  a.fresh = a.owner + batch;
  a.page_of = a.fresh + forks;
  a.kc = static_cast<uint4*>(k_cache);
  a.vc = static_cast<uint4*>(v_cache);
  a.batch = (int)batch;
  a.forks = (int)forks;
  a.max_pages = (int)max_pages;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int e = allow_ring<C8>(op)) return e;
  if (pages <= kSmallForkPages && batch <= kSmallSlots && forks <= kSmallForks && batch * max_pages <= kSmallEntries)
    return launch_pdl(cache_fork_small_kernel<C8>, dim3(grid_for(std::max(batch / 8, forks * layers * 2), kCopyBlocks)),
                      dim3(kCopyThreads), kRing * kChunk + (size_t)pages * 4, st, op, a);
  rc = launch_pdl(cache_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, op, a);
  if (rc) return rc;
  return launch_pdl(cache_fork_apply_kernel<C8>, dim3(grid_for(std::max(batch / 8, forks * layers * 2), kCopyBlocks)), dim3(kCopyThreads),
                    kRing * kChunk, st, op, a);
}

}  // namespace

extern "C" int nkl_cache_fork(void* k_cache, void* v_cache, const int64_t* cache_strides, const int32_t* tables,
                              const int32_t* lens, const int32_t* refs, const int32_t* src, const int32_t* dst,
                              int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* missing,
                              void* workspace, size_t workspace_bytes, int64_t forks, int64_t layers, int64_t batch,
                              int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size,
                              int64_t max_pages, int dtype, void* stream) {
  const char* op = "nkl_cache_fork";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  return fork<false>(op, k_cache, v_cache, cache_strides, nullptr, nullptr, tables, lens, refs, src, dst, tables_out, lens_out,
              refs_out, missing, workspace, workspace_bytes, forks, layers, batch, kv_heads, head_dim, pages, page_size,
              max_pages, 0, dtype, stream);
}

extern "C" int nkl_cache_fork_8bit(void* k_cache, void* v_cache, const int64_t* cache_strides, void* k_scales,
                                   void* v_scales, const int32_t* tables, const int32_t* lens, const int32_t* refs,
                                   const int32_t* src, const int32_t* dst, int32_t* tables_out, int32_t* lens_out,
                                   int32_t* refs_out, int32_t* missing, void* workspace, size_t workspace_bytes,
                                   int64_t forks, int64_t layers, int64_t batch, int64_t kv_heads, int64_t head_dim,
                                   int64_t pages, int64_t page_size, int64_t max_pages, int64_t block, void* stream) {
  return fork<true>("nkl_cache_fork_8bit", k_cache, v_cache, cache_strides, k_scales, v_scales, tables, lens, refs, src, dst,
              tables_out, lens_out, refs_out, missing, workspace, workspace_bytes, forks, layers, batch, kv_heads, head_dim,
              pages, page_size, max_pages, block, kBytes, stream);
}

extern "C" int nkl_cache_free(const int32_t* tables, const int32_t* lens, const int32_t* refs, const int32_t* slots,
                              int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int64_t n_slots,
                              int64_t batch, int64_t pages, int64_t max_pages, void* stream) {
  const char* op = "nkl_cache_free";
  int rc = check_table(op, batch, max_pages);
  if (rc) return rc;
  if (pages < 1 || pages > kMaxInt / 4 || n_slots < 0 || n_slots > kMaxInt / 4)
    return fail(NKL_ERR_SHAPE, "%s: bad number of pages or slots", op);
  if (!refs || !refs_out || (batch && (!tables || !lens || !tables_out || !lens_out)) || (n_slots && !slots))
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  FreeArgs a = {tables,     lens,        refs,          slots,          tables_out, lens_out,
                refs_out,   (int)batch,  (int)n_slots,  (int)max_pages, (int)pages};
  // One block, or a cluster of eight (the portable most), by the entries and counts there are: with
  // 8192 of them 4.4 against 4.8 us, with 24576 9.0 against 4.6, with 196608 49 against 9.6.
  const unsigned blocks = batch * max_pages + pages > 8192 ? 8 : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, cache_free_kernel, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  return NKL_OK;
}

extern "C" size_t nkl_cache_compact_workspace_size(int64_t pages) {
  return pages > 0 ? round256(((size_t)pages * 3 + 1) * 4) : 0;
}

namespace {

template <bool C8>
int compact(const char* op, void* k_cache, void* v_cache, const int64_t* cache_strides, void* k_scales, void* v_scales,
            const int32_t* tables, const int32_t* refs, int32_t* tables_out, int32_t* refs_out, void* workspace,
            size_t workspace_bytes, int64_t layers, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t pages,
            int64_t page_size, int64_t max_pages, int64_t block, int dtype, void* stream) {
  CompactArgs a = {};
  int rc = cache_dims(op, k_cache, v_cache, cache_strides, layers, pages, kv_heads, page_size, head_dim, dtype, &a.d,
                      &a.c);
  if (rc) return rc;
  if (C8 && (rc = page_scales(op, k_scales, v_scales, block, a.d, &a.scales))) return rc;
  rc = check_table(op, batch, max_pages);
  if (rc) return rc;
  if (!refs || !refs_out || (batch && (!tables || !tables_out))) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (!workspace || workspace_bytes < nkl_cache_compact_workspace_size(pages))
    return fail(NKL_ERR_ARG, "%s: workspace too small", op);
  a.tables = tables;
  a.refs = refs;
  a.tables_out = tables_out;
  a.refs_out = refs_out;
  a.place = static_cast<int*>(workspace);
  a.come = a.place + pages;
  a.go = a.come + pages;
  a.moves = a.go + pages;
  a.kc = static_cast<uint4*>(k_cache);
  a.vc = static_cast<uint4*>(v_cache);
  a.entries = batch * max_pages;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (int e = allow_ring<C8>(op)) return e;
  if (pages <= kSmallPages)
    return launch_pdl(cache_compact_small_kernel<C8>,
                      dim3(grid_for(std::max<int64_t>((a.entries + 255) / 256, pages * layers), kCopyBlocks)), dim3(kCopyThreads),
                      kRing * kChunk, st, op, a);
  rc = launch_pdl(cache_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, op, a);
  if (rc) return rc;
  return launch_pdl(cache_compact_apply_kernel<C8>,
                    dim3(grid_for(std::max<int64_t>((a.entries + 255) / 256, pages * layers), kCopyBlocks)), dim3(kCopyThreads),
                    kRing * kChunk, st, op, a);
}

}  // namespace

extern "C" int nkl_cache_compact(void* k_cache, void* v_cache, const int64_t* cache_strides, const int32_t* tables,
                                 const int32_t* refs, int32_t* tables_out, int32_t* refs_out, void* workspace,
                                 size_t workspace_bytes, int64_t layers, int64_t batch, int64_t kv_heads,
                                 int64_t head_dim, int64_t pages, int64_t page_size, int64_t max_pages, int dtype,
                                 void* stream) {
  const char* op = "nkl_cache_compact";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  return compact<false>(op, k_cache, v_cache, cache_strides, nullptr, nullptr, tables, refs, tables_out, refs_out, workspace,
                 workspace_bytes, layers, batch, kv_heads, head_dim, pages, page_size, max_pages, 0, dtype, stream);
}

extern "C" int nkl_cache_compact_8bit(void* k_cache, void* v_cache, const int64_t* cache_strides, void* k_scales,
                                      void* v_scales, const int32_t* tables, const int32_t* refs, int32_t* tables_out,
                                      int32_t* refs_out, void* workspace, size_t workspace_bytes, int64_t layers,
                                      int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                      int64_t page_size, int64_t max_pages, int64_t block, void* stream) {
  return compact<true>("nkl_cache_compact_8bit", k_cache, v_cache, cache_strides, k_scales, v_scales, tables, refs, tables_out,
                 refs_out, workspace, workspace_bytes, layers, batch, kv_heads, head_dim, pages, page_size, max_pages, block,
                 kBytes, stream);
}
