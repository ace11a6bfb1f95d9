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
#include <algorithm>

#include "common.cuh"

namespace nkl {
namespace {

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum over the block (kPlanThreads threads); `total` gets the sum.
// `warp_sums` is shared scratch of 33 ints.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __syncthreads();  // the scratch may still be read from the call before
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    const int w = warp_sums[lane];
    int wi = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, wi, o);
      if (lane >= o) wi += x;
    }
    warp_sums[lane] = wi - w;
    if (lane == 31) warp_sums[32] = wi;
  }
  __syncthreads();
  total = warp_sums[32];
  return warp_sums[warp] + inc - v;
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
};

// One thread per 16-byte vector of a row of k and v.
__global__ void __launch_bounds__(256) cache_append_kernel(const __grid_constant__ AppendArgs a) {
  pdl_enter();
  const int row_vecs = a.d.heads * a.d.vecs;
  const int64_t total = (int64_t)a.d.layers * a.batch * a.tokens * row_vecs;
  const int64_t first = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t b = first; b < a.batch; b += (int64_t)gridDim.x * blockDim.x) {
    const int n = a.count ? min(max(a.count[b], 0), a.tokens) : a.tokens;
    a.lens_out[b] = max(a.lens[b], 0) + n;
  }
  for (int64_t i = first; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / row_vecs;
    const int x = (int)(i - row * row_vecs);
    const int h = x / a.d.vecs, e = x - h * a.d.vecs;
    const int j = (int)(row % a.tokens);
    const int64_t lb = row / a.tokens;
    const int b = (int)(lb % a.batch), l = (int)(lb / a.batch);
    if (a.count && j >= a.count[b]) continue;
    const int src = a.path ? a.path[(int64_t)b * a.tokens + j] : j;
    if (src < 0 || src >= a.tokens) continue;
    const int pos = max(a.lens[b], 0) + j;
    const int p = pos / a.d.page;
    if (p >= a.max_pages) continue;
    const int at = a.tables[(int64_t)b * a.max_pages + p];
    if (at < 0 || at >= a.d.pages) continue;
    const int64_t from = l * a.n_layer + b * a.n_batch + src * a.n_token + h * a.n_head + e;
    const int64_t to = l * a.c.layer + at * a.c.page + h * a.c.head + (pos - p * a.d.page) * a.c.slot + e;
    const uint4 kv = a.k[from], vv = a.v[from];
    a.kc[to] = kv;
    a.vc[to] = vv;
  }
}

// ------------------------------------------------------------------ page copies

// Copies `rows` rows of every head of page `from` to page `to` in one layer of k or v.
__device__ __forceinline__ void copy_page(uint4* c, int from, int to, int rows, const CacheLayout& s,
                                          const CacheDims& d) {
  const int per_head = rows * d.vecs;
  for (int i = threadIdx.x; i < per_head * d.heads; i += blockDim.x) {
    const int h = i / per_head, x = i - h * per_head;
    const int r = x / d.vecs, e = x - r * d.vecs;
    const int64_t at = h * s.head + r * s.slot + e;
    c[to * s.page + at] = c[from * s.page + at];
  }
}

// ------------------------------------------------------------------ reserve

struct ReserveArgs {
  const int *tables, *lens, *refs, *extra;
  int *tables_out, *refs_out, *missing;
  int *need, *first;  // workspace [batch]: pages wanted, and the rank of the first
  int batch, max_pages, pages, page;
};

__global__ void __launch_bounds__(kPlanThreads) cache_reserve_kernel(const __grid_constant__ ReserveArgs a) {
  __shared__ int scratch[33];
  pdl_enter();
  // how many pages each slot has and wants
  int base = 0;
  for (int b0 = 0; b0 < a.batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    int n = 0, have = 0;
    if (b < a.batch) {
      const int64_t want64 = (int64_t)max(a.lens[b], 0) + max(a.extra[b], 0);
      const int64_t want = (want64 + a.page - 1) / a.page;
      while (have < a.max_pages && a.tables[(int64_t)b * a.max_pages + have] >= 0) ++have;
      n = want > have ? (int)min(want, (int64_t)0x3fffffff) - have : 0;
    }
    int total;
    const int at = block_scan(n, scratch, total);
    if (b < a.batch) {
      a.need[b] = n;
      a.first[b] = base + at;
    }
    base = min(base + total, 0x3fffffff);
  }
  const int wanted = base;
  // rows that would not fit their table cannot be served either
  int over = 0;
  for (int b = threadIdx.x; b < a.batch; b += kPlanThreads) {
    int have = 0;
    while (have < a.max_pages && a.tables[(int64_t)b * a.max_pages + have] >= 0) ++have;
    over += max(a.need[b] + have - a.max_pages, 0);
  }
  int over_total, free_total = 0;
  block_scan(over, scratch, over_total);
  for (int p0 = 0; p0 < a.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    int t;
    block_scan(p < a.pages && a.refs[p] == 0, scratch, t);
    free_total += t;
  }
  const int lacking = max(wanted - free_total, over_total);
  const bool ok = lacking <= 0;
  if (threadIdx.x == 0) a.missing[0] = max(lacking, 0);
  for (int64_t i = threadIdx.x; i < (int64_t)a.batch * a.max_pages; i += kPlanThreads) a.tables_out[i] = a.tables[i];
  __syncthreads();
  // the r-th free page goes to the slot whose range of ranks holds r
  int seen = 0;
  for (int p0 = 0; p0 < a.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const bool is_free = p < a.pages && a.refs[p] == 0;
    int t;
    const int r = seen + block_scan(is_free, scratch, t);
    seen += t;
    if (p >= a.pages) continue;
    const bool take = ok && is_free && r < wanted;
    a.refs_out[p] = take ? 1 : a.refs[p];
    if (take) {
      int lo = 0, hi = a.batch - 1;  // the last slot with first <= r and a need
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.first[mid] <= r) lo = mid; else hi = mid - 1;
      }
      int have = 0;
      while (have < a.max_pages && a.tables[(int64_t)lo * a.max_pages + have] >= 0) ++have;
      a.tables_out[(int64_t)lo * a.max_pages + have + r - a.first[lo]] = p;
    }
  }
}

// ------------------------------------------------------------------ fork

struct ForkArgs {
  const int *tables, *lens, *refs, *src, *dst;
  int *tables_out, *lens_out, *refs_out, *missing;
  int *owner, *fresh;  // workspace: fork of each slot [batch], fresh page of each fork [forks] (-1: none)
  uint4 *kc, *vc;
  CacheLayout c;
  CacheDims d;
  int batch, forks, max_pages;
};

// Which forks are valid, the pages they get, and the counts they start from. One block.
__global__ void __launch_bounds__(kPlanThreads) cache_fork_plan_kernel(const __grid_constant__ ForkArgs a) {
  __shared__ int scratch[33];
  pdl_enter();
  for (int b = threadIdx.x; b < a.batch; b += kPlanThreads) a.owner[b] = 0x7fffffff;
  __syncthreads();
  // the first valid fork into a slot is the one that counts
  for (int f = threadIdx.x; f < a.forks; f += kPlanThreads) {
    const int s = a.src[f], t = a.dst[f];
    if (s >= 0 && s < a.batch && t >= 0 && t < a.batch && s != t) atomicMin(&a.owner[t], f);
  }
  __syncthreads();
  int wanted = 0;
  for (int f0 = 0; f0 < a.forks; f0 += kPlanThreads) {
    const int f = f0 + threadIdx.x;
    int need = 0;
    if (f < a.forks) {
      const int s = a.src[f], t = a.dst[f];
      if (s >= 0 && s < a.batch && t >= 0 && t < a.batch && s != t && a.owner[t] == f) {
        const int n = max(a.lens[s], 0);
        need = n % a.d.page != 0 && n / a.d.page < a.max_pages;
      }
    }
    int total;
    const int r = wanted + block_scan(need, scratch, total);
    if (f < a.forks) a.fresh[f] = need ? r : -1;
    wanted += total;
  }
  int seen = 0;
  for (int p0 = 0; p0 < a.d.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const int n = p < a.d.pages ? a.refs[p] : 1;
    if (p < a.d.pages) a.refs_out[p] = n;
    int t;
    block_scan(n == 0, scratch, t);
    seen += t;
  }
  const int lacking = max(wanted - seen, 0);
  if (threadIdx.x == 0) a.missing[0] = lacking;
  if (lacking) {  // nothing is forked
    for (int b = threadIdx.x; b < a.batch; b += kPlanThreads) a.owner[b] = 0x7fffffff;
    for (int f = threadIdx.x; f < a.forks; f += kPlanThreads) a.fresh[f] = -1;
    return;
  }
  // rank -> page: fork f's rank is known, so each fork looks its page up. The ranks are
  // ascending in f; a free page of rank r goes to the fork that holds rank r.
  __syncthreads();
  seen = 0;
  for (int p0 = 0; p0 < a.d.pages && seen < wanted; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const bool is_free = p < a.d.pages && a.refs[p] == 0;
    int t;
    const int r = seen + block_scan(is_free, scratch, t);
    if (is_free && r < wanted) a.owner[a.batch + r] = p;
    seen += t;
  }
  __syncthreads();
  for (int f = threadIdx.x; f < a.forks; f += kPlanThreads)
    if (a.fresh[f] >= 0) a.fresh[f] = a.owner[a.batch + a.fresh[f]];
}

__global__ void __launch_bounds__(256) cache_fork_apply_kernel(const __grid_constant__ ForkArgs a) {
  pdl_enter();
  // tables, lengths and counts
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    const int f = a.owner[b];
    const int64_t row = (int64_t)b * a.max_pages;
    if (f == 0x7fffffff) {
      for (int i = threadIdx.x; i < a.max_pages; i += blockDim.x) a.tables_out[row + i] = a.tables[row + i];
      if (threadIdx.x == 0) a.lens_out[b] = a.lens[b];
      continue;
    }
    const int s = a.src[f], n = max(a.lens[s], 0), full = n / a.d.page, page = a.fresh[f];
    for (int i = threadIdx.x; i < a.max_pages; i += blockDim.x) {
      const int old = a.tables[row + i];
      if (old >= 0 && old < a.d.pages) atomicSub(&a.refs_out[old], 1);
      int now = -1;
      if (i < full) now = a.tables[(int64_t)s * a.max_pages + i];
      else if (i == full) now = page;
      if (now >= 0 && now < a.d.pages) atomicAdd(&a.refs_out[now], 1);
      a.tables_out[row + i] = now;
    }
    if (threadIdx.x == 0) a.lens_out[b] = a.lens[s];
  }
  // the used rows of the last pages
  const int64_t units = (int64_t)a.forks * a.d.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int f = (int)(u / (a.d.layers * 2)), x = (int)(u % (a.d.layers * 2));
    const int to = a.fresh[f];
    if (to < 0) continue;
    const int s = a.src[f], n = max(a.lens[s], 0), full = n / a.d.page;
    const int from = a.tables[(int64_t)s * a.max_pages + full];
    if (from < 0 || from >= a.d.pages) continue;
    copy_page(((x & 1) ? a.vc : a.kc) + (x >> 1) * a.c.layer, from, to, n % a.d.page, a.c, a.d);
  }
}

// ------------------------------------------------------------------ free

struct FreeArgs {
  const int *tables, *lens, *refs, *slots;
  int *tables_out, *lens_out, *refs_out;
  int batch, n_slots, max_pages, pages;
};

__global__ void __launch_bounds__(kPlanThreads) cache_free_kernel(const __grid_constant__ FreeArgs a) {
  pdl_enter();
  for (int p = threadIdx.x; p < a.pages; p += kPlanThreads) a.refs_out[p] = a.refs[p];
  for (int b = threadIdx.x; b < a.batch; b += kPlanThreads) a.lens_out[b] = max(a.lens[b], 0);
  __syncthreads();
  for (int i = threadIdx.x; i < a.n_slots; i += kPlanThreads) {
    const int b = a.slots[i];
    if (b >= 0 && b < a.batch) a.lens_out[b] = -1;  // marks the slot until the end
  }
  __syncthreads();
  for (int64_t i = threadIdx.x; i < (int64_t)a.batch * a.max_pages; i += kPlanThreads) {
    const int b = (int)(i / a.max_pages), p = a.tables[i];
    const bool gone = a.lens_out[b] == -1;
    if (gone && p >= 0 && p < a.pages) atomicSub(&a.refs_out[p], 1);
    a.tables_out[i] = gone ? -1 : p;
  }
  __syncthreads();
  for (int b = threadIdx.x; b < a.batch; b += kPlanThreads) a.lens_out[b] = max(a.lens_out[b], 0);
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
};

__global__ void __launch_bounds__(kPlanThreads) cache_compact_plan_kernel(const __grid_constant__ CompactArgs a) {
  __shared__ int scratch[33];
  pdl_enter();
  int live = 0;
  for (int p0 = 0; p0 < a.d.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    int t;
    block_scan(p < a.d.pages && a.refs[p] > 0, scratch, t);
    live += t;
  }
  // live pages from index `live` on move, in order, into the holes below it
  int holes = 0, movers = 0;
  for (int p0 = 0; p0 < a.d.pages; p0 += kPlanThreads) {
    const int p = p0 + threadIdx.x;
    const int n = p < a.d.pages ? a.refs[p] : 0;
    const bool hole = p < live && n <= 0, mover = p >= live && n > 0;
    int t;
    const int x = block_scan((hole ? 1 : 0), scratch, t);
    if (hole) a.go[holes + x] = p;
    holes += t;
    const int y = block_scan((mover ? 1 : 0), scratch, t);
    if (mover) a.come[movers + y] = p;
    movers += t;
    if (p < a.d.pages) {
      a.place[p] = p;
      a.refs_out[p] = p < live && n > 0 ? n : 0;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) a.moves[0] = movers;
  for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
    a.place[a.come[i]] = a.go[i];
    a.refs_out[a.go[i]] = a.refs[a.come[i]];
  }
}

__global__ void __launch_bounds__(256) cache_compact_apply_kernel(const __grid_constant__ CompactArgs a) {
  pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < a.entries; i += (int64_t)gridDim.x * blockDim.x) {
    const int p = a.tables[i];
    a.tables_out[i] = p >= 0 && p < a.d.pages ? a.place[p] : p;
  }
  const int64_t units = (int64_t)a.moves[0] * a.d.layers * 2;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int i = (int)(u / (a.d.layers * 2)), x = (int)(u % (a.d.layers * 2));
    copy_page(((x & 1) ? a.vc : a.kc) + (x >> 1) * a.c.layer, a.come[i], a.go[i], a.d.page, a.c, a.d);
  }
}

// ------------------------------------------------------------------ host

constexpr int64_t kMaxInt = 0x7fffffffLL;

size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

// Checks and converts the cache's description; strides (elements) are layer, page, head, slot.
int cache_dims(const char* op, const void* kc, const void* vc, const int64_t* strides, int64_t layers, int64_t pages,
               int64_t kv_heads, int64_t page_size, int64_t head_dim, int dtype, CacheDims* d, CacheLayout* c) {
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (layers < 1 || pages < 1 || kv_heads < 1 || page_size < 1 || head_dim < 1)
    return fail(NKL_ERR_SHAPE, "%s: layers, pages, heads, page size and head_dim must be positive", op);
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
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

int check_table(const char* op, int64_t batch, int64_t max_pages) {
  if (batch < 0 || max_pages < 1) return fail(NKL_ERR_SHAPE, "%s: batch must not be negative, tables need a column", op);
  if (batch > kMaxInt / 4 || max_pages > kMaxInt / 4 || batch * max_pages > kMaxInt)
    return fail(NKL_ERR_SHAPE, "%s: tables too large", op);
  return NKL_OK;
}

unsigned grid_for(int64_t blocks, int per_sm) {
  return (unsigned)std::max<int64_t>(1, std::min<int64_t>(blocks, (int64_t)sm_count() * per_sm));
}

}  // namespace
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
  const int64_t total = layers * batch * tokens * kv_heads * a.d.vecs;
  return launch_pdl(cache_append_kernel, dim3(grid_for((std::max(total, batch) + 255) / 256, 8)), dim3(256), 0,
                    static_cast<cudaStream_t>(stream), op, a);
}

extern "C" size_t nkl_cache_reserve_workspace_size(int64_t batch) {
  return batch > 0 ? round256((size_t)batch * 8) : 0;
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
  ReserveArgs a = {tables,     lens,       refs,       extra,
                   tables_out, refs_out,   missing,    static_cast<int*>(workspace),
                   static_cast<int*>(workspace) + batch, (int)batch, (int)max_pages, (int)pages, (int)page_size};
  return launch_pdl(cache_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), op, a);
}

extern "C" size_t nkl_cache_fork_workspace_size(int64_t batch, int64_t forks) {
  return batch > 0 && forks >= 0 ? round256(((size_t)batch + 2 * (size_t)forks) * 4) : 0;
}

extern "C" int nkl_cache_fork(void* k_cache, void* v_cache, const int64_t* cache_strides, const int32_t* tables,
                              const int32_t* lens, const int32_t* refs, const int32_t* src, const int32_t* dst,
                              int32_t* tables_out, int32_t* lens_out, int32_t* refs_out, int32_t* missing,
                              void* workspace, size_t workspace_bytes, int64_t forks, int64_t layers, int64_t batch,
                              int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size,
                              int64_t max_pages, int dtype, void* stream) {
  const char* op = "nkl_cache_fork";
  ForkArgs a = {};
  int rc = cache_dims(op, k_cache, v_cache, cache_strides, layers, pages, kv_heads, page_size, head_dim, dtype, &a.d,
                      &a.c);
  if (rc) return rc;
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
  a.owner = static_cast<int*>(workspace);  // [batch], then [forks] pages by rank
  a.fresh = a.owner + batch + forks;
  a.kc = static_cast<uint4*>(k_cache);
  a.vc = static_cast<uint4*>(v_cache);
  a.batch = (int)batch;
  a.forks = (int)forks;
  a.max_pages = (int)max_pages;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  rc = launch_pdl(cache_fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, op, a);
  if (rc) return rc;
  return launch_pdl(cache_fork_apply_kernel, dim3(grid_for(std::max(batch, forks * layers * 2), 8)), dim3(256), 0, st,
                    op, a);
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
  return launch_pdl(cache_free_kernel, dim3(1), dim3(kPlanThreads), 0, static_cast<cudaStream_t>(stream), op, a);
}

extern "C" size_t nkl_cache_compact_workspace_size(int64_t pages) {
  return pages > 0 ? round256(((size_t)pages * 3 + 1) * 4) : 0;
}

extern "C" int nkl_cache_compact(void* k_cache, void* v_cache, const int64_t* cache_strides, const int32_t* tables,
                                 const int32_t* refs, int32_t* tables_out, int32_t* refs_out, void* workspace,
                                 size_t workspace_bytes, int64_t layers, int64_t batch, int64_t kv_heads,
                                 int64_t head_dim, int64_t pages, int64_t page_size, int64_t max_pages, int dtype,
                                 void* stream) {
  const char* op = "nkl_cache_compact";
  CompactArgs a = {};
  int rc = cache_dims(op, k_cache, v_cache, cache_strides, layers, pages, kv_heads, page_size, head_dim, dtype, &a.d,
                      &a.c);
  if (rc) return rc;
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
  rc = launch_pdl(cache_compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, op, a);
  if (rc) return rc;
  return launch_pdl(cache_compact_apply_kernel,
                    dim3(grid_for(std::max<int64_t>((a.entries + 255) / 256, pages * layers * 2), 8)), dim3(256), 0,
                    st, op, a);
}
