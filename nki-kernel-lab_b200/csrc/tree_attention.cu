// tree_attention.cu - attention of drafted tokens over a paged key/value cache.
//
// Sequence b has lens[b] cached positions, whose k and v lie in pages that tables[b] lists,
// and T drafted tokens that form a tree (parents; NULL: a chain). Drafted token i attends to
// every cached position, to itself and to its ancestors:
//   out[b, i, h] = sum_x softmax_x(scale * q[b, i, h] . k_x) v_x
// Query heads share key/value heads (G = heads / kv_heads), so the T * G query rows of a
// key/value head meet each key together: the cache is read once per G * T rows.
//
// CUDA-core kernel (fp32, and bf16 layouts that the tensor-core kernel does not take): a block
// owns 16 query rows of one key/value head and one range of the keys; each warp has 4 rows,
// lane x scores key x of a 32-key tile and then accumulates 4 columns; two tiles are on their
// way (cp.async) while one is worked on. Key ranges split over several blocks leave (max, sum, O)
// in the workspace; tree_combine_kernel joins them in order.
#include <algorithm>
#include <atomic>

#include "attn_math.cuh"
#include "common.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace nkl {
namespace {

constexpr int kMaxDrafted = NKL_MAX_DRAFTED;
constexpr int kRows = 16;
constexpr int kKeys = 32;
constexpr int kThreads = 128;
constexpr int kMaxDim = 128;

struct TreeArgs {
  const void *q, *k_new, *v_new, *k_cache, *v_cache;
  const int *tables, *lens, *parents;
  void* out;
  float* ws_o;    // [split][batch][kv_heads][rows][d]
  float* ws_ml;   // [split][batch][kv_heads][rows][2]
  int64_t q_b, q_t, q_h, n_b, n_t, n_h, c_p, c_h, c_s;  // strides in elements
  int batch, tokens, heads, kv_heads, group, d, pages, page, max_pages, splits, row_blocks;
  float scale;
};

// The four words of token i's visible drafted tokens; all zero for an absent token.
__device__ __forceinline__ void ancestor_bits(const int* parents, int i, uint32_t (&w)[4]) {
  w[0] = w[1] = w[2] = w[3] = 0u;
  if (!parents) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int left = i + 1 - 32 * k;
      w[k] = left >= 32 ? 0xffffffffu : left > 0 ? (1u << left) - 1u : 0u;
    }
    return;
  }
  int up = parents[i];
  if (up < -1) return;
  for (int at = i;;) {
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] |= (at >> 5) == k ? 1u << (at & 31) : 0u;
    if (up < 0 || up >= at) return;  // the root, or no earlier token: treated as the root
    at = up;
    up = parents[at];
    if (up < -1) return;  // the parent is absent
  }
}

template <typename T> __device__ __forceinline__ float4 load4(const T* p);
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <> __device__ __forceinline__ float4 load4<bf16>(const bf16* p) {
  const uint2 r = *reinterpret_cast<const uint2*>(p);
  const float2 a = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.x));
  const float2 b = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&r.y));
  return make_float4(a.x, a.y, b.x, b.y);
}

__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(bf16* p, float4 v) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// 16 bytes from global to shared memory, zeros where `from` is null.
__device__ __forceinline__ void copy16_async(void* to, const void* from, const void* any) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to), size = from ? 16u : 0u;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at), "l"(from ? from : any), "r"(size) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory: queries in fp32, and two tiles of keys and values as they come; a key row is
// 16 bytes longer than its data, so that 32 lanes reading a row each do not collide.
template <typename T>
size_t tree_smem(int d) {
  return (size_t)kRows * d * 4 + 2 * (size_t)kKeys * (2 * d * sizeof(T) + 16);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int VE = Vec16<T>::N;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ __align__(16) float ps[kRows][kKeys];
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x / a.row_blocks, r0 = (blockIdx.x % a.row_blocks) * kRows;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = a.tokens * a.group, quads = a.d / 4, chunks = a.d / VE, pitch = a.d + VE;
  float* const qs = reinterpret_cast<float*>(smem);
  T* const ring = reinterpret_cast<T*>(smem + (size_t)kRows * a.d * 4);
  const int stage_size = kKeys * (pitch + a.d);
  const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
  // this block's tiles: a share of the cached ones, and the drafted ones in the last split
  const int tiles = (n + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);
  const int end = t1 + (split == a.splits - 1 ? (a.tokens + kKeys - 1) / kKeys : 0);

  const float per_row = 1.f / (float)chunks;
  auto fetch = [&](int t) {  // tile t into its place of the ring
    if (t < end) {
      const bool cached = t < t1;
      const int key0 = (cached ? t : t - t1) * kKeys;
      const T* const kp = static_cast<const T*>(cached ? a.k_cache : a.k_new);
      const T* const vp = static_cast<const T*>(cached ? a.v_cache : a.v_new);
      T* const ks = ring + (t & 1) * stage_size;
      T* const vs = ks + kKeys * pitch;
      for (int i = tid; i < kKeys * chunks; i += kThreads) {
        const int r = (int)(((float)i + 0.5f) * per_row), c = (i - r * chunks) * VE, key = key0 + r;  // r = i / chunks
        int64_t at = -1;
        if (!cached) {
          if (key < a.tokens) at = b * a.n_b + key * a.n_t + kvh * a.n_h + c;
        } else if (key < n) {
          const int pi = key / a.page, p = a.tables[(int64_t)b * a.max_pages + pi];
          if (p >= 0 && p < a.pages) at = p * a.c_p + kvh * a.c_h + (key - pi * a.page) * a.c_s + c;
        }
        copy16_async(ks + r * pitch + c, at >= 0 ? kp + at : nullptr, kp);
        copy16_async(vs + r * a.d + c, at >= 0 ? vp + at : nullptr, vp);
      }
    }
    copies_commit();  // also where there is nothing: the count of groups goes on
  };
  fetch(t0);
  fetch(t0 + 1);

  const T* q = static_cast<const T*>(a.q) + b * a.q_b;
  for (int i = tid; i < kRows * quads; i += kThreads) {
    const int r = i / quads, c = (i - r * quads) * 4, row = r0 + r;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) x = load4<T>(q + (row / a.group) * a.q_t + (kvh * a.group + row % a.group) * a.q_h + c);
    *reinterpret_cast<float4*>(qs + r * a.d + c) = x;
  }
  const int* const parents = a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  uint32_t seen[4][4];  // drafted tokens visible to each of the warp's rows
  bool here[4];
  float m[4], l[4];
  float4 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + warp * 4 + i;
    const int token = row / a.group;
    here[i] = row < rows && (!parents || parents[token] >= -1);
    seen[i][0] = seen[i][1] = seen[i][2] = seen[i][3] = 0u;
    if (here[i] && end > t1) ancestor_bits(parents, token, seen[i]);
    m[i] = -INFINITY;
    l[i] = 0.f;
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // With head_dim up to 64 the warp's halves take the columns twice, for every second key each.
  const bool halves = quads <= 16;
  const int col = (halves ? lane & 15 : lane) * 4, key_of = halves ? lane >> 4 : 0, key_step = halves ? 2 : 1;

  for (int t = t0; t < end; ++t) {
    const bool cached = t < t1;
    const int key0 = (cached ? t : t - t1) * kKeys;
    const T* const ks = ring + (t & 1) * stage_size;
    const T* const vs = ks + kKeys * pitch;
    copies_wait<1>();
    __syncthreads();
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = 0; c < a.d; c += 4) {
      const float4 kx = load4<T>(ks + lane * pitch + c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 qx = *reinterpret_cast<const float4*>(qs + (warp * 4 + i) * a.d + c);
        s[i] = fmaf(qx.x, kx.x, fmaf(qx.y, kx.y, fmaf(qx.z, kx.z, fmaf(qx.w, kx.w, s[i]))));
      }
    }
    const int word = (key0 >> 5) & 3;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t drafts = word == 0 ? seen[i][0] : word == 1 ? seen[i][1] : word == 2 ? seen[i][2] : seen[i][3];
      const bool sees = here[i] && (cached ? key0 + lane < n : ((drafts >> lane) & 1u) != 0u);
      const float x = sees ? s[i] * a.scale : -INFINITY;
      const float top = fmaxf(m[i], warp_max(x));
      const float ref = top == -INFINITY ? 0.f : top;  // nothing seen so far
      const float p = sees ? expf(x - ref) : 0.f;
      const float keep = expf(m[i] - ref);
      l[i] = l[i] * keep + warp_sum(p);
      o[i].x *= keep; o[i].y *= keep; o[i].z *= keep; o[i].w *= keep;
      m[i] = top;
      ps[warp * 4 + i][lane] = p;
    }
    __syncwarp();
    if (col < a.d && cached) {
#pragma unroll 4
      for (int x = key_of; x < kKeys; x += key_step) {
        const float4 v = load4<T>(vs + x * a.d + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = ps[warp * 4 + i][x];
          o[i].x = fmaf(p, v.x, o[i].x);
          o[i].y = fmaf(p, v.y, o[i].y);
          o[i].z = fmaf(p, v.z, o[i].z);
          o[i].w = fmaf(p, v.w, o[i].w);
        }
      }
    } else if (col < a.d) {
      // a drafted token that a row does not see leaves no trace in it, whatever its v holds
      for (int x = key_of; x < kKeys && key0 + x < a.tokens; x += key_step) {
        const float4 v = load4<T>(vs + x * a.d + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t drafts = word == 0 ? seen[i][0] : word == 1 ? seen[i][1] : word == 2 ? seen[i][2] : seen[i][3];
          if (!((drafts >> x) & 1u)) continue;
          const float p = ps[warp * 4 + i][x];
          o[i].x = fmaf(p, v.x, o[i].x);
          o[i].y = fmaf(p, v.y, o[i].y);
          o[i].z = fmaf(p, v.z, o[i].z);
          o[i].w = fmaf(p, v.w, o[i].w);
        }
      }
    }
    __syncthreads();  // every warp is through with this tile's place
    fetch(t + 2);
  }
  copies_wait<0>();

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (halves) {
      o[i].x += __shfl_xor_sync(0xffffffffu, o[i].x, 16);
      o[i].y += __shfl_xor_sync(0xffffffffu, o[i].y, 16);
      o[i].z += __shfl_xor_sync(0xffffffffu, o[i].z, 16);
      o[i].w += __shfl_xor_sync(0xffffffffu, o[i].w, 16);
    }
    const int row = r0 + warp * 4 + i;
    if (row >= rows) continue;
    if (a.splits == 1) {
      const float inv = here[i] ? 1.f / l[i] : 0.f;  // an absent token's row is zero
      const int64_t at = (((int64_t)b * a.tokens + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d;
      if (key_of == 0 && col < a.d)
        store4(static_cast<T*>(a.out) + at + col, make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv));
    } else {
      const int64_t at = (((int64_t)split * a.batch + b) * a.kv_heads + kvh) * rows + row;
      if (key_of == 0 && col < a.d) store4(a.ws_o + at * a.d + col, o[i]);
      if (lane == 0) {
        a.ws_ml[2 * at] = m[i];
        a.ws_ml[2 * at + 1] = l[i];
      }
    }
  }
}

constexpr int kMaxSplits = 256;

// Joins the splits of each row, in split order: one warp per row, lane = 4 columns.
template <typename T>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ TreeArgs a) {
  __shared__ float weight[4][kMaxSplits];
  pdl_enter();
  const int rows = a.tokens * a.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 4 + warp, all = (int64_t)a.batch * a.kv_heads * rows;
  if (row >= all) return;
  const int r = (int)(row % rows), kvh = (int)(row / rows % a.kv_heads), b = (int)(row / rows / a.kv_heads);
  const float2* const ml = reinterpret_cast<const float2*>(a.ws_ml) + row;
  float m = -INFINITY, l = 0.f;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, ml[s * all].x);
  m = warp_max(m);
  for (int s = lane; s < a.splits; s += 32) {
    const float2 x = ml[s * all];
    const float w = x.x == -INFINITY ? 0.f : expf(x.x - m);
    weight[warp][s] = w;
    l = fmaf(w, x.y, l);
  }
  l = warp_sum(l);
  __syncwarp();
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (lane * 4 < a.d) {
    const float* const po = a.ws_o + row * a.d + lane * 4;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
      const float w = weight[warp][s];
      const float4 x = load4<float>(po + s * all * a.d);
      o.x = fmaf(w, x.x, o.x);
      o.y = fmaf(w, x.y, o.y);
      o.z = fmaf(w, x.z, o.z);
      o.w = fmaf(w, x.w, o.w);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;  // 0: an absent token
  const int64_t at = (((int64_t)b * a.tokens + r / a.group) * a.heads + kvh * a.group + r % a.group) * a.d;
  if (lane * 4 < a.d)
    store4(static_cast<T*>(a.out) + at + lane * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

}  // namespace

#include "tree_attention_tc.cuh"

namespace {

// ------------------------------------------------------------------ host

// Blocks that share a sequence's keys: up to four for each SM, each with at least 64 keys, the
// two tiles it has on their way at once, of the longest sequence that the tables can hold.
int split_count(int64_t batch, int64_t kv_heads, int64_t row_blocks, int64_t capacity) {
  const int64_t blocks = batch * kv_heads * row_blocks;
  const int64_t want = (4 * (int64_t)sm_count() + blocks - 1) / std::max<int64_t>(blocks, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (capacity + 63) / 64, kMaxSplits}));
}

// Allows a kernel more than 48 KB of shared memory, once per device.
template <typename K>
int allow_smem(K* kernel, size_t bytes, const char* op) {
  static std::atomic<bool> set[64] = {};  // idempotent
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && set[dev].load(std::memory_order_acquire)) return NKL_OK;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
  if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  return NKL_OK;
}

size_t split_bytes(int64_t splits, int64_t batch, int64_t heads, int64_t tokens, int64_t d) {
  return splits > 1 ? ((size_t)splits * batch * heads * tokens * (d + 2) * 4 + 255) & ~size_t(255) : 0;
}

bool tree_sizes_ok(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t page_size,
                   int64_t max_pages) {
  return batch >= 0 && batch <= 65535 && tokens >= 0 && tokens <= kMaxDrafted && heads >= 1 && heads <= 65535 &&
         kv_heads >= 1 && heads % kv_heads == 0 && head_dim >= 8 && head_dim <= kMaxDim && head_dim % 8 == 0 &&
         page_size >= 1 && page_size <= 65536 && max_pages >= 1 && max_pages * page_size <= (1LL << 30);
}

}  // namespace

int tree_read_and_clear_device_error() {
  unsigned int v = 0, zero = 0;
  if (cudaMemcpyFromSymbol(&v, g_tree_dev_error, sizeof(v)) != cudaSuccess) return -1;
  if (v && cudaMemcpyToSymbol(g_tree_dev_error, &zero, sizeof(zero)) != cudaSuccess) return -1;
  return (int)v;
}

}  // namespace nkl

using namespace nkl;

extern "C" size_t nkl_attention_tree_workspace_size(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                    int64_t head_dim, int64_t page_size, int64_t max_pages,
                                                    int dtype) {
  if (!valid_dtype(dtype) || !tree_sizes_ok(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages) ||
      batch == 0 || tokens == 0)
    return 0;
  // strides and the scale's sign, which are not known here, may still choose the CUDA-core kernel
  const TcPlan p = tc_plan(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages, dtype);
  const int64_t row_blocks = (tokens * (heads / kv_heads) + kRows - 1) / kRows;
  return std::max(p.on ? p.bytes : 0, split_bytes(split_count(batch, kv_heads, row_blocks, page_size * max_pages),
                                                  batch, heads, tokens, head_dim));
}

extern "C" int nkl_attention_tree(const void* q, const int64_t* q_strides, const void* k_new, const void* v_new,
                                  const int64_t* new_strides, const void* k_cache, const void* v_cache,
                                  const int64_t* cache_strides, const int32_t* tables, const int32_t* lens,
                                  const int32_t* parents, void* out, void* workspace, size_t workspace_bytes,
                                  int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                  int64_t pages, int64_t page_size, int64_t max_pages, float scale, int dtype,
                                  void* stream) {
  const char* op = "nkl_attention_tree";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (tokens > kMaxDrafted)
    return fail(NKL_ERR_SHAPE, "%s: %lld drafted tokens, at most %d are taken", op, (long long)tokens, kMaxDrafted);
  if (!tree_sizes_ok(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages) || pages < 1 ||
      pages > 0x7fffffffLL)
    return fail(NKL_ERR_SHAPE,
                "%s: batch %lld, tokens %lld, heads %lld / %lld, head_dim %lld, page size %lld or table width %lld not "
                "supported (kv heads divide heads; head_dim a multiple of 8 up to %d; up to 2^30 positions)",
                op, (long long)batch, (long long)tokens, (long long)heads, (long long)kv_heads, (long long)head_dim,
                (long long)page_size, (long long)max_pages, kMaxDim);
  if (batch == 0 || tokens == 0) return NKL_OK;
  if (!q || !k_new || !v_new || !k_cache || !v_cache || !tables || !lens || !out)
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  for (const void* p : {q, k_new, v_new, k_cache, v_cache, static_cast<const void*>(out)})
    if (!is_aligned(p, 16)) return fail(NKL_ERR_ALIGN, "%s: tensors need 16-byte alignment", op);
  TreeArgs a = {};
  int64_t s[9] = {tokens * heads * head_dim,    heads * head_dim,                 head_dim,
                  tokens * kv_heads * head_dim, kv_heads * head_dim,              head_dim,
                  kv_heads * page_size * head_dim, page_size * head_dim, head_dim};
  const int64_t n[9] = {batch, tokens, heads, batch, tokens, kv_heads, pages, kv_heads, page_size};
  const int64_t* given[3] = {q_strides, new_strides, cache_strides};
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  for (int i = 0; i < 9; ++i) {
    if (given[i / 3]) s[i] = given[i / 3][i % 3];
    if (n[i] > 1 && (s[i] < 0 || s[i] % per))
      return fail(NKL_ERR_ALIGN, "%s: stride %lld is not a multiple of 16 bytes", op, (long long)s[i]);
  }
  a.q = q; a.k_new = k_new; a.v_new = v_new; a.k_cache = k_cache; a.v_cache = v_cache;
  a.tables = tables; a.lens = lens; a.parents = parents; a.out = out;
  a.q_b = s[0]; a.q_t = s[1]; a.q_h = s[2];
  a.n_b = s[3]; a.n_t = s[4]; a.n_h = s[5];
  a.c_p = s[6]; a.c_h = s[7]; a.c_s = s[8];
  a.batch = (int)batch; a.tokens = (int)tokens; a.heads = (int)heads; a.kv_heads = (int)kv_heads;
  a.group = (int)(heads / kv_heads); a.d = (int)head_dim; a.pages = (int)pages; a.page = (int)page_size;
  a.max_pages = (int)max_pages; a.scale = scale;
  const TcPlan p = tc_plan(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages, dtype);
  bool tc = p.on && scale > 0.f && scale < INFINITY;  // the running maximum is one of scaled scores
  for (int i = 0; i < 9; ++i) tc = tc && (n[i] == 1 || (s[i] > 0 && s[i] < (1LL << 38)));  // tensor map strides
  if (tc) {
    if (p.bytes) {
      if (!workspace || workspace_bytes < p.bytes) return fail(NKL_ERR_ARG, "%s: workspace too small", op);
      if (!is_aligned(workspace, 256)) return fail(NKL_ERR_ALIGN, "%s: workspace not 256-byte aligned", op);
    }
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    cudaStream_t on = static_cast<cudaStream_t>(stream);
    // a dimension of one position is never stepped over, but its stride still has to be a valid one
    int64_t* const steps[9] = {&a.q_b, &a.q_t, &a.q_h, &a.n_b, &a.n_t, &a.n_h, &a.c_p, &a.c_h, &a.c_s};
    for (int i = 0; i < 9; ++i)
      if (n[i] == 1) *steps[i] = head_dim;
    if (head_dim == 128) return p.nq == 1 ? tc_launch<128, 1>(a, p, ws, on) : tc_launch<128, 2>(a, p, ws, on);
    return p.nq == 1 ? tc_launch<64, 1>(a, p, ws, on) : tc_launch<64, 2>(a, p, ws, on);
  }
  a.row_blocks = (int)((tokens * a.group + kRows - 1) / kRows);
  a.splits = split_count(batch, kv_heads, a.row_blocks, page_size * max_pages);
  const size_t need = split_bytes(a.splits, batch, heads, tokens, head_dim);
  if (need) {
    if (!workspace || workspace_bytes < need) return fail(NKL_ERR_ARG, "%s: workspace too small", op);
    if (!is_aligned(workspace, 256)) return fail(NKL_ERR_ALIGN, "%s: workspace not 256-byte aligned", op);
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = a.ws_o + (size_t)a.splits * batch * heads * tokens * head_dim;
  }
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)(a.splits * a.row_blocks), (unsigned)kv_heads, (unsigned)batch);
  int rc;
  if (dtype == NKL_FLOAT32) {
    rc = allow_smem(tree_attention_kernel<float>, tree_smem<float>(kMaxDim), op);
    if (!rc) rc = launch_pdl(tree_attention_kernel<float>, grid, dim3(kThreads), tree_smem<float>((int)head_dim), st, op, a);
  } else {
    rc = launch_pdl(tree_attention_kernel<bf16>, grid, dim3(kThreads), tree_smem<bf16>((int)head_dim), st, op, a);
  }
  if (rc || a.splits == 1) return rc;
  const int64_t rows = batch * heads * tokens;
  const dim3 join((unsigned)((rows + 3) / 4));
  return dtype == NKL_FLOAT32 ? launch_pdl(tree_combine_kernel<float>, join, dim3(128), 0, st, op, a)
                              : launch_pdl(tree_combine_kernel<bf16>, join, dim3(128), 0, st, op, a);
}
