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
// lane x scores key x of a 32-key tile and then accumulates 4 columns. Key ranges split over
// several blocks leave (max, sum, O) in the workspace; tree_combine_kernel joins them in order.
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

template <typename T>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  __shared__ __align__(16) float qs[kRows][kMaxDim];
  __shared__ __align__(16) float ks[kKeys][kMaxDim + 4];
  __shared__ __align__(16) float vs[kKeys][kMaxDim];
  __shared__ __align__(16) float ps[kRows][kKeys];
  __shared__ int64_t base[kKeys];
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int split = blockIdx.x / a.row_blocks, r0 = (blockIdx.x % a.row_blocks) * kRows;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = a.tokens * a.group, quads = a.d / 4;
  const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
  // this block's tiles: a share of the cached ones, and the drafted ones in the last split
  const int tiles = (n + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);
  const int new_tiles = split == a.splits - 1 ? (a.tokens + kKeys - 1) / kKeys : 0;

  const T* q = static_cast<const T*>(a.q) + b * a.q_b;
  for (int i = tid; i < kRows * quads; i += kThreads) {
    const int r = i / quads, c = (i - r * quads) * 4, row = r0 + r;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) x = load4<T>(q + (row / a.group) * a.q_t + (kvh * a.group + row % a.group) * a.q_h + c);
    *reinterpret_cast<float4*>(&qs[r][c]) = x;
  }
  uint32_t seen[4][4];  // drafted tokens visible to each of the warp's rows
  bool here[4];
  float m[4], l[4];
  float4 o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + warp * 4 + i;
    seen[i][0] = seen[i][1] = seen[i][2] = seen[i][3] = 0u;
    if (row < rows) ancestor_bits(a.parents ? a.parents + (int64_t)b * a.tokens : nullptr, row / a.group, seen[i]);
    here[i] = (seen[i][0] | seen[i][1] | seen[i][2] | seen[i][3]) != 0u;
    m[i] = -INFINITY;
    l[i] = 0.f;
    o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }

  for (int t = t0; t < t1 + new_tiles; ++t) {
    const bool cached = t < t1;
    const int key0 = (cached ? t : t - t1) * kKeys;
    __syncthreads();
    if (tid < kKeys) {
      int64_t at = -1;
      const int key = key0 + tid;
      if (!cached) {
        if (key < a.tokens) at = b * a.n_b + key * a.n_t + kvh * a.n_h;
      } else if (key < n) {
        const int p = a.tables[(int64_t)b * a.max_pages + key / a.page];
        if (p >= 0 && p < a.pages) at = p * a.c_p + kvh * a.c_h + (key % a.page) * a.c_s;
      }
      base[tid] = at;
    }
    __syncthreads();
    const T* kp = static_cast<const T*>(cached ? a.k_cache : a.k_new);
    const T* vp = static_cast<const T*>(cached ? a.v_cache : a.v_new);
    for (int i = tid; i < kKeys * quads; i += kThreads) {
      const int r = i / quads, c = (i - r * quads) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
      if (base[r] >= 0) {
        x = load4<T>(kp + base[r] + c);
        y = load4<T>(vp + base[r] + c);
      }
      *reinterpret_cast<float4*>(&ks[r][c]) = x;
      *reinterpret_cast<float4*>(&vs[r][c]) = y;
    }
    __syncthreads();
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (int c = 0; c < a.d; c += 4) {
      const float4 kx = *reinterpret_cast<const float4*>(&ks[lane][c]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 qx = *reinterpret_cast<const float4*>(&qs[warp * 4 + i][c]);
        s[i] = fmaf(qx.x, kx.x, fmaf(qx.y, kx.y, fmaf(qx.z, kx.z, fmaf(qx.w, kx.w, s[i]))));
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      bool sees = here[i];
      if (cached) sees &= key0 + lane < n;
      else sees &= (seen[i][(key0 >> 5) & 3] >> lane) & 1u;
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
    if (lane < quads && !cached) {
      // a drafted token that a row does not see leaves no trace in it, whatever its v holds
      for (int x = 0; x < kKeys && key0 + x < a.tokens; ++x) {
        const float4 v = *reinterpret_cast<const float4*>(&vs[x][lane * 4]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (!((seen[i][(key0 >> 5) & 3] >> x) & 1u)) continue;
          const float pk = ps[warp * 4 + i][x];
          o[i].x = fmaf(pk, v.x, o[i].x);
          o[i].y = fmaf(pk, v.y, o[i].y);
          o[i].z = fmaf(pk, v.z, o[i].z);
          o[i].w = fmaf(pk, v.w, o[i].w);
        }
      }
    } else if (lane < quads) {
      for (int x = 0; x < kKeys; x += 4) {
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = *reinterpret_cast<const float4*>(&vs[x + k][lane * 4]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float4 p = *reinterpret_cast<const float4*>(&ps[warp * 4 + i][x]);
          const float pk[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            o[i].x = fmaf(pk[k], v[k].x, o[i].x);
            o[i].y = fmaf(pk[k], v[k].y, o[i].y);
            o[i].z = fmaf(pk[k], v[k].z, o[i].z);
            o[i].w = fmaf(pk[k], v[k].w, o[i].w);
          }
        }
      }
    }
  }

#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = r0 + warp * 4 + i;
    if (row >= rows) continue;
    if (a.splits == 1) {
      const float inv = here[i] ? 1.f / l[i] : 0.f;  // an absent token's row is zero
      const int64_t at = (((int64_t)b * a.tokens + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d;
      if (lane < quads)
        store4(static_cast<T*>(a.out) + at + lane * 4, make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv));
    } else {
      const int64_t at = (((int64_t)split * a.batch + b) * a.kv_heads + kvh) * rows + row;
      if (lane < quads) store4(a.ws_o + at * a.d + lane * 4, o[i]);
      if (lane == 0) {
        a.ws_ml[2 * at] = m[i];
        a.ws_ml[2 * at + 1] = l[i];
      }
    }
  }
}

// Joins the splits of each row, in split order: one warp per row, lane = 4 columns.
template <typename T>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ TreeArgs a) {
  pdl_enter();
  const int rows = a.tokens * a.group, lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5), all = (int64_t)a.batch * a.kv_heads * rows;
  if (row >= all) return;
  const int r = (int)(row % rows), kvh = (int)(row / rows % a.kv_heads), b = (int)(row / rows / a.kv_heads);
  float m = -INFINITY;
  for (int s = lane; s < a.splits; s += 32) m = fmaxf(m, a.ws_ml[2 * (s * all + row)]);
  m = warp_max(m);
  float l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (m != -INFINITY) {
    for (int s = 0; s < a.splits; ++s) {
      const int64_t at = s * all + row;
      const float w = expf(a.ws_ml[2 * at] - m);
      if (w == 0.f) continue;
      l = fmaf(w, a.ws_ml[2 * at + 1], l);
      if (lane * 4 < a.d) {
        const float4 x = load4<float>(a.ws_o + at * a.d + lane * 4);
        o.x = fmaf(w, x.x, o.x);
        o.y = fmaf(w, x.y, o.y);
        o.z = fmaf(w, x.z, o.z);
        o.w = fmaf(w, x.w, o.w);
      }
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  const int64_t at = (((int64_t)b * a.tokens + r / a.group) * a.heads + kvh * a.group + r % a.group) * a.d;
  if (lane * 4 < a.d)
    store4(static_cast<T*>(a.out) + at + lane * 4, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

}  // namespace

#include "tree_attention_tc.cuh"

namespace {

// ------------------------------------------------------------------ host

// Blocks that share a sequence's keys: enough of them to give every SM a few, each with at
// least 64 keys of the longest sequence that the tables can hold.
int split_count(int64_t batch, int64_t kv_heads, int64_t row_blocks, int64_t capacity) {
  const int64_t blocks = batch * kv_heads * row_blocks;
  const int64_t want = (3 * (int64_t)sm_count() + blocks - 1) / std::max<int64_t>(blocks, 1);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, (capacity + 63) / 64, 256}));
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
  int rc = dtype == NKL_FLOAT32 ? launch_pdl(tree_attention_kernel<float>, grid, dim3(kThreads), 0, st, op, a)
                                : launch_pdl(tree_attention_kernel<bf16>, grid, dim3(kThreads), 0, st, op, a);
  if (rc || a.splits == 1) return rc;
  const int64_t rows = batch * heads * tokens;
  const dim3 join((unsigned)((rows + 3) / 4));
  return dtype == NKL_FLOAT32 ? launch_pdl(tree_combine_kernel<float>, join, dim3(128), 0, st, op, a)
                              : launch_pdl(tree_combine_kernel<bf16>, join, dim3(128), 0, st, op, a);
}
