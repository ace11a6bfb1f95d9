// tree_attention.cu - attention of drafted tokens over a paged key/value cache.
//
// Sequence b has lens[b] cached positions, whose k and v lie in pages that tables[b] lists,
// and T drafted tokens that form a tree (parents; NULL: a chain). Drafted token i attends to
// every cached position, to itself and to its ancestors:
//   out[b, i, h] = sum_x softmax_x(scale * q[b, i, h] . k_x) v_x
// Query heads share key/value heads (G = heads / kv_heads), so the T * G query rows of a
// key/value head meet each key together: the cache is read once per G * T rows.
//
// fp32, and bf16 layouts that the tcgen05 kernel does not take: a block owns 16 query rows of
// one key/value head and one range of the keys, in tiles of 32, two of them on their way
// (cp.async) while one is worked on. Each of its four warps takes 8 keys of every tile, with a
// maximum, sum and O of its own, and multiplies with mma.sync m16n8k8 in tf32, a tile of rows as
// high as the block's. Values are split as x = hi + lo, both tf32, and three of the four products
// summed (lo lo is 2^-22 of the result), which keeps fp32's accuracy. A tile of head_dim 64 takes
// four blocks of an SM 3200 cycles, against 5500 with fp32 multiply-adds, which the many
// instructions around them bound; now the products do (16 cycles each on a quarter of an SM, 192 of
// them for each quarter). bf16 values are tf32 values: there lo is zero and only P is split. The
// products of one tile are summed in the tensor core, the tiles in fp32 registers: an accumulator
// that ran through long rows would gather the tensor core's roundings. Key ranges split over
// several blocks leave (max, sum, O) in the workspace; tree_combine_kernel joins them in order.
// Measured, calls in a row: 5 sequences of up to 1999 positions, 7 tokens, 8 heads over 4 of 64: 19 us,
// a minimum of 2 us by bytes; about 9 us of it are the chain lengths -> table -> rows and the join. 16
// of 700, 33 tokens, 32 heads over 8 of 128: 391 us, bound by the products.
#include <algorithm>
#include <cstddef>
#include <atomic>

#include <cuda_fp16.h>

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

// x = hi + lo, hi rounded to tf32 and lo exact (its low bits are dropped by the product).
struct Split {
  uint32_t hi, lo;
};
__device__ __forceinline__ Split split_tf32(float x) {
  uint32_t hi;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
  return {hi, __float_as_uint(x - __uint_as_float(hi))};
}
// x = hi + lo for every x: where rounding would overflow, hi is cut off instead, and an infinity or
// NaN is hi alone.
__device__ __forceinline__ Split split_any(float x) {
  const Split s = split_tf32(x);
  if (fabsf(__uint_as_float(s.hi)) < INFINITY) return s;
  if (!(fabsf(x) < INFINITY)) return {__float_as_uint(x + x), 0u};
  const uint32_t hi = __float_as_uint(x) & 0xffffe000u;
  return {hi, __float_as_uint(x - __uint_as_float(hi))};
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Shared memory: the queries' hi and lo parts, and two tiles of keys and values. Rows are 16
// bytes longer than their data, so that the lanes of a fragment load do not collide. The ring
// is reused for the warps' results.
template <typename T>
struct TreeShared {
  int pitch, stage;
  size_t q_bytes, bytes;
  __host__ __device__ explicit TreeShared(int d) {
    pitch = d + 16 / (int)sizeof(T);
    stage = 2 * kKeys * pitch;  // elements of a tile's keys and values
    q_bytes = (size_t)kRows * (d + 4) * 8;
    const size_t ring = 2 * (size_t)stage * sizeof(T), results = 4 * (size_t)kRows * (d + 2) * 4;
    bytes = q_bytes + (ring > results ? ring : results);
  }
};

// ND: 8 columns each, of head_dim up to 8 ND.
template <typename T, int ND>
__global__ void __launch_bounds__(kThreads) tree_attention_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int VE = Vec16<T>::N;
  constexpr bool kExact = sizeof(T) == 2;  // q, k and v are tf32 values as they are
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t4 = lane & 3;  // a fragment's row and column of this lane
  const int split = blockIdx.x / a.row_blocks, r0 = (blockIdx.x % a.row_blocks) * kRows;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int rows = a.tokens * a.group, nd = a.d / 8, chunks = a.d / VE, q_pitch = a.d + 4;
  const TreeShared<T> lay(a.d);
  float2* const qs = reinterpret_cast<float2*>(smem);  // (hi, lo)
  T* const ring = reinterpret_cast<T*>(smem + lay.q_bytes);
  const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
  // this block's tiles: a share of the cached ones, and the drafted ones in the last split
  const int tiles = (n + kKeys - 1) / kKeys;
  const int per = (tiles + a.splits - 1) / a.splits;
  const int t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);
  const int end = t1 + (split == a.splits - 1 ? (a.tokens + kKeys - 1) / kKeys : 0);

  // Where the 32 rows of a tile lie (one thread looks one up), and their copies.
  __shared__ int64_t place[2][kKeys];
  auto look_up = [&](int t, int r) -> int64_t {
    const bool cached = t < t1;
    const int key = (cached ? t : t - t1) * kKeys + r;
    if (t >= end) return -1;
    if (!cached) return key < a.tokens ? b * a.n_b + key * a.n_t + kvh * a.n_h : -1;
    if (key >= n) return -1;
    const int pi = key / a.page, p = a.tables[(int64_t)b * a.max_pages + pi];
    return p >= 0 && p < a.pages ? p * a.c_p + kvh * a.c_h + (key - pi * a.page) * a.c_s : -1;
  };
  const float per_row = 1.f / (float)chunks;
  auto fetch = [&](int t) {  // tile t into its place of the ring
    if (t < end) {
      const bool cached = t < t1;
      const T* const kp = static_cast<const T*>(cached ? a.k_cache : a.k_new);
      const T* const vp = static_cast<const T*>(cached ? a.v_cache : a.v_new);
      T* const ks = ring + (t & 1) * lay.stage;
      T* const vs = ks + kKeys * lay.pitch;
#pragma unroll 4
      for (int i = tid; i < kKeys * chunks; i += kThreads) {
        const int r = (int)(((float)i + 0.5f) * per_row), c = (i - r * chunks) * VE;  // r = i / chunks
        const int64_t at = place[t & 1][r];
        copy16_async(ks + r * lay.pitch + c, at >= 0 ? kp + at + c : nullptr, kp);
        copy16_async(vs + r * lay.pitch + c, at >= 0 ? vp + at + c : nullptr, vp);
      }
    }
    copies_commit();  // also where there is nothing: the count of groups goes on
  };
  const T* q = static_cast<const T*>(a.q) + b * a.q_b;
  for (int i = tid; i < kRows * chunks; i += kThreads) {
    const int r = (int)(((float)i + 0.5f) * per_row), c = (i - r * chunks) * VE, row = r0 + r, token = row / a.group;
    Vec16<T> x;
    x.raw = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows)
      x.raw = *reinterpret_cast<const uint4*>(q + token * a.q_t + (kvh * a.group + row - token * a.group) * a.q_h + c);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      const Split s = split_any(x.get(e));
      qs[r * q_pitch + c + e] = make_float2(__uint_as_float(s.hi), __uint_as_float(s.lo));
    }
  }

  // the lane's two rows, g and g + 8
  const int* const parents = a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  uint32_t seen[2][4];  // drafted tokens visible to them
  bool here[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = r0 + g + 8 * i, token = row / a.group;
    here[i] = row < rows && (!parents || parents[token] >= -1);
    seen[i][0] = seen[i][1] = seen[i][2] = seen[i][3] = 0u;
    if (here[i] && end > t1) ancestor_bits(parents, token, seen[i]);
  }
  float m[2], l[2], o[ND][4];
  // A value that is infinite, NaN or rounds to infinity has parts whose products are no sum of its
  // own (inf - inf, 0 inf), and 0 times it is no 0 for a row that does not see its key. All that
  // leaves a sum that is not finite, so the tiles go through the tensor core unchecked, and a block
  // with such a sum goes through them again in fp32, a key that a row does not see left out.
  for (bool plain = false;; plain = true) {
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;
#pragma unroll
    for (int j = 0; j < ND; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    if (tid < 2 * kKeys) place[(t0 + (tid >> 5)) & 1][lane] = look_up(t0 + (tid >> 5), lane);
    __syncthreads();
    fetch(t0);
    fetch(t0 + 1);
    for (int t = t0; t < end; ++t) {
      const bool cached = t < t1;
      const int key0 = (cached ? t : t - t1) * kKeys;
      const T* const ks = ring + (t & 1) * lay.stage + (warp * 8) * lay.pitch;  // this warp's 8 keys
      const T* const vs = ks + kKeys * lay.pitch;
      const int64_t next = warp == 0 ? look_up(t + 2, lane) : 0;
      copies_wait<1>();
      __syncthreads();
      // scores: c[0], c[1] of row g, keys 2 t4 and 2 t4 + 1; c[2], c[3] of row g + 8. The three
      // products have sums of their own, so that they do not wait for one another.
      float c[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f}, c2[4] = {0.f, 0.f, 0.f, 0.f};
      if (!plain) {
#pragma unroll 4
        for (int s = 0; s < nd; ++s) {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {  // (g, t4), (g + 8, t4), (g, t4 + 4), (g + 8, t4 + 4)
            const float2 x = qs[(g + 8 * (i & 1)) * q_pitch + 8 * s + t4 + 4 * (i >> 1)];
            hi[i] = __float_as_uint(x.x);
            lo[i] = __float_as_uint(x.y);
          }
          const float k0 = to_f32(ks[g * lay.pitch + 8 * s + t4]), k1 = to_f32(ks[g * lay.pitch + 8 * s + t4 + 4]);
          if constexpr (kExact) {
            mma_tf32(c, hi, __float_as_uint(k0), __float_as_uint(k1));
          } else {
            const Split x = split_tf32(k0), y = split_tf32(k1);
            mma_tf32(c1, lo, x.hi, y.hi);
            mma_tf32(c2, hi, x.lo, y.lo);
            mma_tf32(c, hi, x.hi, y.hi);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += c1[i] + c2[i];
      } else {
#pragma unroll 1
        for (int e = 0; e < a.d; ++e) {
          const float2 x = qs[g * q_pitch + e], y = qs[(g + 8) * q_pitch + e];
          const float k0 = to_f32(ks[2 * t4 * lay.pitch + e]), k1 = to_f32(ks[(2 * t4 + 1) * lay.pitch + e]);
          c[0] = fmaf(x.x + x.y, k0, c[0]);
          c[1] = fmaf(x.x + x.y, k1, c[1]);
          c[2] = fmaf(y.x + y.y, k0, c[2]);
          c[3] = fmaf(y.x + y.y, k1, c[3]);
        }
      }
      const int word = (key0 >> 5) & 3;
      float p[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint32_t drafts = word == 0 ? seen[i][0] : word == 1 ? seen[i][1] : word == 2 ? seen[i][2] : seen[i][3];
        float x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = warp * 8 + 2 * t4 + j;
          const bool sees = here[i] && (cached ? key0 + key < n : ((drafts >> key) & 1u) != 0u);
          x[j] = sees ? c[2 * i + j] * a.scale : -INFINITY;
        }
        float top = fmaxf(x[0], x[1]);
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m[i]);
        const float ref = top == -INFINITY ? 0.f : top;  // nothing seen so far
        const float keep = expf(m[i] - ref);
        p[2 * i] = x[0] == -INFINITY ? 0.f : expf(x[0] - ref);
        p[2 * i + 1] = x[1] == -INFINITY ? 0.f : expf(x[1] - ref);
        l[i] = l[i] * keep + (p[2 * i] + p[2 * i + 1]);  // this lane's keys; the four lanes' sums meet at the end
        m[i] = top;
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          o[j][2 * i] *= keep;
          o[j][2 * i + 1] *= keep;
        }
      }
      if (!plain) {
        // P as the first operand: the columns t4 and t4 + 4 of a fragment stand for the keys 2 t4
        // and 2 t4 + 1, so the scores' registers are in place and V's rows are taken in that order
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Split x = split_tf32(p[2 * (i & 1) + (i >> 1)]);
          hi[i] = x.hi;
          lo[i] = x.lo;
        }
#pragma unroll
        for (int j = 0; j < ND; ++j) {
          if (j >= nd) break;
          const float v0 = to_f32(vs[(2 * t4) * lay.pitch + 8 * j + g]), v1 = to_f32(vs[(2 * t4 + 1) * lay.pitch + 8 * j + g]);
          float y[4] = {0.f, 0.f, 0.f, 0.f};
          if constexpr (kExact) {
            mma_tf32(y, lo, __float_as_uint(v0), __float_as_uint(v1));
            mma_tf32(y, hi, __float_as_uint(v0), __float_as_uint(v1));
          } else {
            const Split s0 = split_tf32(v0), s1 = split_tf32(v1);
            mma_tf32(y, lo, s0.hi, s1.hi);
            mma_tf32(y, hi, s0.lo, s1.lo);
            mma_tf32(y, hi, s0.hi, s1.hi);
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) o[j][k] += y[k];
        }
      } else {
#pragma unroll 1
        for (int x = 0; x < 8 && key0 + warp * 8 + x < (cached ? n : a.tokens); ++x) {
          const int from = (lane & ~3) | (x >> 1);  // the lane that has this key's P of the row
          float w[2];
          bool sees[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float w0 = __shfl_sync(0xffffffffu, p[2 * i], from), w1 = __shfl_sync(0xffffffffu, p[2 * i + 1], from);
            const uint32_t drafts = word == 0 ? seen[i][0] : word == 1 ? seen[i][1] : word == 2 ? seen[i][2] : seen[i][3];
            w[i] = x & 1 ? w1 : w0;
            sees[i] = here[i] && (cached || ((drafts >> (warp * 8 + x)) & 1u));
          }
#pragma unroll
          for (int j = 0; j < ND; ++j) {
            if (j >= nd) break;
            const float v0 = to_f32(vs[x * lay.pitch + 8 * j + 2 * t4]), v1 = to_f32(vs[x * lay.pitch + 8 * j + 2 * t4 + 1]);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              o[j][2 * i] = sees[i] ? fmaf(w[i], v0, o[j][2 * i]) : o[j][2 * i];
              o[j][2 * i + 1] = sees[i] ? fmaf(w[i], v1, o[j][2 * i + 1]) : o[j][2 * i + 1];
            }
          }
        }
      }
      if (warp == 0) place[t & 1][lane] = next;
      __syncthreads();  // every warp is through with this tile's place
      fetch(t + 2);
    }
    copies_wait<0>();
    bool finite = true;
#pragma unroll
    for (int j = 0; j < ND; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) finite &= fabsf(o[j][k]) < INFINITY;
    if (!__syncthreads_or(!finite) || plain) break;
  }

  // the four warps' (max, sum, O) through shared memory, in their order
  float* const ro = reinterpret_cast<float*>(ring);                // [warp][row][d]
  float* const rml = ro + (size_t)4 * kRows * a.d;                 // [warp][row][2]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = warp * kRows + g + 8 * i;
    if (t4 == 0) {
      rml[2 * r] = m[i];
      rml[2 * r + 1] = l[i];
    }
#pragma unroll
    for (int j = 0; j < ND; ++j)
      if (j < nd) *reinterpret_cast<float2*>(ro + (size_t)r * a.d + 8 * j + 2 * t4) = make_float2(o[j][2 * i], o[j][2 * i + 1]);
  }
  __syncthreads();
  const int quads = a.d / 4;
  for (int i = tid; i < kRows * quads; i += kThreads) {
    const int r = i / quads, c = (i - r * quads) * 4, row = r0 + r;
    if (row >= rows) break;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = fmaxf(top, rml[2 * (w * kRows + r)]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = rml[2 * (w * kRows + r)];
      if (mw == -INFINITY && rml[2 * (w * kRows + r) + 1] == 0.f) continue;  // nothing seen (a sum of NaN: only NaN was)
      const float f = expf(mw - top);
      const float4 y = *reinterpret_cast<const float4*>(ro + (size_t)(w * kRows + r) * a.d + c);
      sum = fmaf(f, rml[2 * (w * kRows + r) + 1], sum);
      x.x = fmaf(f, y.x, x.x);
      x.y = fmaf(f, y.y, x.y);
      x.z = fmaf(f, y.z, x.z);
      x.w = fmaf(f, y.w, x.w);
    }
    if (a.splits == 1) {
      const bool present = !parents || parents[row / a.group] >= -1;
      const float inv = present ? 1.f / sum : 0.f;
      const int64_t at = (((int64_t)b * a.tokens + row / a.group) * a.heads + kvh * a.group + row % a.group) * a.d + c;
      store4(static_cast<T*>(a.out) + at, make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    } else {
      const int64_t at = (((int64_t)split * a.batch + b) * a.kv_heads + kvh) * rows + row;
      store4(a.ws_o + at * a.d + c, x);
      if (c == 0) {
        a.ws_ml[2 * at] = top;
        a.ws_ml[2 * at + 1] = sum;
      }
    }
  }
}

constexpr int kMaxSplits = 256;

// Joins the splits of each row: WARPS warps take them in turn (and half warps, with head_dim
// up to 64, every second one of these), so that a row of many splits is one round of loads; the
// partial sums are added in a fixed order.
// BASE2: the maxima are logarithms to base 2.
template <typename T, int WARPS, bool BASE2>
__global__ void __launch_bounds__(128) tree_combine_kernel(const __grid_constant__ TreeArgs a) {
  constexpr int kRowsHere = 4 / WARPS;
  __shared__ float weight[kRowsHere][kMaxSplits];
  __shared__ float4 part[4][32];
  pdl_enter();
  const int rows = a.tokens * a.group, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int mine = warp / WARPS, wi = warp % WARPS;  // this warp's row of the block's, and its share of it
  const int64_t all = (int64_t)a.batch * a.kv_heads * rows, row = min((int64_t)blockIdx.x * kRowsHere + mine, all - 1);
  const float2* const ml = reinterpret_cast<const float2*>(a.ws_ml) + row;
  constexpr int kPer = kMaxSplits / 32;
  float2 x[kPer];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const int s = k * 32 + lane;
    x[k] = s < a.splits ? ml[s * all] : make_float2(-INFINITY, 0.f);
    m = fmaxf(m, x[k].x);
  }
  m = warp_max(m);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const float w = x[k].x == -INFINITY ? 0.f : BASE2 ? exp2f(x[k].x - m) : expf(x[k].x - m);
    if (wi == 0) weight[mine][k * 32 + lane] = w;
    l = fmaf(w, x[k].y, l);
  }
  l = warp_sum(l);
  __syncthreads();
  const bool halves = a.d <= 64;
  const int c = (halves ? lane & 15 : lane) * 4;
  const int first = halves ? wi * 2 + (lane >> 4) : wi, step = halves ? 2 * WARPS : WARPS;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < a.d) {
    const float* const po = a.ws_o + row * a.d + c;
#pragma unroll 8
    for (int s = first; s < a.splits; s += step) {
      const float w = weight[mine][s];
      const float4 y = *reinterpret_cast<const float4*>(po + s * all * a.d);
      o.x = fmaf(w, y.x, o.x);
      o.y = fmaf(w, y.y, o.y);
      o.z = fmaf(w, y.z, o.z);
      o.w = fmaf(w, y.w, o.w);
    }
  }
  if (halves) {
    o.x += __shfl_xor_sync(0xffffffffu, o.x, 16);
    o.y += __shfl_xor_sync(0xffffffffu, o.y, 16);
    o.z += __shfl_xor_sync(0xffffffffu, o.z, 16);
    o.w += __shfl_xor_sync(0xffffffffu, o.w, 16);
  }
  if (WARPS > 1) {
    part[warp][lane] = o;
    __syncthreads();
    if (wi != 0) return;
#pragma unroll
    for (int w = 1; w < WARPS; ++w) {
      const float4 y = part[warp + w][lane];
      o.x += y.x;
      o.y += y.y;
      o.z += y.z;
      o.w += y.w;
    }
  }
  if ((int64_t)blockIdx.x * kRowsHere + mine >= all || c >= a.d || (halves && lane >= 16)) return;
  const int r = (int)(row % rows), kvh = (int)(row / rows % a.kv_heads), b = (int)(row / rows / a.kv_heads);
  const bool present = !a.parents || a.parents[(int64_t)b * a.tokens + r / a.group] >= -1;
  const float inv = present ? 1.f / l : 0.f;
  if (!present) o = make_float4(0.f, 0.f, 0.f, 0.f);  // whatever the cache holds
  const int64_t at = (((int64_t)b * a.tokens + r / a.group) * a.heads + kvh * a.group + r % a.group) * a.d + c;
  store4(static_cast<T*>(a.out) + at, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

}  // namespace

#include "tree_attention_tc.cuh"
#include "tree_attention_8bit.cuh"
#include "tree_attention_8bit_ring.cuh"

namespace {

// ------------------------------------------------------------------ host

// Blocks that share a sequence's keys. Each takes whole tiles, so many that there are no more than
// four blocks for each SM where all sequences are as long as the tables allow: that is what runs at
// once at head_dim up to 64 (by registers; at 128 shared memory holds two). Measured in fp32 on calls
// in a row against five blocks an SM of at least two tiles: geometric mean over 20 shapes with rows
// of equal length 0.88 of the time, over 120 with lengths from half of that to all of it 0.97 (0.69 to
// 1.4: short rows win, ragged long ones may lose). 32 sequences of 500 25.2 and 27.3 us, 8 of 2000 with
// 4 heads to a key/value head 33.8 and 44.9, one of 300 8.6 and 10.4, one of 8000 17.5 and 17.6, 5 of 1000
// to 1999 with 7 tokens 18.8 and 17.1. In whole tiles, three an SM have 0.95 and 0.99, five 0.98 and 0.98,
// four rounded to the nearest tile instead of up 0.94 and 0.99.
int split_count(int64_t batch, int64_t kv_heads, int64_t row_blocks, int64_t capacity) {
  const int64_t tiles = std::max<int64_t>((capacity + kKeys - 1) / kKeys, 1), room = 4 * (int64_t)sm_count();
  const int64_t share = std::max((tiles * batch * kv_heads * row_blocks + room - 1) / room, (tiles + kMaxSplits - 1) / kMaxSplits);
  return (int)((tiles + share - 1) / share);
}

template <typename T, int ND>
int launch_split(const TreeArgs& a, dim3 grid, cudaStream_t st) {
  const char* op = "nkl_attention_tree";
  static std::atomic<bool> set[64] = {};  // per device: more than 48 KB of shared memory allowed (idempotent)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(tree_attention_kernel<T, ND>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               (int)TreeShared<T>(8 * ND).bytes);
    if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  }
  return launch_pdl(tree_attention_kernel<T, ND>, grid, dim3(kThreads), TreeShared<T>(a.d).bytes, st, op, a);
}

// Joins the splits. Four warps to a row where many splits meet: 5 sequences of up to 1999 positions 18.2 against
// 19.3 us, one of 8000 28.5 against 33.4; one where few do: 16 of 700, 33 tokens, 118 against 121 us.
template <bool BASE2>
int launch_combine(const TreeArgs& a, int dtype, cudaStream_t st, const char* op) {
  const int64_t rows = (int64_t)a.batch * a.heads * a.tokens;
  auto join = [&](auto* kernel, int per_block) {
    return launch_pdl(kernel, dim3((unsigned)((rows + per_block - 1) / per_block)), dim3(128), 0, st, op, a);
  };
  if (a.splits > 8)
    return dtype == NKL_FLOAT32 ? join(tree_combine_kernel<float, 4, BASE2>, 1) : join(tree_combine_kernel<bf16, 4, BASE2>, 1);
  return dtype == NKL_FLOAT32 ? join(tree_combine_kernel<float, 1, BASE2>, 4) : join(tree_combine_kernel<bf16, 1, BASE2>, 4);
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

// What the two entry points check and take over; s and n: strides of q [batch, token, head], the drafted tokens' rows
// [batch, token, head] and the cache [page, head, row], and the sizes stepped over. `done`: nothing to do.
int tree_args(const char* op, TreeArgs& a, int64_t (&s)[9], int64_t (&n)[9], bool& done, const void* q,
              const int64_t* q_strides, const void* k_new, const void* v_new, const int64_t* new_strides,
              const void* k_cache, const void* v_cache, const int64_t* cache_strides, const int32_t* tables,
              const int32_t* lens, const int32_t* parents, void* out, int64_t batch, int64_t tokens, int64_t heads,
              int64_t kv_heads, int64_t head_dim, int64_t pages, int64_t page_size, int64_t max_pages, float scale,
              int dtype, int64_t cache_per, int64_t unit) {
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (tokens > kMaxDrafted)
    return fail(NKL_ERR_SHAPE, "%s: %lld drafted tokens, at most %d are taken", op, (long long)tokens, kMaxDrafted);
  if (!tree_sizes_ok(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages) || head_dim % unit || pages < 1 ||
      pages > 0x7fffffffLL)
    return fail(NKL_ERR_SHAPE,
                "%s: batch %lld, tokens %lld, heads %lld / %lld, head_dim %lld, page size %lld or table width %lld not "
                "supported (kv heads divide heads; head_dim a multiple of %lld up to %d; up to 2^30 positions)",
                op, (long long)batch, (long long)tokens, (long long)heads, (long long)kv_heads, (long long)head_dim,
                (long long)page_size, (long long)max_pages, (long long)unit, kMaxDim);
  done = batch == 0 || tokens == 0;
  if (done) return NKL_OK;
  if (!q || !k_new || !v_new || !k_cache || !v_cache || !tables || !lens || !out)
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  for (const void* p : {q, k_new, v_new, k_cache, v_cache, static_cast<const void*>(out)})
    if (!is_aligned(p, 16)) return fail(NKL_ERR_ALIGN, "%s: tensors need 16-byte alignment", op);
  const int64_t dense[9] = {tokens * heads * head_dim,    heads * head_dim,                 head_dim,
                            tokens * kv_heads * head_dim, kv_heads * head_dim,              head_dim,
                            kv_heads * page_size * head_dim, page_size * head_dim, head_dim};
  const int64_t sizes[9] = {batch, tokens, heads, batch, tokens, kv_heads, pages, kv_heads, page_size};
  const int64_t* given[3] = {q_strides, new_strides, cache_strides};
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  for (int i = 0; i < 9; ++i) {
    s[i] = given[i / 3] ? given[i / 3][i % 3] : dense[i];
    n[i] = sizes[i];
    if (n[i] > 1 && (s[i] < 0 || s[i] % (i < 6 ? per : cache_per)))
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
  return NKL_OK;
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
  // strides and the scale's sign, which are not known here, may still choose the other kernel
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
  TreeArgs a = {};
  int64_t s[9], n[9];
  bool done = false;
  if (int rc = tree_args(op, a, s, n, done, q, q_strides, k_new, v_new, new_strides, k_cache, v_cache, cache_strides, tables,
                         lens, parents, out, batch, tokens, heads, kv_heads, head_dim, pages, page_size, max_pages, scale,
                         dtype, 16 / (int64_t)dtype_size(dtype), 8))
    return rc;
  if (done) return NKL_OK;
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
  if (dtype == NKL_FLOAT32)
    rc = head_dim <= 64 ? launch_split<float, 8>(a, grid, st) : launch_split<float, 16>(a, grid, st);
  else
    rc = head_dim <= 64 ? launch_split<bf16, 8>(a, grid, st) : launch_split<bf16, 16>(a, grid, st);
  if (rc || a.splits == 1) return rc;
  return launch_combine<false>(a, dtype, st, op);
}

extern "C" size_t nkl_attention_tree_8bit_workspace_size(int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads,
                                                         int64_t head_dim, int64_t page_size, int64_t max_pages,
                                                         int dtype) {
  if (!valid_dtype(dtype) || !tree_sizes_ok(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages) ||
      batch == 0 || tokens == 0)
    return 0;
  const TcPlan p = tc_plan(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages, dtype);
  return std::max(p.on ? p.bytes : 0, split_bytes(splits_8bit(batch, kv_heads, tokens * (heads / kv_heads), page_size * max_pages),
                                                  batch, heads, tokens, head_dim));
}

extern "C" int nkl_attention_tree_8bit(const void* q, const int64_t* q_strides, const void* k_new, const void* v_new,
                                       const int64_t* new_strides, const void* k_cache, const void* v_cache,
                                       const int64_t* cache_strides, const void* k_scales, const void* v_scales,
                                       const int32_t* tables, const int32_t* lens, const int32_t* parents, void* out,
                                       void* workspace, size_t workspace_bytes, int64_t batch, int64_t tokens,
                                       int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                       int64_t page_size, int64_t max_pages, int64_t block, float scale, int dtype,
                                       void* stream) {
  const char* op = "nkl_attention_tree_8bit";
  Bits8Args a = {};
  int64_t s[9], n[9];
  bool done = false;
  if (int rc = tree_args(op, a.t, s, n, done, q, q_strides, k_new, v_new, new_strides, k_cache, v_cache, cache_strides, tables,
                         lens, parents, out, batch, tokens, heads, kv_heads, head_dim, pages, page_size, max_pages, scale,
                         dtype, 16, 16))
    return rc;
  if (done) return NKL_OK;
  if (block < 1 || page_size % block)
    return fail(NKL_ERR_SHAPE, "%s: blocks of %lld positions do not divide pages of %lld", op, (long long)block, (long long)page_size);
  if (!k_scales || !v_scales) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  a.k_scales = static_cast<const uint8_t*>(k_scales);
  a.v_scales = static_cast<const uint8_t*>(v_scales);
  a.block = (int)block;
  a.per_page = (int)(page_size / block);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t rows = tokens * a.t.group;
  const TcPlan p = tc_plan(batch, tokens, heads, kv_heads, head_dim, page_size, max_pages, dtype);
  bool tc = p.on && scale > 0.f && scale < INFINITY;
  for (int i = 0; i < 9; ++i) tc = tc && (n[i] == 1 || (s[i] > 0 && s[i] < (1LL << 38)));
  if (tc) {
    if (p.bytes) {
      if (!workspace || workspace_bytes < p.bytes) return fail(NKL_ERR_ARG, "%s: workspace too small", op);
      if (!is_aligned(workspace, 256)) return fail(NKL_ERR_ALIGN, "%s: workspace not 256-byte aligned", op);
    }
    unsigned char* ws = static_cast<unsigned char*>(workspace);
    int64_t* const steps[9] = {&a.t.q_b, &a.t.q_t, &a.t.q_h, &a.t.n_b, &a.t.n_t, &a.t.n_h, &a.t.c_p, &a.t.c_h, &a.t.c_s};
    for (int i = 0; i < 9; ++i)
      if (n[i] == 1) *steps[i] = head_dim;
    const TcScales sc = {k_scales, v_scales, (int)block};
    if (rows <= 8)
      return head_dim == 128 ? ring_launch<128, 1>(a.t, p, ws, st, sc) : ring_launch<64, 1>(a.t, p, ws, st, sc);
    if (rows <= kRingRows)
      return head_dim == 128 ? ring_launch<128, 2>(a.t, p, ws, st, sc) : ring_launch<64, 2>(a.t, p, ws, st, sc);
    if (head_dim == 128) return p.nq == 1 ? tc_launch<128, 1, true>(a.t, p, ws, st, sc) : tc_launch<128, 2, true>(a.t, p, ws, st, sc);
    return p.nq == 1 ? tc_launch<64, 1, true>(a.t, p, ws, st, sc) : tc_launch<64, 2, true>(a.t, p, ws, st, sc);
  }
  const Shape8 shape = shape_8bit(rows);
  a.tiles = shape.tiles;
  a.t.row_blocks = shape.row_blocks;
  a.t.splits = (int)splits_8bit(batch, kv_heads, rows, page_size * max_pages);
  if (const size_t need = split_bytes(a.t.splits, batch, heads, tokens, head_dim)) {
    if (!workspace || workspace_bytes < need) return fail(NKL_ERR_ARG, "%s: workspace too small", op);
    if (!is_aligned(workspace, 256)) return fail(NKL_ERR_ALIGN, "%s: workspace not 256-byte aligned", op);
    a.t.ws_o = static_cast<float*>(workspace);
    a.t.ws_ml = a.t.ws_o + (size_t)a.t.splits * batch * heads * tokens * head_dim;
  }
  const dim3 grid((unsigned)(a.t.splits * a.t.row_blocks), (unsigned)kv_heads, (unsigned)batch);
  const bool fast = page_size % 16 == 0 && block % 16 == 0;
  int rc;
  if (dtype == NKL_FLOAT32)
    rc = head_dim <= 64 ? launch_8bit<float, 1>(a, shape.nt, grid, fast, st) : launch_8bit<float, 2>(a, shape.nt, grid, fast, st);
  else
    rc = head_dim <= 64 ? launch_8bit<bf16, 1>(a, shape.nt, grid, fast, st) : launch_8bit<bf16, 2>(a, shape.nt, grid, fast, st);
  if (rc || a.t.splits == 1) return rc;
  return launch_combine<true>(a.t, dtype, st, op);
}
