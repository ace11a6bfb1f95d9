// rotary.cu - rotary positions, alone and on the way of keys and values into a paged cache.
//
// The first r entries of a head are pairs that turn with the token's position: by the angle
// a = position * freqs[i], pair i being the entries (i, i + r / 2) or, interleaved, (2 i, 2 i + 1):
//   y1 = m (x1 cos a - x2 sin a)      y2 = m (x2 cos a + x1 sin a)
// The rest of the head is copied. The gradient is the same turn by -a. Angles are products in 64
// bits, taken modulo a full turn, as are their sines and cosines, so that far positions lose
// nothing; freqs come from the caller, who may stretch them for long contexts.
//
//   rotary         x -> y
//   rotary_append  q, k -> turned q, k; k (turned) and v to the pages of a cache as well
//   append_8bit    rows of k and v (all of them, or an accepted path's) to a cache in 8 bits
//
// A cache in 8 bits holds e4m3 numbers, and for each block of positions and head a power of two:
// the smallest 2^e, e >= -100, with which the block's largest magnitude is at most 448 2^e. It
// costs an e4m3 number no precision, and a row that was rounded once can be rounded again when its
// block grows past its power of two: only numbers below e4m3's normal range lose bits. Infinities
// and NaN have no place in e4m3; a block that gets one has the power of two NaN, and reads as NaN.
//
// A group of tokens of one sequence (one or more whole blocks of an 8-bit cache) is a thread
// block's. It computes the tokens' sines and cosines once, into shared memory, for all heads:
// 64 angles of a token cost as much as some 40 heads' rows. Rows without a block of their own go
// through all threads, each with two vectors at places half of r apart; a block of an 8-bit
// cache is one warp's, which copies its rows to shared memory as they are, finds the largest magnitude of
// the turned ones, and turns them again to round them (in fp32 they would not fit into registers; held there in
// bf16 they were unpacked once for both, and spilled: a prompt of 4 x 4096 239 us, so 190 at first; places looked up once a
// block, rows gone through by pointers in loops that are not unrolled: 156). A warp has two buffers of rows where they are
// of 4 KB or less (168 us with one); three thread blocks to an SM, with 85 registers to a thread, took 187 and more.
//
// Measured (6.57 TB/s is what a copy of memory reaches): x and its gradient, bf16, 4 x 4096 tokens of 64 heads of 128
// 186 us (1.07 GB: 163 by bytes; 183 with sines and cosines in 32 bits); q, k, v of 32 heads, turned, k and v to a cache in 8 bits, 4 x 4096 tokens 156 us
// (808 MB: 123), bound by issue and by what a thread block's two phases (queries, then blocks) do not overlap. x alone, bf16, 4 x
// 4096 tokens of 64 heads of 64 (269 MB: 41): whole heads in halves 50 us, interleaved 59, half of each head 65 (halves: entries that
// stay are loaded and stored twice) and 59 (interleaved), where a thread has half as many bytes on their way. The smallest calls:
// 2.5 us on the GPU for x alone, 5 to 6 with a cache (lengths -> tables -> rows), and 6 to 9 of the host's.
#include <algorithm>
#include <atomic>
#include <cuda_fp8.h>

#include "common.cuh"

namespace nkl {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kHeld = 8192;      // bytes of rows that a warp holds, at most
constexpr int kMaxTokens = 32;   // whose angles are held at a time
constexpr int kMaxHead = 256;
constexpr int kMaxHead8 = 128;   // in 8 bits: as the attention
constexpr int kLowest = -100;    // of the powers of two
constexpr uint8_t kNanScale = 255;
constexpr int kMostTokens = 1 << 24;  // of a call
constexpr int kMostLen = 0x7fffffff - 2 * kMostTokens;

constexpr int kMostSmem = 2 * kMaxTokens * (kMaxHead / 2) * 4 + kWarps * kHeld;

enum Kind { kPlain, kSame, kBits8 };  // where rows go: no cache, one of their type, one of 8 bits

struct RotaryArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *k_cache, *v_cache;
  uint8_t *k_scales, *v_scales;
  const int *positions, *parents, *tables, *lens, *path, *count;
  int* lens_out;
  const double* freqs;
  int64_t q_b, q_t, q_h, n_l, n_b, n_t, n_h, c_l, c_p, c_h, c_s;  // strides in elements
  int batch, tokens, heads, kv_heads, d, half, layers, pages, page, max_pages, block;
  int group, groups;  // tokens of a thread block; thread blocks of a sequence
  int chunk;          // tokens whose angles are held at a time
  int buffer, two;    // bytes of a warp's rows; whether it has two such buffers
  int per_token;      // whether positions are given for each token
  int splits;         // thread blocks that share the heads of a group
  int inverse;
  float magnitude;
};

// A lane's part of a row: VE entries at o0 and, of the half layout's pairs, VE more at o1.
template <typename T, int VE> struct Raw;
template <> struct Raw<bf16, 8> { typedef uint4 type; };
template <> struct Raw<float, 4> { typedef uint4 type; };
template <> struct Raw<bf16, 4> { typedef uint2 type; };

template <typename T, int VE, bool INTER>
struct Part {
  typedef typename Raw<T, VE>::type V;
  int o0, o1, f;  // o1: o0 where there are none; f: the first pair, -1: entries that stay as they are
  __device__ __forceinline__ Part(int item, int half) {
    if (INTER) {
      o1 = o0 = item * VE;
      f = o0 < 2 * half ? o0 / 2 : -1;
    } else {
      const int pairs = half / VE;
      o0 = item < pairs ? item * VE : 2 * half + (item - pairs) * VE;
      f = item < pairs ? o0 : -1;
      o1 = item < pairs ? o0 + half : o0;
    }
  }
  static __device__ __forceinline__ int items(int d, int half) { return INTER ? d / VE : half / VE + (d - 2 * half) / VE; }
  __device__ __forceinline__ void load(const T* row, V& x, V& y) const {
    x = *reinterpret_cast<const V*>(row + o0);
    if (!INTER) y = *reinterpret_cast<const V*>(row + o1);
  }
  static __device__ __forceinline__ void unpack(const V& x, float (&a)[VE]) {
    const uint32_t* const w = reinterpret_cast<const uint32_t*>(&x);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; ++i) a[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        a[2 * i] = __uint_as_float(w[i] << 16);
        a[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ V pack(const float (&a)[VE]) {
    V x;
    uint32_t* const w = reinterpret_cast<uint32_t*>(&x);
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VE; ++i) w[i] = __float_as_uint(a[i]);
    } else {
#pragma unroll
      for (int i = 0; i < VE / 2; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a[2 * i], a[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    return x;
  }
  // The cosines and sines of its pairs, of a token's c and s.
  static constexpr int kPairs = INTER ? VE / 2 : VE;
  struct Angles {
    float c[kPairs], s[kPairs];
  };
  __device__ __forceinline__ void load(const float* c, const float* s, Angles& to) const {
    if (f < 0) return;
    if constexpr (kPairs % 4 == 0) {  // f is a multiple of 4
#pragma unroll
      for (int i = 0; i < kPairs; i += 4) {
        *reinterpret_cast<float4*>(to.c + i) = *reinterpret_cast<const float4*>(c + f + i);
        *reinterpret_cast<float4*>(to.s + i) = *reinterpret_cast<const float4*>(s + f + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        to.c[i] = c[f + i];
        to.s[i] = s[f + i];
      }
    }
  }
  // The entries at o0 and o1, turned.
  __device__ __forceinline__ void turn(const V& x, const V& y, const Angles& by, float (&a)[VE], float (&b)[VE]) const {
    unpack(x, a);
    if (!INTER) unpack(y, b);
    if (f < 0) return;
#pragma unroll
    for (int i = 0; i < kPairs; ++i) {
      float &u = INTER ? a[2 * i] : a[i], &w = INTER ? a[2 * i + 1] : b[i];
      const float p = u, q = w;
      u = p * by.c[i] - q * by.s[i];
      w = q * by.c[i] + p * by.s[i];
    }
  }
  __device__ __forceinline__ void store(T* row, const float (&a)[VE], const float (&b)[VE]) const {
    *reinterpret_cast<V*>(row + o0) = pack(a);
    if (!INTER) *reinterpret_cast<V*>(row + o1) = pack(b);
  }
};

__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_issued() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_landed() {  // all but the last N groups
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float max_nan(float a, float b) {  // NaN (0x7fffffff) if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }  // -126 <= e <= 127

// e4m3 codes of VE values times 2^-e; with `keep` 0 they are zeros, for a block whose power is NaN: 0 times a number that
// is none would be e4m3's code for NaN, which the attention does not look for.
template <int VE>
__device__ __forceinline__ void store_codes(uint8_t* to, const float (&a)[VE], float inv, uint32_t keep) {
  uint32_t w[VE / 4];
#pragma unroll
  for (int i = 0; i < VE / 4; ++i) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a[4 * i] * inv, a[4 * i + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(a[4 * i + 2] * inv, a[4 * i + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[i] = (lo | hi << 16) & keep;
  }
  if constexpr (VE == 8) *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(to) = w[0];
}

// The power of two's code for a largest magnitude given by its bits.
__device__ __forceinline__ int scale_code(uint32_t top) {
  if (top >= 0x7f800000u) return kNanScale;
  return max((int)(top >> 23) - 135 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0), kLowest) + 127;
}

// Four codes times 2^-shift.
__device__ __forceinline__ uint32_t round_again(uint32_t w, float factor) {
  uint32_t out = 0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    out |= (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(f.x * factor, f.y * factor), __NV_SATFINITE, __NV_E4M3) << (16 * i);
  }
  return out;
}

// Of an angle given as a part of a turn, in [-1/2, 1/2]: the Taylor series in 64 bits, within an eighth of a turn of the
// nearest quarter (first terms left out: 7e-12 and 5e-13). In 32 bits they would be off by up to two steps, which
// brings more keys over the border between two e4m3 numbers than the products' roundings do.
__device__ __forceinline__ void sine_cosine(double turns, double& sine, double& cosine) {
  const double quarter = rint(4. * turns), x = (turns - 0.25 * quarter) * 6.283185307179586, z = x * x;
  const double s = x + x * z * (-1. / 6 + z * (1. / 120 + z * (-1. / 5040 + z * (1. / 362880 - z * (1. / 39916800)))));
  const double c = 1. + z * (-1. / 2 + z * (1. / 24 + z * (-1. / 720 + z * (1. / 40320 + z * (-1. / 3628800 + z * (1. / 479001600))))));
  const int q = (int)quarter & 3;
  const double u = q & 1 ? c : s, v = q & 1 ? s : c;
  sine = q & 2 ? -u : u;
  cosine = (q + 1) & 2 ? -v : v;
}

// Position below its sequence's first of token j: its depth in a tree of drafted tokens (0 for a
// child of the last cached position, an absent token and a child of one, as in the attention).
__device__ __forceinline__ int depth_of(const int* parents, int j) {
  if (!parents) return j;
  int up = parents[j], n = 0;
  for (int at = j; up >= 0 && up < at && parents[up] >= -1; ++n) {
    at = up;
    up = parents[at];
  }
  return parents[j] < -1 ? 0 : n;
}

template <typename T, int VE, bool INTER, int KIND>
__global__ void __launch_bounds__(kThreads, 2) rotary_kernel(const __grid_constant__ RotaryArgs a) {
  typedef Part<T, VE, INTER> P;
  typedef typename P::V V;
  extern __shared__ __align__(16) float angles[];  // [cosine, sine][chunk][half]
  __shared__ int s_at[kMaxTokens];                 // the chunk's positions
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int i = blockIdx.x % a.groups, bl = blockIdx.x / a.groups, b = bl % a.batch, layer = bl / a.batch;
  float* const cosines = angles;
  float* const sines = angles + a.chunk * a.half;
  const int items = P::items(a.d, a.half);
  const int capacity = a.max_pages * a.page;
  // (a length past the tables is a position all the same; what ends it keeps the sums below in 32 bits)
  const int given = KIND == kPlain ? 0 : max(a.lens[b], 0), len = min(given, kMostLen);
  const int count = KIND == kPlain ? a.tokens : a.count ? min(max(a.count[b], 0), a.tokens) : a.tokens;
  if (KIND == kBits8 && a.lens_out && layer == 0 && i == 0 && blockIdx.y == 0 && tid == 0) a.lens_out[b] = given + count;
  // the group's tokens [j0, j1), of which those before `kept` go to the cache
  int j0, j1, first = 0;  // first: an 8-bit cache's position where the group begins
  if (KIND == kBits8) {
    first = (len / a.block) * a.block + i * a.group;
    j0 = max(first - len, 0);
    j1 = min(first + a.group - len, a.q || a.k_out ? a.tokens : count);
  } else {
    j0 = i * a.group;
    j1 = min(j0 + a.group, a.tokens);
  }
  if (j0 >= j1) return;
  auto page_of = [&](int position) {  // -1: none
    if (position >= capacity) return -1;
    const int p = a.tables[(int64_t)b * a.max_pages + position / a.page];
    return p >= 0 && p < a.pages ? p : -1;
  };
  const int* const parents = KIND == kPlain && a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  auto fill_angles = [&](int t0, int n) {  // of the tokens t0 .. t0 + n - 1; the caller synchronises
    if (!a.freqs) return;
    if (KIND == kPlain && parents) {
      if (tid < n) s_at[tid] = a.positions[b] + depth_of(parents, t0 + tid);
      __syncthreads();
    }
    for (int x = tid; x < n * a.half; x += kThreads) {
      const int t = x / a.half, f = x - t * a.half;
      int at;
      if (KIND != kPlain) at = len + t0 + t;
      else if (parents) at = s_at[t];
      else at = a.per_token ? a.positions[(int64_t)b * a.tokens + t0 + t] : a.positions[b] + t0 + t;
      double turns = (double)at * a.freqs[f] * 0.15915494309189533577;  // 1 / (2 pi)
      turns -= rint(turns);
      double sine, cosine;
      sine_cosine(turns, sine, cosine);
      cosines[x] = (float)(cosine * a.magnitude);
      sines[x] = (float)((a.inverse ? -sine : sine) * a.magnitude);
    }
  };
  const T* const q = static_cast<const T*>(a.q) + b * a.q_b;
  const T* const k = static_cast<const T*>(a.k) + layer * a.n_l + b * a.n_b;
  const T* const v = static_cast<const T*>(a.v) + layer * a.n_l + b * a.n_b;
  // Rows without a block: head h of a.heads (q), then k's and v's, of the tokens t0 .. t0 + n - 1;
  // this thread block's share of the heads.
  auto rows = [&](int t0, int n, bool ready) {
    const int all = a.heads + (KIND == kSame ? 2 * a.kv_heads : 0);
    const int h0 = (int)((int64_t)all * blockIdx.y / a.splits), h1 = (int)((int64_t)all * (blockIdx.y + 1) / a.splits);
    // A thread stays with its entries and with a token, whose cosines and sines it keeps, and goes from head to head.
    // (Counting rows through, with divisions for token and head and the cosines from shared memory for each: 29
    // instructions to a pair, and 110 us for 4 x 4096 tokens of 64 heads of 128; so 92.)
    const int per = kThreads / items, row0 = tid / items;
    const int tokens = min(n, per), step = per / tokens;  // tokens of a pass, and its heads
    const int my_t = row0 % tokens, my_h = row0 / tokens;
    const P part(tid - row0 * items, a.half);
    constexpr int kAhead = 4;
    for (int ts = 0; ts < n; ts += tokens) {
      const int t = t0 + ts + my_t;
      const bool on = row0 < per && my_h < step && ts + my_t < n;
      const T* const q_t = q + t * a.q_t;
      const T* const kv_t = k + t * a.n_t;
      T* const out = static_cast<T*>(a.q_out) + ((int64_t)b * a.tokens + t) * a.heads * a.d;
      T* const k_out = static_cast<T*>(a.k_out) + ((int64_t)b * a.tokens + t) * a.kv_heads * a.d;
      const int at = len + t, page = KIND == kSame && on && t < count ? page_of(at) : -1;
      const int64_t cached = KIND == kSame ? page * a.c_p + (at % a.page) * a.c_s : 0;
      typename P::Angles by;
      for (int hb = h0; hb < h1 || !ready; hb += kAhead * step) {
        V x[kAhead], y[kAhead];
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
          const int h = hb + my_h + s * step;
          if (!on || h >= h1) continue;
          const T* from = q_t + h * a.q_h;
          if (KIND == kSame && h >= a.heads)
            from = h < a.heads + a.kv_heads ? kv_t + (h - a.heads) * a.n_h : v + t * a.n_t + (h - a.heads - a.kv_heads) * a.n_h;
          part.load(from, x[s], y[s]);
        }
        if (!ready) {  // the first rows are on their way while the angles are computed
          fill_angles(t0, n);
          __syncthreads();
          ready = true;
        }
        if (hb == h0 && on) part.load(cosines + (t - t0) * a.half, sines + (t - t0) * a.half, by);
#pragma unroll
        for (int s = 0; s < kAhead; ++s) {
          const int h = hb + my_h + s * step;
          if (!on || h >= h1) continue;
          float e[VE], o[VE];
          if (KIND == kSame && h >= a.heads + a.kv_heads) {
            P::unpack(x[s], e);
            if (!INTER) P::unpack(y[s], o);
          } else {
            part.turn(x[s], y[s], by, e, o);
          }
          if (h < a.heads) part.store(out + h * a.d, e, o);
          if (KIND == kSame && h >= a.heads) {
            const bool key = h < a.heads + a.kv_heads;
            const int g = h - a.heads - (key ? 0 : a.kv_heads);
            if (key) part.store(k_out + g * a.d, e, o);
            if (page >= 0) part.store(static_cast<T*>(key ? a.k_cache : a.v_cache) + cached + g * a.c_h, e, o);
          }
        }
      }
    }
  };
  if (KIND != kBits8) {
    rows(j0, j1 - j0, false);
    return;
  }

  // ---------------------------------------------------------------- blocks of an 8-bit cache
  const int* const path = a.path ? a.path + (int64_t)b * a.tokens : nullptr;
  const int per = 32 / items, row0 = lane / items;
  const P part(lane - row0 * items, a.half);
  const int subs = a.group / a.block;  // blocks of the group
  const int units = 2 * a.kv_heads * subs;
  const int u0 = (int)((int64_t)units * blockIdx.y / a.splits), u1 = (int)((int64_t)units * (blockIdx.y + 1) / a.splits);
  const int nb = a.page / a.block;  // blocks of a page
  // a warp's two buffers of rows, dense, filled 16 bytes at a time
  uint8_t* const held = reinterpret_cast<uint8_t*>(sines + a.chunk * a.half) + (a.two + 1) * warp * a.buffer;
  const int row_bytes = a.d * (int)sizeof(T), chunks = row_bytes / 16, per_c = 32 / chunks, row_c = lane / chunks;
  struct Unit {
    bool key;
    int g, p0;  // head, first position
  };
  auto unit_of = [&](int u) {
    const int sub = subs == 1 ? 0 : u / (2 * a.kv_heads), kg = u - sub * 2 * a.kv_heads;
    return Unit{kg < a.kv_heads, kg < a.kv_heads ? kg : kg - a.kv_heads, first + sub * a.block};
  };
  // source row of token j for the cache, -1: none
  auto source = [&](int j) {
    if (j >= count) return -1;
    const int r = path ? path[j] : j;
    return r >= 0 && r < a.tokens ? r : -1;
  };
  // Of the tokens t0 .. t0 + n - 1, how many a unit looks at: without a path those that go to the cache are the first.
  auto kept = [&](int t0, int n) { return path ? n : min(n, count - t0); };
  // Their rows into a buffer, as one group of copies.
  auto fetch = [&](const Unit& u, int t0, int n, int buf) {
    const bool out = u.key && a.k_out;
    const int m = row_c < per_c ? (out ? n : kept(t0, n)) : 0, col = lane - row_c * chunks;
    const T* const from = (u.key ? k : v) + u.g * a.n_h + col * (16 / (int)sizeof(T));
    uint32_t to = (uint32_t)__cvta_generic_to_shared(held + buf * a.buffer) + (uint32_t)(row_c * row_bytes + col * 16);
    if (out || !path) {
      const T* row = from + (t0 + row_c) * a.n_t;
      const int64_t step = per_c * a.n_t;
      for (int t = row_c; t < m; t += per_c, row += step, to += per_c * row_bytes) copy16(to, row);
    } else {
      for (int t = row_c; t < m; t += per_c, to += per_c * row_bytes)
        if (const int r = source(t0 + t); r >= 0) copy16(to, from + r * a.n_t);
    }
    copies_issued();
  };
  // A row of a buffer, turned by the cosines and sines at c and s.
  auto values = [&](bool turned, const uint8_t* row, const float* c, const float* s, float (&e)[VE], float (&o)[VE]) {
    V x, y;
    part.load(reinterpret_cast<const T*>(row), x, y);
    if (turned) {
      typename P::Angles by;
      part.load(c, s, by);
      part.turn(x, y, by, e, o);
    } else {
      P::unpack(x, e);
      if (!INTER) P::unpack(y, o);
    }
  };
  // The largest magnitude's bits, of the rows that go to the cache; turned keys to k_out. c0: the chunk's first token.
  auto largest = [&](const Unit& u, int t0, int n, int c0, int buf) {
    float top = 0.f;
    const bool out = u.key && a.k_out, turned = u.key && a.freqs;
    const int nc = kept(t0, n), m = row0 < per ? (out ? n : nc) : 0;
    const int64_t k_row = (int64_t)a.kv_heads * a.d;
    T* to = static_cast<T*>(a.k_out) + (((int64_t)b * a.tokens + t0 + row0) * a.kv_heads + u.g) * a.d;
    const uint8_t* row = held + buf * a.buffer + row0 * row_bytes;
    const float *c = cosines + (t0 + row0 - c0) * a.half, *s = c + (sines - cosines);
#pragma unroll 1
    for (int t = row0; t < m; t += per, row += per * row_bytes, to += per * k_row, c += per * a.half, s += per * a.half) {
      if (path && !out && source(t0 + t) < 0) continue;  // not read
      float e[VE], o[VE];
      values(turned, row, c, s, e, o);
      if (out) part.store(to, e, o);
      float most = 0.f;
#pragma unroll
      for (int z = 0; z < VE; ++z) {
        most = max_nan(most, fabsf(e[z]));
        if (!INTER) most = max_nan(most, fabsf(o[z]));
      }
      if (path ? source(t0 + t) >= 0 : t < nc) top = max_nan(top, most);
    }
    return __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  };
  auto write = [&](const Unit& u, int t0, int n, int c0, int buf, uint8_t* rows8, int code) {
    const float inv = code == kNanScale ? 0.f : power_of_two(127 - code);
    const uint32_t keep = code == kNanScale ? 0u : ~0u;
    const bool turned = u.key && a.freqs;
    const int m = row0 < per ? kept(t0, n) : 0;
    uint8_t* to = rows8 + (len + t0 - u.p0 + row0) * a.c_s;
    const uint8_t* row = held + buf * a.buffer + row0 * row_bytes;
    const float *c = cosines + (t0 + row0 - c0) * a.half, *s = c + (sines - cosines);
#pragma unroll 1
    for (int t = row0; t < m; t += per, row += per * row_bytes, to += per * a.c_s, c += per * a.half, s += per * a.half) {
      if (path && source(t0 + t) < 0) continue;
      float e[VE], o[VE];
      values(turned, row, c, s, e, o);
      store_codes<VE>(to + part.o0, e, inv, keep);
      if (!INTER) store_codes<VE>(to + part.o1, o, inv, keep);
    }
  };
  // The block's power of two, given the largest magnitude that comes to it; rows that were in it
  // are rounded again if it grows. Returns the code.
  auto settle = [&](const Unit& u, uint32_t top, uint8_t* rows8, uint8_t* scale) {
    int code = scale_code(top);
    const int old = len - u.p0;  // rows of the block that were there
    if (old > 0) {
      const int was = *scale;
      if (was == kNanScale || code == kNanScale) {
        code = kNanScale;
      } else if (code > was) {
        const float factor = code - was > 126 ? 0.f : power_of_two(was - code);
        const int words = a.d / 4;
        for (int z = lane; z < old * words; z += 32) {
          const int r = z / words, w = z - r * words;
          uint32_t* const at = reinterpret_cast<uint32_t*>(rows8 + r * a.c_s) + w;
          *at = round_again(*at, factor);
        }
      } else {
        code = was;
      }
    }
    __syncwarp();
    if (lane == 0) *scale = (uint8_t)code;
    return code;
  };
  int placed = -1, page = -1, in_page = 0, in_scales = 0;  // the place of the last units' first position
  auto place = [&](const Unit& u, uint8_t*& rows8, uint8_t*& scale) {  // of the block's first row
    if (u.p0 != placed) {
      placed = u.p0;
      page = page_of(u.p0);
      in_page = u.p0 % a.page;
      in_scales = in_page / a.block;
    }
    const int p = max(page, 0);
    rows8 = static_cast<uint8_t*>(u.key ? a.k_cache : a.v_cache) + layer * a.c_l + p * a.c_p + u.g * a.c_h + in_page * a.c_s;
    scale = (u.key ? a.k_scales : a.v_scales) + (((int64_t)layer * a.pages + p) * a.kv_heads + u.g) * nb + in_scales;
    return page >= 0;
  };
  // whether any row of the tokens [t0, t1) goes to the cache (an accepted path may leave rows out)
  auto any_row = [&](int t0, int t1) {
    if (!path) return t0 < count;
    bool any = false;
    for (int t = t0 + lane; t < t1; t += 32) any |= source(t) >= 0;
    return __any_sync(0xffffffffu, any) != 0;
  };
  if (a.group <= a.chunk) {  // the blocks' rows are held
    auto span = [&](const Unit& u, int& t0) {  // its tokens
      t0 = max(u.p0 - len, 0);
      return min(u.p0 + a.block - len, j1) - t0;
    };
    auto fetch_unit = [&](int z, int buf) {
      int t0;
      const Unit u = unit_of(min(z, units - 1));
      const int n = span(u, t0);
      fetch(u, t0, z < u1 ? n : 0, buf);
    };
    fetch_unit(u0 + warp, 0);  // on their way while the queries are turned
    if (a.q) {
      rows(j0, j1 - j0, false);
    } else {
      fill_angles(j0, j1 - j0);
      __syncthreads();
    }
    int buf = 0;
    for (int z = u0 + warp; z < u1; z += kWarps) {
      const Unit u = unit_of(z);
      int t0;
      const int n = span(u, t0);
      if (a.two) {
        fetch_unit(z + kWarps, buf ^ 1);
        copies_landed<1>();
      } else {
        copies_landed<0>();
      }
      __syncwarp();
      if (n > 0) {
        uint8_t *rows8, *scale;
        const bool there = place(u, rows8, scale) && any_row(t0, t0 + n);
        const uint32_t top = largest(u, t0, n, j0, buf);
        if (there) write(u, t0, n, j0, buf, rows8, settle(u, top, rows8, scale));
      }
      __syncwarp();  // the buffer is read
      if (a.two) buf ^= 1;
      else fetch_unit(z + kWarps, 0);
    }
    return;
  }
  // Long blocks, one to a group: once through the tokens for the largest magnitudes, once more for
  // the codes. A warp keeps its units' magnitudes.
  __shared__ uint32_t s_top[2 * 256];
  for (int z = u0 + tid; z < u1; z += kThreads) s_top[z - u0] = 0u;
  for (int pass = 0; pass < 2; ++pass) {
    for (int c0 = j0; c0 < j1; c0 += a.chunk) {
      const int n = min(a.chunk, j1 - c0);
      __syncthreads();
      if (pass == 0 && a.q) {
        rows(c0, n, false);
      } else {
        fill_angles(c0, n);
        __syncthreads();
      }
      for (int z = u0 + warp; z < u1; z += kWarps) {
        const Unit u = unit_of(z);
        uint8_t *rows8, *scale;
        const bool there = place(u, rows8, scale) && any_row(j0, j1);
        if (pass == 1 && !there) continue;
        fetch(u, c0, n, 0);
        copies_landed<0>();
        __syncwarp();
        if (pass == 0) {
          const uint32_t top = max(largest(u, c0, n, c0, 0), s_top[z - u0]);
          __syncwarp();
          if (lane == 0) s_top[z - u0] = top;
        } else {
          int code;
          if (c0 == j0) code = settle(u, s_top[z - u0], rows8, scale);
          else code = *scale;
          write(u, c0, n, c0, 0, rows8, code);
        }
        __syncwarp();
      }
    }
  }
}

// ------------------------------------------------------------------ host

template <auto Kernel>
int launch_kernel(const RotaryArgs& a, dim3 grid, size_t smem, cudaStream_t st, const char* op) {
  // per device: the shared memory attribute is set (idempotent), for every call: 48 KB without it are together with the
  // kernel's own 2 KB
  static std::atomic<bool> set[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  }
  return launch_pdl(Kernel, grid, dim3(kThreads), smem, st, op, a);
}

// Vectors of 16 bytes, or of 8 where the half layout's pairs are not so many bytes apart.
template <typename T, int KIND>
int launch_rotary(RotaryArgs& a, bool interleaved, cudaStream_t st, const char* op) {
  constexpr int full = 16 / (int)sizeof(T);
  const int ve = interleaved || a.half % full == 0 ? full : 4;
  const int items = interleaved ? a.d / ve : a.half / ve + (a.d - 2 * a.half) / ve;
  const int64_t sequences = (int64_t)a.batch * a.layers;
  if (KIND == kBits8) {
    // 16 tokens to a thread block where the cache's blocks are short
    const int subs = std::max(1, 16 / a.block);
    const int row_bytes = a.d * (int)sizeof(T), held = std::min(kMaxTokens, kHeld / row_bytes);
    a.group = a.block <= held ? a.block * subs : a.block;
    a.chunk = a.group <= kMaxTokens ? (a.block <= held ? a.group : held) : held;
    a.groups = (a.tokens + a.group - 2) / a.group + 1;
    a.buffer = std::min(a.block, held) * row_bytes;
    a.two = a.buffer <= kHeld / 2;
  } else {
    // Tokens share a thread block's launch and the angles' latency where there are enough of them.
    a.group = 1;
    while (a.group < 8 && sequences * a.tokens >= 2LL * a.group * 4 * sm_count()) a.group *= 2;
    a.chunk = a.group;
    a.groups = (a.tokens + a.group - 1) / a.group;
  }
  const int64_t blocks = sequences * a.groups;
  if (blocks > 0x7fffffffLL) return fail(NKL_ERR_SHAPE, "%s: too many tokens", op);
  // Where thread blocks are few, several share a group's heads, as long as each has rows for its threads.
  const int64_t heads = a.heads + (KIND == kPlain ? 0 : 2 * a.kv_heads);
  a.splits = 1;
  while (a.splits < 16 && blocks * a.splits * 2 <= 2LL * sm_count() && heads * a.group * items >= 2LL * a.splits * kThreads) a.splits *= 2;
  if (KIND == kBits8 && a.group > a.chunk)  // s_top
    while ((2 * a.kv_heads + a.splits - 1) / a.splits > 512) ++a.splits;
  const size_t smem = (size_t)2 * a.chunk * a.half * 4 + (size_t)(a.two + 1) * kWarps * a.buffer;
  const dim3 grid((unsigned)blocks, (unsigned)a.splits);
  if (interleaved) return launch_kernel<rotary_kernel<T, full, true, KIND>>(a, grid, smem, st, op);
  if constexpr (full == 8)
    if (ve == 4) return launch_kernel<rotary_kernel<T, 4, false, KIND>>(a, grid, smem, st, op);
  return launch_kernel<rotary_kernel<T, full, false, KIND>>(a, grid, smem, st, op);
}

template <int KIND>
int launch_rotary(RotaryArgs& a, int interleaved, int dtype, void* stream, const char* op) {
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == NKL_FLOAT32 ? launch_rotary<float, KIND>(a, interleaved != 0, st, op)
                              : launch_rotary<bf16, KIND>(a, interleaved != 0, st, op);
}

// Strides of a tensor (NULL: dense) into `s`, checked to be whole vectors of 16 bytes.
int take_strides(const char* op, const int64_t* given, int n, const int64_t* sizes, int64_t row, int64_t per, int64_t* s) {
  int64_t step = row;
  for (int i = n - 1; i >= 0; --i) {
    s[i] = given ? given[i] : step;
    step *= std::max<int64_t>(sizes[i], 1);
    if (sizes[i] > 1 && (s[i] < 0 || s[i] % per))
      return fail(NKL_ERR_ALIGN, "%s: stride %lld is not a multiple of 16 bytes", op, (long long)s[i]);
  }
  return NKL_OK;
}

bool rotary_sizes_ok(int64_t batch, int64_t tokens, int64_t heads, int64_t d, int64_t r) {
  return batch >= 0 && batch <= 0x7fffffLL && tokens >= 0 && tokens <= kMostTokens && heads >= 1 && heads <= 65535 &&
         d >= 8 && d <= kMaxHead && d % 8 == 0 && r >= 0 && r <= d && r % 8 == 0;
}

bool cache_sizes_ok(int64_t layers, int64_t kv_heads, int64_t pages, int64_t page, int64_t max_pages) {
  return layers >= 1 && layers <= 65535 && kv_heads >= 1 && kv_heads <= 65535 && pages >= 1 && pages <= 0x7fffffffLL &&
         page >= 1 && page <= 65536 && max_pages >= 1 && max_pages * page <= (1LL << 30);
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_rotary(const void* x, const int64_t* x_strides, const int32_t* positions, const int32_t* parents,
                          const double* freqs, void* out, int64_t batch, int64_t tokens, int64_t heads,
                          int64_t head_dim, int64_t rotary_dim, int per_token, int interleaved, int inverse,
                          float magnitude, int dtype, void* stream) {
  const char* op = "nkl_rotary";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (!rotary_sizes_ok(batch, tokens, heads, head_dim, rotary_dim) || rotary_dim == 0)
    return fail(NKL_ERR_SHAPE, "%s: batch %lld, tokens %lld, heads %lld, head_dim %lld or rotary_dim %lld not supported "
                "(multiples of 8, head_dim up to %d)", op, (long long)batch, (long long)tokens, (long long)heads,
                (long long)head_dim, (long long)rotary_dim, kMaxHead);
  if (parents && (per_token || tokens > NKL_MAX_DRAFTED))
    return fail(NKL_ERR_ARG, "%s: a tree has up to %d tokens and one position to a sequence", op, NKL_MAX_DRAFTED);
  if (batch == 0 || tokens == 0) return NKL_OK;
  if (!x || !positions || !freqs || !out) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  for (const void* p : {x, static_cast<const void*>(out)})
    if (!is_aligned(p, 16)) return fail(NKL_ERR_ALIGN, "%s: tensors need 16-byte alignment", op);
  RotaryArgs a = {};
  const int64_t sizes[3] = {batch, tokens, heads};
  int64_t s[3];
  if (int rc = take_strides(op, x_strides, 3, sizes, head_dim, 16 / (int64_t)dtype_size(dtype), s)) return rc;
  a.q = x; a.q_out = out; a.positions = positions; a.parents = parents; a.freqs = freqs;
  a.q_b = s[0]; a.q_t = s[1]; a.q_h = s[2];
  a.batch = (int)batch; a.tokens = (int)tokens; a.heads = (int)heads; a.d = (int)head_dim; a.half = (int)(rotary_dim / 2);
  a.layers = 1; a.per_token = per_token; a.inverse = inverse; a.magnitude = magnitude;
  return launch_rotary<kPlain>(a, interleaved, dtype, stream, op);
}

extern "C" int nkl_rotary_append(const void* q, const int64_t* q_strides, const void* k, const void* v,
                                 const int64_t* kv_strides, void* k_cache, void* v_cache, const int64_t* cache_strides,
                                 void* k_scales, void* v_scales, const int32_t* tables, const int32_t* lens,
                                 const int32_t* count, const double* freqs, void* q_out, void* k_out, int64_t batch,
                                 int64_t tokens, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t rotary_dim,
                                 int64_t pages, int64_t page_size, int64_t max_pages, int64_t block, int interleaved,
                                 float magnitude, int dtype, void* stream) {
  const char* op = "nkl_rotary_append";
  const bool bits8 = k_scales || v_scales;
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (!rotary_sizes_ok(batch, tokens, heads, head_dim, rotary_dim) || rotary_dim == 0 ||
      !cache_sizes_ok(1, kv_heads, pages, page_size, max_pages) ||
      (bits8 && (head_dim % 16 || head_dim > kMaxHead8 || block < 1 || page_size % block)))
    return fail(NKL_ERR_SHAPE, "%s: batch %lld, tokens %lld, heads %lld / %lld, head_dim %lld, rotary_dim %lld, page size "
                "%lld, table width %lld or block %lld not supported (multiples of 8, head_dim up to %d; in 8 bits "
                "multiples of 16 up to %d, blocks divide pages)", op, (long long)batch, (long long)tokens, (long long)heads,
                (long long)kv_heads, (long long)head_dim, (long long)rotary_dim, (long long)page_size,
                (long long)max_pages, (long long)block, kMaxHead, kMaxHead8);
  if (batch == 0 || tokens == 0) return NKL_OK;
  if (!q || !k || !v || !k_cache || !v_cache || !tables || !lens || !freqs || !q_out || !k_out || (bits8 && (!k_scales || !v_scales)))
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  for (const void* p : {q, k, v, static_cast<const void*>(k_cache), static_cast<const void*>(v_cache),
                        static_cast<const void*>(q_out), static_cast<const void*>(k_out)})
    if (!is_aligned(p, 16)) return fail(NKL_ERR_ALIGN, "%s: tensors need 16-byte alignment", op);
  RotaryArgs a = {};
  const int64_t per = 16 / (int64_t)dtype_size(dtype);
  int64_t s[3], n[3], c[3];
  const int64_t qs[3] = {batch, tokens, heads}, ns[3] = {batch, tokens, kv_heads}, cs[3] = {pages, kv_heads, page_size};
  if (int rc = take_strides(op, q_strides, 3, qs, head_dim, per, s)) return rc;
  if (int rc = take_strides(op, kv_strides, 3, ns, head_dim, per, n)) return rc;
  if (int rc = take_strides(op, cache_strides, 3, cs, head_dim, bits8 ? 16 : per, c)) return rc;
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.k_out = k_out; a.k_cache = k_cache; a.v_cache = v_cache;
  a.k_scales = static_cast<uint8_t*>(k_scales); a.v_scales = static_cast<uint8_t*>(v_scales);
  a.tables = tables; a.lens = lens; a.count = count; a.freqs = freqs;
  a.q_b = s[0]; a.q_t = s[1]; a.q_h = s[2];
  a.n_b = n[0]; a.n_t = n[1]; a.n_h = n[2];
  a.c_p = c[0]; a.c_h = c[1]; a.c_s = c[2];
  a.batch = (int)batch; a.tokens = (int)tokens; a.heads = (int)heads; a.kv_heads = (int)kv_heads; a.d = (int)head_dim;
  a.half = (int)(rotary_dim / 2); a.layers = 1; a.pages = (int)pages; a.page = (int)page_size;
  a.max_pages = (int)max_pages; a.block = (int)block; a.magnitude = magnitude;
  return bits8 ? launch_rotary<kBits8>(a, interleaved, dtype, stream, op)
               : launch_rotary<kSame>(a, interleaved, dtype, stream, op);
}

extern "C" int nkl_cache_append_8bit(const void* k, const void* v, const int64_t* kv_strides, void* k_cache,
                                     void* v_cache, const int64_t* cache_strides, void* k_scales, void* v_scales,
                                     const int32_t* tables, const int32_t* lens, const int32_t* path,
                                     const int32_t* count, int32_t* lens_out, int64_t layers, int64_t batch,
                                     int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t pages,
                                     int64_t page_size, int64_t max_pages, int64_t block, int dtype, void* stream) {
  const char* op = "nkl_cache_append_8bit";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (!rotary_sizes_ok(batch, tokens, 1, head_dim, 0) || !cache_sizes_ok(layers, kv_heads, pages, page_size, max_pages) ||
      head_dim % 16 || head_dim > kMaxHead8 || block < 1 || page_size % block)
    return fail(NKL_ERR_SHAPE, "%s: layers %lld, batch %lld, tokens %lld, kv heads %lld, head_dim %lld, page size %lld, table "
                "width %lld or block %lld not supported (head_dim a multiple of 16 up to %d, blocks divide pages)", op,
                (long long)layers, (long long)batch, (long long)tokens, (long long)kv_heads, (long long)head_dim,
                (long long)page_size, (long long)max_pages, (long long)block, kMaxHead8);
  if (batch == 0) return NKL_OK;
  if ((tokens && (!k || !v)) || !k_cache || !v_cache || !k_scales || !v_scales || !tables || !lens || !lens_out)
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  for (const void* p : {k, v, static_cast<const void*>(k_cache), static_cast<const void*>(v_cache)})
    if (!is_aligned(p, 16)) return fail(NKL_ERR_ALIGN, "%s: tensors need 16-byte alignment", op);
  RotaryArgs a = {};
  int64_t n[4], c[4];
  const int64_t ns[4] = {layers, batch, tokens, kv_heads}, cs[4] = {layers, pages, kv_heads, page_size};
  if (int rc = take_strides(op, kv_strides, 4, ns, head_dim, 16 / (int64_t)dtype_size(dtype), n)) return rc;
  if (int rc = take_strides(op, cache_strides, 4, cs, head_dim, 16, c)) return rc;
  a.k = k; a.v = v; a.k_cache = k_cache; a.v_cache = v_cache;
  a.k_scales = static_cast<uint8_t*>(k_scales); a.v_scales = static_cast<uint8_t*>(v_scales);
  a.tables = tables; a.lens = lens; a.path = path; a.count = count; a.lens_out = lens_out;
  a.n_l = n[0]; a.n_b = n[1]; a.n_t = n[2]; a.n_h = n[3];
  a.c_l = c[0]; a.c_p = c[1]; a.c_h = c[2]; a.c_s = c[3];
  a.batch = (int)batch; a.tokens = (int)tokens; a.kv_heads = (int)kv_heads; a.d = (int)head_dim;
  a.layers = (int)layers; a.pages = (int)pages; a.page = (int)page_size; a.max_pages = (int)max_pages;
  a.block = (int)block; a.magnitude = 1.f;
  return launch_rotary<kBits8>(a, 0, dtype, stream, op);
}
