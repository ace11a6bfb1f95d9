// tree_attention_8bit.cuh - the tree attention over a cache in 8 bits, by mma.sync; included by
// tree_attention.cu.
//
// Cached k and v are e4m3 numbers with a power of two for each block of positions and head. They go
// from global memory into registers, 16 bytes to a lane, and from there, as f16 (which has every
// e4m3 number), into the products, without shared memory and without barriers. Both products have the
// cache's values as their first operand, 16 rows high, and 8 query rows as their second, so that a decoding
// step's few rows waste little:
//   S^T = K Q^T      the lanes of a row hold other entries of a head than the fragment's layout says, in
//                    Q and K alike, so that a lane's 16 bytes of K are the fragments of four products
//   O^T += V^T P^T   two keys' bytes are interleaved to pairs; a lane's 16 bytes of a key are its rows of eight
//                    products, and it ends up with 16 entries in a row of O. P is transposed by movmatrix
// A warp meets its 8 or 16 query rows with one window of 32 keys after the other, the windows
// dealt out over a block's warps; their (max, sum, O) meet in shared memory, those of several blocks
// in the workspace (tree_combine_kernel).
//
// Powers of two: K's multiply the scores. V's move the exponent of the weights, p 2^e, before these
// are rounded to f16, which therefore have a maximum of their own, beside that of the scores. Q is
// scaled by a power of two per row, so that f16 holds it; fp32 queries and weights are two f16
// numbers. Both maxima may lag behind by 2^8: sums are rescaled when a row's grow by more.
// The drafted tokens' own k and v multiply in bf16, fp32 ones in three parts.
//
// This kernel takes fp32 and the bf16 layouts that neither tree_attention_8bit_ring.cuh (up to 16 query rows to a
// key/value head) nor tree_attention_tc.cuh does. Measured, fp32: 1 token, 16 sequences of up to 4000, 32 heads over 8 of
// 128 67 us (15 by bytes), 7 tokens, 5 of up to 1999, 8 heads over 4 of 64 24 us: queries and weights are two f16 numbers
// each, so that a product is two, or three with the first's rest; bf16, 3 tokens, 4 of up to 3000, 12 heads over 4 of 80
// 18 us. What bounds it is issue: converting and interleaving a tile costs more than its products.
#pragma once

namespace {

constexpr int kThreads8 = 128;
constexpr int kWarps8 = kThreads8 / 32;
constexpr int kWindow = 32;     // keys that a warp looks up at a time
constexpr float kLag8 = 8.f;    // log2 of how far the maxima may lag
constexpr float kRaise = 6.f;   // weights are up to 2^(kLag8 + kRaise): f16 ends at 2^16, and below 2^-14 it loses bits
static_assert(kLag8 + kRaise < 16.f, "weights for O are f16 numbers");

struct Bits8Args {
  TreeArgs t;  // c_p, c_h, c_s: in bytes
  const uint8_t *k_scales, *v_scales;
  int block, per_page;  // positions of a block, blocks of a page
  int tiles;            // of 8 NT query rows, which a block's warps share
};

// Four e4m3 numbers as two pairs of f16.
__device__ __forceinline__ void e4m3_pairs(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n .reg .b16 x, y;\n mov.b32 {x, y}, %2;\n cvt.rn.f16x2.e4m3x2 %0, x;\n cvt.rn.f16x2.e4m3x2 %1, y;\n}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
// An 8 x 8 matrix, row g at the lanes 4 g .. 4 g + 3, transposed.
__device__ __forceinline__ uint32_t transpose(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_b16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t half_pair(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What rounding left of two numbers; of infinities and NaN nothing.
__device__ __forceinline__ float2 rest_half(uint32_t h, float lo, float hi) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  return make_float2(fabsf(lo) < INFINITY ? lo - f.x : 0.f, fabsf(hi) < INFINITY ? hi - f.y : 0.f);
}
__device__ __forceinline__ float2 rest_bf16(uint32_t h, float lo, float hi) {
  const float x = __uint_as_float(h << 16), y = __uint_as_float(h & 0xffff0000u);
  return make_float2(fabsf(x) < INFINITY ? lo - x : 0.f, fabsf(y) < INFINITY ? hi - y : 0.f);
}
// Two numbers as bf16 pairs, N parts that add up to them.
template <int N>
__device__ __forceinline__ void bf16_parts(float lo, float hi, uint32_t (&p)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    p[i] = bf16_pair(lo, hi);
    if (N == 3 && i == 0) {  // near the largest numbers the first part is cut off, not rounded
      if (((p[0] & 0x7fffu) == 0x7f80u) && fabsf(lo) < INFINITY) p[0] = (p[0] & 0xffff0000u) | (__float_as_uint(lo) >> 16);
      if (((p[0] & 0x7fff0000u) == 0x7f800000u) && fabsf(hi) < INFINITY) p[0] = (p[0] & 0xffffu) | (__float_as_uint(hi) & 0xffff0000u);
    }
    const float2 r = rest_bf16(p[i], lo, hi);
    lo = r.x;
    hi = r.y;
  }
}

// 2^x for a whole number, 0 below 2^-126.
constexpr float kRound = 12582912.f;  // 1.5 2^23: added, it rounds to whole numbers
__device__ __forceinline__ float power2(float x) {
  return __uint_as_float(__float_as_uint(fminf(fmaxf(x, -127.f), 127.f) + (kRound + 127.f)) << 23);
}

// The sums of a lane: rows 2 t4 and 2 t4 + 1 (the last index of m, mv, l) of NT tiles of 8 query rows. m: the
// rows' reference for sums l of 2^(s - m), over the lane's keys; mv: that for O, sums of 2^(s + e - mv + kRaise) v. Both
// are whole numbers (of a maximum that is over the lag; if the whole number below it had to be, a row whose maximum lies
// between would look for it at every tile: 18 sequences of 8192, 73.7 us for 66.4), and a power of two comes to a weight by its exponent alone: the weights' bits do not depend on how a
// block's numbers are shared out between e4m3 codes and their power of two, which changes when the block grows.
// O's products j hold two entries of a head: o[t][j][i] and o[t][j][2 + i].
template <int NT, int DC>
struct Sums8 {
  float m[NT][2], mv[NT][2], l[NT][2], o[NT][4 * DC][4];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = mv[t][0] = mv[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int j = 0; j < 4 * DC; ++j) o[t][j][0] = o[t][j][1] = o[t][j][2] = o[t][j][3] = 0.f;
    }
  }
  // Weights of 16 keys: x[t][2 k + i] the score of key 8 k + g with row 2 t4 + i of tile t, e[k] the key's power of
  // two for O. Comes back with x the weights for O.
  __device__ __forceinline__ void weigh(float (&x)[NT][4], const float (&e)[2]) {
    bool grows = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) grows |= x[t][2 * k + i] > m[t][i] + kLag8 || x[t][2 * k + i] + e[k] > mv[t][i] + kLag8;
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float top = fmaxf(x[t][i], x[t][2 + i]), tv = fmaxf(x[t][i] + e[0], x[t][2 + i] + e[1]);
#pragma unroll
          for (int z = 4; z < 32; z *= 2) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
            tv = fmaxf(tv, __shfl_xor_sync(0xffffffffu, tv, z));
          }
          const bool over = top > m[t][i] + kLag8, over_v = tv > mv[t][i] + kLag8;
          top = floorf(top);
          tv = floorf(tv);
          if (over) {  // a row goes by its own scores alone
            l[t][i] *= fast_exp2(m[t][i] - top);
            m[t][i] = top;
          }
          float f = 1.f;
          if (over_v) {
            f = fast_exp2(mv[t][i] - tv);
            mv[t][i] = tv;
          }
#pragma unroll
          for (int j = 0; j < 4 * DC; ++j) {
            o[t][j][i] *= f;
            o[t][j][2 + i] *= f;
          }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float rm = m[t][i] == -INFINITY ? 0.f : m[t][i], rv = mv[t][i] == -INFINITY ? 0.f : mv[t][i] - kRaise;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float& s = x[t][2 * k + i];
          const float z = s - rm, d = e[k] + (rm - rv), p = fast_exp2(z);
          l[t][i] += p;
          if (d <= 100.f) {  // where p is 0, so is p 2^d in f16
            s = p * power2(d);
          } else {  // v's block has by far the largest numbers: p may be 0 too early; or d is NaN
            const float least = z < -2000.f ? -2000.f : z, whole = least + kRound - kRound;
            s = (fast_exp2(least - whole) + (d - d)) * power2(whole + d);
          }
        }
      }
  }
};

// Four consecutive numbers as they lie, and in fp32.
template <typename T> struct Four;
template <> struct Four<float> { typedef float4 type; };
template <> struct Four<bf16> { typedef uint2 type; };
__device__ __forceinline__ float4 in_f32(float4 x) { return x; }
__device__ __forceinline__ float4 in_f32(uint2 w) {
  return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                     __uint_as_float(w.y & 0xffff0000u));
}
// Loads without branches, so that they go out together: where `there` does not hold, `any` is read and zeros come back.
template <typename T>
__device__ __forceinline__ typename Four<T>::type load_four(const T* p, bool there, const T* any) {
  typename Four<T>::type x = *reinterpret_cast<const typename Four<T>::type*>(there ? p : any);
  if (!there) x = typename Four<T>::type{};
  return x;
}
__device__ __forceinline__ float2 load_two(const float* p, bool there, const float* any) {
  const float2 x = *reinterpret_cast<const float2*>(there ? p : any);
  return there ? x : make_float2(0.f, 0.f);
}
__device__ __forceinline__ float2 load_two(const bf16* p, bool there, const bf16* any) {
  const uint32_t w = *reinterpret_cast<const uint32_t*>(there ? p : any);
  return there ? make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)) : make_float2(0.f, 0.f);
}
__device__ __forceinline__ float4 four_of(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 four_of(const bf16* p) { return in_f32(*reinterpret_cast<const uint2*>(p)); }

// The drafted tokens first, first + 1, .. (16 at a time, then the ones `step` further on) against a warp's rows r0
// .. r0 + 8 NT - 1 of a key/value head: query(r, real) says where row r's q lies and whether it is one, entry(s) where
// the lane's four entries of product s are, col(j) its two of O's product j. Returns whether a v was not finite.
template <typename T, int NT, int DC, typename Query, typename Entry, typename Col>
__device__ __forceinline__ bool drafted_8bit(const TreeArgs& a, int b, int kvh, int r0, int first, int step, Query query,
                                             Entry entry, Col col, Sums8<NT, DC>& sums) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kParts = kF32 ? 3 : 1;   // of k and v, in bf16
  constexpr int kPParts = kF32 ? 3 : 2;  // of the weights
  const int lane = threadIdx.x & 31, g = lane >> 2, t4 = lane & 3;
  const int* const parents = a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  const T* const kn = static_cast<const T*>(a.k_new) + b * a.n_b + kvh * a.n_h;
  const T* const vn = static_cast<const T*>(a.v_new) + b * a.n_b + kvh * a.n_h;
  bool bad = false;
#pragma unroll 1
  for (int k0 = first; k0 < a.tokens; k0 += step) {
    float x[NT][4] = {};
    const T* qp[NT];
    bool real[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) qp[t] = query(8 * t + g, real[t]);
#pragma unroll
    for (int s0 = 0; s0 < 4 * DC; s0 += 4) {  // four products' loads at a time
      typename Four<T>::type kr[4][2], qr[4][NT];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int e = entry(s0 + s);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int key = k0 + 8 * k + g;
          kr[s][k] = load_four(kn + key * a.n_t + e, key < a.tokens && e < a.d, kn);
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) qr[s][t] = load_four(qp[t] + e, real[t] && e < a.d, qp[t]);
      }
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        uint32_t ka[kParts][4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float4 y = in_f32(kr[s][k]);
          uint32_t p[kParts];
          bf16_parts(y.x, y.y, p);
#pragma unroll
          for (int z = 0; z < kParts; ++z) ka[z][k] = p[z];
          bf16_parts(y.z, y.w, p);
#pragma unroll
          for (int z = 0; z < kParts; ++z) ka[z][2 + k] = p[z];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const float4 y = in_f32(qr[s][t]);
          uint32_t q0[kParts], q1[kParts];
          bf16_parts(y.x, y.y, q0);
          bf16_parts(y.z, y.w, q1);
#pragma unroll
          for (int sum = kParts - 1; sum >= 0; --sum)  // the smallest products first
#pragma unroll
            for (int z = 0; z <= sum; ++z) mma_b16(x[t], ka[z], q0[sum - z], q1[sum - z]);
        }
      }
    }
    const float none[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * t + 2 * t4 + i;
        bool there;
        const T* const row = query(r, there);
        uint32_t w[4] = {0u, 0u, 0u, 0u};
        if (there) ancestor_bits(parents, (r0 + r) / a.group, w);
        const int word = k0 >> 5;
        const uint32_t bits = word == 0 ? w[0] : word == 1 ? w[1] : word == 2 ? w[2] : w[3];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int key = k0 + 8 * k + g;
          float& y = x[t][2 * k + i];
          // an infinity's product with a part that is zero is no part of its product
          if (kF32 && !(fabsf(y) < INFINITY) && there && key < a.tokens) {
            y = 0.f;
            for (int c = 0; c < a.d; ++c) y = fmaf(to_f32(row[c]), to_f32(kn[key * a.n_t + c]), y);
          }
          y = (bits >> (key & 31)) & 1u ? y * (a.scale * kLog2e) : -INFINITY;
        }
      }
    sums.weigh(x, none);
    uint32_t p[NT][kPParts][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        uint32_t y[kPParts];
        bf16_parts(x[t][2 * k], x[t][2 * k + 1], y);
#pragma unroll
        for (int z = 0; z < kPParts; ++z) p[t][z][k] = transpose(y[z]);
      }
    bool here[4];  // an absent token's v is left out
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k0 + 2 * t4 + (i & 1) + 8 * (i >> 1);
      here[i] = key < a.tokens && (!parents || parents[key] >= -1);
    }
#pragma unroll
    for (int j0 = 0; j0 < 4 * DC; j0 += 4) {
      float2 v[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 2 * t4 + (i & 1) + 8 * (i >> 1), c = col(j0 + j);
          v[j][i] = load_two(vn + key * a.n_t + c, here[i] && c < a.d, vn);
        }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // weights of 0 must meet no infinity, which is put in at the end
          if (!(fabsf(v[j][i].x) < INFINITY)) {
            bad = true;
            v[j][i].x = 0.f;
          }
          if (!(fabsf(v[j][i].y) < INFINITY)) {
            bad = true;
            v[j][i].y = 0.f;
          }
        }
        uint32_t va[kParts][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // keys 2 t4, 2 t4 + 1 (i < 2) or 8 more, the first entry or the second
          uint32_t y[kParts];
          const float2 p = v[j][2 * (i >> 1)], q = v[j][2 * (i >> 1) + 1];
          bf16_parts((i & 1) ? p.y : p.x, (i & 1) ? q.y : q.x, y);
#pragma unroll
          for (int q2 = 0; q2 < kParts; ++q2) va[q2][i] = y[q2];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int sum = (kF32 ? 2 : 1); sum >= 0; --sum)
#pragma unroll
            for (int q = 0; q < kParts && q <= sum; ++q)
              mma_b16(sums.o[t][j0 + j], va[q], p[t][sum - q][0], p[t][sum - q][1]);
      }
    }
  }
  return bad;
}

// A warp's query rows as the second operand of the products: row g of each tile, scaled by a power of two so that
// f16 holds it, and (fp32) what that leaves of it; factor: of the scores of the rows 2 t4 and 2 t4 + 1.
template <typename T, int NT, int DC>
struct Queries8 {
  static constexpr bool kF32 = sizeof(T) == 4;
  uint32_t hi[NT][4 * DC][2], lo[NT][kF32 ? 4 * DC : 1][2];
  float factor[NT][2];
  typename Four<T>::type raw[NT][4 * DC];  // as they lie
  template <typename Query, typename Entry>
  __device__ __forceinline__ void fetch(const TreeArgs& a, Query query, Entry entry) {
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      bool real;
      const T* const qp = query(8 * t + ((threadIdx.x & 31) >> 2), real);
#pragma unroll
      for (int s = 0; s < 4 * DC; ++s) raw[t][s] = load_four(qp + entry(s), real && entry(s) < a.d, qp);
    }
  }
  __device__ __forceinline__ void turn(const TreeArgs& a) {
    const int t4 = threadIdx.x & 3;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float top = 0.f;
#pragma unroll
      for (int s = 0; s < 4 * DC; ++s) {
        const float4 x = in_f32(raw[t][s]);
        for (float y : {x.x, x.y, x.z, x.w}) top = fmaxf(top, fabsf(y) < INFINITY ? fabsf(y) : 0.f);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max((int)(__float_as_uint(top) >> 23) - 127, -112);  // 2^e <= top
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
      const float f = a.scale * kLog2e * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
      factor[t][0] = __shfl_sync(0xffffffffu, f, 8 * t4);
      factor[t][1] = __shfl_sync(0xffffffffu, f, 8 * t4 + 4);
#pragma unroll
      for (int s = 0; s < 4 * DC; ++s) {
        float4 x = in_f32(raw[t][s]);
        x = make_float4(x.x * up, x.y * up, x.z * up, x.w * up);
        hi[t][s][0] = half_pair(x.x, x.y);
        hi[t][s][1] = half_pair(x.z, x.w);
        if constexpr (kF32) {
          const float2 u = rest_half(hi[t][s][0], x.x, x.y), v = rest_half(hi[t][s][1], x.z, x.w);
          lo[t][s][0] = half_pair(u.x, u.y);
          lo[t][s][1] = half_pair(v.x, v.y);
        }
      }
    }
  }
};

// DC: head_dim up to 64 DC. FAST: pages and blocks are multiples of 16 positions, so that the 16 keys of a
// product lie in a row and share their powers of two. NT: tiles of 8 query rows to a warp.
template <typename T, int DC, bool FAST, int NT>
__global__ void __launch_bounds__(kThreads8, NT == 1 && sizeof(T) == 2 ? 4 : 2)
attention_8bit_kernel(const __grid_constant__ Bits8Args args) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kCols = 8 * DC;          // entries of V that a lane has of a key
  constexpr int kRowsW = 8 * NT;         // a warp's query rows
  extern __shared__ __align__(16) float joined[];
  __shared__ int s_bad;                  // a drafted v that is not finite
  const TreeArgs& a = args.t;
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int tile = warp % args.tiles, stream = warp / args.tiles, streams = kWarps8 / args.tiles;
  const int rows = a.tokens * a.group, r0 = (rb * args.tiles + tile) * kRowsW;
  const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
  const int windows = (n + kWindow - 1) / kWindow, per = (windows + a.splits - 1) / a.splits;
  const int w0 = min(split * per, windows), w1 = min(w0 + per, windows);
  const int* const parents = a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // Query row r of the warp's: where it lies, and whether it is one (an absent token's is not looked at).
  auto query = [&](int r, bool& real) {
    const int row = r0 + r, token = row / a.group;
    real = row < rows && (!parents || parents[token] >= -1);
    return static_cast<const T*>(a.q) + b * a.q_b + (real ? token * a.q_t + (kvh * a.group + row - token * a.group) * a.q_h : 0);
  };
  // Four consecutive entries of the lane's: step s takes those at entry(s).
  auto entry = [&](int s) { return (t4 + 4 * (s >> 2)) * 16 + (s & 3) * 4; };
  Queries8<T, NT, DC> q;
  q.fetch(a, query, entry);
  q.turn(a);

  Sums8<NT, DC> rows_of_sums;
  rows_of_sums.clear();
  auto& m = rows_of_sums.m;
  auto& mv = rows_of_sums.mv;
  auto& l = rows_of_sums.l;
  auto& o = rows_of_sums.o;

  auto col = [&](int j) { return g * kCols + 2 * j; };
  if (split == a.splits - 1 && drafted_8bit<T, NT, DC>(a, b, kvh, r0, stream * 16, streams * 16, query, entry, col, rows_of_sums))
    s_bad = 1;

  // ------------------------------------------------ the cached keys
  const uint8_t* const kc = static_cast<const uint8_t*>(a.k_cache);
  const uint8_t* const vc = static_cast<const uint8_t*>(a.v_cache);
  // What a lane finds out about one key of a window: where its rows lie (-1: nowhere, they read as
  // zeros), k's power of two, and the exponent of v's.
  struct Found {
    int64_t at;
    float ks, ve;
  };
  auto page_of = [&](int w) {
    const int key = w * kWindow + lane;
    if (w >= w1 || key >= n) return -1;
    const int p = a.tables[(int64_t)b * a.max_pages + key / a.page];
    return p >= 0 && p < a.pages ? p : -1;
  };
  auto look_up = [&](int w, int p) {
    Found f = {-1, 1.f, 0.f};
    if (p < 0) return f;
    const int slot = (w * kWindow + lane) % a.page;
    const int64_t at = ((int64_t)p * a.kv_heads + kvh) * args.per_page + slot / args.block;
    const int ks = args.k_scales[at], vs = args.v_scales[at];
    f.at = p * a.c_p + kvh * a.c_h + slot * a.c_s;
    f.ks = ks == 255 ? NAN : ks == 0 ? 5.877472e-39f : __uint_as_float((uint32_t)ks << 23);  // 2^-127: below the normal numbers
    f.ve = vs == 255 ? NAN : (float)(vs - 127);
    return f;
  };
  struct Keys {
    uint4 k[2][DC], v[4];  // K of keys g, g + 8; V of keys 2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9 (8 bytes if DC is 1)
  };
  auto load_v = [&](const uint8_t* p, bool there) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (there && g * kCols < a.d) {
      if constexpr (DC == 2) {
        x = *reinterpret_cast<const uint4*>(p + g * 16);
      } else {
        const uint2 y = *reinterpret_cast<const uint2*>(p + g * 8);
        x.x = y.x;
        x.y = y.y;
      }
    }
    return x;
  };
  // Group h (0 or 1) of 16 keys of the window w that `f` describes.
  auto fetch = [&](const Found& f, int w, int h, Keys& x) {
    const int left = n - w * kWindow - 16 * h;  // keys there
    const int64_t base = FAST ? __shfl_sync(0xffffffffu, f.at, 16 * h) : 0;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int key = 8 * k + g;
      const int64_t at = FAST ? base + key * a.c_s : __shfl_sync(0xffffffffu, f.at, 16 * h + key);
      const bool there = w < w1 && key < left && (FAST ? base : at) >= 0;
#pragma unroll
      for (int c = 0; c < DC; ++c)
        x.k[k][c] = there && (t4 + 4 * c) * 16 < a.d ? *reinterpret_cast<const uint4*>(kc + at + (t4 + 4 * c) * 16) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 2 * t4 + (i & 1) + 8 * (i >> 1);
      const int64_t at = FAST ? base + key * a.c_s : __shfl_sync(0xffffffffu, f.at, 16 * h + key);
      x.v[i] = load_v(vc + at, w < w1 && key < left && (FAST ? base : at) >= 0);
    }
  };
  auto meet = [&](const Found& f, int w, int h, const Keys& x) {
    const int left = n - w * kWindow - 16 * h;
    if (left <= 0) return;
    float s[NT][4] = {};
#pragma unroll
    for (int c = 0; c < DC; ++c) {
      const uint32_t k0[4] = {x.k[0][c].x, x.k[0][c].y, x.k[0][c].z, x.k[0][c].w};
      const uint32_t k1[4] = {x.k[1][c].x, x.k[1][c].y, x.k[1][c].z, x.k[1][c].w};
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        uint32_t ka[4];
        e4m3_pairs(k0[z], ka[0], ka[2]);
        e4m3_pairs(k1[z], ka[1], ka[3]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (kF32) mma_f16(s[t], ka, q.lo[t][4 * c + z][0], q.lo[t][4 * c + z][1]);
          mma_f16(s[t], ka, q.hi[t][4 * c + z][0], q.hi[t][4 * c + z][1]);
        }
      }
    }
    float e[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int key = 8 * k + g, from = 16 * h + (FAST ? 0 : key);
      const float ks = __shfl_sync(0xffffffffu, f.ks, from), ve = __shfl_sync(0xffffffffu, f.ve, from);
      e[k] = key < left ? ve : 0.f;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) s[t][2 * k + i] = key < left ? s[t][2 * k + i] * q.factor[t][i] * ks : -INFINITY;
    }
    rows_of_sums.weigh(s, e);
    uint32_t p[NT][2], pl[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t y = half_pair(s[t][2 * k], s[t][2 * k + 1]);
        p[t][k] = transpose(y);
        if constexpr (kF32) {
          const float2 r = rest_half(y, s[t][2 * k], s[t][2 * k + 1]);
          pl[t][k] = transpose(half_pair(r.x, r.y));
        }
      }
    const uint32_t vw[4][4] = {{x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w}, {x.v[1].x, x.v[1].y, x.v[1].z, x.v[1].w},
                               {x.v[2].x, x.v[2].y, x.v[2].z, x.v[2].w}, {x.v[3].x, x.v[3].y, x.v[3].z, x.v[3].w}};
#pragma unroll
    for (int z = 0; z < kCols / 4; ++z)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t va[4];
        e4m3_pairs(__byte_perm(vw[0][z], vw[1][z], y ? 0x7362 : 0x5140), va[0], va[1]);
        e4m3_pairs(__byte_perm(vw[2][z], vw[3][z], y ? 0x7362 : 0x5140), va[2], va[3]);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (kF32) mma_f16(o[t][2 * z + y], va, pl[t][0], pl[t][1]);
          mma_f16(o[t][2 * z + y], va, p[t][0], p[t][1]);
        }
      }
  };
  {
    // The table entry of a window is read two windows ahead, the powers of two one ahead, the rows half
    // a window ahead.
    int w = w0 + stream;
    Found now = look_up(w, page_of(w));
    int next_page = page_of(w + streams);
    Keys x, y;
    if (w < w1) fetch(now, w, 0, x);
#pragma unroll 1
    for (; w < w1; w += streams) {
      const Found next = look_up(w + streams, next_page);
      next_page = page_of(w + 2 * streams);
      fetch(now, w, 1, y);
      meet(now, w, 0, x);
      fetch(next, w + streams, 0, x);
      meet(now, w, 1, y);
      now = next;
    }
  }

  // ------------------------------------------------ the warps' (max, sum, O), in their order
  const int d = a.d, all = args.tiles * kRowsW;          // the block's rows
  float* const ro = joined;                              // [stream][row][d]
  float* const rml = ro + (size_t)streams * all * d;     // [stream][row][2]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int z = 4; z < 32; z *= 2) l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], z);
      const int r = stream * all + tile * kRowsW + 8 * t + 2 * t4 + i;
      if (g == 0) {
        rml[2 * r] = m[t][i];
        rml[2 * r + 1] = l[t][i];
      }
      const float f = mv[t][i] == -INFINITY ? 1.f : fast_exp2(mv[t][i] - kRaise - m[t][i]);  // O's reference becomes the sums'
      if (g * kCols < d)
#pragma unroll
        for (int j = 0; j < kCols / 2; j += 2)
          *reinterpret_cast<float4*>(ro + (size_t)r * d + g * kCols + 2 * j) =
              make_float4(o[t][j][i] * f, o[t][j][2 + i] * f, o[t][j + 1][i] * f, o[t][j + 1][2 + i] * f);
    }
  __syncthreads();
  const int quads = d / 4;
  for (int i = tid; i < all * quads; i += kThreads8) {
    const int r = i / quads, c = (i - r * quads) * 4, row = rb * all + r;
    if (row >= rows) break;
    float top = -INFINITY, sum = 0.f;
    for (int w = 0; w < streams; ++w) top = fmaxf(top, rml[2 * (w * all + r)]);
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < streams; ++w) {
      const float mw = rml[2 * (w * all + r)], lw = rml[2 * (w * all + r) + 1];
      if (mw == -INFINITY && lw == 0.f) continue;  // nothing seen (a sum of NaN: only NaN was)
      const float f = mw == top ? 1.f : fast_exp2(mw - top);
      const float4 y = *reinterpret_cast<const float4*>(ro + (size_t)(w * all + r) * d + c);
      sum = fmaf(f, lw, sum);
      x.x = fmaf(f, y.x, x.x);
      x.y = fmaf(f, y.y, x.y);
      x.z = fmaf(f, y.z, x.z);
      x.w = fmaf(f, y.w, x.w);
    }
    const int token = row / a.group;
    const bool present = !parents || parents[token] >= -1;
    if (s_bad && present) {
      uint32_t seen[4];
      ancestor_bits(parents, token, seen);
      for (int j = 0; j < a.tokens; ++j) {
        const uint32_t bits = j < 32 ? seen[0] : j < 64 ? seen[1] : j < 96 ? seen[2] : seen[3];
        if (!((bits >> (j & 31)) & 1u)) continue;
        const float4 v = four_of(static_cast<const T*>(a.v_new) + b * a.n_b + j * a.n_t + kvh * a.n_h + c);
        x.x += fabsf(v.x) < INFINITY ? 0.f : v.x;
        x.y += fabsf(v.y) < INFINITY ? 0.f : v.y;
        x.z += fabsf(v.z) < INFINITY ? 0.f : v.z;
        x.w += fabsf(v.w) < INFINITY ? 0.f : v.w;
      }
    }
    if (a.splits == 1) {
      const float inv = 1.f / sum;
      const float4 y = present ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f);
      store4(static_cast<T*>(a.out) + (((int64_t)b * a.tokens + token) * a.heads + kvh * a.group + row % a.group) * d + c, y);
    } else {
      const int64_t at = (((int64_t)split * a.batch + b) * a.kv_heads + kvh) * rows + row;
      store4(a.ws_o + at * d + c, x);
      if (c == 0) {
        a.ws_ml[2 * at] = top;
        a.ws_ml[2 * at + 1] = sum;
      }
    }
  }
}

// ------------------------------------------------------------------ host

// How a block's warps share query rows and keys: tiles of 8 rows (16 from 9 rows on), as many as there are, up to
// the warps, which share the keys if there are fewer.
struct Shape8 {
  int nt, tiles, row_blocks, streams;
};
Shape8 shape_8bit(int64_t rows) {
  Shape8 s;
  s.nt = rows <= 8 ? 1 : 2;
  s.tiles = rows <= 16 ? 1 : rows <= 32 ? 2 : kWarps8;
  s.row_blocks = (int)((rows + 8 * s.nt * s.tiles - 1) / (8 * s.nt * s.tiles));
  s.streams = kWarps8 / s.tiles;
  return s;
}

// Blocks that share a sequence's keys, of at least two windows to a warp, as long as there are no
// more than kRoom8 for each SM where all sequences are as long as the tables allow.
// (bf16, 32 heads over 8 of 128: 8 to an SM, three of them at a time, took 123 us for 150 over 32 sequences of up to
// 8192 positions, but 47 for 34 over 64 of about 700.)
constexpr int kRoom8 = 4, kLeast8 = 2;
int64_t splits_8bit(int64_t batch, int64_t kv_heads, int64_t rows, int64_t capacity) {
  const Shape8 s = shape_8bit(rows);
  const int64_t windows = std::max<int64_t>((capacity + kWindow - 1) / kWindow, 1);
  const int64_t room = std::max<int64_t>(kRoom8 * (int64_t)sm_count() / (batch * kv_heads * s.row_blocks), 1);
  return std::max<int64_t>(1, std::min({room, (windows + kLeast8 * s.streams - 1) / (kLeast8 * s.streams), (int64_t)kMaxSplits}));
}

template <typename T, int DC>
int launch_8bit(const Bits8Args& a, int nt, dim3 grid, bool fast, cudaStream_t st) {
  const char* op = "nkl_attention_tree_8bit";
  const size_t smem = (size_t)kWarps8 * 8 * nt * (a.t.d + 2) * 4;
  static_assert((size_t)kWarps8 * 16 * (128 + 2) * 4 <= 48 * 1024, "no attribute needed");
  auto go = [&](auto* kernel) { return launch_pdl(kernel, grid, dim3(kThreads8), smem, st, op, a); };
  if (nt == 1) return fast ? go(attention_8bit_kernel<T, DC, true, 1>) : go(attention_8bit_kernel<T, DC, false, 1>);
  return fast ? go(attention_8bit_kernel<T, DC, true, 2>) : go(attention_8bit_kernel<T, DC, false, 2>);
}

}  // namespace
