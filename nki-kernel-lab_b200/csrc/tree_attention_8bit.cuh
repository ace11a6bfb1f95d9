// tree_attention_8bit.cuh - the tree attention over a cache in 8 bits, by mma.sync; included by
// tree_attention.cu.
//
// Cached k and v are e4m3 numbers with a power of two for each block of positions and head. They go
// from global memory into registers, 16 bytes to a lane, and from there, as f16 (which has every
// e4m3 number), into the products, without shared memory and without barriers:
//   S = Q K^T  the lanes of a row hold other entries of a head than the fragment's layout says, in
//              Q and K alike, so that a lane's 16 bytes of K are the fragments of four products
//   O += P V   two keys' bytes are interleaved to pairs; a lane's 16 bytes are its column of 16
//              products, and it ends up with 16 entries in a row of O
// A warp meets one tile of 16 query rows with one window of 32 keys after the other, the windows
// dealt out over a block's warps; their (max, sum, O) meet in shared memory, those of several blocks
// in the workspace (tree_combine_kernel).
//
// Powers of two: K's multiply the scores. V's move the exponent of the weights, p 2^e, before these
// are rounded to f16, which therefore have a maximum of their own, beside that of the scores. Q is
// scaled by a power of two per row, so that f16 holds it; fp32 queries and weights are two f16
// numbers. Both maxima may lag behind by 2^8: sums are rescaled when a row's grow by more.
// The drafted tokens' own k and v multiply in bf16, fp32 ones in three parts.
#pragma once

namespace {

constexpr int kThreads8 = 128;
constexpr int kWarps8 = kThreads8 / 32;
constexpr int kWindow = 32;     // keys that a warp looks up at a time
constexpr float kLag8 = 8.f;    // log2 of how far the maxima may lag
constexpr float kRaise = 6.f;   // weights are up to 2^(kLag8 + kRaise): f16 ends at 2^16, and below 2^-14 it loses bits

struct Bits8Args {
  TreeArgs t;  // c_p, c_h, c_s: in bytes
  const uint8_t *k_scales, *v_scales;
  int block, per_page;  // positions of a block, blocks of a page
  int tiles;            // tiles of 16 query rows that a block's warps share
};

__device__ __forceinline__ uint32_t e4m3_pair(uint32_t two) {  // the lower 16 bits
  uint32_t r;
  asm("{\n .reg .b16 x;\n mov.b32 {x, _}, %1;\n cvt.rn.f16x2.e4m3x2 %0, x;\n}" : "=r"(r) : "r"(two));
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

// DC: head_dim up to 64 DC. FAST: pages and blocks are multiples of 16 positions, so that the 16 keys of a
// product lie in a row and share their powers of two.
template <typename T, int DC, bool FAST>
__global__ void __launch_bounds__(kThreads8, 2) attention_8bit_kernel(const __grid_constant__ Bits8Args args) {
  constexpr bool kF32 = sizeof(T) == 4;
  constexpr int kParts = kF32 ? 3 : 1;   // of drafted k and v, in bf16
  constexpr int kSteps = 4 * DC;         // products over the entries of a head
  constexpr int kCols = 8 * DC;          // entries of V that a lane has of a key, and products P V
  extern __shared__ __align__(16) float joined[];
  __shared__ int s_bad;                  // a drafted v that is not finite
  const TreeArgs& a = args.t;
  pdl_enter();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3;
  const int split = blockIdx.x / a.row_blocks, rb = blockIdx.x % a.row_blocks;
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int tile = warp % args.tiles, stream = warp / args.tiles, streams = kWarps8 / args.tiles;
  const int rows = a.tokens * a.group, r0 = (rb * args.tiles + tile) * 16;
  const int n = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.max_pages * a.page);
  const int windows = (n + kWindow - 1) / kWindow, per = (windows + a.splits - 1) / a.splits;
  const int w0 = min(split * per, windows), w1 = min(w0 + per, windows);
  const int* const parents = a.parents ? a.parents + (int64_t)b * a.tokens : nullptr;
  if (tid == 0) s_bad = 0;
  __syncthreads();

  // the lane's rows, g and g + 8: where their q lies
  const T* qp[2];
  bool real[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int row = r0 + g + 8 * i, token = row / a.group;
    real[i] = row < rows && (!parents || parents[token] >= -1);  // an absent token's q is not looked at
    qp[i] = static_cast<const T*>(a.q) + b * a.q_b + (real[i] ? token * a.q_t + (kvh * a.group + row - token * a.group) * a.q_h : 0);
  }
  // Four consecutive entries of the lane's: step s takes those at entry(s).
  auto entry = [&](int s) { return (t4 + 4 * (s >> 2)) * 16 + (s & 3) * 4; };
  auto four = [&](const T* p) {
    float4 x;
    if constexpr (kF32) {
      x = *reinterpret_cast<const float4*>(p);
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      x = make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u));
    }
    return x;
  };
  uint32_t qh[kSteps][4], ql[kF32 ? kSteps : 1][4];
  float factor[2];  // of a row's scores
  {
    float top[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        if (!real[i] || entry(s) >= a.d) continue;
        const float4 x = four(qp[i] + entry(s));
        for (float y : {x.x, x.y, x.z, x.w}) top[i] = fmaxf(top[i], fabsf(y) < INFINITY ? fabsf(y) : 0.f);
      }
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 1));
      top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], 2));
      const int e = max((int)(__float_as_uint(top[i]) >> 23) - 127, -112);  // 2^e <= top
      const float up = __uint_as_float((uint32_t)(14 - e + 127) << 23);
      factor[i] = a.scale * kLog2e * __uint_as_float((uint32_t)(e - 14 + 127) << 23);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (real[i] && entry(s) < a.d) x = four(qp[i] + entry(s));
        x = make_float4(x.x * up, x.y * up, x.z * up, x.w * up);
        qh[s][i] = half_pair(x.x, x.y);
        qh[s][2 + i] = half_pair(x.z, x.w);
        if constexpr (kF32) {
          const float2 u = rest_half(qh[s][i], x.x, x.y), v = rest_half(qh[s][2 + i], x.z, x.w);
          ql[s][i] = half_pair(u.x, u.y);
          ql[s][2 + i] = half_pair(v.x, v.y);
        }
      }
    }
  }

  // m: the rows' reference for sums l of 2^(s - m); v: that for O, sums of 2^(s + e - v + kRaise) v
  float m[2] = {-INFINITY, -INFINITY}, mv[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, o[kCols][4];
#pragma unroll
  for (int j = 0; j < kCols; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  // Weights of 16 keys: x[2 k + ..] the scores of rows g (0, 1) and g + 8 (2, 3) with keys 8 k + 2 t4 and
  // the one after it, e[..] their powers of two for O. Comes back with x the weights for O.
  auto weigh = [&](float (&x)[2][4], const float (&e)[2][2]) {
    bool grows = false;
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) grows |= x[k][i] > m[i >> 1] + kLag8 || x[k][i] + e[k][i & 1] > mv[i >> 1] + kLag8;
    if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float top = fmaxf(fmaxf(x[0][2 * i], x[0][2 * i + 1]), fmaxf(x[1][2 * i], x[1][2 * i + 1]));
        float tv = fmaxf(fmaxf(x[0][2 * i] + e[0][0], x[0][2 * i + 1] + e[0][1]), fmaxf(x[1][2 * i] + e[1][0], x[1][2 * i + 1] + e[1][1]));
#pragma unroll
        for (int z = 1; z < 4; z *= 2) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
          tv = fmaxf(tv, __shfl_xor_sync(0xffffffffu, tv, z));
        }
        if (top > m[i] + kLag8) {  // a row goes by its own scores alone
          l[i] *= fast_exp2(m[i] - top);
          m[i] = top;
        }
        float f = 1.f;
        if (tv > mv[i] + kLag8) {
          f = fast_exp2(mv[i] - tv);
          mv[i] = tv;
        }
#pragma unroll
        for (int j = 0; j < kCols; ++j) {
          o[j][2 * i] *= f;
          o[j][2 * i + 1] *= f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float rm = m[i] == -INFINITY ? 0.f : m[i], rv = mv[i] == -INFINITY ? 0.f : mv[i] - kRaise;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          float& s = x[k][2 * i + z];
          l[i] += fast_exp2(s - rm);
          s = fast_exp2(s + e[k][z] - rv);
        }
    }
  };

  // ------------------------------------------------ the drafted tokens
  if (split == a.splits - 1) {
    uint32_t seen[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int token = (r0 + g + 8 * i) / a.group;
      seen[i][0] = seen[i][1] = seen[i][2] = seen[i][3] = 0u;
      if (real[i]) ancestor_bits(parents, token, seen[i]);
    }
    const T* const kn = static_cast<const T*>(a.k_new) + b * a.n_b + kvh * a.n_h;
    const T* const vn = static_cast<const T*>(a.v_new) + b * a.n_b + kvh * a.n_h;
    bool bad = false;
#pragma unroll 1
    for (int k0 = stream * 16; k0 < a.tokens; k0 += streams * 16) {
      float x[2][4] = {};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t q[kParts][4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (real[i] && entry(s) < a.d) y = four(qp[i] + entry(s));
          uint32_t p[kParts];
          bf16_parts(y.x, y.y, p);
#pragma unroll
          for (int z = 0; z < kParts; ++z) q[z][i] = p[z];
          bf16_parts(y.z, y.w, p);
#pragma unroll
          for (int z = 0; z < kParts; ++z) q[z][2 + i] = p[z];
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int key = k0 + 8 * k + g;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          if (key < a.tokens && entry(s) < a.d) y = four(kn + key * a.n_t + entry(s));
          uint32_t p0[kParts], p1[kParts];
          bf16_parts(y.x, y.y, p0);
          bf16_parts(y.z, y.w, p1);
#pragma unroll
          for (int sum = kParts - 1; sum >= 0; --sum)  // the smallest products first
#pragma unroll
            for (int z = 0; z <= sum; ++z) mma_b16(x[k], q[z], p0[sum - z], p1[sum - z]);
        }
      }
      if constexpr (kF32) {
        // an infinity's product with a part that is zero is no part of its product
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int key = k0 + 8 * k + 2 * t4 + (i & 1);
            if (fabsf(x[k][i]) < INFINITY || !real[i >> 1] || key >= a.tokens) continue;
            float y = 0.f;
            for (int c = 0; c < a.d; ++c) y = fmaf(qp[i >> 1][c], kn[key * a.n_t + c], y);
            x[k][i] = y;
          }
      }
      const float none[2][2] = {};
      const int word = k0 >> 5, first = k0 & 31;
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t (&w)[4] = seen[i >> 1];
          const uint32_t bits = word == 0 ? w[0] : word == 1 ? w[1] : word == 2 ? w[2] : w[3];
          x[k][i] = (bits >> (first + 8 * k + 2 * t4 + (i & 1))) & 1u ? x[k][i] * (a.scale * kLog2e) : -INFINITY;
        }
      weigh(x, none);
      uint32_t p[kF32 ? 3 : 2][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t y[kF32 ? 3 : 2];
        bf16_parts(x[i >> 1][2 * (i & 1)], x[i >> 1][2 * (i & 1) + 1], y);
#pragma unroll
        for (int z = 0; z < (kF32 ? 3 : 2); ++z) p[z][i] = y[z];
      }
#pragma unroll
      for (int j = 0; j < kCols; j += 4) {
        float v[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = k0 + 2 * t4 + (i & 1) + 8 * (i >> 1), c = g * kCols + j;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          // an absent token's v is left out; weights of 0 must meet no infinity, which is put in at the end
          if (key < a.tokens && c < a.d && (!parents || parents[key] >= -1)) y = four(vn + key * a.n_t + c);
          v[i][0] = y.x; v[i][1] = y.y; v[i][2] = y.z; v[i][3] = y.w;
#pragma unroll
          for (int z = 0; z < 4; ++z)
            if (!(fabsf(v[i][z]) < INFINITY)) {
              bad = true;
              v[i][z] = 0.f;
            }
        }
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          uint32_t v0[kParts], v1[kParts];
          bf16_parts(v[0][z], v[1][z], v0);
          bf16_parts(v[2][z], v[3][z], v1);
          if constexpr (kF32) {
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)
#pragma unroll
              for (int y = 0; y <= sum; ++y) mma_b16(o[j + z], p[y], v0[sum - y], v1[sum - y]);
          } else {
            mma_b16(o[j + z], p[1], v0[0], v1[0]);
            mma_b16(o[j + z], p[0], v0[0], v1[0]);
          }
        }
      }
    }
    if (bad) s_bad = 1;
  }

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
    float s[2][4] = {};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int c = 0; c < DC; ++c) {
        const uint32_t words[4] = {x.k[k][c].x, x.k[k][c].y, x.k[k][c].z, x.k[k][c].w};
#pragma unroll
        for (int z = 0; z < 4; ++z) {
          const uint32_t b0 = e4m3_pair(words[z]), b1 = e4m3_pair(words[z] >> 16);
          if constexpr (kF32) mma_f16(s[k], ql[4 * c + z], b0, b1);
          mma_f16(s[k], qh[4 * c + z], b0, b1);
        }
      }
    float e[2][2];
    float ks = 0.f, ve = 0.f;
    if (FAST) {
      ks = __shfl_sync(0xffffffffu, f.ks, 16 * h);
      ve = __shfl_sync(0xffffffffu, f.ve, 16 * h);
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int key = 8 * k + 2 * t4 + z;
        if (!FAST) {
          ks = __shfl_sync(0xffffffffu, f.ks, 16 * h + key);
          ve = __shfl_sync(0xffffffffu, f.ve, 16 * h + key);
        }
        e[k][z] = key < left ? ve : 0.f;
        s[k][z] = key < left ? s[k][z] * factor[0] * ks : -INFINITY;
        s[k][2 + z] = key < left ? s[k][2 + z] * factor[1] * ks : -INFINITY;
      }
    weigh(s, e);
    uint32_t p[4], pl[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float lo = s[i >> 1][2 * (i & 1)], hi = s[i >> 1][2 * (i & 1) + 1];
      p[i] = half_pair(lo, hi);
      if constexpr (kF32) {
        const float2 r = rest_half(p[i], lo, hi);
        pl[i] = half_pair(r.x, r.y);
      }
    }
    const uint32_t vw[4][4] = {{x.v[0].x, x.v[0].y, x.v[0].z, x.v[0].w}, {x.v[1].x, x.v[1].y, x.v[1].z, x.v[1].w},
                               {x.v[2].x, x.v[2].y, x.v[2].z, x.v[2].w}, {x.v[3].x, x.v[3].y, x.v[3].z, x.v[3].w}};
#pragma unroll
    for (int z = 0; z < kCols / 4; ++z)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const uint32_t u0 = __byte_perm(vw[0][z], vw[1][z], y ? 0x7362 : 0x5140), u1 = __byte_perm(vw[2][z], vw[3][z], y ? 0x7362 : 0x5140);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const uint32_t b0 = e4m3_pair(q ? u0 >> 16 : u0), b1 = e4m3_pair(q ? u1 >> 16 : u1);
          float (&to)[4] = o[4 * z + 2 * y + q];
          if constexpr (kF32) mma_f16(to, pl, b0, b1);
          mma_f16(to, p, b0, b1);
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
  const int d = a.d, all = args.tiles * 16;  // the block's rows
  float* const ro = joined;                              // [stream][row][d]
  float* const rml = ro + (size_t)streams * all * d;     // [stream][row][2]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    const int r = stream * all + tile * 16 + g + 8 * i;
    if (t4 == 0) {
      rml[2 * r] = m[i];
      rml[2 * r + 1] = l[i];
    }
    const float f = mv[i] == -INFINITY ? 1.f : fast_exp2(mv[i] - kRaise - m[i]);  // O's reference becomes the sums'
#pragma unroll
    for (int z = 0; z < 2; ++z) {  // entries c .. c + kCols - 1
      const int c = (2 * t4 + z) * kCols;
      if (c >= d) continue;
#pragma unroll
      for (int j = 0; j < kCols; j += 4)
        *reinterpret_cast<float4*>(ro + (size_t)r * d + c + j) =
            make_float4(o[j][2 * i + z] * f, o[j + 1][2 * i + z] * f, o[j + 2][2 * i + z] * f, o[j + 3][2 * i + z] * f);
    }
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
        const float4 v = four(static_cast<const T*>(a.v_new) + b * a.n_b + j * a.n_t + kvh * a.n_h + c);
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

// Tiles of 16 query rows that a block's warps share: as many as there are, up to its warps.
int tiles_8bit(int64_t rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : kWarps8; }

// Blocks that share a sequence's keys, of at least two windows to a warp, as long as there are no
// more than four for each SM where all sequences are as long as the tables allow.
int64_t splits_8bit(int64_t batch, int64_t kv_heads, int64_t rows, int64_t capacity) {
  const int64_t tiles = tiles_8bit(rows), row_blocks = (rows + 16 * tiles - 1) / (16 * tiles), streams = kWarps8 / tiles;
  const int64_t windows = std::max<int64_t>((capacity + kWindow - 1) / kWindow, 1);
  const int64_t room = std::max<int64_t>(4 * (int64_t)sm_count() / (batch * kv_heads * row_blocks), 1);
  return std::max<int64_t>(1, std::min({room, (windows + 2 * streams - 1) / (2 * streams), (int64_t)kMaxSplits}));
}

template <typename T, int DC>
int launch_8bit(const Bits8Args& a, dim3 grid, bool fast, cudaStream_t st) {
  const char* op = "nkl_attention_tree_8bit";
  const size_t smem = (size_t)kWarps8 * 16 * (a.t.d + 2) * 4;
  static_assert((size_t)kWarps8 * 16 * (128 + 2) * 4 <= 48 * 1024, "no attribute needed");
  return fast ? launch_pdl(attention_8bit_kernel<T, DC, true>, grid, dim3(kThreads8), smem, st, op, a)
              : launch_pdl(attention_8bit_kernel<T, DC, false>, grid, dim3(kThreads8), smem, st, op, a);
}

}  // namespace
