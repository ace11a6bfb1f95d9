// attn_math.cuh - arithmetic and register helpers shared by the tensor-core attention kernels.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

namespace nkl {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Packed fp32 pairs (lo, hi) for fma.rn.f32x2 / add.rn.f32x2: each lane is an ordinary fp32
// FMA / add, so the values equal those of the scalar forms, with half the instructions.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 f2_pack(float lo, float hi) {
  return ((f32x2)__float_as_uint(hi) << 32) | __float_as_uint(lo);
}
__device__ __forceinline__ f32x2 f2_pack_bits(uint32_t lo, uint32_t hi) { return ((f32x2)hi << 32) | lo; }
__device__ __forceinline__ float f2_lo(f32x2 a) { return __uint_as_float((uint32_t)a); }
__device__ __forceinline__ float f2_hi(f32x2 a) { return __uint_as_float((uint32_t)(a >> 32)); }
__device__ __forceinline__ f32x2 f2_fma(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 f2_add(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ f32x2 f2_mul(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// P = 2^(s * scale_log2 - m) for the scores v[0..N), packed as bf16 pairs into v[0..N/2)
// (pair (c, c+1) lands in v[c/2], a score already consumed). The row sum runs in `acc`
// packed accumulators (acc = 1 or 2); accumulator j's lanes take the pairs with
// (c/2) % acc == j, low lane the even scores, high lane the odd ones. Returns the
// accumulators themselves so each caller combines them in its own order.
template <int N, int ACC>
__device__ __forceinline__ void exp_pack(uint32_t* v, float scale_log2, float neg_m, f32x2 (&rs)[ACC]) {
  const f32x2 k2 = f2_pack(scale_log2, scale_log2), m2 = f2_pack(neg_m, neg_m);
#pragma unroll
  for (int j = 0; j < ACC; ++j) rs[j] = 0ull;
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const f32x2 x2 = f2_fma(f2_pack_bits(v[c], v[c + 1]), k2, m2);
    const float p0 = fast_exp2(f2_lo(x2)), p1 = fast_exp2(f2_hi(x2));
    rs[(c >> 1) % ACC] = f2_add(rs[(c >> 1) % ACC], f2_pack(p0, p1));
    __nv_bfloat162 h2 = __floats2bfloat162_rn(p0, p1);
    v[c >> 1] = *reinterpret_cast<uint32_t*>(&h2);
  }
}

// exp_pack with the row sum taken over the rounded exponentials: what the product with V
// sums up is then divided by the sum of just those weights, so the roundings of the weights
// cancel where V varies little and a row that sees one key gets it exactly.
template <int N, int ACC>
__device__ __forceinline__ void exp_pack_rounded(uint32_t* v, float scale_log2, float neg_m, f32x2 (&rs)[ACC]) {
  const f32x2 k2 = f2_pack(scale_log2, scale_log2), m2 = f2_pack(neg_m, neg_m);
#pragma unroll
  for (int j = 0; j < ACC; ++j) rs[j] = 0ull;
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const f32x2 x2 = f2_fma(f2_pack_bits(v[c], v[c + 1]), k2, m2);
    __nv_bfloat162 h2 = __floats2bfloat162_rn(fast_exp2(f2_lo(x2)), fast_exp2(f2_hi(x2)));
    const uint32_t h = *reinterpret_cast<uint32_t*>(&h2);
    rs[(c >> 1) % ACC] = f2_add(rs[(c >> 1) % ACC], f2_pack_bits(h << 16, h & 0xffff0000u));
    v[c >> 1] = h;
  }
}

// exp_pack in two parts: hi the exponentials cut off to bf16, lo what that left, rounded (2^-15 of
// the exponential); the sum is over the exponentials in fp32. Neither part is negative, and lo has
// 2^-40 of the exponential added, so that it is zero only where that is: an infinity in V times
// either part is that infinity, and no NaN (0 inf, inf - inf) comes of their sum.
template <int N, int ACC>
__device__ __forceinline__ void exp_pack_two(const uint32_t* v, uint32_t* hi, uint32_t* lo, float scale_log2,
                                             float neg_m, f32x2 (&rs)[ACC]) {
  const f32x2 k2 = f2_pack(scale_log2, scale_log2), m2 = f2_pack(neg_m, neg_m);
  const f32x2 minus = f2_pack(-1.f, -1.f), little = f2_pack(0x1p-40f, 0x1p-40f);
#pragma unroll
  for (int j = 0; j < ACC; ++j) rs[j] = 0ull;
#pragma unroll
  for (int c = 0; c < N; c += 2) {
    const f32x2 x2 = f2_fma(f2_pack_bits(v[c], v[c + 1]), k2, m2);
    const f32x2 p2 = f2_pack(fast_exp2(f2_lo(x2)), fast_exp2(f2_hi(x2)));
    rs[(c >> 1) % ACC] = f2_add(rs[(c >> 1) % ACC], p2);
    const uint32_t h = __byte_perm((uint32_t)p2, (uint32_t)(p2 >> 32), 0x7632);
    const f32x2 l2 = f2_fma(p2, little, f2_fma(f2_pack_bits(h << 16, h & 0xffff0000u), minus, p2));
    __nv_bfloat162 b2 = __floats2bfloat162_rn(f2_lo(l2), f2_hi(l2));
    hi[c >> 1] = h;
    lo[c >> 1] = *reinterpret_cast<uint32_t*>(&b2);
  }
}

// Marks r[0..N) as defined here: placed after tcgen05.wait::ld, it keeps every use of
// registers written by an asynchronous tcgen05.ld behind the wait that completes it.
template <int N>
__device__ __forceinline__ void reg_fence(uint32_t* r) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ float max3f(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
      "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
      "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

}  // namespace
}  // namespace nkl
