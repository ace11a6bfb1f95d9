// sample.cu - the next token of each row of logits: temperature, top-k, top-p, min-p, from given
// uniform numbers.
//
// A row's tokens in order of their logits, of equal ones the lowest index first, have the weights
//   w = floor(2^31 exp((x - max) / T)), or one more or less
// What is drawn from is the longest beginning of that order that every filter allows: top-k its k first
// tokens; top-p the fewest whose weights come to the share p of the top-k's; min-p those of at least
// p times the first one's weight. Of it the token is the first one, by index, with which
// the cumulative weight is over the uniform number's share of the sum. Weights, shares and uniform
// numbers are whole multiples of 2^-31, so that sums do not depend on their order, and equal
// inputs give equal tokens on every launch. NaN counts as minus infinity, and minus infinity is never
// drawn; T of 0 (or below, or NaN) takes the first token.
//
// A cluster of up to eight blocks takes a row; each holds its part in shared memory, first as logits,
// then as weights, which are computed once, to a unit of their last place (a float's 24 bits would shift
// a border between two tokens of a long row now and then). The order's end is found without sorting: a histogram of
// weights and counts over 1024 ranges of the weight, a thirty-second of it wide, tells the range where it
// is. Up to 768 tokens of that range go to every block, by distributed shared memory, and each finds
// the end among them for itself; more are taken apart by histograms over 512 parts of the range, added up over
// the blocks, and so on, until a part is one weight. Of equal ones as many stay as it takes, by logit and then by index.
//
// Measured (temperature 0.8, top-p 0.95): fp32: one row of 32768 14 us, 64 rows of 131072 63 us (34 MB: 5 us by bytes),
// with settings of their own, some of which need no filter, 46. What bounds it is the chain of phases: maximum -> weights and histogram -> the end's range ->
// its tokens -> sums -> draw, each with a barrier of the block, most with one of the cluster (1700 to 2000 cycles), and
// 69 instructions to 32 tokens in the first two, of which the weights' powers take most. With 64-bit
// atomics in the histogram (which loop) instead of two of 32 it took 291 us, with further rounds over the cluster instead of the
// list of a range's tokens 79.
#include <algorithm>
#include <atomic>

#include "attn_math.cuh"
#include "common.cuh"

namespace nkl {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 1024;       // of the first round: 992 are used
constexpr int kParts = 512;       // of a range, in the rounds after it
constexpr int kList = 768;        // tokens of a range that are gathered
constexpr int kStep = 128;        // tokens that a warp looks at at once, four to a lane
constexpr int kPerBlock = 45056;  // tokens that a block holds: 176 KB; blocks of up to kPerHalf go two to an SM
constexpr int kPerHalf = 16384;
constexpr int kTable = 256;
constexpr u64 kOne = 1ull << 31;
constexpr u64 kNone = ~0ull;

struct SampleArgs {
  const void* logits;
  int64_t stride;  // of the rows, in elements
  const float *uniforms, *temperatures, *top_ps, *min_ps;  // arrays of the rows, or NULL: the number below
  const int* top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int* token;
  float* prob;
  int batch, vocab, part;  // part: tokens of a block, whole steps of its warps
};

// Keys in the order of the numbers; -0 counts as 0. NaN and minus infinity do not come here.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ uint32_t whole_share(float x) {  // of [0, 1], in multiples of 2^-31
  return x > 0.f ? (uint32_t)(fminf(x, 1.f) * 2147483648.f) : 0u;
}
__device__ __forceinline__ u64 share_of(u64 total, u64 share) {
  return (total >> 31) * share + (((total & (kOne - 1)) * share) >> 31);
}

// The first round's range of a weight w > 0: by the upper 5 bits behind the leading one; 0 is the highest.
constexpr uint32_t kTopBits = 158u << 23;  // 2^31 as a float
__device__ __forceinline__ int range_of(uint32_t w) { return (int)((kTopBits - __float_as_uint(__uint2float_rz(w))) >> 18); }
// Its least and largest weight.
__device__ __forceinline__ uint32_t least_of(int range) {
  const float f = __uint_as_float(max(kTopBits - ((uint32_t)(range + 1) << 18) + 1u, 1u));
  return max((uint32_t)ceilf(f), 1u);
}
__device__ __forceinline__ uint32_t most_of(int range) {
  const float f = __uint_as_float(kTopBits - ((uint32_t)range << 18) + 1u);  // the next float
  return min((uint32_t)ceilf(f) - 1u, (uint32_t)kOne);
}

__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void put(u64* p, uint32_t rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void put(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void put(uint4* p, uint32_t rank, uint4 v) {
  asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(remote(p, rank)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void add_remote(u64* p, uint32_t rank, u64 v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void add_remote(uint32_t* p, uint32_t rank, uint32_t v) {
  asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t get(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
  return v;
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// 2^31 2^(-j / kTable): the whole part, and the rest as a float. By Taylor's series for e^-x, x below ln 2.
struct Table {
  uint32_t whole[kTable];
  float rest[kTable];
  constexpr Table() : whole(), rest() {
    for (int j = 0; j < kTable; ++j) {
      const double x = 0.69314718055994530942 * j / kTable;
      double e = 1.0;
      for (int n = 24; n > 0; --n) e = 1.0 - x / n * e;
      e *= 2147483648.0;
      whole[j] = (uint32_t)e;
      rest[j] = (float)(e - whole[j]);
    }
  }
};
__device__ constexpr Table kPowers;

template <int N>
struct Sums {  // over the cluster: weights and counts of the ranges
  u64 w[N];
  uint32_t c[N];
};
struct Shared {
  uint32_t lo[kBins], hi[kBins], count[kBins];  // the block's: weights in halves of 16 bits, which 2^16 tokens do not overflow
  Sums<kBins> first;
  union {
    Sums<kParts> next[2];  // in turn; all zero when they are added to
    uint4 list[kList];     // a range's tokens: key, weight, index
  };
  uint32_t part_lo[kParts], part_hi[kParts], part_count[kParts];
  uint2 table[kTable];   // 2^31 2^(-j / kTable): whole part, and the rest as a float
  u64 all[2][kMaxCluster][3];  // what each block has to tell the others, in turn
  u64 scan[kWarps][3];
  int bin, slots;
  uint32_t ahead;
  u64 before[2], in[2];
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint32_t weights[];  // the part's: logits at first
  __shared__ Shared s;
  cluster_started();
  pdl_enter();
  uint32_t blocks, rank;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(blocks));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const int b = blockIdx.x / blocks, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int x0 = min((int)rank * a.part, a.vocab), n = min(a.part, a.vocab - x0);
  const T* const row = static_cast<const T*>(a.logits) + b * a.stride + x0;
  const float temperature = a.temperatures ? a.temperatures[b] : a.temperature;
  const float top_p = a.top_ps ? a.top_ps[b] : a.top_p, min_p = a.min_ps ? a.min_ps[b] : a.min_p;
  const int top_k = a.top_ks ? a.top_ks[b] : a.top_k;
  // this warp's tokens: [lo, hi) of the block's, whole steps; behind n there is nothing to draw
  const int per = a.part / kWarps, lo = warp * per, hi = min(lo + per, (n + kStep - 1) / kStep * kStep);
  if (tid < kTable) s.table[tid] = make_uint2(kPowers.whole[tid], __float_as_uint(kPowers.rest[tid]));
  for (int i = tid; i < kBins; i += kThreads) s.lo[i] = s.hi[i] = s.count[i] = 0u;
  for (int i = tid; i < 2 * kParts; i += kThreads) {
    s.next[i / kParts].w[i % kParts] = 0ull;
    s.next[i / kParts].c[i % kParts] = 0u;
  }

  // A block's numbers, the same in all its threads, to every block. The places take turns: what a call wrote is
  // read before the next call's barrier, and written again after it.
  int turn = 0;
  auto tell = [&](u64 x, u64 y, u64 z) -> const u64(&)[kMaxCluster][3] {
    u64(&to)[kMaxCluster][3] = s.all[turn];
    turn ^= 1;
    if (tid < (int)blocks) {
      put(&to[rank][0], tid, x);
      put(&to[rank][1], tid, y);
      put(&to[rank][2], tid, z);
    }
    cluster_sync();
    return to;
  };
  // Sums of the warps' numbers over the block, in every thread.
  auto block_sums = [&](u64 x, u64 y, u64 (&sum)[2]) {
    x = warp_sum64(x);
    y = warp_sum64(y);
    __syncthreads();
    if (lane == 0) {
      s.scan[warp][0] = x;
      s.scan[warp][1] = y;
    }
    __syncthreads();
    sum[0] = sum[1] = 0;
    for (int k = 0; k < kWarps; ++k) {
      sum[0] += s.scan[k][0];
      sum[1] += s.scan[k][1];
    }
  };

  // ---------------------------------------------------------------- logits and their maximum
  float top = -INFINITY;
  {
    constexpr int VE = Vec16<T>::N;
    const bool vec = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    const int whole = vec ? min(hi, n) : lo;
#pragma unroll 4
    for (int i = lo + lane * VE; i < whole; i += 32 * VE) {
      float x[VE];
      if (i + VE <= n) {
        Vec16<T> v;
        v.raw = *reinterpret_cast<const uint4*>(row + i);
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = v.get(e);
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = i + e < n ? to_f32(row[i + e]) : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
#pragma unroll
        for (int z = 0; z < 4; ++z) top = fmaxf(top, x[e + z]);
        *reinterpret_cast<float4*>(weights + i + e) = make_float4(x[e], x[e + 1], x[e + 2], x[e + 3]);
      }
    }
    if (vec) {  // what is left of the last step
      const int end = (n + VE - 1) / VE * VE;
      for (int i = max(lo, end) + lane; i < hi; i += 32) weights[i] = __float_as_uint(-INFINITY);
    } else {
#pragma unroll 4
      for (int i = lo + lane; i < hi; i += 32) {
        const float x = i < n ? to_f32(row[i]) : -INFINITY;
        weights[i] = __float_as_uint(x);
        top = fmaxf(top, x);
      }
    }
  }
  auto block_max = [&](uint32_t x) {
    x = __reduce_max_sync(0xffffffffu, x);
    __syncthreads();
    if (lane == 0) s.scan[warp][0] = x;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, (uint32_t)s.scan[lane & (kWarps - 1)][0]);
  };
  // (fmaxf passes NaN over; a key of 0 stands for minus infinity)
  uint32_t top_key = block_max(top > -INFINITY ? key_of(top) : 0u);
  cluster_wait_started();
  {
    const auto& all = tell(top_key, 0, 0);
    for (uint32_t r = 0; r < blocks; ++r) top_key = max(top_key, (uint32_t)all[r][0]);
  }
  if (top_key == 0u || !(temperature > 0.f) || top_k == 1) {
    uint32_t first = 0xffffffffu;  // the lowest index of the maximum
    if (top_key != 0u)
      for (int i = tid; i < n; i += kThreads) {
        const float x = __uint_as_float(weights[i]);
        if (x > -INFINITY && key_of(x) == top_key) first = min(first, (uint32_t)(x0 + i));
      }
    first = ~block_max(~first);
    const auto& all = tell(first, 0, 0);
    for (uint32_t r = 0; r < blocks; ++r) first = min(first, (uint32_t)all[r][0]);
    if (rank == 0 && tid == 0) {
      a.token[b] = top_key == 0u ? -1 : (int)first;
      a.prob[b] = top_key == 0u ? 0.f : 1.f;
    }
    return;
  }

  // ---------------------------------------------------------------- weights
  const bool by_count = top_k > 0 && top_k < a.vocab, by_share = top_p < 1.f;
  const bool ranges = by_count || by_share;
  const uint32_t least = min_p > 0.f ? max((uint32_t)__double2ull_ru((double)fminf(min_p, 1.f) * 2147483648.0), 1u) : 1u;
  u64 total, fit;  // of all weights; how many tokens weigh at least `least`
  {
    const float top_x = __uint_as_float(top_key & 0x80000000u ? top_key & 0x7fffffffu : ~top_key);
    // exp(z) = 2^(-k / kTable) 2^(y / kTable), k whole, |y| <= 1/2 + a little. z comes to 2^-33 of a whole in pairs of
    // floats: x - max and what rounding left of it, times a constant in two parts. Two tokens at a time.
    const double rate = min(kTable / 0.69314718055994530942 / (double)temperature, 3e38);
    const float ch = (float)rate, cl = (float)(rate - (double)ch);
    const f32x2 up = f2_pack(ch, ch), down = f2_pack(-ch, -ch), rest = f2_pack(cl, cl), minus = f2_pack(-1.f, -1.f);
    const f32x2 ntop = f2_pack(-top_x, -top_x), magic = f2_pack(12582912.f, 12582912.f), back = f2_pack(-12582912.f, -12582912.f);
    constexpr double l = 0.69314718055994530942 / kTable;
    const f32x2 a1 = f2_pack((float)l, (float)l), a2 = f2_pack((float)(l * l / 2), (float)(l * l / 2)),
                a3 = f2_pack((float)(l * l * l / 6), (float)(l * l * l / 6));
    auto weigh = [&](float x0, float x1, uint32_t& w0, uint32_t& w1) {
      const f32x2 x = f2_pack(x0, x1), d = f2_add(x, ntop), g = f2_fma(x, minus, d);
      const f32x2 e = f2_add(f2_fma(f2_fma(g, minus, d), minus, x), f2_fma(g, minus, ntop));  // d + e = x - max
      const f32x2 u = f2_mul(d, down);  // how far below, in steps of the table
      const f32x2 t = f2_fma(e, up, f2_fma(d, rest, f2_fma(d, up, u)));
      const f32x2 k = f2_add(u, magic), y = f2_add(f2_fma(u, minus, f2_add(k, back)), t);
      const f32x2 q = f2_mul(y, f2_fma(y, f2_fma(y, a3, a2), a1));  // 2^(y / kTable) - 1
      auto one = [&](float far, float at, float more) -> uint32_t {
        if (!(far < 31.5f * kTable)) return 0u;  // below 2^-31; NaN
        const int i = __float_as_int(at) - 0x4b400000;
        const uint2 p = s.table[i & (kTable - 1)];
        const uint32_t w = p.x + (uint32_t)__float2int_rd(fmaf(__uint2float_rn(p.x), more, __uint_as_float(p.y)));
        return w >> (i / kTable);
      };
      w0 = one(f2_lo(u), f2_lo(k), f2_lo(q));
      w1 = one(f2_hi(u), f2_hi(k), f2_hi(q));
    };
    const bool infinite = !(top_x < INFINITY);
    auto add = [&](uint32_t y) {
      if (y == 0u) return;
      const int range = range_of(y);
      atomicAdd(&s.lo[range], y & 0xffffu);
      atomicAdd(&s.hi[range], y >> 16);
      atomicAdd(&s.count[range], 1u);
    };
    u64 sum = 0;
    uint32_t some = 0;
    for (int i = lo + lane * 4; i < hi; i += kStep) {
      uint4& at = *reinterpret_cast<uint4*>(weights + i);
      const uint4 x = at;
      uint4 y;
      weigh(__uint_as_float(x.x), __uint_as_float(x.y), y.x, y.y);
      weigh(__uint_as_float(x.z), __uint_as_float(x.w), y.z, y.w);
      if (infinite) {
        const uint32_t one = (uint32_t)kOne, in = __float_as_uint(INFINITY);
        y = make_uint4(x.x == in ? one : 0u, x.y == in ? one : 0u, x.z == in ? one : 0u, x.w == in ? one : 0u);
      }
      at = y;
      sum += ((u64)y.x + y.y) + ((u64)y.z + y.w);
      if (least > 1u) some += (uint32_t)(y.x >= least) + (uint32_t)(y.y >= least) + (uint32_t)(y.z >= least) + (uint32_t)(y.w >= least);
      else if (by_count) some += (uint32_t)(y.x > 0u) + (uint32_t)(y.y > 0u) + (uint32_t)(y.z > 0u) + (uint32_t)(y.w > 0u);
      if (ranges) {
        add(y.x);
        add(y.y);
        add(y.z);
        add(y.w);
      }
    }
    u64 mine[2];
    block_sums(sum, some, mine);
    const auto& all = tell(mine[0], mine[1], 0);
    total = fit = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
      total += all[r][0];
      fit += all[r][1];
    }
  }

  // ---------------------------------------------------------------- where the order ends
  // The scan of N ranges, two or one to a thread: what is in them, and up to and with them.
  u64 w[2] = {0, 0}, c[2] = {0, 0}, w_to = 0, c_to = 0;
  auto scan = [&](int each, auto weight, auto number) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      w[k] = k < each ? weight(each * tid + k) : 0;
      c[k] = k < each ? number(each * tid + k) : 0;
    }
    w_to = w[0] + w[1];
    uint32_t n_to = (uint32_t)(c[0] + c[1]);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(0xffffffffu, w_to, o);
      const uint32_t q = __shfl_up_sync(0xffffffffu, n_to, o);
      if (lane >= o) {
        w_to += p;
        n_to += q;
      }
    }
    __syncthreads();
    if (lane == 31) {
      s.scan[warp][0] = w_to;
      s.scan[warp][1] = n_to;
    }
    if (tid == 0) s.bin = -1;
    __syncthreads();
    c_to = n_to;
    for (int k = 0; k < warp; ++k) {
      w_to += s.scan[k][0];
      c_to += s.scan[k][1];
    }
  };
  // The range, in scanned sums, where the count comes to `count` or the weights to `need`; -1: none. w0 and c0:
  // what is before all of them, and then before the range; wb and cb: what is in it.
  auto cross = [&](int each, u64 count, u64 need, u64& w0, u64& c0, u64& wb, u64& cb) {
    const u64 we = w0 + w_to, ce = c0 + c_to, ws = we - w[0] - w[1], cs = ce - c[0] - c[1];
    if (ws < need && cs < count && (we >= need || ce >= count)) {
      const bool one = ws + w[0] >= need || cs + c[0] >= count;
      s.bin = each * tid + (one ? 0 : 1);
      s.before[0] = ws + (one ? 0 : w[0]);
      s.before[1] = cs + (one ? 0 : c[0]);
      s.in[0] = one ? w[0] : w[1];
      s.in[1] = one ? c[0] : c[1];
    }
    __syncthreads();
    const int bin = s.bin;
    if (bin >= 0) {
      w0 = s.before[0];
      c0 = s.before[1];
      wb = s.in[0];
      cb = s.in[1];
    }
    return bin;  // a scan's first barrier comes before the next crossing
  };
  int buffer = 0;
  // From the values [v0, v1] on, of which there are cb, to the one where the order ends: each(f) calls f(value,
  // weight) for the warp's tokens there.
  auto narrow = [&](uint32_t v0, uint32_t v1, u64 count, u64 need, u64& w0, u64& c0, u64& wb, u64& cb, auto each) {
    while (v0 < v1) {
      const int shift = max(0, 32 - __clz(v1 - v0) - 9);
      for (int i = tid; i < kParts; i += kThreads) s.part_lo[i] = s.part_hi[i] = s.part_count[i] = 0u;
      __syncthreads();
      each([&](uint32_t v, uint32_t y) {
        if (v < v0 || v > v1) return;
        const int part = (int)((v1 - v) >> shift);
        atomicAdd(&s.part_lo[part], y & 0xffffu);
        atomicAdd(&s.part_hi[part], y >> 16);
        atomicAdd(&s.part_count[part], 1u);
      });
      __syncthreads();
      auto& sums = s.next[buffer];
      for (int i = tid; i < kParts; i += kThreads) {
        if (s.part_count[i] == 0u) continue;
        const u64 y = s.part_lo[i] + ((u64)s.part_hi[i] << 16);
        for (uint32_t r = 0; r < blocks; ++r) {
          add_remote(&sums.w[i], r, y);
          add_remote(&sums.c[i], r, s.part_count[i]);
        }
      }
      cluster_sync();
      scan(kParts / kThreads, [&](int i) { return sums.w[i]; }, [&](int i) { return sums.c[i]; });
      for (int i = tid; i < kParts; i += kThreads) {  // for the round after the next one, whose barrier is behind the next one's
        sums.w[i] = 0ull;
        sums.c[i] = 0u;
      }
      buffer ^= 1;
      const int part = cross(kParts / kThreads, count, need, w0, c0, wb, cb);
      v1 -= (uint32_t)part << shift;
      v0 = shift ? max(v0, v1 - min(v1 - v0, (1u << shift) - 1u)) : v1;
    }
    return v0;
  };
  // Tokens that weigh more than `border` stay, and of those that weigh as much the `ties` first ones of `tied`.
  uint32_t border = least - 1u;
  u64 ties = 0, tied = 0;
  auto all_weights = [&](auto f) {
    for (int i = lo + lane * 4; i < hi; i += kStep) {
      const uint4 x = *reinterpret_cast<const uint4*>(weights + i);
      f(x.x, x.x);
      f(x.y, x.y);
      f(x.z, x.z);
      f(x.w, x.w);
    }
  };
  auto key_at = [&](int i) { return key_of(to_f32(row[i])); };
  // A range of few tokens: they go to every block, which then finds the end for itself. With `apply` the weights of
  // this block's tokens behind the end become 0. Returns the weights up to the end.
  bool listed = false, narrowed = false;  // what the shared place was used for last
  auto end_in_list = [&](int range, u64 count, u64 need, u64 w0, u64 c0, int number, bool apply) {
    // where this block's begin in the list: behind those of the blocks before it
    uint32_t mine = lane < (int)blocks ? get(&s.count[range], lane) : 0u, to = mine;
#pragma unroll
    for (int o = 1; o < kMaxCluster; o <<= 1) {
      const uint32_t p = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += p;
    }
    const int end = (int)__shfl_sync(0xffffffffu, to, rank), begin = end - (int)__shfl_sync(0xffffffffu, mine, rank);
    if (tid == 0) {
      s.slots = begin;
      s.ahead = 0u;
    }
    if (listed || narrowed) cluster_sync();  // others may still read theirs
    __syncthreads();
    listed = true;
    constexpr int kKeyShift = sizeof(T) == 2 ? 16 : 0;  // a bf16's key is its upper half
    const uint32_t y0 = least_of(range), y1 = most_of(range);
    for (int i = lo + lane * 4; i < hi; i += kStep) {
      const uint4 x = *reinterpret_cast<const uint4*>(weights + i);
      const uint32_t y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        if (y[z] < y0 || y[z] > y1) continue;
        const uint4 e = make_uint4(key_at(i + z) >> kKeyShift, y[z], (uint32_t)(i + z), 0u);
        const int slot = atomicAdd(&s.slots, 1);
        for (uint32_t r = 0; r < blocks; ++r) put(&s.list[slot], r, e);
      }
    }
    cluster_sync();
    const bool one = tid < number, two = tid + kThreads < number;
    const uint4 none = make_uint4(0u, 0u, 0u, 0u), e0 = one ? s.list[tid] : none, e1 = two ? s.list[tid + kThreads] : none;
    auto pair_max = [&](uint32_t p, uint32_t q) {  // of two numbers of a thread, over the block
      p = __reduce_max_sync(0xffffffffu, p);
      q = __reduce_max_sync(0xffffffffu, q);
      __syncthreads();
      if (lane == 0) s.scan[warp][2] = (u64)p << 32 | q;
      __syncthreads();
      const u64 x = s.scan[lane & (kWarps - 1)][2];
      return make_uint2(__reduce_max_sync(0xffffffffu, (uint32_t)(x >> 32)), __reduce_max_sync(0xffffffffu, (uint32_t)x));
    };
    const uint2 most = pair_max(max(e0.x, e1.x), max(one ? ~e0.x : 0u, two ? ~e1.x : 0u));
    uint32_t v1 = most.x, v0 = ~most.y;
    u64 wb = 0, cb = 0;
    do {  // as in narrow, among the block's own copy
      const int shift = max(0, 32 - __clz(v1 - v0) - 9);
      for (int i = tid; i < kParts; i += kThreads) s.part_lo[i] = s.part_hi[i] = s.part_count[i] = 0u;
      __syncthreads();
      auto add = [&](const uint4& e, bool there) {
        if (!there || e.x < v0 || e.x > v1) return;
        const int part = (int)((v1 - e.x) >> shift);
        atomicAdd(&s.part_lo[part], e.y & 0xffffu);
        atomicAdd(&s.part_hi[part], e.y >> 16);
        atomicAdd(&s.part_count[part], 1u);
      };
      add(e0, one);
      add(e1, two);
      __syncthreads();
      scan(kParts / kThreads, [&](int i) { return s.part_lo[i] + ((u64)s.part_hi[i] << 16); }, [&](int i) { return s.part_count[i]; });
      const int part = cross(kParts / kThreads, count, need, w0, c0, wb, cb);
      v1 -= (uint32_t)part << shift;
      v0 = shift ? max(v0, v1 - min(v1 - v0, (1u << shift) - 1u)) : v1;
    } while (v0 < v1);
    // tokens of one logit, so of one weight: as many stay as it takes, the lowest indices
    const uint32_t y = (uint32_t)(wb / cb);
    u64 stay = min(cb, count == kNone ? kNone : count - c0);
    if (need != kNone) stay = min(stay, (need - w0 + y - 1) / y);
    if (apply) {
      const uint32_t before = (uint32_t)(one && tid < begin && e0.x == v1) + (uint32_t)(two && tid + kThreads < begin && e1.x == v1);
      if (before) atomicAdd(&s.ahead, before);
      __syncthreads();
      const u64 ahead = s.ahead;
      auto settle = [&](const uint4& e, int at) {
        if (at < begin || at >= end || e.x > v1) return;
        bool out = e.x < v1;
        if (!out && stay < cb) {
          u64 place = ahead;
          for (int j = begin; j < end; ++j) place += s.list[j].x == v1 && s.list[j].z < e.z;
          out = place >= stay;
        }
        if (out) weights[e.z] = 0u;
      };
      if (one) settle(e0, tid);
      if (two) settle(e1, tid + kThreads);
      __syncthreads();
    }
    return w0 + stay * y;
  };
  u64 scanned[6] = {};
  // Ends the order where its count comes to `count` or its weights to `need`; returns the weights in it.
  auto end_order = [&](u64 count, u64 need, bool apply) {
    __syncthreads();
    if (tid == 0) s.bin = -1;
    __syncthreads();
    w[0] = scanned[0], w[1] = scanned[1], c[0] = scanned[2], c[1] = scanned[3], w_to = scanned[4], c_to = scanned[5];
    u64 w0 = 0, c0 = 0, wb = 0, cb = 0;
    const int range = cross(kBins / kThreads, count, need, w0, c0, wb, cb);
    ties = tied = 0;
    if (range < 0) {
      border = least - 1u;  // nothing ends it but what weighs nothing
      return total;
    }
    if (cb > 1 && cb <= (u64)kList) {
      border = least_of(range) - 1u;
      return end_in_list(range, count, need, w0, c0, (int)cb, apply);
    }
    if (cb > 1 && listed) {  // the list's place is that of the sums
      for (int i = tid; i < 2 * kParts; i += kThreads) {
        s.next[i / kParts].w[i % kParts] = 0ull;
        s.next[i / kParts].c[i % kParts] = 0u;
      }
      cluster_sync();
      listed = false;
    }
    narrowed = cb > 1;
    // one token: its weight is the range's sum
    const uint32_t at = cb == 1 ? (uint32_t)wb : narrow(least_of(range), most_of(range), count, need, w0, c0, wb, cb, all_weights);
    border = at;
    tied = cb;
    ties = min(cb, count == kNone ? kNone : count - c0);
    if (need != kNone) ties = min(ties, (need - w0 + at - 1) / at);
    return w0 + ties * at;
  };
  if (ranges && (by_share || fit > (u64)top_k)) {
    // each block's share of the ranges over all blocks, to all blocks
    const int share = kBins / (int)blocks;
    for (int i = tid; i < share; i += kThreads) {
      const int bin = (int)rank * share + i;
      u64 y = 0;
      uint32_t m = 0;
      for (uint32_t r = 0; r < blocks; ++r) {
        y += get(&s.lo[bin], r) + ((u64)get(&s.hi[bin], r) << 16);
        m += get(&s.count[bin], r);
      }
      for (uint32_t r = 0; r < blocks; ++r) {
        put(&s.first.w[bin], r, y);
        put(&s.first.c[bin], r, m);
      }
    }
    cluster_sync();
    scan(kBins / kThreads, [&](int i) { return s.first.w[i]; }, [&](int i) { return s.first.c[i]; });
    scanned[0] = w[0], scanned[1] = w[1], scanned[2] = c[0], scanned[3] = c[1], scanned[4] = w_to, scanned[5] = c_to;
    const u64 k = by_count ? (u64)top_k : kNone;
    u64 need = kNone;
    if (by_share) need = max(share_of(by_count ? end_order(k, kNone, false) : total, whole_share(top_p)), (u64)1);
    end_order(least > 1u ? min(k, fit) : k, need, true);
  }

  // ---------------------------------------------------------------- the draw
  // Not all that weigh as much as the last one stay: those of the highest logits, and of equal ones of
  // the lowest indices. `last`: the key at the end; `room`: how many with it stay of this warp's tokens.
  const bool split = ties < tied;
  uint32_t last = 0u;
  u64 room = 0;
  if (split) {
    auto tied_keys = [&](auto f) {
      for (int i = lo + lane; i < min(hi, n); i += 32)
        if (weights[i] == border) f(key_at(i), 1u);
    };
    uint32_t low = 0xffffffffu, high = 0u;
    tied_keys([&](uint32_t v, uint32_t) {
      low = min(low, v);
      high = max(high, v);
    });
    low = ~block_max(~low);
    high = block_max(high);
    {
      const auto& all = tell(low, high, 0);
      for (uint32_t r = 0; r < blocks; ++r) {
        low = min(low, (uint32_t)all[r][0]);
        high = max(high, (uint32_t)all[r][1]);
      }
    }
    u64 w0 = 0, c0 = 0, wb = 0, cb = 0;
    // (an end found in a list splits nothing: the sums' place is theirs)
    last = narrow(low, high, ties, kNone, w0, c0, wb, cb, tied_keys);
    u64 mine = 0;
    tied_keys([&](uint32_t v, uint32_t) { mine += v == last; });
    mine = warp_sum64(mine);
    __syncthreads();
    if (lane == 0) s.scan[warp][2] = mine;
    __syncthreads();
    u64 before = 0, block = 0;
    for (int k = 0; k < kWarps; ++k) {
      if (k < warp) before += s.scan[k][2];
      block += s.scan[k][2];
    }
    const auto& all = tell(block, 0, 0);
    for (uint32_t r = 0; r < rank; ++r) before += all[r][0];
    room = ties - c0 > before ? ties - c0 - before : 0;
  }
  // The weights that stay of the warp's step from i on, four to a lane; `left`: of `room`.
  auto kept = [&](int i, u64& left) {
    uint4 x = *reinterpret_cast<const uint4*>(weights + i + lane * 4);
    if (!split) {
      const uint32_t from = tied ? border : border + 1u;
      return make_uint4(x.x >= from ? x.x : 0u, x.y >= from ? x.y : 0u, x.z >= from ? x.z : 0u, x.w >= from ? x.w : 0u);
    }
    uint32_t y[4] = {x.x, x.y, x.z, x.w}, at = 0u;  // at: which of the four are at the end
    u64 mine = 0;
#pragma unroll
    for (int z = 0; z < 4; ++z) {
      if (y[z] > border) continue;
      if (y[z] == border) {
        const uint32_t key = key_at(i + lane * 4 + z);
        if (key > last) continue;
        if (key == last) {
          at |= 1u << z;
          ++mine;
          continue;
        }
      }
      y[z] = 0u;
    }
    u64 to = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += p;
    }
    u64 rank_of = to - mine;
#pragma unroll
    for (int z = 0; z < 4; ++z)
      if ((at >> z) & 1u) {
        if (rank_of >= left) y[z] = 0u;
        ++rank_of;
      }
    left -= min(left, (u64)__shfl_sync(0xffffffffu, to, 31));
    return make_uint4(y[0], y[1], y[2], y[3]);
  };
  u64 sum = 0, left = room;
  for (int i = lo; i < hi; i += kStep) {
    const uint4 x = kept(i, left);
    sum += (u64)x.x + x.y + x.z + x.w;
  }
  sum = warp_sum64(sum);
  __syncthreads();
  if (lane == 0) s.scan[warp][0] = sum;
  __syncthreads();
  u64 block = 0, at = 0;
  for (int k = 0; k < kWarps; ++k) {
    if (k < warp) at += s.scan[k][0];
    block += s.scan[k][0];
  }
  const auto& each = tell(block, 0, 0);  // no block's shared memory is looked at by another from here on
  u64 all = 0;
  for (uint32_t r = 0; r < blocks; ++r) {
    if (r < rank) at += each[r][0];
    all += each[r][0];
  }
  const u64 u = min((u64)whole_share(a.uniforms[b]), kOne - 1), t = share_of(all, u);
  if (t < at || t >= at + sum) return;  // another warp has it
  left = room;
  for (int i = lo; i < hi; i += kStep) {
    const uint4 x = kept(i, left);
    const uint32_t y[4] = {x.x, x.y, x.z, x.w};
    const u64 mine = (u64)x.x + x.y + x.z + x.w;
    u64 to = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 p = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += p;
    }
    u64 from = at + to - mine;
    if (t >= from && t < from + mine) {
#pragma unroll
      for (int z = 0; z < 4; ++z) {
        if (t >= from && t < from + y[z]) {
          a.token[b] = x0 + i + lane * 4 + z;
          a.prob[b] = (float)((double)y[z] / (double)all);
        }
        from += y[z];
      }
    }
    at += __shfl_sync(0xffffffffu, to, 31);
    if (t < at) return;
  }
}

template <typename T>
int launch_sample(SampleArgs& a, cudaStream_t st) {
  const char* op = "nkl_sample";
  // Blocks to a row: as many as it takes for two blocks to fit on an SM (fp32 128 x 131072 121 us with 8, 124 with 4);
  // more, up to eight, as long as no SM gets a third block and each has 2048 tokens (64 x 32768 22 us with 4, 28 with 2, 37
  // with 8; 16 x 8192 13.8 with 4, 15.7 with 8; one row of 32768 14 with 8, 29 with 1).
  int blocks = 1;
  while (blocks < kMaxCluster && (a.vocab > blocks * kPerHalf ||
                                  ((int64_t)a.batch * blocks <= sm_count() && a.vocab >= 4096 * blocks)))
    blocks *= 2;
  a.part = ((a.vocab + blocks - 1) / blocks + kWarps * kStep - 1) / (kWarps * kStep) * (kWarps * kStep);
  const size_t smem = (size_t)a.part * 4;
  static std::atomic<bool> set[64] = {};  // per device: the shared memory attribute is set (idempotent)
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64 || !set[dev].load(std::memory_order_acquire)) {
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kPerBlock * 4);
    if (e != cudaSuccess) return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
    if (dev >= 0 && dev < 64) set[dev].store(true, std::memory_order_release);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<T>, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NKL_ERR_CUDA, "%s: %s", op, cudaGetErrorString(e));
  }
  return NKL_OK;
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_sample(const void* logits, int64_t row_stride, const float* uniforms, const float* temperatures,
                          const int32_t* top_ks, const float* top_ps, const float* min_ps, float temperature, int top_k,
                          float top_p, float min_p, int32_t* token, float* prob, int64_t batch, int64_t vocab, int dtype,
                          void* stream) {
  const char* op = "nkl_sample";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (batch < 0 || batch > (1LL << 27) || vocab < 1 || vocab > NKL_MAX_VOCAB)
    return fail(NKL_ERR_SHAPE, "%s: batch %lld or vocabulary %lld out of range (up to %d tokens)", op, (long long)batch,
                (long long)vocab, NKL_MAX_VOCAB);
  if (batch == 0) return NKL_OK;
  if (!logits || !uniforms || !token || !prob) return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (batch > 1 && row_stride < 0) return fail(NKL_ERR_SHAPE, "%s: row stride %lld", op, (long long)row_stride);
  if (!is_aligned(logits, dtype_size(dtype))) return fail(NKL_ERR_ALIGN, "%s: misaligned logits", op);
  SampleArgs a = {};
  a.logits = logits; a.stride = row_stride; a.uniforms = uniforms;
  a.temperatures = temperatures; a.top_ks = top_ks; a.top_ps = top_ps; a.min_ps = min_ps;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.token = token; a.prob = prob; a.batch = (int)batch; a.vocab = (int)vocab;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == NKL_FLOAT32 ? launch_sample<float>(a, st) : launch_sample<bf16>(a, st);
}
