// sample.cu - the next token of each row of logits: temperature, top-k, top-p, min-p, from given
// uniform numbers.
//
// A row's tokens in order of their logits, of equal ones the lowest index first, have the weights
//   w = floor(2^31 exp((x - max) / T))
// What is drawn from is the longest beginning of that order that every filter allows: top-k its k first
// tokens; top-p the fewest whose weights come to the share p of the top-k's; min-p those of at least
// p times the first one's weight. Of it the token is the first one, by index, with which
// the cumulative weight is over the uniform number's share of the sum. Weights, shares and uniform
// numbers are whole multiples of 2^-31, so that sums do not depend on their order, and equal
// inputs give equal tokens on every launch. NaN counts as minus infinity, and minus infinity is never
// drawn; T of 0 (or below, or NaN) takes the first token.
//
// A cluster of up to eight blocks takes a row; each holds its part in shared memory as keys whose order
// is the logits'. The order's end is found without sorting: a histogram of weights and counts
// over 1024 ranges of the logit (by distance from the maximum, which spreads them out), in it the
// range where the first filter ends the order; then, among that range's keys, over 1024 ranges of the
// key, until a range is one key; of equal ones the lowest indices stay. Blocks add their
// histograms up through distributed shared memory, an eighth of the ranges each.
#include <algorithm>
#include <atomic>

#include "common.cuh"

namespace nkl {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBins = 1024;
constexpr int kPerBlock = 49152;  // keys that a block holds: 192 KB
constexpr u64 kOne = 1ull << 31;
constexpr uint32_t kNever = 0u;   // the key of minus infinity and NaN: below all others

struct SampleArgs {
  const void* logits;
  int64_t stride;  // of the rows, in elements
  const float *uniforms, *temperatures, *top_ps, *min_ps;  // arrays of the rows, or NULL: the number below
  const int* top_ks;
  float temperature, top_p, min_p;
  int top_k;
  int* token;
  float* prob;
  int batch, vocab, part;  // part: keys of a block
};

// Keys in the order of the numbers; -0 counts as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  if (!(x > -INFINITY)) return kNever;
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// exp(z) for z <= 0, to some 2^-52 of it, times 2^31 and rounded down: exp(z) = 2^n 2^(j / 64) e^r, n and j
// whole, |r| <= ln 2 / 128, with e^r by its series.
__device__ __forceinline__ uint32_t weight_of(double z, const double* table) {
  if (!(z > -22.0)) return 0u;  // below 2^-31
  const double t = z * 92.332482616893656877;  // 64 / ln 2
  const double k = rint(t);
  const int i = (int)k;
  const double r = fma(k, -0.010830424696249145, z);  // ln 2 / 64
  const double e = fma(fma(fma(fma(fma(r, 1.0 / 120, 1.0 / 24), r, 1.0 / 6), r, 0.5), r, 1.0), r, 1.0);
  const double power = __hiloint2double(((i >> 6) + 31 + 1023) << 20, 0);  // 2^(n + 31)
  return __double2uint_rd(e * table[i & 63] * power);
}

__device__ __forceinline__ uint32_t whole_share(float x) {  // of [0, 1], in multiples of 2^-31
  return x > 0.f ? (uint32_t)(fminf(x, 1.f) * 2147483648.f) : 0u;
}
__device__ __forceinline__ u64 share_of(u64 total, u64 share) {
  return (total >> 31) * share + (((total & (kOne - 1)) * share) >> 31);
}

__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return at;
}
__device__ __forceinline__ void put(u64* p, uint32_t rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
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

struct Histogram {  // a range's weights as two halves of 16 and 15 bits, which do not overflow for 2^16 keys
  uint32_t lo[kBins], hi[kBins], count[kBins];
};
struct Shared {
  Histogram h;
  double table[64];
  u64 all[2][kMaxCluster][2];                // what each block has to tell the others, in turn
  u64 bins[kMaxCluster][kBins / kMaxCluster][2];  // sums over the blocks: weights and counts of each range
  u64 scan[kWarps][2];
  uint32_t reduce[kWarps];
  int bin, token;
  u64 before[2];
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint32_t keys[];
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
  const int asked = a.top_ks ? a.top_ks[b] : a.top_k;
  if (tid < 64) s.table[tid] = exp2((double)tid / 64);

  // Every block's (x, y) to every block. The places take turns: what a call wrote is read before the next
  // call's barrier, and written again after it.
  int turn = 0;
  auto tell = [&](u64 x, u64 y) -> const u64(&)[kMaxCluster][2] {
    u64(&to)[kMaxCluster][2] = s.all[turn];
    turn ^= 1;
    if (tid < (int)blocks) {
      put(&to[rank][0], tid, x);
      put(&to[rank][1], tid, y);
    }
    cluster_sync();
    return to;
  };

  // ---------------------------------------------------------------- keys and their maximum
  uint32_t top = kNever;
  int first = 0x7fffffff;
  {
    constexpr int VE = Vec16<T>::N;
    const bool vec = reinterpret_cast<uintptr_t>(row) % 16 == 0;
    const int whole = vec ? n / VE * VE : 0;
#pragma unroll 4
    for (int i = tid * VE; i < whole; i += kThreads * VE) {
      Vec16<T> v;
      v.raw = *reinterpret_cast<const uint4*>(row + i);
#pragma unroll
      for (int e = 0; e < VE; e += 4) {
        const uint4 k = make_uint4(key_of(v.get(e)), key_of(v.get(e + 1)), key_of(v.get(e + 2)), key_of(v.get(e + 3)));
        *reinterpret_cast<uint4*>(keys + i + e) = k;
        top = max(top, max(max(k.x, k.y), max(k.z, k.w)));
      }
    }
    for (int i = whole + tid; i < n; i += kThreads) {
      const uint32_t k = key_of(to_f32(row[i]));
      keys[i] = k;
      top = max(top, k);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if (lane == 0) s.reduce[warp] = top;
  __syncthreads();
  top = __reduce_max_sync(0xffffffffu, s.reduce[lane & (kWarps - 1)]);
  // the first index of the block's maximum: the first token of the order, if it is the row's
  for (int i = tid; i < n && first == 0x7fffffff; i += kThreads)
    if (keys[i] == top) first = x0 + i;
  first = (int)__reduce_min_sync(0xffffffffu, (uint32_t)first);
  __syncthreads();
  if (lane == 0) s.reduce[warp] = (uint32_t)first;
  __syncthreads();
  first = (int)__reduce_min_sync(0xffffffffu, s.reduce[lane & (kWarps - 1)]);
  cluster_wait_started();
  {
    const auto& all = tell(top, (u64)first);
    for (uint32_t r = 0; r < blocks; ++r) {
      const uint32_t its = (uint32_t)all[r][0];
      if (its > top || (its == top && (int)all[r][1] < first)) first = (int)all[r][1];
      top = max(top, its);
    }
  }
  if (top == kNever || !(temperature > 0.f) || asked == 1) {
    if (rank == 0 && tid == 0) {
      a.token[b] = top == kNever ? -1 : first;
      a.prob[b] = top == kNever ? 0.f : 1.f;
    }
    return;
  }

  const double highest = (double)value_of(top), rate = 1.0 / (double)temperature;
  auto weigh = [&](uint32_t key) -> uint32_t {
    if (key == kNever) return 0u;
    return key == top ? (uint32_t)kOne : weight_of(((double)value_of(key) - highest) * rate, s.table);
  };
  const bool by_count = asked > 0 && asked < a.vocab, by_share = top_p < 1.f;
  // min-p's least weight: a token stays if its weight is at least that
  const uint32_t least = min_p > 0.f ? (uint32_t)__double2ull_ru((double)fminf(min_p, 1.f) * 2147483648.0) : 0u;

  // ---------------------------------------------------------------- where the order ends
  // Tokens above `border` stay, of those at it the `ties` first ones.
  uint32_t border = kNever;
  u64 ties = ~0ull;
  // One descent: the place in the order where the count reaches `count` or the weights reach `need`
  // (whichever is first), among the keys of [lo, hi].
  auto descend = [&](u64 count, u64 need) {
    uint32_t lo = 1u, hi = top;
    u64 c0 = 0, w0 = 0;  // of the keys above hi
    for (int round = 0;; ++round) {
      // ranges of the first round: distance from the maximum, in steps of T / 32, the last one open
      // (32 T below it weights are 0); then equal parts of [lo, hi]
      const float step = 32.f / temperature;
      const uint32_t span = hi - lo;
      const int shift = max(0, 32 - __clz(span) - 10);
      auto bin_of = [&](uint32_t key) {  // 0: the highest
        if (round == 0) {
          const float d = (value_of(top) - value_of(key)) * step;
          return key == top ? 0 : d < (float)(kBins - 1) ? (int)d : kBins - 1;  // NaN and infinity: the last
        }
        return (int)((hi - key) >> shift);
      };
      for (int i = tid; i < kBins; i += kThreads) s.h.lo[i] = s.h.hi[i] = s.h.count[i] = 0u;
      __syncthreads();
      for (int base = 0; base < n; base += kThreads) {
        const int i = base + tid;
        const uint32_t key = i < n ? keys[i] : kNever;
        const bool in = key >= lo && key <= hi;
        const int bin = in ? bin_of(key) : -1;
        const uint32_t w = in && by_share ? weigh(key) : 0u;
        // equal ranges of a warp are added up first: rows of few different logits would queue up
        const unsigned same = __match_any_sync(0xffffffffu, bin);
        if (same == 0xffffffffu) {
          const u64 sum = warp_sum64(w);
          if (lane == 0 && bin >= 0) {
            atomicAdd(&s.h.count[bin], 32u);
            atomicAdd(&s.h.lo[bin], (uint32_t)(sum & 0xffffu));
            atomicAdd(&s.h.hi[bin], (uint32_t)(sum >> 16));
          }
        } else if (in) {
          atomicAdd(&s.h.count[bin], 1u);
          if (by_share) {
            atomicAdd(&s.h.lo[bin], w & 0xffffu);
            atomicAdd(&s.h.hi[bin], w >> 16);
          }
        }
      }
      cluster_sync();
      // this block's ranges, over all blocks; to all blocks
      const int per = kBins / (int)blocks;
      for (int i = tid; i < per; i += kThreads) {
        const int bin = (int)rank * per + i;
        u64 w = 0, c = 0;
        for (uint32_t r = 0; r < blocks; ++r) {
          w += get(&s.h.lo[bin], r) + ((u64)get(&s.h.hi[bin], r) << 16);
          c += get(&s.h.count[bin], r);
        }
        for (uint32_t r = 0; r < blocks; ++r) {
          u64* const to = &s.bins[0][0][0] + 2 * bin;
          put(to, r, w);
          put(to + 1, r, c);
        }
      }
      cluster_sync();
      // the range where the order ends: two ranges to a thread
      const u64* const sums = &s.bins[0][0][0];
      u64 w[2], c[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        w[k] = sums[2 * (2 * tid + k)];
        c[k] = sums[2 * (2 * tid + k) + 1];
      }
      u64 wi = w[0] + w[1], ci = c[0] + c[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const u64 p = __shfl_up_sync(0xffffffffu, wi, o), q = __shfl_up_sync(0xffffffffu, ci, o);
        if (lane >= o) {
          wi += p;
          ci += q;
        }
      }
      if (lane == 31) {
        s.scan[warp][0] = wi;
        s.scan[warp][1] = ci;
      }
      if (tid == 0) s.bin = -1;
      __syncthreads();
      wi += w0;
      ci += c0;
      for (int k = 0; k < warp; ++k) {
        wi += s.scan[k][0];
        ci += s.scan[k][1];
      }
      // inclusive up to the thread's second range; the range that crosses first
      const u64 w_before = wi - w[0] - w[1], c_before = ci - c[0] - c[1];
      if (w_before < need && c_before < count && (wi >= need || ci >= count)) {
        const bool one = w_before + w[0] >= need || c_before + c[0] >= count;
        s.bin = 2 * tid + (one ? 0 : 1);
        s.before[0] = w_before + (one ? 0 : w[0]);
        s.before[1] = c_before + (one ? 0 : c[0]);
      }
      __syncthreads();
      const int bin = s.bin;
      if (bin < 0) {  // no end: the whole order
        border = kNever;
        ties = ~0ull;
        return;
      }
      w0 = s.before[0];
      c0 = s.before[1];
      if (round == 0) {
        // the range's keys: from its lowest to its highest, found among the keys
        uint32_t low = 0xffffffffu, high = 0u;
        for (int i = tid; i < n; i += kThreads) {
          const uint32_t key = keys[i];
          if (key == kNever || bin_of(key) != bin) continue;
          low = min(low, key);
          high = max(high, key);
        }
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        __syncthreads();
        if (lane == 0) s.scan[warp][0] = (u64)low << 32 | high;
        __syncthreads();
        for (int k = 0; k < kWarps; ++k) {
          low = min(low, (uint32_t)(s.scan[k][0] >> 32));
          high = max(high, (uint32_t)s.scan[k][0]);
        }
        const auto& all = tell(low, high);
        for (uint32_t r = 0; r < blocks; ++r) {
          low = min(low, (uint32_t)all[r][0]);
          high = max(high, (uint32_t)all[r][1]);
        }
        lo = low;
        hi = high;
      } else {
        const uint32_t to = hi - ((uint32_t)bin << shift);
        lo = max(lo, shift ? to - min(to - lo, (1u << shift) - 1u) : to);
        hi = to;
      }
      __syncthreads();  // the histogram and the sums are used again
      if (lo == hi) {   // one key: of its tokens as many stay as it takes
        const uint32_t w = weigh(lo);
        u64 t = count - c0;
        if (by_share && need != ~0ull && w > 0) t = min(t, (need - w0 + w - 1) / w);
        border = lo;
        ties = t;
        return;
      }
    }
  };
  auto stays = [&](uint32_t key) { return key > border; };

  // the sum over the cluster of a block's value, thread by thread
  auto total_of = [&](u64 mine, u64& before) {
    mine = warp_sum64(mine);
    __syncthreads();
    if (lane == 0) s.scan[warp][0] = mine;
    __syncthreads();
    u64 block = 0;
    for (int k = 0; k < kWarps; ++k) block += s.scan[k][0];
    const auto& each = tell(block, 0);
    u64 all = 0;
    before = 0;
    for (uint32_t r = 0; r < blocks; ++r) {
      if (r == rank) before = all;
      all += each[r][0];
    }
    return all;
  };
  u64 need = ~0ull, before;
  if (by_count) {
    descend((u64)asked, ~0ull);
    if (by_share) {  // the top-k's weights
      u64 sum = 0;
      for (int i = tid; i < n; i += kThreads) sum += stays(keys[i]) ? weigh(keys[i]) : 0u;
      sum = total_of(sum, before) + (ties == ~0ull ? 0 : ties * weigh(border));
      need = max(share_of(sum, whole_share(top_p)), (u64)1);
      descend((u64)asked, need);
    }
  } else if (by_share) {
    u64 sum = 0;
    for (int i = tid; i < n; i += kThreads) sum += weigh(keys[i]);
    sum = total_of(sum, before);
    need = max(share_of(sum, whole_share(top_p)), (u64)1);
    descend(~0ull, need);
  }

  // ---------------------------------------------------------------- the draw
  // Of the tokens at the border those of the lowest indices stay: how many a block has of them, and the
  // blocks before it.
  u64 left = 0;
  if (ties != ~0ull) {
    u64 mine = 0;
    for (int i = tid; i < n; i += kThreads) mine += keys[i] == border;
    total_of(mine, before);
    left = ties > before ? ties - before : 0;  // that this block's keep
  }
  // Warps take contiguous parts: the kept weights in index order.
  const int per = (n + kWarps * 32 - 1) / (kWarps * 32) * 32, lo = min(warp * per, n), hi = min(lo + per, n);
  u64 tied = 0;  // at the border, in this warp's part
  if (ties != ~0ull) {
    for (int i = lo + lane; i < hi; i += 32) tied += keys[i] == border;
    tied = warp_sum64(tied);
    __syncthreads();
    if (lane == 0) s.scan[warp][1] = tied;
    __syncthreads();
    u64 at = 0;
    for (int k = 0; k < warp; ++k) at += s.scan[k][1];
    left = left > at ? left - at : 0;  // that this warp's part keeps
  }
  auto kept = [&](int i, u64& room) -> uint32_t {  // the warp's, 32 in a row from i; room: border tokens that may stay
    const uint32_t key = i + lane < hi ? keys[i + lane] : kNever;
    bool stay = key > border && key != kNever;
    if (ties != ~0ull) {
      const unsigned at = __ballot_sync(0xffffffffu, key == border && i + lane < hi);
      if (key == border) stay = (u64)__popc(at & ((1u << lane) - 1u)) < room;
      room -= min(room, (u64)__popc(at));
    }
    const uint32_t w = stay ? weigh(key) : 0u;
    return w >= least ? w : 0u;
  };
  u64 sum = 0, room = left;
  for (int i = lo; i < hi; i += 32) sum += kept(i, room);
  sum = warp_sum64(sum);
  __syncthreads();
  if (lane == 0) s.scan[warp][0] = sum;
  __syncthreads();
  u64 block = 0, at = 0;
  for (int k = 0; k < kWarps; ++k) {
    if (k < warp) at += s.scan[k][0];
    block += s.scan[k][0];
  }
  const auto& each = tell(block, 0);  // no block's shared memory is looked at by another from here on
  u64 total = 0;
  for (uint32_t r = 0; r < blocks; ++r) {
    if (r < rank) at += each[r][0];
    total += each[r][0];
  }
  const u64 u = min((u64)whole_share(a.uniforms[b]), kOne - 1), t = share_of(total, u);
  if (t < at || t >= at + sum) return;
  room = left;
  for (int i = lo; i < hi; i += 32) {
    const uint32_t w = kept(i, room);
    u64 to = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += y;
    }
    if (t >= at + to - w && t < at + to) {
      a.token[b] = x0 + i + lane;
      a.prob[b] = (float)((double)w / (double)total);
    }
    at += __shfl_sync(0xffffffffu, to, 31);
    if (t < at) return;
  }
}

template <typename T>
int launch_sample(SampleArgs& a, cudaStream_t st) {
  const char* op = "nkl_sample";
  // Blocks to a row: as many as its keys need; more, up to eight, as long as there are no more than two for
  // each SM and each has 1024 keys.
  int blocks = 1;
  while (blocks < kMaxCluster && ((a.vocab + blocks - 1) / blocks > kPerBlock ||
                                  ((int64_t)a.batch * blocks * 2 <= 2LL * sm_count() && a.vocab >= 2 * blocks * 1024)))
    blocks *= 2;
  a.part = ((a.vocab + blocks - 1) / blocks + 15) / 16 * 16;
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
