// verify.cu - verification of drafted tokens against the target's probabilities.
//
// A sequence has T drafted tokens and T + 1 rows of target probabilities: row 0 follows the
// last accepted token, row i + 1 follows drafted token i. From given uniform numbers the
// walk accepts a path of drafted tokens and draws the token after it, such that the tokens
// are distributed as the target's:
//   chain with draft rows q   token i is accepted if u_i q_i(x_i) < p_i(x_i); at the first
//                             rejection the next token has weights max(p_i - q_i, 0)
//   tree (or no draft rows)   the children of the current node are tried in index order: x_c
//                             is accepted if u_c m < p(x_c), m being the mass that the
//                             rejected ones before it left; with none accepted the next
//                             token has the weights p without the rejected tokens
// The next token is the first x whose cumulative weight exceeds u_T times their sum.
//
// All of it is done in whole numbers: p, q and u are taken as multiples of 2^-31 (rounded
// down; an fp32 softmax row is itself no better than 2^-24 of its largest value), sums are
// 64 bit. Sums of whole numbers do not depend on their order, so the drawn token is the same
// for every launch shape, which a cumulative sum in fp32 is not.
//
// A cluster of blocks takes one sequence. Each block walks for itself (some hundred values,
// from L2); then each warp sums a contiguous part of the one row (with q: two) that the next
// token is drawn from, the blocks exchange their sums through shared memory, and the block that
// holds the drawn place reads the part of the warp where it lies once more, from L2, a step for
// each of its warps. So each of those rows is read from HBM once.
//
// Measured, fp32, GPU time: 64 chains of 8 over 131072 (two rows each, 67 MB) 20.5 us, of which
// 10.3 us by bytes; the rest is the chain launch -> tokens -> gathered probabilities -> first
// vectors of the rows, and after them exchange -> part, which does not overlap the reading. With the
// part read by its warp alone, four steps at a time, it was 26.1 us; with one block to a sequence
// and one element a lane at a time 204 us. One tree of 24 over 32768 is that chain and no more:
// 7.8 us, with one block 40 us.
#include "common.cuh"

namespace nkl {
namespace {

constexpr int kMaxDrafted = NKL_MAX_DRAFTED;
constexpr int kVerifyThreads = 512;
constexpr int kVerifyWarps = kVerifyThreads / 32;
constexpr unsigned long long kOne = 1ull << 31;

// p in [0, 1] as a multiple of 2^-31; NaN and negative values are 0.
__device__ __forceinline__ uint32_t whole(float p) {
  return p > 0.f ? (uint32_t)(fminf(p, 1.f) * 2147483648.f) : 0u;
}
__device__ __forceinline__ unsigned long long whole_u(float u) {
  return min((unsigned long long)whole(u), kOne - 1);
}

struct VerifyArgs {
  const void *probs, *draft;
  const int* tokens;
  const float* uniforms;
  const int* parents;
  int *path, *count, *token;
  int batch, drafted, vocab;
};

typedef unsigned long long u64;

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Weights of N elements x0 .. x0 + N - 1 of a row, less those of q; 0 from the row's end on.
// VEC: rows are 16-byte aligned and whole vectors long.
template <typename T, bool VEC, int N>
__device__ __forceinline__ void load_row(const T* p, int x0, int end, uint32_t (&w)[N]) {
  static_assert(N == Vec16<T>::N, "one vector");
  if constexpr (VEC) {
    Vec16<T> v;
    v.raw = x0 < end ? *reinterpret_cast<const uint4*>(p + x0) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = whole(v.get(e));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) w[e] = x0 + e < end ? whole(to_f32(p[x0 + e])) : 0u;
  }
}

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// Stores to the same shared variable of another block of the cluster.
__device__ __forceinline__ void store_remote(u64* p, uint32_t rank, u64 v) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}
constexpr int kMaxCluster = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  constexpr int VE = Vec16<T>::N;
  __shared__ int s_token[kMaxDrafted], s_parent[kMaxDrafted], s_next[kMaxDrafted + 1];
  __shared__ uint32_t s_mass[kMaxDrafted], s_left[kMaxDrafted];
  __shared__ int s_last;
  __shared__ u64 s_sum[kVerifyWarps], s_all[kVerifyWarps];
  __shared__ u64 s_blocks[kMaxCluster][2];  // the cluster's sums and sums of whole rows
  cluster_started();
  pdl_enter();
  const int blocks = (int)cluster_size(), rank = (int)cluster_rank();
  const int b = blockIdx.x / blocks, n = a.drafted, V = a.vocab;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* probs = static_cast<const T*>(a.probs) + (int64_t)b * (n + 1) * V;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + (int64_t)b * n * V : nullptr;
  const float* u = a.uniforms + (int64_t)b * (n + 1);

  // each drafted token's mass in its parent's row; parent -2 marks one that cannot be accepted
  u64 my_u = 0;
  if (tid < n) {
    const int x = a.tokens[(int64_t)b * n + tid];
    int up = a.parents ? a.parents[(int64_t)b * n + tid] : tid - 1;
    if (up >= tid) up = -1;
    if (x < 0 || x >= V || up < -1) up = -2;
    my_u = whole_u(u[tid]);
    s_token[tid] = x;
    s_parent[tid] = up;
    s_mass[tid] = up >= -1 ? whole(to_f32(probs[(int64_t)(up + 1) * V + x])) : 0u;
    // what the chain's test compares with; the tree's is found below
    s_left[tid] = draft ? (up >= -1 ? whole(to_f32(draft[(int64_t)tid * V + x])) : 0u) : (uint32_t)kOne;
  }
  if (tid <= n) s_next[tid] = 0x7fffffff;
  const u64 last_u = whole_u(u[n]);
  __syncthreads();
  if (!draft && a.parents) {
    // a token that an earlier brother has had already has no mass left
    for (int i = warp; i < n; i += kVerifyWarps) {
      const int up = s_parent[i], x = s_token[i];
      bool again = false;
      for (int j = lane; j < i; j += 32) again |= s_parent[j] == up && s_token[j] == x;
      if (__any_sync(0xffffffffu, again) && lane == 0) s_mass[i] = 0u;  // read by no one before the barrier
    }
    __syncthreads();
    // the mass that the brothers before a token leave, if they are rejected
    for (int i = warp; i < n; i += kVerifyWarps) {
      const int up = s_parent[i];
      u64 out = 0;
      for (int j = lane; j < i; j += 32) out += s_parent[j] == up ? s_mass[j] : 0u;
      out = warp_sum64(out);
      if (lane == 0) s_left[i] = (uint32_t)(kOne - min(out, kOne));
    }
    __syncthreads();
  }
  // s_next[node + 1]: the node's first child that is accepted when the walk stands there
  if (tid < n && s_parent[tid] >= -1 && my_u * s_left[tid] < s_mass[tid] * kOne) atomicMin(&s_next[s_parent[tid] + 1], tid);
  __syncthreads();
  if (tid == 0) {
    int at = -1, c = 0;
    for (int i; (i = s_next[at + 1]) != 0x7fffffff; at = i, ++c)
      if (rank == 0) a.path[(int64_t)b * n + c] = i;
    s_last = at;
    if (rank == 0) {
      a.count[b] = c;
      for (; c < n; ++c) a.path[(int64_t)b * n + c] = -1;
    }
  }
  __syncthreads();
  const int last = s_last;

  // the next token's weights: row p of the last accepted token, less q or the rejected tokens
  const T* p = probs + (int64_t)(last + 1) * V;
  const T* q = draft && last + 1 < n && s_parent[last + 1] >= -1 ? draft + (int64_t)(last + 1) * V : nullptr;
  const int step = 32 * VE, parts = blocks * kVerifyWarps;
  const int per_warp = (V + parts * step - 1) / (parts * step) * step;
  const int64_t begin = (int64_t)(rank * kVerifyWarps + warp) * per_warp;
  const int lo = (int)min(begin, (int64_t)V), hi = min(lo + per_warp, V);
  u64 sum = 0, all = 0;
  if (q) {
#pragma unroll 4
    for (int x = lo + lane * VE; x < hi; x += step) {
      uint32_t pw[VE], qw[VE];
      load_row<T, VEC>(p, x, hi, pw);
      load_row<T, VEC>(q, x, hi, qw);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        all += pw[e];
        sum += pw[e] > qw[e] ? pw[e] - qw[e] : 0u;
      }
    }
  } else {
#pragma unroll 4
    for (int x = lo + lane * VE; x < hi; x += step) {
      uint32_t pw[VE];
      load_row<T, VEC>(p, x, hi, pw);
#pragma unroll
      for (int e = 0; e < VE; ++e) all += pw[e];
    }
  }
  all = warp_sum64(all);
  sum = q ? warp_sum64(sum) : all;
  if (!draft) {
    u64 out = 0;
    for (int i = lane; i < n; i += 32)
      if (s_parent[i] == last && s_token[i] >= lo && s_token[i] < hi) out += s_mass[i];
    sum -= warp_sum64(out);
  }
  if (lane == 0) {
    s_sum[warp] = sum;
    s_all[warp] = all;
  }
  __syncthreads();
  cluster_wait_started();  // no wait by now: the row has been read since
  if (warp == 0) {  // the block's sums to every block
    const u64 x = warp_sum64(lane < kVerifyWarps ? s_sum[lane] : 0), y = warp_sum64(lane < kVerifyWarps ? s_all[lane] : 0);
    if (lane < blocks) {
      store_remote(&s_blocks[rank][0], lane, x);
      store_remote(&s_blocks[rank][1], lane, y);
    }
  }
  cluster_sync();
  u64 total = 0, total_all = 0;
  for (int r = 0; r < blocks; ++r) {
    total += s_blocks[r][0];
    total_all += s_blocks[r][1];
  }
  const bool plain = total == 0;  // nothing left: the row itself
  if (plain) total = total_all;
  if (total == 0) {
    if (rank == 0 && tid == 0) a.token[b] = -1;
    return;
  }
  const u64 t = (total >> 31) * last_u + (((total & (kOne - 1)) * last_u) >> 31);
  u64 before = 0;
  for (int r = 0; r < rank; ++r) before += s_blocks[r][plain];
  if (t < before || t >= before + s_blocks[rank][plain]) return;  // another block has it
  // the warp that has it, whose part the block's warps read again, a step each
  int owner = 0;
  for (; owner < kVerifyWarps - 1; ++owner) {
    const u64 x = plain ? s_all[owner] : s_sum[owner];
    if (t < before + x) break;
    before += x;
  }
  __syncthreads();  // the sums' place is used again
  const int64_t from = (int64_t)(rank * kVerifyWarps + owner) * per_warp;
  const int part_lo = (int)min(from, (int64_t)V), part_hi = min(part_lo + per_warp, V);
  for (int base = part_lo; base < part_hi; base += kVerifyWarps * step) {
    const int x0 = base + warp * step + lane * VE;
    uint32_t w[VE];
    load_row<T, VEC>(p, x0, part_hi, w);
    if (q && !plain) {
      uint32_t qw[VE];
      load_row<T, VEC>(q, x0, part_hi, qw);
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = w[e] > qw[e] ? w[e] - qw[e] : 0u;
    }
    if (!draft && !plain) {
      for (int j = 0; j < n; ++j) {
        if (s_parent[j] != last) continue;
#pragma unroll
        for (int e = 0; e < VE; ++e) w[e] = s_token[j] == x0 + e ? 0u : w[e];
      }
    }
    u64 mine = 0;
#pragma unroll
    for (int e = 0; e < VE; ++e) mine += w[e];
    u64 to = mine;  // the sum up to this lane
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 y = __shfl_up_sync(0xffffffffu, to, o);
      if (lane >= o) to += y;
    }
    if (lane == 31) s_sum[warp] = to;
    __syncthreads();
    u64 at = before;
    for (int k = 0; k < kVerifyWarps; ++k) {
      if (k < warp) at += s_sum[k];
      before += s_sum[k];
    }
    at += to - mine;
    if (t >= at && t < at + mine) {  // one lane of the block at most
      int e = 0;
#pragma unroll
      for (int k = 0; k < VE; ++k) {
        at += w[k];
        if (at <= t) e = k + 1;
      }
      a.token[b] = x0 + e;
    }
    if (t < before) return;
    __syncthreads();
  }
}

template <typename T>
int launch_verify(const VerifyArgs& a, cudaStream_t st) {
  // Blocks per sequence: up to eight, as long as there are no more than three for each SM (two
  // fit at once) and a warp's part still has a step of its own. Measured over 131072, chains, with
  // 1, 2, 4, 8 blocks: 4 sequences 24.4, 14.6, 10.0, 7.6 us; 32: 47, 27, 17, 13.7; 64: 50, 29, 20.7,
  // 25.6; 100: 52, 33, 27, 34; 200: 57, 43, 43, 52; 400: 73, 71, 69, 85.
  int blocks = kMaxCluster;
  while (blocks > 1 && ((int64_t)a.batch * blocks > 3LL * sm_count() ||
                        (int64_t)blocks * kVerifyWarps * 32 * Vec16<T>::N > 2LL * a.vocab))
    blocks /= 2;
  const bool vec = a.vocab % Vec16<T>::N == 0 && is_aligned(a.probs, 16) && (!a.draft || is_aligned(a.draft, 16));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.batch * blocks));
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim = {(unsigned)blocks, 1, 1};
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, verify_kernel<T, true>, a) : cudaLaunchKernelEx(&cfg, verify_kernel<T, false>, a);
  if (e != cudaSuccess) {
    (void)cudaGetLastError();
    return fail(NKL_ERR_CUDA, "nkl_verify_drafts: %s", cudaGetErrorString(e));
  }
  return NKL_OK;
}

}  // namespace
}  // namespace nkl

using namespace nkl;

extern "C" int nkl_verify_drafts(const void* probs, const void* draft_probs, const int32_t* tokens,
                                 const float* uniforms, const int32_t* parents, int32_t* path, int32_t* count,
                                 int32_t* token, int64_t batch, int64_t drafted, int64_t vocab, int dtype,
                                 void* stream) {
  const char* op = "nkl_verify_drafts";
  if (!valid_dtype(dtype)) return fail(NKL_ERR_DTYPE, "%s: unsupported dtype %d", op, dtype);
  if (batch < 0 || batch > (1LL << 27) || vocab < 1 || vocab > (1LL << 30))
    return fail(NKL_ERR_SHAPE, "%s: batch %lld or vocabulary %lld out of range", op, (long long)batch, (long long)vocab);
  if (drafted < 0 || drafted > kMaxDrafted)
    return fail(NKL_ERR_SHAPE, "%s: %lld drafted tokens, at most %d are taken", op, (long long)drafted, kMaxDrafted);
  if (draft_probs && parents) return fail(NKL_ERR_ARG, "%s: draft probabilities go with a chain, not with a tree", op);
  if (batch == 0) return NKL_OK;
  if (!probs || !uniforms || !count || !token || (drafted && (!tokens || !path)))
    return fail(NKL_ERR_ARG, "%s: NULL pointer", op);
  if (!is_aligned(probs, dtype_size(dtype)) || (draft_probs && !is_aligned(draft_probs, dtype_size(dtype))))
    return fail(NKL_ERR_ALIGN, "%s: misaligned probabilities", op);
  VerifyArgs a = {probs, draft_probs, tokens,     uniforms,     parents,   path,
                  count, token,       (int)batch, (int)drafted, (int)vocab};
  if (drafted == 0) a.draft = nullptr;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == NKL_FLOAT32 ? launch_verify<float>(a, st) : launch_verify<bf16>(a, st);
}
