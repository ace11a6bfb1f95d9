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

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// One block per sequence.
template <typename T>
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(const __grid_constant__ VerifyArgs a) {
  __shared__ int s_token[kMaxDrafted], s_parent[kMaxDrafted], s_next[kMaxDrafted + 1];
  __shared__ uint32_t s_mass[kMaxDrafted];
  __shared__ int s_last, s_count;
  __shared__ unsigned long long s_sum[kVerifyWarps], s_all[kVerifyWarps];
  pdl_enter();
  const int b = blockIdx.x, n = a.drafted, V = a.vocab;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* probs = static_cast<const T*>(a.probs) + (int64_t)b * (n + 1) * V;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + (int64_t)b * n * V : nullptr;
  const float* u = a.uniforms + (int64_t)b * (n + 1);

  // each drafted token's mass in its parent's row; parent -2 marks one that cannot be accepted
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int x = a.tokens[(int64_t)b * n + i];
    int up = a.parents ? a.parents[(int64_t)b * n + i] : i - 1;
    if (up >= i) up = -1;
    if (x < 0 || x >= V || up < -1) up = -2;
    s_token[i] = x;
    s_parent[i] = up;
    s_mass[i] = up >= -1 ? whole(to_f32(probs[(int64_t)(up + 1) * V + x])) : 0u;
  }
  for (int i = tid; i <= n; i += kVerifyThreads) s_next[i] = 0x7fffffff;
  __syncthreads();
  // s_next[node + 1]: the node's first child that is accepted when the walk stands there
  for (int i = tid; i < n; i += kVerifyThreads) {
    const int up = s_parent[i], x = s_token[i];
    if (up < -1) continue;
    unsigned long long left = kOne, mass = s_mass[i];
    if (draft) {
      left = whole(to_f32(draft[(int64_t)i * V + x]));
    } else {
      for (int j = 0; j < i; ++j) {
        if (s_parent[j] != up) continue;
        if (s_token[j] == x) mass = 0;  // a token already rejected
        bool again = false;
        for (int k = 0; k < j; ++k) again |= s_parent[k] == up && s_token[k] == s_token[j];
        if (!again) left -= min((unsigned long long)s_mass[j], left);
      }
    }
    if (whole_u(u[i]) * left < mass * kOne) atomicMin(&s_next[up + 1], i);
  }
  __syncthreads();
  if (tid == 0) {
    int at = -1, c = 0;
    for (int i; (i = s_next[at + 1]) != 0x7fffffff; at = i) a.path[(int64_t)b * n + c++] = i;
    s_last = at;
    s_count = c;
    a.count[b] = c;
  }
  __syncthreads();
  const int last = s_last;
  for (int i = s_count + tid; i < n; i += kVerifyThreads) a.path[(int64_t)b * n + i] = -1;

  // the next token's weights: row p of the last accepted token, less q or the rejected tokens
  const T* p = probs + (int64_t)(last + 1) * V;
  const T* q = draft && last + 1 < n && s_parent[last + 1] >= -1 ? draft + (int64_t)(last + 1) * V : nullptr;
  const int per_warp = ((V + kVerifyWarps - 1) / kVerifyWarps + 31) & ~31;
  const int lo = min(warp * per_warp, V), hi = min(lo + per_warp, V);
  unsigned long long sum = 0, all = 0;
  for (int x = lo + lane; x < hi; x += 32) {
    const uint32_t pw = whole(to_f32(p[x]));
    all += pw;
    if (q) {
      const uint32_t qw = whole(to_f32(q[x]));
      sum += pw > qw ? pw - qw : 0u;
    }
  }
  all = warp_sum64(all);
  sum = q ? warp_sum64(sum) : all;
  if (!draft) {
    unsigned long long out = 0;
    for (int i = lane; i < n; i += 32) {
      if (s_parent[i] != last || s_token[i] < lo || s_token[i] >= hi) continue;
      bool again = false;
      for (int k = 0; k < i; ++k) again |= s_parent[k] == last && s_token[k] == s_token[i];
      if (!again) out += s_mass[i];
    }
    sum -= warp_sum64(out);
  }
  if (lane == 0) {
    s_sum[warp] = sum;
    s_all[warp] = all;
  }
  __syncthreads();
  unsigned long long total = 0, whole_row = 0;
  for (int w = 0; w < kVerifyWarps; ++w) {
    total += s_sum[w];
    whole_row += s_all[w];
  }
  const bool plain = total == 0;  // nothing left: the row itself
  if (plain) total = whole_row;
  if (total == 0) {
    if (tid == 0) a.token[b] = -1;
    return;
  }
  const unsigned long long ul = whole_u(u[n]);
  const unsigned long long t = (total >> 31) * ul + (((total & (kOne - 1)) * ul) >> 31);
  unsigned long long before = 0;
  int w = 0;
  for (; w < kVerifyWarps; ++w) {
    const unsigned long long s = plain ? s_all[w] : s_sum[w];
    if (before + s > t) break;
    before += s;
  }
  if (w != warp) return;
  for (int x0 = lo; x0 < hi; x0 += 32) {
    const int x = x0 + lane;
    unsigned long long v = 0;
    if (x < hi) {
      uint32_t pw = whole(to_f32(p[x]));
      if (!plain) {
        if (q) {
          const uint32_t qw = whole(to_f32(q[x]));
          pw = pw > qw ? pw - qw : 0u;
        } else if (!draft) {
          for (int i = 0; i < n; ++i)
            if (s_parent[i] == last && s_token[i] == x) pw = 0;
        }
      }
      v = pw;
    }
    unsigned long long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned long long y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + inc > t);
    if (hit) {
      if (lane == 0) a.token[b] = x0 + __ffs(hit) - 1;
      return;
    }
    before += __shfl_sync(0xffffffffu, inc, 31);
  }
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
  if (batch < 0 || batch > 0x7fffffffLL || vocab < 1 || vocab > (1LL << 30))
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
  if (dtype == NKL_FLOAT32)
    return launch_pdl(verify_kernel<float>, dim3((unsigned)batch), dim3(kVerifyThreads), 0, st, op, a);
  return launch_pdl(verify_kernel<bf16>, dim3((unsigned)batch), dim3(kVerifyThreads), 0, st, op, a);
}
