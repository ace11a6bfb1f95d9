// torch_ops.cpp - PyTorch operators (namespace nkilab) of the decoding entry points of the C ABI.
//
// A decoding loop calls these once per layer or step on little data, so the checks of the
// arguments are C++: the host's time is what bounds the smallest calls. Each operator takes
// CUDA tensors, allocates its outputs with the caching allocator and launches the C entry point
// on the current stream; there is no CPU implementation. Wrong values raise ValueError, wrong
// types TypeError, tensors on the wrong device RuntimeError, a refusal of the C ABI a
// RuntimeError that begins with the entry point's name (nkilab.ops makes it an NklError).
#include <ATen/core/Tensor.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/library.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "../../include/nkilab.h"

namespace {

using at::Tensor;
using OptTensor = const std::optional<Tensor>&;

void check(const char* fn, int status) {
  TORCH_CHECK(status == NKL_OK, fn, " failed (", status, "): ", nkl_last_error());
}

int dtype_code(const Tensor& t) {
  if (t.scalar_type() == at::kBFloat16) return NKL_BFLOAT16;
  TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, "nkilab kernels support float32 and bfloat16, got ", t.scalar_type());
  return NKL_FLOAT32;
}

// A dense int32 tensor of this shape on the device.
const int32_t* ints(const char* name, const Tensor& t, c10::Device dev, at::IntArrayRef shape) {
  TORCH_CHECK_TYPE(t.scalar_type() == at::kInt, name, " must be int32, got ", t.scalar_type());
  TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", not on ", dev);
  TORCH_CHECK_VALUE(t.sizes() == shape, name, " has shape ", t.sizes(), ", expected ", shape);
  TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
  return static_cast<const int32_t*>(t.data_ptr());
}

const int32_t* ints(const char* name, OptTensor t, c10::Device dev, at::IntArrayRef shape) {
  return t.has_value() ? ints(name, *t, dev, shape) : nullptr;
}

int32_t* out_ints(const Tensor& t) { return static_cast<int32_t*>(t.data_ptr()); }

// Straight from the caching allocator, past the dispatcher.
Tensor new_tensor(at::IntArrayRef shape, at::ScalarType type, c10::Device dev) {
  return at::detail::empty_cuda(shape, type, dev, std::nullopt);
}
Tensor new_ints(at::IntArrayRef shape, c10::Device dev) { return new_tensor(shape, at::kInt, dev); }

void same(const Tensor& t, const Tensor& ref) {
  TORCH_CHECK_TYPE(t.scalar_type() == ref.scalar_type(), "mixed dtypes: ", t.scalar_type(), " vs ", ref.scalar_type());
  TORCH_CHECK(t.device() == ref.device(), "tensors on different devices: ", t.device(), " vs ", ref.device());
}

// Whether t's rows are contiguous and 16-byte aligned, so that a kernel can read it as it lies.
bool rows16(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  const auto st = t.strides();
  if (st.back() != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  for (size_t i = 0; i + 1 < st.size(); ++i)
    if (st[i] % per) return false;
  return true;
}

// t, or a copy of it whose rows are contiguous and that begins where a kernel can read it.
Tensor readable(const Tensor& t) {
  if (rows16(t)) return t;
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

int check_caches(const Tensor& k, const Tensor& v, int64_t dims) {
  TORCH_CHECK_VALUE(k.dim() == dims && k.sizes() == v.sizes(), "caches ", k.sizes(), " and ", v.sizes(),
                    ": need equal shapes of ", dims, " dimensions");
  TORCH_CHECK_TYPE(k.scalar_type() == v.scalar_type() && k.device() == v.device(),
                   "k and v caches differ in dtype or device");
  TORCH_CHECK(k.strides() == v.strides() && k.stride(-1) == 1, "caches need equal strides and contiguous rows");
  return dtype_code(k);
}

// The caches' type and their powers of two, for a cache in 8 bits: [.., pages, kv heads, blocks of a page].
struct Scales {
  void *k, *v;
  int64_t block;
};
Scales check_scales(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k, const Tensor& v, int64_t dims) {
  TORCH_CHECK_VALUE(k_cache.dim() == dims && k_cache.sizes() == v_cache.sizes(), "caches ", k_cache.sizes(), " and ",
                    v_cache.sizes(), ": need equal shapes of ", dims, " dimensions");
  const c10::Device dev = k_cache.device();
  for (const Tensor* c : {&k_cache, &v_cache}) {
    TORCH_CHECK_TYPE(c->scalar_type() == at::kFloat8_e4m3fn, "a cache with scales is float8_e4m3fn, got ", c->scalar_type());
    TORCH_CHECK(c->device() == dev, "k and v caches on different devices");
  }
  TORCH_CHECK(k_cache.strides() == v_cache.strides() && k_cache.stride(-1) == 1, "caches need equal strides and contiguous rows");
  TORCH_CHECK_VALUE(k.sizes() == v.sizes(), "scales ", k.sizes(), " and ", v.sizes(), ": need equal shapes");
  for (const Tensor* s : {&k, &v}) {
    TORCH_CHECK_TYPE(s->scalar_type() == at::kFloat8_e8m0fnu, "scales must be float8_e8m0fnu, got ", s->scalar_type());
    TORCH_CHECK(s->device() == dev, "scales are on ", s->device(), ", not on ", dev);
    TORCH_CHECK_VALUE(s->dim() == dims - 1 && s->sizes().slice(0, dims - 2) == k_cache.sizes().slice(0, dims - 2) &&
                          s->size(-1) >= 1 && k_cache.size(-2) % s->size(-1) == 0,
                      "scales ", k.sizes(), " and ", v.sizes(), ", caches ", k_cache.sizes(),
                      ": need one for each block of a page and head, and whole blocks");
    TORCH_CHECK(s->is_contiguous(), "scales must be contiguous");
  }
  return {k.data_ptr(), v.data_ptr(), k_cache.size(-2) / k.size(-1)};
}

void same_device(const Tensor& t, c10::Device dev) {
  TORCH_CHECK(t.device() == dev, "tensors on different devices: ", t.device(), " vs ", dev);
}

// The frequencies of a rotation: as many pairs as entries of a head.
const double* check_freqs(const Tensor& freqs, c10::Device dev, int64_t d) {
  TORCH_CHECK_TYPE(freqs.scalar_type() == at::kDouble, "freqs must be float64, got ", freqs.scalar_type());
  same_device(freqs, dev);
  TORCH_CHECK_VALUE(freqs.dim() == 1 && freqs.size(0) >= 1 && 2 * freqs.size(0) <= d, "freqs ", freqs.sizes(),
                    ": need one dimension of up to ", d / 2);
  TORCH_CHECK(freqs.is_contiguous(), "freqs must be contiguous");
  return static_cast<const double*>(freqs.data_ptr());
}

// Rows k and v as the kernels read them: equal strides, aligned rows.
std::pair<Tensor, Tensor> rows_of(const Tensor& k, const Tensor& v) {
  if (k.strides() == v.strides() && rows16(k) && rows16(v)) return {k, v};
  return {readable(k.contiguous()), readable(v.contiguous())};
}

struct Table {
  c10::Device dev;
  int64_t B, M, P;
  const int32_t *tables, *lens, *refs;
};

Table check_table(const Tensor& tables, OptTensor lens, const Tensor& refs) {
  TORCH_CHECK_VALUE(tables.dim() == 2 && refs.dim() == 1 && tables.size(1) >= 1 && refs.size(0) >= 1, "tables ",
                    tables.sizes(), ", refs ", refs.sizes(), ": need [B, pages of a slot] and [pages]");
  const c10::Device dev = tables.device();
  const int64_t B = tables.size(0), M = tables.size(1), P = refs.size(0);
  return {dev, B, M, P, ints("tables", tables, dev, {B, M}), ints("lens", lens, dev, {B}), ints("refs", refs, dev, {P})};
}

// A call's workspace, for as long as the object lives: until the call's last launch is queued.
struct Workspace {
  void* data = nullptr;
  Tensor hold;
  std::unique_lock<std::mutex> lock;
};

// Calls of one stream share one, grown on demand. A call of two launches hands values from one to
// the next through it, and another host thread may queue on the same stream (the default one
// is every thread's), so a call holds the stream's lock from here to its last launch: the stream
// then runs whole calls one after another. A call under capture into a graph gets a workspace
// of the graph's own pool, so graphs never share.
Workspace workspace(c10::Device dev, cudaStream_t stream, size_t bytes) {
  Workspace w;
  if (bytes == 0) return w;
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
    w.hold = new_tensor({(int64_t)bytes}, at::kByte, dev);
  } else {
    struct Kept {
      std::mutex mutex;
      Tensor tensor;
    };
    static std::mutex mutex;
    // never destroyed: the CUDA context may be gone before static destructors run
    static auto* const all = new std::map<std::pair<int, cudaStream_t>, Kept>;
    Kept* kept;
    {
      std::lock_guard<std::mutex> lock(mutex);
      kept = &(*all)[{dev.index(), stream}];
    }
    w.lock = std::unique_lock<std::mutex>(kept->mutex);
    if (!kept->tensor.defined() || (size_t)kept->tensor.numel() < bytes)
      kept->tensor = new_tensor({(int64_t)bytes}, at::kByte, dev);
    w.hold = kept->tensor;
  }
  w.data = w.hold.data_ptr();
  return w;
}

Tensor attention_tree(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache,
                      const Tensor& v_cache, const Tensor& tables, const Tensor& lens, OptTensor parents, double scale) {
  const int dt = check_caches(k_cache, v_cache, 4);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && k_in.sizes() == v_in.sizes(), "q ", q_in.sizes(), ", k ",
                    k_in.sizes(), ", v ", v_in.sizes(), ": need [B, T, heads, head_dim]");
  const int64_t B = q_in.size(0), T = q_in.size(1), H = q_in.size(2), d = q_in.size(3);
  const int64_t P = k_cache.size(0), Hkv = k_cache.size(1), page = k_cache.size(2);
  TORCH_CHECK_VALUE(k_in.size(0) == B && k_in.size(1) == T && k_in.size(2) == Hkv && k_in.size(3) == d &&
                        k_cache.size(3) == d && Hkv > 0 && H % Hkv == 0,
                    "q ", q_in.sizes(), ", k ", k_in.sizes(), ", cache ", k_cache.sizes(),
                    ": sizes do not match, or the cache's heads do not divide q's");
  same(q_in, k_cache);
  same(k_in, k_cache);
  same(v_in, k_cache);
  TORCH_CHECK_VALUE(T <= NKL_MAX_DRAFTED, T, " drafted tokens, at most ", NKL_MAX_DRAFTED, " are taken");
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(1) >= 1, "tables ", tables.sizes(), ": need [B, pages of a slot]");
  const c10::Device dev = k_cache.device();
  const int64_t M = tables.size(1);
  const int32_t* tb = ints("tables", tables, dev, {B, M});
  const int32_t* ln = ints("lens", lens, dev, {B});
  const int32_t* up = ints("parents", parents, dev, {B, T});
  const Tensor q = readable(q_in);
  const auto [k, v] = rows_of(k_in, v_in);
  const c10::cuda::CUDAGuard guard(dev);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  Tensor out = new_tensor({B, T, H, d}, q.scalar_type(), dev);
  const size_t bytes = nkl_attention_tree_workspace_size(B, T, H, Hkv, d, page, M, dt);
  const Workspace ws = workspace(dev, st, bytes);
  check("nkl_attention_tree",
        nkl_attention_tree(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                           k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), tb, ln, up, out.data_ptr(),
                           ws.data, bytes, B, T, H, Hkv, d, P, page, M, (float)scale, dt, st));
  return out;
}

Tensor attention_tree_8bit(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache,
                           const Tensor& v_cache, const Tensor& k_scales, const Tensor& v_scales, const Tensor& tables,
                           const Tensor& lens, OptTensor parents, double scale) {
  const Scales sc = check_scales(k_cache, v_cache, k_scales, v_scales, 4);
  const int dt = dtype_code(q_in);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && k_in.sizes() == v_in.sizes(), "q ", q_in.sizes(), ", k ",
                    k_in.sizes(), ", v ", v_in.sizes(), ": need [B, T, heads, head_dim]");
  const int64_t B = q_in.size(0), T = q_in.size(1), H = q_in.size(2), d = q_in.size(3);
  const int64_t P = k_cache.size(0), Hkv = k_cache.size(1), page = k_cache.size(2);
  TORCH_CHECK_VALUE(k_in.size(0) == B && k_in.size(1) == T && k_in.size(2) == Hkv && k_in.size(3) == d &&
                        k_cache.size(3) == d && Hkv > 0 && H % Hkv == 0,
                    "q ", q_in.sizes(), ", k ", k_in.sizes(), ", cache ", k_cache.sizes(),
                    ": sizes do not match, or the cache's heads do not divide q's");
  same(k_in, q_in);
  same(v_in, q_in);
  const c10::Device dev = k_cache.device();
  same_device(q_in, dev);
  TORCH_CHECK_VALUE(T <= NKL_MAX_DRAFTED, T, " drafted tokens, at most ", NKL_MAX_DRAFTED, " are taken");
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(1) >= 1, "tables ", tables.sizes(), ": need [B, pages of a slot]");
  const int64_t M = tables.size(1);
  const int32_t* tb = ints("tables", tables, dev, {B, M});
  const int32_t* ln = ints("lens", lens, dev, {B});
  const int32_t* up = ints("parents", parents, dev, {B, T});
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor q = readable(q_in);
  const auto [k, v] = rows_of(k_in, v_in);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  Tensor out = new_tensor({B, T, H, d}, q.scalar_type(), dev);
  const size_t bytes = nkl_attention_tree_8bit_workspace_size(B, T, H, Hkv, d, page, M, dt);
  const Workspace ws = workspace(dev, st, bytes);
  check("nkl_attention_tree_8bit",
        nkl_attention_tree_8bit(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                                k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), sc.k, sc.v, tb, ln, up,
                                out.data_ptr(), ws.data, bytes, B, T, H, Hkv, d, P, page, M, sc.block, (float)scale, dt,
                                st));
  return out;
}

Tensor cache_append(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                    const Tensor& tables, const Tensor& lens, OptTensor path, OptTensor count) {
  const int dt = check_caches(k_cache, v_cache, 5);
  const int64_t L = k_cache.size(0), P = k_cache.size(1), Hkv = k_cache.size(2), page = k_cache.size(3),
                d = k_cache.size(4);
  TORCH_CHECK_VALUE(k_in.dim() == 5 && k_in.sizes() == v_in.sizes() && k_in.size(0) == L && k_in.size(3) == Hkv &&
                        k_in.size(4) == d,
                    "k ", k_in.sizes(), ", v ", v_in.sizes(), ", cache ", k_cache.sizes(),
                    ": need rows [layers, B, T, kv heads, head_dim]");
  const int64_t B = k_in.size(1), T = k_in.size(2);
  same(k_in, k_cache);
  same(v_in, k_cache);
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(1) >= 1, "tables ", tables.sizes(), ": need [B, pages of a slot]");
  const c10::Device dev = k_cache.device();
  const int64_t M = tables.size(1);
  const int32_t* tb = ints("tables", tables, dev, {B, M});
  const int32_t* ln = ints("lens", lens, dev, {B});
  const int32_t* pt = ints("path", path, dev, {B, T});
  const int32_t* ct = ints("count", count, dev, {B});
  const auto [k, v] = rows_of(k_in, v_in);
  const c10::cuda::CUDAGuard guard(dev);
  Tensor lens_out = new_ints({B}, dev);
  check("nkl_cache_append",
        nkl_cache_append(k.data_ptr(), v.data_ptr(), k.strides().data(), k_cache.data_ptr(), v_cache.data_ptr(),
                         k_cache.strides().data(), tb, ln, pt, ct, out_ints(lens_out), L, B, T, Hkv, d, P, page, M, dt,
                         c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return lens_out;
}

Tensor cache_append_8bit(const Tensor& k_in, const Tensor& v_in, const Tensor& k_cache, const Tensor& v_cache,
                         const Tensor& k_scales, const Tensor& v_scales, const Tensor& tables, const Tensor& lens,
                         OptTensor path, OptTensor count) {
  const Scales sc = check_scales(k_cache, v_cache, k_scales, v_scales, 5);
  const int64_t L = k_cache.size(0), P = k_cache.size(1), Hkv = k_cache.size(2), page = k_cache.size(3),
                d = k_cache.size(4);
  TORCH_CHECK_VALUE(k_in.dim() == 5 && k_in.sizes() == v_in.sizes() && k_in.size(0) == L && k_in.size(3) == Hkv &&
                        k_in.size(4) == d,
                    "k ", k_in.sizes(), ", v ", v_in.sizes(), ", cache ", k_cache.sizes(),
                    ": need rows [layers, B, T, kv heads, head_dim]");
  const int dt = dtype_code(k_in);
  const int64_t B = k_in.size(1), T = k_in.size(2);
  same(v_in, k_in);
  same_device(k_in, k_cache.device());
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(1) >= 1, "tables ", tables.sizes(), ": need [B, pages of a slot]");
  const c10::Device dev = k_cache.device();
  const int64_t M = tables.size(1);
  const int32_t* tb = ints("tables", tables, dev, {B, M});
  const int32_t* ln = ints("lens", lens, dev, {B});
  const int32_t* pt = ints("path", path, dev, {B, T});
  const int32_t* ct = ints("count", count, dev, {B});
  const c10::cuda::CUDAGuard guard(dev);
  const auto [k, v] = rows_of(k_in, v_in);
  Tensor lens_out = new_ints({B}, dev);
  check("nkl_cache_append_8bit",
        nkl_cache_append_8bit(k.data_ptr(), v.data_ptr(), k.strides().data(), k_cache.data_ptr(), v_cache.data_ptr(),
                              k_cache.strides().data(), sc.k, sc.v, tb, ln, pt, ct, out_ints(lens_out), L, B, T, Hkv, d, P,
                              page, M, sc.block, dt, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return lens_out;
}

Tensor rotary(const Tensor& x_in, const Tensor& positions, const Tensor& freqs, OptTensor parents, bool interleaved,
              double magnitude, bool inverse) {
  const int dt = dtype_code(x_in);
  TORCH_CHECK_VALUE(x_in.dim() == 4, "x ", x_in.sizes(), ": need [B, T, heads, head_dim]");
  const int64_t B = x_in.size(0), T = x_in.size(1), H = x_in.size(2), d = x_in.size(3);
  const c10::Device dev = x_in.device();
  const bool per_token = positions.dim() == 2;
  const int32_t* at = per_token ? ints("positions", positions, dev, {B, T}) : ints("positions", positions, dev, {B});
  const int32_t* up = ints("parents", parents, dev, {B, T});
  const double* f = check_freqs(freqs, dev, d);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor x = readable(x_in);
  Tensor out = new_tensor({B, T, H, d}, x.scalar_type(), dev);
  check("nkl_rotary", nkl_rotary(x.data_ptr(), x.strides().data(), at, up, f, out.data_ptr(), B, T, H, d, 2 * freqs.size(0),
                                 per_token, interleaved, inverse, (float)magnitude, dt,
                                 c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return out;
}

std::tuple<Tensor, Tensor> rotary_append(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                                         const Tensor& k_cache, const Tensor& v_cache, OptTensor k_scales,
                                         OptTensor v_scales, const Tensor& tables, const Tensor& lens, const Tensor& freqs,
                                         OptTensor count, bool interleaved, double magnitude) {
  TORCH_CHECK_VALUE(k_scales.has_value() == v_scales.has_value(), "scales: need both or none");
  Scales sc = {nullptr, nullptr, 0};
  if (k_scales.has_value()) {
    sc = check_scales(k_cache, v_cache, *k_scales, *v_scales, 4);
  } else {
    check_caches(k_cache, v_cache, 4);
    same(k_in, k_cache);
  }
  const int dt = dtype_code(q_in);
  TORCH_CHECK_VALUE(q_in.dim() == 4 && k_in.dim() == 4 && k_in.sizes() == v_in.sizes(), "q ", q_in.sizes(), ", k ",
                    k_in.sizes(), ", v ", v_in.sizes(), ": need [B, T, heads, head_dim]");
  const int64_t B = q_in.size(0), T = q_in.size(1), H = q_in.size(2), d = q_in.size(3);
  const int64_t P = k_cache.size(0), Hkv = k_cache.size(1), page = k_cache.size(2);
  TORCH_CHECK_VALUE(k_in.size(0) == B && k_in.size(1) == T && k_in.size(2) == Hkv && k_in.size(3) == d &&
                        k_cache.size(3) == d,
                    "q ", q_in.sizes(), ", k ", k_in.sizes(), ", cache ", k_cache.sizes(), ": sizes do not match");
  same(k_in, q_in);
  same(v_in, q_in);
  const c10::Device dev = k_cache.device();
  same_device(q_in, dev);
  TORCH_CHECK_VALUE(tables.dim() == 2 && tables.size(1) >= 1, "tables ", tables.sizes(), ": need [B, pages of a slot]");
  const int64_t M = tables.size(1);
  const int32_t* tb = ints("tables", tables, dev, {B, M});
  const int32_t* ln = ints("lens", lens, dev, {B});
  const int32_t* ct = ints("count", count, dev, {B});
  const double* f = check_freqs(freqs, dev, d);
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor q = readable(q_in);
  const auto [k, v] = rows_of(k_in, v_in);
  Tensor q_out = new_tensor({B, T, H, d}, q.scalar_type(), dev), k_out = new_tensor({B, T, Hkv, d}, q.scalar_type(), dev);
  check("nkl_rotary_append",
        nkl_rotary_append(q.data_ptr(), q.strides().data(), k.data_ptr(), v.data_ptr(), k.strides().data(),
                          k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), sc.k, sc.v, tb, ln, ct, f,
                          q_out.data_ptr(), k_out.data_ptr(), B, T, H, Hkv, d, 2 * freqs.size(0), P, page, M, sc.block,
                          interleaved, (float)magnitude, dt, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {q_out, k_out};
}

std::tuple<Tensor, Tensor, Tensor> cache_reserve(const Tensor& tables, const Tensor& lens, const Tensor& refs,
                                                 const Tensor& extra, int64_t page_size) {
  const Table t = check_table(tables, lens, refs);
  const int32_t* ex = ints("extra", extra, t.dev, {t.B});
  const c10::cuda::CUDAGuard guard(t.dev);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(t.dev.index()).stream();
  Tensor tables_out = new_ints({t.B, t.M}, t.dev), refs_out = new_ints({t.P}, t.dev), missing = new_ints({1}, t.dev);
  const size_t bytes = nkl_cache_reserve_workspace_size(t.B);
  const Workspace ws = workspace(t.dev, st, bytes);
  check("nkl_cache_reserve", nkl_cache_reserve(t.tables, t.lens, t.refs, ex, out_ints(tables_out), out_ints(refs_out),
                                               out_ints(missing), ws.data, bytes, t.B, t.P, page_size, t.M, st));
  return {tables_out, refs_out, missing};
}

// k_scales and v_scales: of a cache in 8 bits, else undefined.
std::tuple<Tensor, Tensor, Tensor, Tensor> fork(const Tensor& k_cache, const Tensor& v_cache, const Tensor* k_scales,
                                                const Tensor* v_scales, const Tensor& tables, const Tensor& lens,
                                                const Tensor& refs, const Tensor& src, const Tensor& dst) {
  Scales sc = {nullptr, nullptr, 0};
  int dt = 0;
  if (k_scales) sc = check_scales(k_cache, v_cache, *k_scales, *v_scales, 5);
  else dt = check_caches(k_cache, v_cache, 5);
  const Table t = check_table(tables, lens, refs);
  TORCH_CHECK_VALUE(k_cache.size(1) == t.P, "the cache has ", k_cache.size(1), " pages, refs ", t.P);
  TORCH_CHECK(k_cache.device() == t.dev, "tensors on different devices: ", k_cache.device(), " vs ", t.dev);
  TORCH_CHECK_VALUE(src.dim() == 1, "src ", src.sizes(), ": need one dimension");
  const int64_t F = src.size(0);
  const int32_t* from = ints("src", src, t.dev, {F});
  const int32_t* to = ints("dst", dst, t.dev, {F});
  const c10::cuda::CUDAGuard guard(t.dev);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(t.dev.index()).stream();
  Tensor tables_out = new_ints({t.B, t.M}, t.dev), lens_out = new_ints({t.B}, t.dev), refs_out = new_ints({t.P}, t.dev),
         missing = new_ints({1}, t.dev);
  const size_t bytes = nkl_cache_fork_workspace_size(t.B, F);
  const Workspace ws = workspace(t.dev, st, bytes);
  const int64_t L = k_cache.size(0), Hkv = k_cache.size(2), page = k_cache.size(3), d = k_cache.size(4);
  if (k_scales)
    check("nkl_cache_fork_8bit",
          nkl_cache_fork_8bit(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), sc.k, sc.v, t.tables, t.lens,
                              t.refs, from, to, out_ints(tables_out), out_ints(lens_out), out_ints(refs_out),
                              out_ints(missing), ws.data, bytes, F, L, t.B, Hkv, d, t.P, page, t.M, sc.block, st));
  else
    check("nkl_cache_fork",
          nkl_cache_fork(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), t.tables, t.lens, t.refs, from, to,
                         out_ints(tables_out), out_ints(lens_out), out_ints(refs_out), out_ints(missing), ws.data, bytes, F,
                         L, t.B, Hkv, d, t.P, page, t.M, dt, st));
  return {tables_out, lens_out, refs_out, missing};
}

std::tuple<Tensor, Tensor, Tensor, Tensor> cache_fork(const Tensor& k_cache, const Tensor& v_cache, const Tensor& tables,
                                                      const Tensor& lens, const Tensor& refs, const Tensor& src,
                                                      const Tensor& dst) {
  return fork(k_cache, v_cache, nullptr, nullptr, tables, lens, refs, src, dst);
}

std::tuple<Tensor, Tensor, Tensor, Tensor> cache_fork_8bit(const Tensor& k_cache, const Tensor& v_cache,
                                                           const Tensor& k_scales, const Tensor& v_scales,
                                                           const Tensor& tables, const Tensor& lens, const Tensor& refs,
                                                           const Tensor& src, const Tensor& dst) {
  return fork(k_cache, v_cache, &k_scales, &v_scales, tables, lens, refs, src, dst);
}

std::tuple<Tensor, Tensor, Tensor> cache_free(const Tensor& tables, const Tensor& lens, const Tensor& refs,
                                              const Tensor& slots) {
  const Table t = check_table(tables, lens, refs);
  TORCH_CHECK_VALUE(slots.dim() == 1, "slots ", slots.sizes(), ": need one dimension");
  const int32_t* sl = ints("slots", slots, t.dev, slots.sizes());
  const c10::cuda::CUDAGuard guard(t.dev);
  Tensor tables_out = new_ints({t.B, t.M}, t.dev), lens_out = new_ints({t.B}, t.dev), refs_out = new_ints({t.P}, t.dev);
  check("nkl_cache_free", nkl_cache_free(t.tables, t.lens, t.refs, sl, out_ints(tables_out), out_ints(lens_out),
                                         out_ints(refs_out), slots.size(0), t.B, t.P, t.M,
                                         c10::cuda::getCurrentCUDAStream(t.dev.index()).stream()));
  return {tables_out, lens_out, refs_out};
}

std::tuple<Tensor, Tensor> compact(const Tensor& k_cache, const Tensor& v_cache, const Tensor* k_scales,
                                   const Tensor* v_scales, const Tensor& tables, const Tensor& refs) {
  Scales sc = {nullptr, nullptr, 0};
  int dt = 0;
  if (k_scales) sc = check_scales(k_cache, v_cache, *k_scales, *v_scales, 5);
  else dt = check_caches(k_cache, v_cache, 5);
  const Table t = check_table(tables, std::nullopt, refs);
  TORCH_CHECK_VALUE(k_cache.size(1) == t.P, "the cache has ", k_cache.size(1), " pages, refs ", t.P);
  TORCH_CHECK(k_cache.device() == t.dev, "tensors on different devices: ", k_cache.device(), " vs ", t.dev);
  const c10::cuda::CUDAGuard guard(t.dev);
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(t.dev.index()).stream();
  Tensor tables_out = new_ints({t.B, t.M}, t.dev), refs_out = new_ints({t.P}, t.dev);
  const size_t bytes = nkl_cache_compact_workspace_size(t.P);
  const Workspace ws = workspace(t.dev, st, bytes);
  const int64_t L = k_cache.size(0), Hkv = k_cache.size(2), page = k_cache.size(3), d = k_cache.size(4);
  if (k_scales)
    check("nkl_cache_compact_8bit",
          nkl_cache_compact_8bit(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), sc.k, sc.v, t.tables,
                                 t.refs, out_ints(tables_out), out_ints(refs_out), ws.data, bytes, L, t.B, Hkv, d, t.P, page,
                                 t.M, sc.block, st));
  else
    check("nkl_cache_compact",
          nkl_cache_compact(k_cache.data_ptr(), v_cache.data_ptr(), k_cache.strides().data(), t.tables, t.refs,
                            out_ints(tables_out), out_ints(refs_out), ws.data, bytes, L, t.B, Hkv, d, t.P, page, t.M, dt, st));
  return {tables_out, refs_out};
}

std::tuple<Tensor, Tensor> cache_compact(const Tensor& k_cache, const Tensor& v_cache, const Tensor& tables,
                                         const Tensor& refs) {
  return compact(k_cache, v_cache, nullptr, nullptr, tables, refs);
}

std::tuple<Tensor, Tensor> cache_compact_8bit(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scales,
                                              const Tensor& v_scales, const Tensor& tables, const Tensor& refs) {
  return compact(k_cache, v_cache, &k_scales, &v_scales, tables, refs);
}

std::tuple<Tensor, Tensor, Tensor> verify_drafts(const Tensor& probs_in, const Tensor& tokens, const Tensor& uniforms_in,
                                                 OptTensor parents, OptTensor draft_in) {
  const int dt = dtype_code(probs_in);
  TORCH_CHECK_VALUE(tokens.dim() == 2 && probs_in.dim() == 3 && probs_in.size(0) == tokens.size(0) &&
                        probs_in.size(1) == tokens.size(1) + 1,
                    "probs ", probs_in.sizes(), ", tokens ", tokens.sizes(), ": need [B, T + 1, vocabulary] and [B, T]");
  const int64_t B = tokens.size(0), T = tokens.size(1), V = probs_in.size(2);
  TORCH_CHECK_VALUE(!(parents.has_value() && draft_in.has_value()), "draft probabilities go with a chain, not with a tree");
  TORCH_CHECK_VALUE(T <= NKL_MAX_DRAFTED, T, " drafted tokens, at most ", NKL_MAX_DRAFTED, " are taken");
  const c10::Device dev = probs_in.device();
  const int32_t* tk = ints("tokens", tokens, dev, {B, T});
  const int32_t* up = ints("parents", parents, dev, {B, T});
  TORCH_CHECK_VALUE(uniforms_in.scalar_type() == at::kFloat && uniforms_in.dim() == 2 && uniforms_in.size(0) == B &&
                        uniforms_in.size(1) == T + 1 && uniforms_in.device() == dev,
                    "uniforms: need float32 [", B, ", ", T + 1, "] on ", dev, ", got ", uniforms_in.scalar_type(), " ",
                    uniforms_in.sizes(), " on ", uniforms_in.device());
  const Tensor probs = probs_in.contiguous(), uniforms = uniforms_in.contiguous();
  Tensor draft;
  if (draft_in.has_value()) {
    TORCH_CHECK_VALUE(draft_in->scalar_type() == probs.scalar_type() && draft_in->dim() == 3 && draft_in->size(0) == B &&
                          draft_in->size(1) == T && draft_in->size(2) == V && draft_in->device() == dev,
                      "draft_probs: need ", probs.scalar_type(), " [", B, ", ", T, ", ", V, "] on ", dev, ", got ",
                      draft_in->scalar_type(), " ", draft_in->sizes(), " on ", draft_in->device());
    draft = draft_in->contiguous();
  }
  const c10::cuda::CUDAGuard guard(dev);
  Tensor path = new_ints({B, T}, dev), count = new_ints({B}, dev), token = new_ints({B}, dev);
  check("nkl_verify_drafts",
        nkl_verify_drafts(probs.data_ptr(), draft.defined() ? draft.data_ptr() : nullptr, tk,
                          static_cast<const float*>(uniforms.data_ptr()), up, out_ints(path), out_ints(count),
                          out_ints(token), B, T, V, dt, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {path, count, token};
}

std::tuple<Tensor, Tensor> sample(const Tensor& logits_in, const Tensor& uniforms, OptTensor temperatures,
                                  OptTensor top_ks, OptTensor top_ps, OptTensor min_ps, double temperature,
                                  int64_t top_k, double top_p, double min_p) {
  const int dt = dtype_code(logits_in);
  TORCH_CHECK_VALUE(logits_in.dim() == 2 && logits_in.size(1) >= 1, "logits ", logits_in.sizes(), ": need [B, vocabulary]");
  const c10::Device dev = logits_in.device();
  const int64_t B = logits_in.size(0), V = logits_in.size(1);
  auto floats = [&](const char* name, const Tensor& t) {
    TORCH_CHECK_TYPE(t.scalar_type() == at::kFloat, name, " must be float32, got ", t.scalar_type());
    TORCH_CHECK(t.device() == dev, name, " is on ", t.device(), ", not on ", dev);
    TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == B, name, " has shape ", t.sizes(), ", expected [", B, "]");
    TORCH_CHECK(t.is_contiguous(), name, " must be contiguous");
    return static_cast<const float*>(t.data_ptr());
  };
  auto each = [&](const char* name, OptTensor t) { return t.has_value() ? floats(name, *t) : nullptr; };
  const float* u = floats("uniforms", uniforms);
  const float *ts = each("temperature", temperatures), *ps = each("top_p", top_ps), *ms = each("min_p", min_ps);
  const int32_t* ks = ints("top_k", top_ks, dev, {B});
  const c10::cuda::CUDAGuard guard(dev);
  const Tensor logits = logits_in.stride(1) == 1 || V == 1 ? logits_in : logits_in.contiguous();
  Tensor token = new_ints({B}, dev), prob = new_tensor({B}, at::kFloat, dev);
  check("nkl_sample",
        nkl_sample(logits.data_ptr(), logits.stride(0), u, ts, ks, ps, ms, (float)temperature,
                   (int)std::max<int64_t>(std::min<int64_t>(top_k, INT32_MAX), 0), (float)top_p, (float)min_p,
                   out_ints(token), static_cast<float*>(prob.data_ptr()), B, V, dt,
                   c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  return {token, prob};
}

// Whether a forward derivative is on its way through t.
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// An operator without derivatives refuses tangents at the call, before it writes anything.
void no_tangent(const char* name, std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs) TORCH_CHECK_NOT_IMPLEMENTED(!has_tangent(*t), name, " has no forward derivative");
}

// The attention has no backward pass: with inputs that require a gradient, one through it raises.
Tensor no_backward(Tensor out, const char* name, std::initializer_list<Tensor> inputs) {
  const std::vector<Tensor> in(inputs);
  bool any = false;
  for (const Tensor& t : in) any |= torch::autograd::compute_requires_grad(t);
  if (any) {
    const std::shared_ptr<torch::autograd::Node> node(
        new torch::autograd::NotImplemented(name, torch::autograd::collect_next_edges(in)), torch::autograd::deleteNode);
    torch::autograd::set_history(out, node);
  }
  return out;
}

Tensor attention_tree_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_cache,
                               const Tensor& v_cache, const Tensor& tables, const Tensor& lens, OptTensor parents,
                               double scale) {
  no_tangent("nkilab::attention_tree", {&q, &k, &v, &k_cache, &v_cache});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nkilab::attention_tree", "")
                             .typed<decltype(attention_tree_autograd)>();
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(q, k, v, k_cache, v_cache, tables, lens, parents, scale);
  }
  if (!torch::autograd::compute_requires_grad(q, k, v, k_cache, v_cache)) return out;
  return no_backward(out, "nkilab::attention_tree", {q, k, v, k_cache, v_cache});
}

Tensor attention_tree_8bit_autograd(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& k_cache,
                                    const Tensor& v_cache, const Tensor& k_scales, const Tensor& v_scales,
                                    const Tensor& tables, const Tensor& lens, OptTensor parents, double scale) {
  no_tangent("nkilab::attention_tree_8bit", {&q, &k, &v});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nkilab::attention_tree_8bit", "")
                             .typed<decltype(attention_tree_8bit_autograd)>();
  Tensor out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(q, k, v, k_cache, v_cache, k_scales, v_scales, tables, lens, parents, scale);
  }
  if (!torch::autograd::compute_requires_grad(q, k, v)) return out;
  return no_backward(out, "nkilab::attention_tree_8bit", {q, k, v});
}

std::tuple<Tensor, Tensor> sample_autograd(const Tensor& logits, const Tensor& uniforms, OptTensor temperatures,
                                           OptTensor top_ks, OptTensor top_ps, OptTensor min_ps, double temperature,
                                           int64_t top_k, double top_p, double min_p) {
  const Tensor t = temperatures.value_or(Tensor());
  no_tangent("nkilab::sample", {&logits, &t});
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("nkilab::sample", "").typed<decltype(sample)>();
  std::tuple<Tensor, Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(logits, uniforms, temperatures, top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p);
  }
  if (torch::autograd::compute_requires_grad(logits, t)) no_backward(std::get<1>(out), "nkilab::sample", {logits, t});
  return out;
}

// The gradient of a turn by an angle is the turn by the opposite one, so a pass back through it
// is the operator itself, and can be passed back through in turn.
Tensor rotary_op(const Tensor& x, const Tensor& positions, const Tensor& freqs, OptTensor parents, bool interleaved,
                 double magnitude, bool inverse) {
  static const auto op =
      c10::Dispatcher::singleton().findSchemaOrThrow("nkilab::rotary", "").typed<decltype(rotary)>();
  return op.call(x, positions, freqs, parents, interleaved, magnitude, inverse);
}

struct Rotary : public torch::autograd::Function<Rotary> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& positions,
                        const Tensor& freqs, const std::optional<Tensor>& parents, bool interleaved, double magnitude,
                        bool inverse) {
    ctx->save_for_backward({positions, freqs, parents.value_or(Tensor())});
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["magnitude"] = magnitude;
    ctx->saved_data["inverse"] = inverse;
    at::AutoDispatchBelowADInplaceOrView below;
    return rotary_op(x, positions, freqs, parents, interleaved, magnitude, inverse);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 const torch::autograd::variable_list& grads) {
    const auto saved = ctx->get_saved_variables();
    std::optional<Tensor> parents;
    if (saved[2].defined()) parents = saved[2];
    const Tensor grad = rotary_op(grads[0], saved[0], saved[1], parents, ctx->saved_data["interleaved"].toBool(),
                                  ctx->saved_data["magnitude"].toDouble(), !ctx->saved_data["inverse"].toBool());
    return {grad, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor rotary_autograd(const Tensor& x, const Tensor& positions, const Tensor& freqs, OptTensor parents,
                       bool interleaved, double magnitude, bool inverse) {
  TORCH_CHECK(!torch::autograd::compute_requires_grad(freqs) && !has_tangent(freqs), "nkilab::rotary: freqs have no gradient");
  if (has_tangent(x)) {  // the turn is linear: the tangent turns as its x does
    const Tensor tangent = rotary_op(x._fw_grad(0), positions, freqs, parents, interleaved, magnitude, inverse);
    const Tensor out = rotary_autograd(x._fw_primal(0), positions, freqs, parents, interleaved, magnitude, inverse);
    out._set_fw_grad(tangent, 0, /*is_inplace_op=*/false);
    return out;
  }
  if (!torch::autograd::compute_requires_grad(x)) {  // past the graph's bookkeeping: the smallest calls are bound by it
    at::AutoDispatchBelowADInplaceOrView below;
    return rotary_op(x, positions, freqs, parents, interleaved, magnitude, inverse);
  }
  return Rotary::apply(x, positions, freqs, parents, interleaved, magnitude, inverse);
}

// The appends are for decoding: what comes out of one that inputs with gradients went into raises
// when a backward pass gets there.
std::tuple<Tensor, Tensor> rotary_append_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                                                  const Tensor& k_cache, const Tensor& v_cache, OptTensor k_scales,
                                                  OptTensor v_scales, const Tensor& tables, const Tensor& lens,
                                                  const Tensor& freqs, OptTensor count, bool interleaved,
                                                  double magnitude) {
  no_tangent("nkilab::rotary_append", {&q, &k, &v, &freqs});
  static const auto op = c10::Dispatcher::singleton()
                             .findSchemaOrThrow("nkilab::rotary_append", "")
                             .typed<decltype(rotary_append)>();
  std::tuple<Tensor, Tensor> out;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    out = op.call(q, k, v, k_cache, v_cache, k_scales, v_scales, tables, lens, freqs, count, interleaved, magnitude);
  }
  if (torch::autograd::compute_requires_grad(q, k, v)) {
    const std::shared_ptr<torch::autograd::Node> node(
        new torch::autograd::NotImplemented("nkilab::rotary_append", torch::autograd::collect_next_edges(q, k, v)),
        torch::autograd::deleteNode);
    std::vector<Tensor> both = {std::get<0>(out), std::get<1>(out)};
    torch::autograd::set_history(both, node);
  }
  return out;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(nkilab, m) {
  m.def("attention_tree(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor tables, Tensor lens, "
        "Tensor? parents, float scale) -> Tensor");
  m.def("attention_tree_8bit(Tensor q, Tensor k, Tensor v, Tensor k_cache, Tensor v_cache, Tensor k_scales, Tensor v_scales, "
        "Tensor tables, Tensor lens, Tensor? parents, float scale) -> Tensor");
  m.def("cache_append(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor tables, Tensor lens, "
        "Tensor? path, Tensor? count) -> Tensor");
  m.def("cache_append_8bit(Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, "
        "Tensor(d!) v_scales, Tensor tables, Tensor lens, Tensor? path, Tensor? count) -> Tensor");
  m.def("rotary(Tensor x, Tensor positions, Tensor freqs, Tensor? parents, bool interleaved, float magnitude, "
        "bool inverse) -> Tensor");
  m.def("rotary_append(Tensor q, Tensor k, Tensor v, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scales, "
        "Tensor(d!)? v_scales, Tensor tables, Tensor lens, Tensor freqs, Tensor? count, bool interleaved, "
        "float magnitude) -> (Tensor, Tensor)");
  m.def("cache_reserve(Tensor tables, Tensor lens, Tensor refs, Tensor extra, int page_size) -> (Tensor, Tensor, Tensor)");
  m.def("cache_fork(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor tables, Tensor lens, Tensor refs, Tensor src, "
        "Tensor dst) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("cache_free(Tensor tables, Tensor lens, Tensor refs, Tensor slots) -> (Tensor, Tensor, Tensor)");
  m.def("cache_compact(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor tables, Tensor refs) -> (Tensor, Tensor)");
  m.def("cache_fork_8bit(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales, Tensor tables, "
        "Tensor lens, Tensor refs, Tensor src, Tensor dst) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("cache_compact_8bit(Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!) k_scales, Tensor(d!) v_scales, Tensor tables, "
        "Tensor refs) -> (Tensor, Tensor)");
  m.def("sample(Tensor logits, Tensor uniforms, Tensor? temperatures, Tensor? top_ks, Tensor? top_ps, Tensor? min_ps, "
        "float temperature, int top_k, float top_p, float min_p) -> (Tensor, Tensor)");
  m.def("verify_drafts(Tensor probs, Tensor tokens, Tensor uniforms, Tensor? parents, Tensor? draft_probs) "
        "-> (Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(nkilab, CUDA, m) {
  m.impl("attention_tree", &attention_tree);
  m.impl("attention_tree_8bit", &attention_tree_8bit);
  m.impl("cache_append", &cache_append);
  m.impl("cache_append_8bit", &cache_append_8bit);
  m.impl("rotary", &rotary);
  m.impl("rotary_append", &rotary_append);
  m.impl("cache_reserve", &cache_reserve);
  m.impl("cache_fork", &cache_fork);
  m.impl("cache_free", &cache_free);
  m.impl("cache_compact", &cache_compact);
  m.impl("cache_fork_8bit", &cache_fork_8bit);
  m.impl("cache_compact_8bit", &cache_compact_8bit);
  m.impl("verify_drafts", &verify_drafts);
  m.impl("sample", &sample);
}

TORCH_LIBRARY_IMPL(nkilab, Autograd, m) {
  m.impl("attention_tree", &attention_tree_autograd);
  m.impl("attention_tree_8bit", &attention_tree_8bit_autograd);
  m.impl("rotary", &rotary_autograd);
  m.impl("rotary_append", &rotary_append_autograd);
  m.impl("sample", &sample_autograd);
}
