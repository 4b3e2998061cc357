// The host path of the package's hot calls: allocate the results, launch
// through the C ABI, wait for the one value that a call needs on the host.
// Bound with pybind11 for the Python layer, which keeps the API, its argument
// checks and their messages; nothing here is reached with arguments that layer
// has not accepted.
//
// Bound by call overhead: with ctypes and Python bookkeeping a forward took
// about 20 us of host time between the routing's read-back and its launch, in
// which the GPU is idle; these take about 8.

#include <ATen/core/CachingHostAllocator.h>
#include <torch/extension.h>

#include <string>
#include <tuple>
#include <vector>

#include "swattn.h"
#include "swattn_cache.h"
#include "swattn_internal.h"

namespace {

using at::Tensor;
using std::optional;
namespace py = pybind11;

void check(int status, const char* what) {
  TORCH_CHECK(status == SWATTN_OK, what, " failed with status ", status, ": ", swattn_last_error());
}

void* as_stream(int64_t s) { return reinterpret_cast<void*>(static_cast<intptr_t>(s)); }

Tensor bytes(const Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, like.options().dtype(at::kByte));
}

// An output like t: the one that the Python layer made, where a tensor subclass
// has a say in that, or a new one.
Tensor like(const Tensor& t, const optional<Tensor>& made) {
  return made.has_value() ? *made : at::empty(t.sizes(), t.options());
}

const int32_t* i32(const Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }
const int32_t* i32(const optional<Tensor>& t) { return t.has_value() ? i32(*t) : nullptr; }

// Pinned host memory for a compaction's counts.  One buffer per thread: a call
// waits for its counts before it returns, so that a thread has at most one
// compaction in flight.  After a HIP error a kernel may still be queued that
// reports there: the buffer is then left to it for good.
template <int kWords>
struct HostWords {
  c10::DataPtr ptr;
  int32_t* get() {
    if (!ptr) ptr = at::getHostAllocator(at::kCUDA)->allocate(kWords * sizeof(int32_t));
    return static_cast<int32_t*>(ptr.get());
  }
  void abandon() {
    (void)ptr.release_context();
    ptr = c10::DataPtr();
  }
};
thread_local HostWords<SWATTN_COMPACT_HOST_WORDS> t_words;
thread_local HostWords<SWATTN_KEY_WEIGHTS_HOST_WORDS> t_check_words;

// (full, local) of a byte mask (dtype -1) or of router logits.
std::tuple<Tensor, Tensor> compact(const Tensor& x, int64_t dtype, double threshold,
                                   int64_t stream) {
  const int64_t n = x.numel();
  const Tensor out = at::empty({n}, x.options().dtype(at::kInt));
  const size_t ws_bytes = swattn_compact_workspace_bytes(n);
  Tensor ws;
  if (ws_bytes > 0) ws = bytes(x, ws_bytes);
  int32_t* host = t_words.get();
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_compact_wait(x.const_data_ptr(), static_cast<int32_t>(dtype), n,
                                 static_cast<float>(threshold), out.data_ptr<int32_t>(), host,
                                 ws_bytes > 0 ? ws.data_ptr() : nullptr, ws_bytes,
                                 as_stream(stream));
  }
  if (status > 0) t_words.abandon();
  check(status, dtype < 0 ? "swattn_compact" : "swattn_compact_logits");
  const int64_t nf = host[0];
  return {out.narrow(0, 0, nf), out.narrow(0, nf, n - nf)};
}

// Whether q, k, v meet every precondition of the prefill (the Python layer
// finds out which one fails and raises for it, also for arguments that are no
// tensors).
bool qkv_ok(const py::object& qo, const py::object& ko, const py::object& vo) {
  if (!THPVariable_Check(qo.ptr()) || !THPVariable_Check(ko.ptr()) || !THPVariable_Check(vo.ptr()))
    return false;
  const Tensor& q = THPVariable_Unpack(qo.ptr());
  const Tensor& k = THPVariable_Unpack(ko.ptr());
  const Tensor& v = THPVariable_Unpack(vo.ptr());
  return q.scalar_type() == at::kBFloat16 && k.scalar_type() == at::kBFloat16 &&
         v.scalar_type() == at::kBFloat16 && q.is_cuda() && k.is_cuda() && v.is_cuda() &&
         q.layout() == at::kStrided && k.layout() == at::kStrided && v.layout() == at::kStrided &&
         q.is_contiguous() && k.is_contiguous() && v.is_contiguous() && q.dim() == 4 &&
         k.dim() == 4 && v.dim() == 4 && k.sizes() == v.sizes() && q.size(0) == k.size(0) &&
         q.size(3) == 128 && k.size(3) == 128 && k.size(2) > 0 && q.size(2) % k.size(2) == 0 &&
         q.device() == k.device() && q.device() == v.device();
}

std::tuple<Tensor, Tensor> prefill_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                           const Tensor& full, const Tensor& local,
                                           const optional<Tensor>& full_starts,
                                           const optional<Tensor>& local_starts,
                                           const optional<Tensor>& causal_ends, int64_t window,
                                           double scale_log2, int64_t stream,
                                           const optional<Tensor>& out_made) {
  const int32_t batch = static_cast<int32_t>(q.size(0)), hq = static_cast<int32_t>(q.size(2));
  const int32_t hkv = static_cast<int32_t>(k.size(2)), dim = static_cast<int32_t>(q.size(3));
  const int64_t sq = q.size(1), skv = k.size(1), nf = full.numel(), nl = local.numel();
  const Tensor out = like(q, out_made);
  const Tensor lse = at::empty({q.size(0), sq, q.size(2)}, q.options().dtype(at::kFloat));
  const int32_t w = static_cast<int32_t>(window);
  // The larger workspace that lets the kernel split long full items by key
  // range when they would otherwise set its length (few KV heads).
  const size_t ws_bytes =
      swattn_prefill_split_workspace_bytes(batch, sq, skv, hq, hkv, dim, w, nf, nl);
  const Tensor ws = bytes(q, ws_bytes);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_prefill_fwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), i32(full),
                   nf, i32(local), nl, i32(full_starts), i32(local_starts),
                   i32(causal_ends), out.data_ptr(), lse.data_ptr<float>(), batch, sq, skv,
                   hq, hkv, dim, w, static_cast<float>(scale_log2), ws.data_ptr(), ws_bytes,
                   as_stream(stream));
  }
  check(status, "swattn_prefill_fwd");
  return {out, lse};
}

// The seven fields of a SwitchAttentionMetadata, in its order; the sequences'
// offsets, checked and at most SWATTN_METADATA_HOST_MAX_SEQS of them, travel as
// kernel arguments.
std::vector<Tensor> metadata(const std::vector<int32_t>& cu_q, const std::vector<int32_t>& cu_kv,
                             int64_t q_len, int64_t kv_len, int64_t window, at::Device device,
                             int64_t stream) {
  const auto opts = at::TensorOptions().dtype(at::kInt).device(device);
  std::vector<Tensor> f;
  f.reserve(7);
  for (const int64_t n : {q_len, kv_len, q_len, kv_len, q_len, q_len, q_len})
    f.push_back(at::empty({n}, opts));
  auto out = [&](int i) { return f[i].data_ptr<int32_t>(); };
  check(swattn_build_metadata_host(cu_q.data(), cu_kv.data(), static_cast<int32_t>(cu_q.size()) - 1,
                                   q_len, kv_len, static_cast<int32_t>(window), out(0), out(1),
                                   out(2), out(3), out(4), out(5), out(6), as_stream(stream)),
        "swattn_build_metadata");
  return f;
}

std::tuple<Tensor, Tensor, Tensor> prefill_backward(
    const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& out, const Tensor& lse,
    const Tensor& grad, const Tensor& full, const Tensor& local,
    const optional<Tensor>& full_starts, const optional<Tensor>& local_starts,
    const optional<Tensor>& causal_ends, int64_t window, double scale_log2, int64_t stream,
    const optional<Tensor>& dq_made, const optional<Tensor>& dk_made,
    const optional<Tensor>& dv_made) {
  const int32_t batch = static_cast<int32_t>(q.size(0)), hq = static_cast<int32_t>(q.size(2));
  const int32_t hkv = static_cast<int32_t>(k.size(2)), dim = static_cast<int32_t>(q.size(3));
  const int64_t sq = q.size(1), skv = k.size(1), nf = full.numel(), nl = local.numel();
  // The lists cover every query position once (checked by the caller), and the
  // kernels write every listed row (0 for a row with no key): no fill.
  const Tensor dq = like(q, dq_made), dk = like(k, dk_made), dv = like(v, dv_made);
  const int32_t w = static_cast<int32_t>(window);
  const size_t ws_bytes = swattn_prefill_bwd_workspace_bytes(batch, skv, hq, hkv, dim, w, nf, nl);
  const Tensor ws = bytes(q, ws_bytes > 0 ? ws_bytes : 1);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_prefill_bwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(),
                   out.const_data_ptr(), lse.const_data_ptr<float>(),
                   grad.const_data_ptr(), i32(full), nf, i32(local), nl, i32(full_starts),
                   i32(local_starts), i32(causal_ends), dq.data_ptr(), dk.data_ptr(),
                   dv.data_ptr(), batch, sq, skv, hq, hkv, dim, w,
                   static_cast<float>(scale_log2), ws.data_ptr(), ws_bytes,
                   as_stream(stream));
  }
  check(status, "swattn_prefill_bwd");
  return {dq, dk, dv};
}

std::tuple<Tensor, Tensor> decode_forward(const Tensor& q, const Tensor& k, const Tensor& v,
                                          const Tensor& lens, const Tensor& full, int64_t window,
                                          double scale_log2, int64_t stream,
                                          const optional<Tensor>& out_made) {
  const int32_t batch = static_cast<int32_t>(q.size(0)), hq = static_cast<int32_t>(q.size(2));
  const int32_t hkv = static_cast<int32_t>(k.size(2)), dim = static_cast<int32_t>(q.size(3));
  const Tensor out = like(q, out_made);
  const Tensor lse = at::empty({q.size(0), 1, q.size(2)}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = swattn_decode_workspace_bytes(batch, k.size(1), hq, hkv);
  const Tensor ws = bytes(q, ws_bytes);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_decode_fwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), i32(lens),
                  static_cast<const uint8_t*>(full.const_data_ptr()), out.data_ptr(),
                  lse.data_ptr<float>(), batch, k.size(1), hq, hkv, dim,
                  static_cast<int32_t>(window), static_cast<float>(scale_log2),
                  ws.data_ptr(), ws_bytes, as_stream(stream));
  }
  check(status, "swattn_decode_fwd");
  return {out, lse};
}

// The 8-bit KV cache (codes [B, L, Hkv, 128], scales [B, Hkv, blocks]).
const float* f32(const Tensor& t) { return static_cast<const float*>(t.const_data_ptr()); }

struct CacheShape {
  int32_t batch, hkv, dim;
  int64_t len;
  explicit CacheShape(const Tensor& k)
      : batch(static_cast<int32_t>(k.size(0))), hkv(static_cast<int32_t>(k.size(2))),
        dim(static_cast<int32_t>(k.size(3))), len(k.size(1)) {}
};

// Whether a cache's tensors meet every precondition (the Python layer finds out
// which one fails and raises for it).
bool cache_ok(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t block) {
  if (!(block == 16 || block == 32 || block == 64 || block == 128)) return false;
  if (!(k.is_cuda() && k.layout() == at::kStrided && k.dim() == 4 && k.numel() > 0 && k.size(3) == 128 &&
        (k.scalar_type() == at::kChar || k.scalar_type() == at::kFloat8_e4m3fn)))
    return false;
  const int64_t want[3] = {k.size(0), k.size(2), (k.size(1) + block - 1) / block};
  return v.scalar_type() == k.scalar_type() && v.layout() == at::kStrided && v.sizes() == k.sizes() &&
         ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.layout() == at::kStrided &&
         vs.layout() == at::kStrided && ks.sizes() == at::IntArrayRef(want, 3) && vs.sizes() == ks.sizes() &&
         k.is_contiguous() && v.is_contiguous() && ks.is_contiguous() && vs.is_contiguous() &&
         v.device() == k.device() && ks.device() == k.device() && vs.device() == k.device();
}

// Whether contiguous tensors that a call writes share no memory with each other
// or with those that it reads.
bool apart(const std::vector<Tensor>& written, const std::vector<Tensor>& read) {
  const auto overlap = [](const Tensor& a, const Tensor& b) {
    const char* pa = static_cast<const char*>(a.const_data_ptr());
    const char* pb = static_cast<const char*>(b.const_data_ptr());
    return a.device() == b.device() && pa < pb + b.nbytes() && pb < pa + a.nbytes();
  };
  for (size_t i = 0; i < written.size(); ++i) {
    for (size_t j = 0; j < i; ++j)
      if (overlap(written[i], written[j])) return false;
    for (const Tensor& t : read)
      if (overlap(written[i], t)) return false;
  }
  return true;
}

bool lens_ok(const Tensor& t, const Tensor& k) {
  return t.scalar_type() == at::kInt && t.layout() == at::kStrided && t.dim() == 1 && t.size(0) == k.size(0) &&
         t.is_contiguous() && t.device() == k.device();
}

// Whether a whole call's arguments meet every precondition, in their usual form:
// where not, the Python layer looks closer and raises, or makes them so.
bool append_ok(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t block,
               const Tensor& new_k, const Tensor& new_v, const Tensor& lens, const optional<Tensor>& counts) {
  return cache_ok(k, v, ks, vs, block) && new_k.scalar_type() == at::kBFloat16 &&
         new_v.scalar_type() == at::kBFloat16 && new_k.layout() == at::kStrided &&
         new_v.layout() == at::kStrided && new_k.device() == k.device() && new_v.device() == k.device() &&
         new_k.dim() == 4 && new_v.sizes() == new_k.sizes() && new_k.size(0) == k.size(0) &&
         new_k.size(1) <= k.size(1) && new_k.size(2) == k.size(2) && new_k.size(3) == 128 &&
         new_k.is_contiguous() && new_v.is_contiguous() && lens_ok(lens, k) &&
         (!counts.has_value() || lens_ok(*counts, k)) && apart({k, v, ks, vs}, {new_k, new_v, lens});
}

bool read_ok(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t block,
             const optional<Tensor>& starts, const optional<Tensor>& lens) {
  return cache_ok(k, v, ks, vs, block) && (!starts.has_value() || lens_ok(*starts, k)) && (!lens.has_value() || lens_ok(*lens, k));
}

bool evict_ok(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, int64_t block,
              const Tensor& lens, const Tensor& weights) {
  const int64_t want[3] = {k.dim() == 4 ? k.size(0) : 0, k.dim() == 4 ? k.size(2) : 0, k.dim() == 4 ? k.size(1) : 0};
  return cache_ok(k, v, ks, vs, block) && lens_ok(lens, k) && weights.scalar_type() == at::kFloat &&
         weights.layout() == at::kStrided && weights.sizes() == at::IntArrayRef(want, 3) &&
         weights.is_contiguous() && weights.device() == k.device();
}

bool decode_ok(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
               int64_t block, const Tensor& lens, const Tensor& full) {
  return cache_ok(k, v, ks, vs, block) && q.scalar_type() == at::kBFloat16 && q.layout() == at::kStrided &&
         q.dim() == 4 && q.is_contiguous() && q.device() == k.device() && q.size(0) == k.size(0) &&
         q.size(1) == 1 && q.size(3) == 128 && q.size(2) > 0 && q.size(2) % k.size(2) == 0 &&
         q.size(2) / k.size(2) <= 8 && lens_ok(lens, k) && full.scalar_type() == at::kBool &&
         full.layout() == at::kStrided && full.dim() == 1 && full.size(0) == k.size(0) &&
         full.is_contiguous() && full.device() == k.device();
}

// The new lengths.  cu: packed offsets on the device, or host_cu (not empty).
Tensor cache_append(const Tensor& new_k, const Tensor& new_v, const optional<Tensor>& cu,
                    const std::vector<int32_t>& host_cu, const optional<Tensor>& counts, const Tensor& lens, const Tensor& k, const Tensor& v,
                    const Tensor& ks, const Tensor& vs, int64_t rows, int64_t block, int64_t code,
                    int64_t stream) {
  const CacheShape c(k);
  const Tensor out = at::empty({k.size(0)}, lens.options());
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    if (!host_cu.empty())
      status = swattn_cache_append_host(new_k.const_data_ptr(), new_v.const_data_ptr(), host_cu.data(),
                                        i32(lens), k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(),
                                        vs.data_ptr<float>(), out.data_ptr<int32_t>(), c.batch, rows,
                                        new_k.size(1), c.len, c.hkv, c.dim, static_cast<int32_t>(block),
                                        static_cast<int32_t>(code), as_stream(stream));
    else
      status = swattn_cache_append(new_k.const_data_ptr(), new_v.const_data_ptr(), i32(cu), i32(counts),
                                   i32(lens), k.data_ptr(), v.data_ptr(), ks.data_ptr<float>(),
                                   vs.data_ptr<float>(), out.data_ptr<int32_t>(), c.batch, rows,
                                   new_k.size(1), c.len, c.hkv, c.dim, static_cast<int32_t>(block),
                                   static_cast<int32_t>(code), as_stream(stream));
  }
  check(status, "swattn_cache_append");
  return out;
}

std::tuple<Tensor, Tensor> cache_read(const Tensor& k, const Tensor& v, const Tensor& ks,
                                      const Tensor& vs, const optional<Tensor>& starts, int64_t start,
                                      const optional<Tensor>& lens, int64_t rows, int64_t block,
                                      int64_t code, int64_t stream) {
  const CacheShape c(k);
  const auto opts = k.options().dtype(at::kBFloat16);
  const Tensor out_k = at::empty({k.size(0), rows, k.size(2), k.size(3)}, opts);
  const Tensor out_v = at::empty(out_k.sizes(), opts);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_cache_read(k.const_data_ptr(), v.const_data_ptr(), f32(ks), f32(vs), i32(starts), start,
                               i32(lens), out_k.data_ptr(), out_v.data_ptr(), c.batch, rows, c.len, c.hkv,
                               c.dim, static_cast<int32_t>(block), static_cast<int32_t>(code),
                               as_stream(stream));
  }
  check(status, "swattn_cache_read");
  return {out_k, out_v};
}

std::tuple<Tensor, Tensor> cache_decode(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& ks,
                                        const Tensor& vs, const Tensor& lens, const Tensor& full,
                                        const optional<Tensor>& weights, int64_t window, int64_t block,
                                        int64_t code, double scale_log2, int64_t stream,
                                        const optional<Tensor>& out_made) {
  const CacheShape c(k);
  const int32_t hq = static_cast<int32_t>(q.size(2));
  const Tensor out = like(q, out_made);
  const Tensor lse = at::empty({q.size(0), 1, q.size(2)}, q.options().dtype(at::kFloat));
  const size_t ws_bytes =
      swattn_cache_decode_workspace_bytes(c.batch, c.len, hq, c.hkv, weights.has_value() ? 1 : 0);
  const Tensor ws = bytes(q, ws_bytes);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_cache_decode_fwd(q.const_data_ptr(), k.const_data_ptr(), v.const_data_ptr(), f32(ks), f32(vs),
                                     i32(lens), static_cast<const uint8_t*>(full.const_data_ptr()),
                                     out.data_ptr(), lse.data_ptr<float>(),
                                     weights.has_value() ? weights->data_ptr<float>() : nullptr, c.batch,
                                     c.len, hq, c.hkv, c.dim, static_cast<int32_t>(window),
                                     static_cast<int32_t>(block), static_cast<int32_t>(code),
                                     static_cast<float>(scale_log2), ws.data_ptr(), ws_bytes,
                                     as_stream(stream));
  }
  check(status, "swattn_cache_decode_fwd");
  return {out, lse};
}

// With `unchecked` lists also their check's bits.
std::tuple<Tensor, int64_t> prefill_key_weights(const Tensor& q, const Tensor& k, const Tensor& lse, const Tensor& full,
                           const Tensor& local, const optional<Tensor>& full_starts,
                           const optional<Tensor>& local_starts, const optional<Tensor>& causal_ends,
                           int64_t window, double scale_log2, bool unchecked, int64_t stream) {
  const CacheShape c(k);
  const int32_t hq = static_cast<int32_t>(q.size(2));
  const int64_t nf = full.numel(), nl = local.numel();
  int32_t* host = unchecked ? t_check_words.get() : nullptr;
  int32_t flags = 0;
  const Tensor out = at::empty({k.size(0), k.size(2), k.size(1)}, q.options().dtype(at::kFloat));
  const size_t ws_bytes = swattn_prefill_key_weights_workspace_bytes(c.batch, c.len, hq, c.hkv, c.dim, nf, nl);
  const Tensor ws = bytes(q, ws_bytes > 0 ? ws_bytes : 1);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    const void *qp = q.const_data_ptr(), *kp = k.const_data_ptr();
    const int32_t w = static_cast<int32_t>(window);
    const float scale = static_cast<float>(scale_log2);
    status = unchecked
                 ? swattn_prefill_key_weights_checked(
                       qp, kp, f32(lse), i32(full), nf, i32(local), nl, i32(full_starts), i32(local_starts),
                       i32(causal_ends), out.data_ptr<float>(), c.batch, q.size(1), c.len, hq, c.hkv, c.dim, w,
                       scale, ws.data_ptr(), ws_bytes, as_stream(stream), host, &flags)
                 : swattn_prefill_key_weights(
                       qp, kp, f32(lse), i32(full), nf, i32(local), nl, i32(full_starts), i32(local_starts),
                       i32(causal_ends), out.data_ptr<float>(), c.batch, q.size(1), c.len, hq, c.hkv, c.dim, w,
                       scale, ws.data_ptr(), ws_bytes, as_stream(stream));
  }
  if (status > 0 && unchecked) t_check_words.abandon();
  check(status, "swattn_prefill_key_weights");
  return {out, flags};
}

// The new lengths.
Tensor cache_evict(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs,
                   const Tensor& weights, const Tensor& lens, const Tensor& out_k, const Tensor& out_v,
                   const Tensor& out_ks, const Tensor& out_vs, const Tensor& out_weights, int64_t block,
                   int64_t code, int64_t budget, int64_t recent, int64_t stream) {
  const CacheShape c(k);
  const Tensor out = at::empty({k.size(0)}, lens.options());
  const size_t ws_bytes = swattn_cache_evict_workspace_bytes(c.batch, c.hkv, budget);
  const Tensor ws = bytes(k, ws_bytes);
  int status = 0;
  {
    pybind11::gil_scoped_release release;
    status = swattn_cache_evict(k.const_data_ptr(), v.const_data_ptr(), f32(ks), f32(vs), f32(weights),
                                i32(lens), out_k.data_ptr(), out_v.data_ptr(), out_ks.data_ptr<float>(),
                                out_vs.data_ptr<float>(), out_weights.data_ptr<float>(),
                                out.data_ptr<int32_t>(), c.batch, c.len, out_k.size(1), c.hkv, c.dim,
                                static_cast<int32_t>(block), static_cast<int32_t>(code), budget, recent,
                                ws.data_ptr(), ws_bytes, as_stream(stream));
  }
  check(status, "swattn_cache_evict");
  return out;
}

// The same into a new cache of `rows` rows: (k, v, k_scales, v_scales, weights, lengths).
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> cache_evict_new(
    const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs, const Tensor& weights,
    const Tensor& lens, int64_t rows, int64_t block, int64_t code, int64_t budget, int64_t recent,
    int64_t stream) {
  const Tensor out_k = at::empty({k.size(0), rows, k.size(2), k.size(3)}, k.options());
  const Tensor out_v = at::empty(out_k.sizes(), k.options());
  const Tensor out_ks = at::empty({k.size(0), k.size(2), (rows + block - 1) / block}, ks.options());
  const Tensor out_vs = at::empty(out_ks.sizes(), ks.options());
  const Tensor out_weights = at::empty({k.size(0), k.size(2), rows}, weights.options());
  const Tensor out_lens = cache_evict(k, v, ks, vs, weights, lens, out_k, out_v, out_ks, out_vs, out_weights,
                                      block, code, budget, recent, stream);
  return {out_k, out_v, out_ks, out_vs, out_weights, out_lens};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("compact", &compact);
  m.def("qkv_ok", &qkv_ok);
  m.def("prefill_forward", &prefill_forward);
  m.def("metadata", &metadata);
  m.def("prefill_backward", &prefill_backward);
  m.def("decode_forward", &decode_forward);
  m.def("cache_ok", &cache_ok);
  m.def("apart", &apart);
  m.def("append_ok", &append_ok);
  m.def("read_ok", &read_ok);
  m.def("decode_ok", &decode_ok);
  m.def("evict_ok", &evict_ok);
  m.def("cache_append", &cache_append);
  m.def("cache_read", &cache_read);
  m.def("cache_decode", &cache_decode);
  m.def("prefill_key_weights", &prefill_key_weights);
  m.def("cache_evict", &cache_evict);
  m.def("cache_evict_new", &cache_evict_new);
}
