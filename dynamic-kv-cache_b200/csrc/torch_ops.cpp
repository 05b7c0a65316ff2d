// Host fast path of the per-layer calls a GPUCache makes (append, attend, append +
// attend): the same argument checks and the same C-ABI entry points as the ctypes
// binding in src/gpu_kernels.py, made from C++ so that one eager call costs a few
// microseconds of host time instead of ~25 (ctypes marshals ~35 arguments, and every
// stride and pointer query is a Python call). The reference launches its Triton
// kernels from Python once per layer (src/gpu_cache.py:90-92, 99-103), so this host
// cost is paid on every layer of every frame.
#include <torch/extension.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <map>
#include <mutex>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "dkv.h"

namespace {

// Pointers of one cache: p4, m4, p8, m8, p16, rows, codes, status.
using Ptrs = std::vector<int64_t>;
using Caps = std::vector<int64_t>;

void* vp(int64_t p) { return reinterpret_cast<void*>(static_cast<uintptr_t>(p)); }

void check(int rc) {
  if (rc == DKV_OK) return;
  const char* m = dkv_last_error();
  if (rc == DKV_ECUDA) throw std::runtime_error(m);
  throw pybind11::value_error(m);
}

// bf16 [1, heads, n, 64] operand whose rows the kernels load 16 bytes at a time
// (else a contiguous copy), as gpu_kernels._rows_ready.
at::Tensor rows_ready(const at::Tensor& x) {
  if (!x.is_cuda()) throw pybind11::value_error("GPU cache requires CUDA, batch one and the configured head dimension");
  if (x.scalar_type() != at::kBFloat16) throw pybind11::value_error("GPU kernels take bfloat16 queries, keys and values");
  if (x.dim() != 4) throw pybind11::value_error("GPU kernels take [1, heads, n, dim] queries, keys and values");
  const bool ok = x.stride(3) == 1 && x.stride(1) % 8 == 0 && x.stride(2) % 8 == 0 &&
                  (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15u) == 0;
  return ok ? x : x.contiguous();
}

void same_device(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v) {
  if (k.device() != q.device() || v.device() != q.device())
    throw pybind11::value_error("queries, keys and values must be on one CUDA device");
}

void check_ptrs(const Ptrs& p, const Caps& c) {
  if (p.size() != 8 || c.size() != 3) throw pybind11::value_error("cache pointers (8) and capacities (3) expected");
}

// Attention workspaces, one per (device, stream): the library leaves the merge
// counters at the head of a workspace zero after every call, so a workspace is
// zero-filled once and reused; calls on one stream never overlap, calls on other
// streams get other workspaces. Outgrown ones stay referenced, so CUDA graphs
// captured with them keep valid addresses.
std::mutex g_ws_mu;
std::map<std::pair<int, cudaStream_t>, at::Tensor> g_ws;
std::vector<at::Tensor> g_retired;

at::Tensor workspace_for(const at::Device& device, cudaStream_t stream, int64_t size) {
  std::lock_guard<std::mutex> lock(g_ws_mu);
  auto& ws = g_ws[{device.index(), stream}];
  if (!ws.defined() || ws.numel() < size) {
    if (ws.defined()) g_retired.push_back(ws);
    ws = at::zeros({size}, at::TensorOptions().dtype(at::kByte).device(device));
  }
  return ws;
}

cudaStream_t current_stream(const at::Tensor& x) {
  return c10::cuda::getCurrentCUDAStream(x.device().index()).stream();
}

}  // namespace

// The workspace of (x's device, current stream) with at least `size` bytes (size > 0).
at::Tensor workspace(const at::Tensor& like, int64_t size) {
  return workspace_for(like.device(), current_stream(like), size);
}

// GPUCache.attend: dkv_packed_attention of q [1, heads*group, n, 64] over the
// cache's packed history plus k / v [1, heads, n, 64]; returns [1, n, heads*group, 64].
at::Tensor attend(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const Ptrs& p,
                  int64_t layer, int64_t past, const Caps& caps, int64_t heads, int64_t block_m, int64_t block_n,
                  int64_t layers) {
  check_ptrs(p, caps);
  const at::Tensor q = rows_ready(q_in), k = rows_ready(k_in), v = rows_ready(v_in);
  same_device(q, k, v);
  const c10::cuda::CUDAGuard guard(q.device());  // the library launches on the current device
  const int64_t nq = q.size(2), hq = q.size(1);
  if (heads <= 0 || hq % heads) throw pybind11::value_error("query heads must be a positive multiple of KV heads");
  const int64_t group = hq / heads;
  at::Tensor out = at::empty({1, nq, hq, q.size(3)}, q.options());
  const cudaStream_t stream = current_stream(q);
  const size_t size = dkv_packed_attention_workspace(past, nq, heads, group, q.size(3));
  void* ws = size ? workspace_for(q.device(), stream, size).data_ptr() : nullptr;
  check(dkv_packed_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), vp(p[0]), vp(p[1]), vp(p[2]), vp(p[3]),
                             vp(p[4]), static_cast<const int32_t*>(vp(p[5])), static_cast<const uint8_t*>(vp(p[6])),
                             out.data_ptr(), q.stride(1), q.stride(2), k.stride(1), k.stride(2), v.stride(1),
                             v.stride(2), layer, past, nq, caps[0], caps[1], caps[2], heads, group, q.size(3),
                             block_m, block_n, layers, ws, size, static_cast<int32_t*>(vp(p[7])), stream));
  return out;
}

// GPUCache.append's launch: dkv_pack_rows of k / v [1, heads, n, 64] at rows
// [row_start, row_start + n) of the `bits` pool.
void pack(const at::Tensor& k_in, const at::Tensor& v_in, const Ptrs& p, int64_t layer, int64_t row_start,
          const Caps& caps, int64_t heads, int64_t bits, int64_t layers) {
  check_ptrs(p, caps);
  const at::Tensor k = rows_ready(k_in), v = rows_ready(v_in);
  same_device(k, k, v);
  const c10::cuda::CUDAGuard guard(k.device());
  check(dkv_pack_rows(k.data_ptr(), v.data_ptr(), vp(p[0]), vp(p[1]), vp(p[2]), vp(p[3]), vp(p[4]), k.stride(1),
                      k.stride(2), v.stride(1), v.stride(2), layer, row_start, k.size(2), caps[0], caps[1], caps[2],
                      heads, k.size(3), bits, layers, static_cast<int32_t*>(vp(p[7])), current_stream(k)));
}

// GPUCache.append_attend: dkv_append_attention (pack + attention of one frame in
// one launch); returns [1, n, heads*group, 64].
at::Tensor append_attend(const at::Tensor& q_in, const at::Tensor& k_in, const at::Tensor& v_in, const Ptrs& p,
                         int64_t layer, int64_t past, int64_t row_start, int64_t bits, bool fill_map,
                         int64_t map_capacity, const Caps& caps, int64_t heads, int64_t block_m, int64_t block_n,
                         int64_t layers) {
  check_ptrs(p, caps);
  const at::Tensor q = rows_ready(q_in), k = rows_ready(k_in), v = rows_ready(v_in);
  same_device(q, k, v);
  const c10::cuda::CUDAGuard guard(q.device());  // the library launches on the current device
  const int64_t nq = q.size(2), hq = q.size(1);
  if (heads <= 0 || hq % heads) throw pybind11::value_error("query heads must be a positive multiple of KV heads");
  const int64_t group = hq / heads;
  at::Tensor out = at::empty({1, nq, hq, q.size(3)}, q.options());
  const cudaStream_t stream = current_stream(q);
  const size_t size = dkv_packed_attention_workspace(past, nq, heads, group, q.size(3));
  void* ws = size ? workspace_for(q.device(), stream, size).data_ptr() : nullptr;
  check(dkv_append_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), vp(p[0]), vp(p[1]), vp(p[2]), vp(p[3]),
                             vp(p[4]), static_cast<int32_t*>(vp(p[5])), static_cast<uint8_t*>(vp(p[6])),
                             out.data_ptr(), q.stride(1), q.stride(2), k.stride(1), k.stride(2), v.stride(1),
                             v.stride(2), layer, past, nq, row_start, bits, fill_map ? 1 : 0, map_capacity, caps[0],
                             caps[1], caps[2], heads, group, q.size(3), block_m, block_n, layers, ws, size,
                             static_cast<int32_t*>(vp(p[7])), stream));
  return out;
}

// The decoder layer's x + y followed by RMSNorm and its weight (dkv_add_rms_norm)
// over the rows of x / y [..., width]: returns (x + y, norm) — (x, norm) without y.
std::vector<at::Tensor> add_rms_norm(const at::Tensor& x_in, const c10::optional<at::Tensor>& y_in,
                                     const at::Tensor& weight_in, double eps) {
  if (!x_in.is_cuda() || x_in.scalar_type() != at::kBFloat16 || weight_in.scalar_type() != at::kBFloat16)
    throw pybind11::value_error("add_rms_norm takes CUDA bfloat16 tensors");
  const int64_t width = x_in.size(-1);
  const at::Tensor x = x_in.contiguous(), w = weight_in.contiguous();
  if (w.numel() != width || w.device() != x.device()) throw pybind11::value_error("add_rms_norm: weight must be [width]");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor h = at::empty_like(x);
  at::Tensor x_out = x;
  const void* yp = nullptr;
  at::Tensor y;
  if (y_in.has_value()) {
    y = y_in->contiguous();
    if (y.sizes() != x.sizes() || y.scalar_type() != at::kBFloat16 || y.device() != x.device())
      throw pybind11::value_error("add_rms_norm: y must match x");
    yp = y.data_ptr();
    x_out = at::empty_like(x);
  }
  const int64_t rows = width ? x.numel() / width : 0;
  check(dkv_add_rms_norm(x.data_ptr(), yp, yp ? x_out.data_ptr() : nullptr, h.data_ptr(), w.data_ptr(), rows,
                         static_cast<int32_t>(width), width, width, width, width, static_cast<float>(eps),
                         current_stream(x)));
  return {x_out, h};
}

// -- 8-bit decoder operators (dkv_fp8_*): e4m3 codes and fp32 scales ------------------

namespace {

constexpr int64_t kGroup = 128;

int64_t groups_of(int64_t width) { return (width + kGroup - 1) / kGroup; }

// The operators have no derivative: an operand (rows, weights, codes or scales) that autograd would
// have to follow is refused, backward (requires_grad) as forward (a dual tensor's tangent).
void no_grad(const at::Tensor& x, const char* what) {
  if (x.requires_grad() && at::GradMode::is_enabled())
    throw pybind11::value_error(std::string(what) + " has no backward pass (call it under torch.no_grad())");
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && x._fw_grad(0).defined())
    throw pybind11::value_error(std::string(what) + " has no derivative: the tangent of an operand would be lost");
}

// bf16 [..., width] as rows the kernels can load 16 bytes at a time; `stride` receives
// the row stride in elements.
at::Tensor bf16_rows(const at::Tensor& x, const char* what, int64_t* stride) {
  if (!x.is_cuda() || x.scalar_type() != at::kBFloat16 || x.dim() < 1)
    throw pybind11::value_error(std::string(what) + " takes CUDA bfloat16 tensors");
  no_grad(x, what);
  const int64_t width = x.size(-1);
  if (x.dim() == 2 && x.size(0) > 0 && x.stride(1) == 1 && x.stride(0) >= width && x.stride(0) % 8 == 0 &&
      (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15u) == 0) {
    *stride = x.stride(0);
    return x;
  }
  *stride = width;
  const at::Tensor c = x.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
}

// e4m3 matrix [..., width] of 16-byte aligned rows; `stride` receives the row stride in bytes.
at::Tensor e4m3_rows(const at::Tensor& q, const char* what, int64_t* stride) {
  if (!q.is_cuda() || q.scalar_type() != at::kFloat8_e4m3fn || q.dim() < 1)
    throw pybind11::value_error(std::string(what) + " takes CUDA float8_e4m3fn codes");
  no_grad(q, what);
  const int64_t width = q.size(-1);
  if (q.dim() == 2 && q.size(0) > 0 && q.stride(1) == 1 && q.stride(0) >= width && q.stride(0) % 16 == 0 &&
      (reinterpret_cast<uintptr_t>(q.data_ptr()) & 15u) == 0) {
    *stride = q.stride(0);
    return q;
  }
  *stride = width;
  const at::Tensor c = q.contiguous();
  return (reinterpret_cast<uintptr_t>(c.data_ptr()) & 15u) == 0 ? c : c.clone();
}

// The scales of e4m3 rows [..., width]: fp32 [..., groups], contiguous.
at::Tensor row_scales(const at::Tensor& s, const at::Tensor& q, const char* what) {
  bool ok = s.scalar_type() == at::kFloat && s.device() == q.device() && s.dim() == q.dim() &&
            s.size(-1) == groups_of(q.size(-1));
  for (int64_t d = 0; ok && d + 1 < q.dim(); ++d) ok = s.size(d) == q.size(d);
  if (!ok) throw pybind11::value_error(std::string(what) + ": rows need fp32 scales [..., ceil(width / 128)] on their device");
  no_grad(s, what);
  return s.contiguous();
}

// The scales of e4m3 weights [n, k]: fp32 [ceil(n / 128), ceil(k / 128)], contiguous.
at::Tensor block_scales(const at::Tensor& s, const at::Tensor& q, const char* what) {
  if (q.dim() != 2 || s.dim() != 2 || s.scalar_type() != at::kFloat || s.device() != q.device() ||
      s.size(0) != groups_of(q.size(0)) || s.size(1) != groups_of(q.size(1)))
    throw pybind11::value_error(std::string(what) +
                                ": weights are [n, k] with fp32 scales [ceil(n / 128), ceil(k / 128)] on their device");
  no_grad(s, what);
  return s.contiguous();
}

std::vector<int64_t> with_last(const at::Tensor& x, int64_t last) {
  std::vector<int64_t> sizes = x.sizes().vec();
  sizes.back() = last;
  return sizes;
}

int64_t rows_of(const at::Tensor& x) { return x.size(-1) ? x.numel() / x.size(-1) : 0; }

int32_t narrow(int64_t v) { return v > INT32_MAX ? INT32_MAX : static_cast<int32_t>(v); }

// An uninitialised tensor on x's device, as at::empty makes it, without the dispatcher's
// round (two or three of them were a quarter of a call's host time).
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& x) {
  return at::detail::empty_cuda(sizes, type, x.device(), c10::nullopt);
}

float* fp(const at::Tensor& t) { return static_cast<float*>(t.data_ptr()); }

}  // namespace

// bf16 rows x [..., width] to (codes [..., width], scales [..., ceil(width / 128)]).
std::vector<at::Tensor> fp8_quantize(const at::Tensor& x_in) {
  int64_t xs;
  const at::Tensor x = bf16_rows(x_in, "fp8_quantize", &xs);
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t width = x.size(-1);
  at::Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, x);
  at::Tensor s = fresh(with_last(x, groups_of(width)), at::kFloat, x);
  check(dkv_fp8_quantize(x.data_ptr(), q.data_ptr(), fp(s), rows_of(x), narrow(width), xs, current_stream(x)));
  return {q, s};
}

// bf16 weights w [n, k] to (codes [n, k], scales [ceil(n / 128), ceil(k / 128)]).
std::vector<at::Tensor> fp8_quantize_weight(const at::Tensor& w_in) {
  if (w_in.dim() != 2) throw pybind11::value_error("fp8_quantize_weight takes weights [n, k]");
  int64_t ws;
  const at::Tensor w = bf16_rows(w_in, "fp8_quantize_weight", &ws);
  const c10::cuda::CUDAGuard guard(w.device());
  const int64_t n = w.size(0), k = w.size(1);
  at::Tensor q = fresh({n, k}, at::kFloat8_e4m3fn, w);
  at::Tensor s = fresh({groups_of(n), groups_of(k)}, at::kFloat, w);
  check(dkv_fp8_quantize_weight(w.data_ptr(), q.data_ptr(), fp(s), narrow(n), narrow(k), ws, current_stream(w)));
  return {q, s};
}

// (x + y, codes, scales of its norm) over the rows of x / y [..., width]; (x, ...) without y.
std::vector<at::Tensor> add_rms_norm_fp8(const at::Tensor& x_in, const c10::optional<at::Tensor>& y_in,
                                         const at::Tensor& weight_in, double eps) {
  int64_t xs, ys = 0, wstride;
  const at::Tensor x = bf16_rows(x_in, "add_rms_norm_fp8", &xs);
  const int64_t width = x.size(-1);
  if (weight_in.dim() != 1 || weight_in.size(0) != width || weight_in.device() != x.device())
    throw pybind11::value_error("add_rms_norm_fp8: weight must be [width]");
  const c10::cuda::CUDAGuard guard(x.device());
  const at::Tensor w = bf16_rows(weight_in, "add_rms_norm_fp8", &wstride);
  at::Tensor y, x_out = x_in;
  if (y_in.has_value()) {
    if (y_in->sizes() != x.sizes() || y_in->device() != x.device())
      throw pybind11::value_error("add_rms_norm_fp8: y must match x");
    y = bf16_rows(*y_in, "add_rms_norm_fp8", &ys);
    x_out = fresh(x.sizes(), at::kBFloat16, x);
  }
  at::Tensor q = fresh(x.sizes(), at::kFloat8_e4m3fn, x);
  at::Tensor s = fresh(with_last(x, groups_of(width)), at::kFloat, x);
  check(dkv_add_rms_norm_fp8(x.data_ptr(), y.defined() ? y.data_ptr() : nullptr,
                             y.defined() ? x_out.data_ptr() : nullptr, q.data_ptr(), fp(s), w.data_ptr(), rows_of(x),
                             narrow(width), xs, ys, width, static_cast<float>(eps), current_stream(x)));
  return {x_out, q, s};
}

// The linear layer of e4m3 rows (q, s) [..., k] and e4m3 weights (w, ws) [n, k]: [..., n] in bf16 or fp32.
at::Tensor fp8_linear(const at::Tensor& q_in, const at::Tensor& s_in, const at::Tensor& w_in, const at::Tensor& ws_in,
                      bool out_f32) {
  int64_t as, wstride;
  const at::Tensor q = e4m3_rows(q_in, "fp8_linear", &as), w = e4m3_rows(w_in, "fp8_linear", &wstride);
  const at::Tensor s = row_scales(s_in, q, "fp8_linear"), wsc = block_scales(ws_in, w, "fp8_linear");
  if (w.device() != q.device() || w.size(1) != q.size(-1))
    throw pybind11::value_error("fp8_linear: rows and weights must share their device and width");
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t n = w.size(0), k = w.size(1);
  at::Tensor out = fresh(with_last(q, n), out_f32 ? at::kFloat : at::kBFloat16, q);
  check(dkv_fp8_linear(q.data_ptr(), fp(s), w.data_ptr(), fp(wsc), out.data_ptr(), out_f32 ? 32 : 16, rows_of(q),
                       narrow(n), narrow(k), as, wstride, current_stream(q)));
  return out;
}

// silu(rows gate^T) * (rows up^T) as (codes [..., n], scales [..., ceil(n / 128)]).
std::vector<at::Tensor> fp8_gate_up(const at::Tensor& q_in, const at::Tensor& s_in, const at::Tensor& g_in,
                                    const at::Tensor& gs_in, const at::Tensor& u_in, const at::Tensor& us_in) {
  int64_t as, gstride, ustride;
  const at::Tensor q = e4m3_rows(q_in, "fp8_gate_up", &as), g = e4m3_rows(g_in, "fp8_gate_up", &gstride),
                   u = e4m3_rows(u_in, "fp8_gate_up", &ustride);
  const at::Tensor s = row_scales(s_in, q, "fp8_gate_up");
  const at::Tensor gsc = block_scales(gs_in, g, "fp8_gate_up"), usc = block_scales(us_in, u, "fp8_gate_up");
  if (g.device() != q.device() || u.device() != q.device() || g.sizes() != u.sizes() || g.size(1) != q.size(-1))
    throw pybind11::value_error("fp8_gate_up: gate and up must have one shape [n, width] on the rows' device");
  const c10::cuda::CUDAGuard guard(q.device());
  const int64_t n = g.size(0), k = g.size(1);
  at::Tensor out = fresh(with_last(q, n), at::kFloat8_e4m3fn, q);
  at::Tensor scale = fresh(with_last(q, groups_of(n)), at::kFloat, q);
  check(dkv_fp8_gate_up(q.data_ptr(), fp(s), g.data_ptr(), fp(gsc), u.data_ptr(), fp(usc), out.data_ptr(), fp(scale),
                        rows_of(q), narrow(n), narrow(k), as, gstride, ustride, current_stream(q)));
  return {out, scale};
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "C++ host path of GPUCache's per-layer calls into libdkv.so";
  m.def("workspace", &workspace);
  m.def("attend", &attend);
  m.def("pack", &pack);
  m.def("append_attend", &append_attend);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("fp8_quantize", &fp8_quantize);
  m.def("fp8_quantize_weight", &fp8_quantize_weight);
  m.def("add_rms_norm_fp8", &add_rms_norm_fp8);
  m.def("fp8_linear", &fp8_linear);
  m.def("fp8_gate_up", &fp8_gate_up);
}
