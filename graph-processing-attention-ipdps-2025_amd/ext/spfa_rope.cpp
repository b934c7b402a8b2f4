// Python module spfa_rope: head norms of queries and keys with the position rotation in one pass.
//   forward(q, k, w_q, w_k, positions, inv_freq, q_out, k_out, eps=1e-6, interleaved=False) -> (q_out, k_out)
//   backward(q, k, w_q, w_k, positions, inv_freq, d_q_out, d_k_out, d_q, d_k, d_w_q, d_w_k, eps=1e-6,
//            interleaved=False) -> (d_q, d_k)
// The reference starts from finished Q and K (Sparse_FlashAttention_CSR/sp_flatt_csr.cpp:28-39); the
// work is done by spfa_qk_norm_rope_forward / _backward in libspfa_hip.so.
#include "spfa_serve_ext.h"

using spfa_ext::OptTensor;

namespace {

spfa_rope_t make_rope(const torch::Tensor& q, const torch::Tensor& k, const OptTensor& w_q, const OptTensor& w_k,
                      const torch::Tensor& positions, const torch::Tensor& inv_freq, double eps, bool interleaved) {
  CHECK_ROWS(q);
  CHECK_ROWS(k);
  CHECK_ROWS(positions);
  CHECK_INPUT(inv_freq);
  const int64_t n = q.dim();
  TORCH_CHECK((n == 3 || n == 4) && k.dim() == n, "q and k must both be [tokens, heads, d] or [batch, tokens, heads, d]");
  TORCH_CHECK(k.size(n - 1) == q.size(n - 1), "q and k must share the head dimension");
  TORCH_CHECK(k.size(n - 3) == q.size(n - 3) && (n == 3 || k.size(0) == q.size(0)), "q and k must have the same tokens");
  TORCH_CHECK(k.scalar_type() == q.scalar_type(), "q and k must have the same dtype");
  CHECK_SAME_DEVICE(k, q);
  CHECK_SAME_DEVICE(positions, q);
  CHECK_SAME_DEVICE(inv_freq, q);
  spfa_rope_t p{};
  p.batch = n == 4 ? q.size(0) : 1;
  p.tokens = q.size(n - 3);
  p.heads_q = q.size(n - 2);
  p.heads_k = k.size(n - 2);
  p.d = q.size(n - 1);
  p.dtype = spfa_ext::serve_dtype(q, "q");
  p.w_dtype = p.dtype;
  p.interleaved = interleaved;
  TORCH_CHECK(eps >= 0.0, "eps must not be negative");
  p.eps = (float)eps;
  p.q = spfa_ext::heads_of(q);
  p.k = spfa_ext::heads_of(k);
  TORCH_CHECK(inv_freq.dim() == 1 && inv_freq.scalar_type() == torch::kFloat32, "inv_freq must be a one-dimensional float32 tensor");
  p.rot = 2 * inv_freq.size(0);
  TORCH_CHECK(p.rot <= p.d, "inv_freq has more frequencies than a head has pairs");
  p.inv_freq = (const float*)inv_freq.data_ptr();
  for (const OptTensor* w : {&w_q, &w_k}) {
    if (!w->has_value()) continue;
    const torch::Tensor& t = **w;
    TORCH_CHECK(t.device().is_cuda() && t.is_contiguous(), "w_q and w_k must be contiguous CUDA tensors");
    CHECK_SAME_DEVICE(t, q);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == p.d, "w_q and w_k must be [d]");
    TORCH_CHECK(t.scalar_type() == q.scalar_type() || t.scalar_type() == torch::kFloat32, "w_q and w_k must have the dtype of q (or float32)");
    p.w_dtype = spfa_ext::elem_dtype(t);
  }
  TORCH_CHECK(!(w_q.has_value() && w_k.has_value()) || w_q->scalar_type() == w_k->scalar_type(), "w_q and w_k must have the same dtype");
  p.w_q = w_q.has_value() ? w_q->data_ptr() : nullptr;
  p.w_k = w_k.has_value() ? w_k->data_ptr() : nullptr;
  p.position_bytes = spfa_ext::signed_index_bytes(positions, "positions");
  if (positions.dim() == 1) {
    TORCH_CHECK(positions.size(0) == p.tokens, "positions must be [tokens], [1, tokens] or [batch, tokens]");
  } else {
    TORCH_CHECK(n == 4 && positions.dim() == 2 && (positions.size(0) == p.batch || positions.size(0) == 1) && positions.size(1) == p.tokens,
                "positions must be [tokens], [1, tokens] or [batch, tokens]");
    p.position_stride = spfa_ext::stride_of(positions, 0);
  }
  p.positions = positions.data_ptr();
  return p;
}

void check_like(const torch::Tensor& t, const torch::Tensor& like, const char* name) {
  TORCH_CHECK(t.device().is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.sizes() == like.sizes() && t.scalar_type() == like.scalar_type(), name, " must have the shape and dtype of ",
              "the tensor it belongs to");
  CHECK_SAME_DEVICE(t, like);
  TORCH_CHECK(t.stride(-1) == 1 || t.size(-1) <= 1, name, " must have unit stride along its last dimension");
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> spfa_rope_forward_py(torch::Tensor q, torch::Tensor k, OptTensor w_q, OptTensor w_k,
                                                              torch::Tensor positions, torch::Tensor inv_freq,
                                                              torch::Tensor q_out, torch::Tensor k_out, double eps,
                                                              bool interleaved) {
  const spfa_rope_t p = make_rope(q, k, w_q, w_k, positions, inv_freq, eps, interleaved);
  check_like(q_out, q, "q_out");
  check_like(k_out, k, "k_out");
  spfa_ext::check_output(q_out, "q_out", {k, k_out, w_q, w_k, positions, inv_freq}, {q});
  spfa_ext::check_output(k_out, "k_out", {q, w_q, w_k, positions, inv_freq}, {k});
  c10::DeviceGuard guard(q.device());
  const spfa_heads_t qo = spfa_ext::heads_of(q_out), ko = spfa_ext::heads_of(k_out);
  spfa_ext::raise_on_error(spfa_qk_norm_rope_forward(&p, &qo, &ko, spfa_ext::current_stream(q)));
  return std::make_tuple(q_out, k_out);
}

// d_w_q, d_w_k: float32 [d], or None where they are not wanted.  All gradients are written.
std::tuple<torch::Tensor, torch::Tensor> spfa_rope_backward_py(torch::Tensor q, torch::Tensor k, OptTensor w_q, OptTensor w_k,
                                                               torch::Tensor positions, torch::Tensor inv_freq,
                                                               torch::Tensor d_q_out, torch::Tensor d_k_out, torch::Tensor d_q,
                                                               torch::Tensor d_k, OptTensor d_w_q, OptTensor d_w_k, double eps,
                                                               bool interleaved) {
  const spfa_rope_t p = make_rope(q, k, w_q, w_k, positions, inv_freq, eps, interleaved);
  check_like(d_q_out, q, "d_q_out");
  check_like(d_k_out, k, "d_k_out");
  check_like(d_q, q, "d_q");
  check_like(d_k, k, "d_k");
  spfa_ext::check_output(d_q, "d_q", {k, d_k_out, d_k, w_q, w_k, positions, inv_freq}, {q, d_q_out});
  spfa_ext::check_output(d_k, "d_k", {q, d_q_out, w_q, w_k, positions, inv_freq}, {k, d_k_out});
  for (const OptTensor* w : {&d_w_q, &d_w_k}) {
    if (!w->has_value()) continue;
    const torch::Tensor& t = **w;
    TORCH_CHECK(t.device().is_cuda() && t.is_contiguous(), "d_w_q and d_w_k must be contiguous CUDA tensors");
    CHECK_SAME_DEVICE(t, q);
    TORCH_CHECK(t.dim() == 1 && t.size(0) == p.d && t.scalar_type() == torch::kFloat32, "d_w_q and d_w_k must be float32 [d]");
  }
  // (in place of its own weights: these have been read when the sums are written)
  if (d_w_q.has_value()) spfa_ext::check_output(*d_w_q, "d_w_q", {q, k, w_k, positions, inv_freq, d_q_out, d_k_out, d_q, d_k, d_w_k}, {w_q});
  if (d_w_k.has_value()) spfa_ext::check_output(*d_w_k, "d_w_k", {q, k, w_q, positions, inv_freq, d_q_out, d_k_out, d_q, d_k}, {w_k});
  c10::DeviceGuard guard(q.device());
  const spfa_heads_t dqo = spfa_ext::heads_of(d_q_out), dko = spfa_ext::heads_of(d_k_out);
  const spfa_heads_t dq = spfa_ext::heads_of(d_q), dk = spfa_ext::heads_of(d_k);
  torch::Tensor ws =
      spfa_ext::make_workspace(spfa_qk_norm_rope_backward_workspace_bytes(p.batch, p.tokens, p.heads_q, p.heads_k, p.d), q);
  spfa_ext::raise_on_error(spfa_qk_norm_rope_backward(&p, &dqo, &dko, &dq, &dk, d_w_q.has_value() ? (float*)d_w_q->data_ptr() : nullptr,
                                                      d_w_k.has_value() ? (float*)d_w_k->data_ptr() : nullptr, ws.data_ptr(),
                                                      (size_t)ws.numel(), spfa_ext::current_stream(q)));
  return std::make_tuple(d_q, d_k);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  namespace py = pybind11;
  mod.def("forward", &spfa_rope_forward_py, "Head norms and position rotation of queries and keys (HIP, gfx950)", py::arg("q"),
          py::arg("k"), py::arg("w_q"), py::arg("w_k"), py::arg("positions"), py::arg("inv_freq"), py::arg("q_out"),
          py::arg("k_out"), py::arg("eps") = 1e-6, py::arg("interleaved") = false);
  mod.def("backward", &spfa_rope_backward_py, "Gradients of forward(...), written to d_q, d_k, d_w_q, d_w_k", py::arg("q"),
          py::arg("k"), py::arg("w_q"), py::arg("w_k"), py::arg("positions"), py::arg("inv_freq"), py::arg("d_q_out"),
          py::arg("d_k_out"), py::arg("d_q"), py::arg("d_k"), py::arg("d_w_q"), py::arg("d_w_k"), py::arg("eps") = 1e-6,
          py::arg("interleaved") = false);
}
