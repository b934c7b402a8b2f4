// Python module spfa_tree: attention of drafted tokens (a tree, a chain, one token) over a paged cache.
//   forward(q, k_cache, v_cache, page_table, ctx_lens, q_offsets, out, tree_mask=None, k_scale=None,
//           v_scale=None, m=None, l=None, scale=None) -> out
// The reference's masks are fixed before the call (CSR, COO, windows; Sparse_FlashAttention_CSR/
// sp_flatt_csr.cpp:28-39); here the mask is the ancestors of each node, over keys that grow from call
// to call.  The work is done by spfa_tree_forward in libspfa_hip.so.
#include <cmath>

#include "spfa_serve_ext.h"

using spfa_ext::OptTensor;

torch::Tensor spfa_tree_forward_py(torch::Tensor q, torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor page_table,
                                   torch::Tensor ctx_lens, torch::Tensor q_offsets, torch::Tensor out, OptTensor tree_mask,
                                   OptTensor k_scale, OptTensor v_scale, OptTensor m, OptTensor l, std::optional<double> scale) {
  CHECK_ROWS(q);
  CHECK_ROWS(out);
  CHECK_CUDA(page_table);
  CHECK_INPUT(ctx_lens);
  CHECK_INPUT(q_offsets);
  TORCH_CHECK(q.dim() == 3, "q must be [rows, heads, d]");
  TORCH_CHECK(q.scalar_type() == torch::kFloat16 || q.scalar_type() == torch::kBFloat16, "q must be float16 or bfloat16 (got ",
              q.scalar_type(), ")");
  TORCH_CHECK(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type(), "out must have the shape and dtype of q");
  CHECK_SAME_DEVICE(out, q);
  const spfa_cache_t c = spfa_ext::make_cache(k_cache, v_cache, k_scale, v_scale, q, "q");
  TORCH_CHECK(q.size(2) == c.d, "q must have the head dimension of the cache");
  TORCH_CHECK(c.heads >= 1 && q.size(1) >= 1 && q.size(1) % c.heads == 0, "the heads of q must be a multiple of the cache's");
  for (const torch::Tensor& t : {page_table, ctx_lens, q_offsets}) {
    TORCH_CHECK(t.scalar_type() == torch::kInt32, "page_table, ctx_lens and q_offsets must be int32");
    CHECK_SAME_DEVICE(t, q);
  }
  TORCH_CHECK(ctx_lens.dim() == 1, "ctx_lens must be [sequences]");
  const int64_t n = ctx_lens.size(0);
  TORCH_CHECK(q_offsets.dim() == 1 && q_offsets.size(0) == n + 1, "q_offsets must be [sequences + 1]");
  TORCH_CHECK(page_table.dim() == 2 && page_table.size(0) == n, "page_table must be [sequences, pages of a sequence]");
  TORCH_CHECK(page_table.stride(1) == 1 || page_table.size(1) <= 1, "page_table must have unit stride along its last dimension");
  TORCH_CHECK(m.has_value() == l.has_value(), "m and l go together");
  spfa_tree_t t{};
  t.q = q.data_ptr();
  t.out = out.data_ptr();
  t.q_stride_row = spfa_ext::stride_of(q, 0);
  t.q_stride_head = spfa_ext::stride_of(q, 1);
  t.out_stride_row = spfa_ext::stride_of(out, 0);
  t.out_stride_head = spfa_ext::stride_of(out, 1);
  t.rows = q.size(0);
  t.heads_q = q.size(1);
  t.n_seqs = n;
  t.q_offsets = (const int32_t*)q_offsets.data_ptr();
  t.ctx_lens = (const int32_t*)ctx_lens.data_ptr();
  t.page_table = (const int32_t*)page_table.data_ptr();
  t.table_width = page_table.size(1);
  t.table_stride = spfa_ext::stride_of(page_table, 0);
  if (tree_mask.has_value()) {
    const torch::Tensor& b = *tree_mask;
    TORCH_CHECK(b.device().is_cuda() && b.is_contiguous(), "tree_mask must be a contiguous CUDA tensor");
    CHECK_SAME_DEVICE(b, q);
    TORCH_CHECK(b.scalar_type() == torch::kInt64 && b.dim() == 2 && b.size(0) == t.rows && b.size(1) >= 1,
                "tree_mask must be int64 [rows, words]");
    t.tree_mask = (const int64_t*)b.data_ptr();
    t.mask_words = b.size(1);
  }
  for (const OptTensor* s : {&m, &l}) {
    if (!s->has_value()) continue;
    const torch::Tensor& x = **s;
    TORCH_CHECK(x.device().is_cuda() && x.is_contiguous(), "m and l must be contiguous CUDA tensors");
    CHECK_SAME_DEVICE(x, q);
    TORCH_CHECK(x.scalar_type() == torch::kFloat32 && x.dim() == 2 && x.size(0) == t.rows && x.size(1) == t.heads_q,
                "m and l must be float32 [rows, heads]");
  }
  t.m = m.has_value() ? (float*)m->data_ptr() : nullptr;
  t.l = l.has_value() ? (float*)l->data_ptr() : nullptr;
  t.scale = scale.has_value() ? (float)*scale : 1.f / std::sqrt((float)c.d);
  // (a row of q is read by every workgroup that has a part of its keys, so out cannot take its place)
  spfa_ext::check_output(out, "out", {q, k_cache, v_cache, page_table, ctx_lens, q_offsets, tree_mask, k_scale, v_scale, m, l});
  if (m.has_value()) {
    spfa_ext::check_output(*m, "m", {q, k_cache, v_cache, page_table, ctx_lens, q_offsets, tree_mask, k_scale, v_scale, l});
    spfa_ext::check_output(*l, "l", {q, k_cache, v_cache, page_table, ctx_lens, q_offsets, tree_mask, k_scale, v_scale});
  }
  c10::DeviceGuard guard(q.device());
  torch::Tensor ws = spfa_ext::make_workspace(spfa_tree_workspace_bytes(&c, &t), q);
  spfa_ext::raise_on_error(spfa_tree_forward(&c, &t, ws.data_ptr(), (size_t)ws.numel(), spfa_ext::current_stream(q)));
  return out;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  namespace py = pybind11;
  mod.def("forward", &spfa_tree_forward_py, "Attention of drafted tokens over a paged cache (HIP, gfx950)", py::arg("q"),
          py::arg("k_cache"), py::arg("v_cache"), py::arg("page_table"), py::arg("ctx_lens"), py::arg("q_offsets"), py::arg("out"),
          py::arg("tree_mask") = py::none(), py::arg("k_scale") = py::none(), py::arg("v_scale") = py::none(),
          py::arg("m") = py::none(), py::arg("l") = py::none(), py::arg("scale") = py::none());
}
