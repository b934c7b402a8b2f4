// Python module spfa_cache: keys and values into a paged cache (plain, int8 or float8_e4m3fn) and back.
//   write(k, v, slots, k_cache, v_cache, k_scale=None, v_scale=None)
//   read(k_cache, v_cache, slots, k_out, v_out, k_scale=None, v_scale=None) -> (k_out, v_out)
// The reference keeps no cache (its calls take whole K and V, Sparse_FlashAttention_CSR/
// sp_flatt_csr.cpp:28-39); the work is done by spfa_cache_write / spfa_cache_read in libspfa_hip.so.
#include "spfa_serve_ext.h"

using spfa_ext::OptTensor;

namespace {

// k, v (or the outputs) [tokens, heads, d] and the slots of their tokens
spfa_cache_t check_call(const torch::Tensor& k, const torch::Tensor& v, const torch::Tensor& slots, const torch::Tensor& k_cache,
                        const torch::Tensor& v_cache, const OptTensor& k_scale, const OptTensor& v_scale, const char* names) {
  TORCH_CHECK(k.device().is_cuda() && v.device().is_cuda(), names, " must be CUDA tensors");
  CHECK_INPUT(slots);
  TORCH_CHECK(k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes(), names, " must both be [tokens, heads, d]");
  TORCH_CHECK(k.scalar_type() == v.scalar_type(), names, " must have the same dtype");
  for (const torch::Tensor& t : {k, v})
    TORCH_CHECK(t.stride(-1) == 1 || t.size(-1) <= 1, names, " must have unit stride along the last dimension");
  CHECK_SAME_DEVICE(v, k);
  CHECK_SAME_DEVICE(slots, k);
  TORCH_CHECK(slots.dim() == 1 && slots.size(0) == k.size(0), "slots must hold one slot per token");
  const spfa_cache_t c = spfa_ext::make_cache(k_cache, v_cache, k_scale, v_scale, k, names);
  TORCH_CHECK(k.size(1) == c.heads && k.size(2) == c.d, names, " must have the heads and the head dimension of the cache");
  return c;
}

}  // namespace

void spfa_cache_write_py(torch::Tensor k, torch::Tensor v, torch::Tensor slots, torch::Tensor k_cache, torch::Tensor v_cache,
                         OptTensor k_scale, OptTensor v_scale) {
  const spfa_cache_t c = check_call(k, v, slots, k_cache, v_cache, k_scale, v_scale, "k and v");
  spfa_ext::check_output(k_cache, "k_cache", {k, v, slots, v_cache, k_scale, v_scale});
  spfa_ext::check_output(v_cache, "v_cache", {k, v, slots, k_scale, v_scale});
  if (c.code != SPFA_CODE_NONE) {
    spfa_ext::check_output(*k_scale, "k_scale", {k, v, slots, v_scale});
    spfa_ext::check_output(*v_scale, "v_scale", {k, v, slots});
  }
  c10::DeviceGuard guard(k.device());
  const spfa_heads_t kh = spfa_ext::heads_of(k), vh = spfa_ext::heads_of(v);
  spfa_ext::raise_on_error(spfa_cache_write(&c, &kh, &vh, k.size(0), slots.data_ptr(),
                                            spfa_ext::signed_index_bytes(slots, "slots"), spfa_ext::current_stream(k)));
}

std::tuple<torch::Tensor, torch::Tensor> spfa_cache_read_py(torch::Tensor k_cache, torch::Tensor v_cache, torch::Tensor slots,
                                                            torch::Tensor k_out, torch::Tensor v_out, OptTensor k_scale,
                                                            OptTensor v_scale) {
  const spfa_cache_t c = check_call(k_out, v_out, slots, k_cache, v_cache, k_scale, v_scale, "k_out and v_out");
  spfa_ext::check_output(k_out, "k_out", {k_cache, v_cache, slots, v_out, k_scale, v_scale});
  spfa_ext::check_output(v_out, "v_out", {k_cache, v_cache, slots, k_scale, v_scale});
  c10::DeviceGuard guard(k_out.device());
  const spfa_heads_t kh = spfa_ext::heads_of(k_out), vh = spfa_ext::heads_of(v_out);
  spfa_ext::raise_on_error(spfa_cache_read(&c, slots.data_ptr(), spfa_ext::signed_index_bytes(slots, "slots"), slots.size(0), &kh,
                                           &vh, spfa_ext::current_stream(k_out)));
  return std::make_tuple(k_out, v_out);
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, mod) {
  namespace py = pybind11;
  mod.def("write", &spfa_cache_write_py, "Keys and values into their slots of a paged cache (HIP, gfx950)", py::arg("k"),
          py::arg("v"), py::arg("slots"), py::arg("k_cache"), py::arg("v_cache"), py::arg("k_scale") = py::none(),
          py::arg("v_scale") = py::none());
  mod.def("read", &spfa_cache_read_py, "Keys and values of the slots of a paged cache (HIP, gfx950)", py::arg("k_cache"),
          py::arg("v_cache"), py::arg("slots"), py::arg("k_out"), py::arg("v_out"), py::arg("k_scale") = py::none(),
          py::arg("v_scale") = py::none());
}
