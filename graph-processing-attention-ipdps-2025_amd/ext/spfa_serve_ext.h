// Host-side glue shared by spfa_rope, spfa_cache and spfa_tree: strided tensors as the C ABI takes
// them.  No device code here.
#pragma once

#include <ATen/MemoryOverlap.h>

#include "spfa_ext_common.h"

namespace spfa_ext {

using OptTensor = std::optional<torch::Tensor>;

// Elements of a row lie next to each other; every other dimension may have any stride.
#define CHECK_ROWS(x)                                                                       \
  CHECK_CUDA(x);                                                                            \
  TORCH_CHECK(x.dim() > 0 && (x.stride(-1) == 1 || x.size(-1) <= 1), #x " must have unit stride along its last dimension")

#define CHECK_SAME_DEVICE(x, y) TORCH_CHECK((x).device() == (y).device(), "all tensors must be on the same device")

// stride of a dimension, 0 where there is nothing to stride over
inline int64_t stride_of(const torch::Tensor& t, int64_t dim) { return t.size(dim) <= 1 ? 0 : t.stride(dim); }

// [tokens, heads, d] or [batch, tokens, heads, d]
inline spfa_heads_t heads_of(const torch::Tensor& t) {
  const int64_t n = t.dim();
  return spfa_heads_t{t.data_ptr(), n == 4 ? stride_of(t, 0) : 0, stride_of(t, n - 3), stride_of(t, n - 2)};
}

// The very same elements in the same places (the stride of a dimension of one element is nobody's).
inline bool same_place(const torch::Tensor& a, const torch::Tensor& b) {
  if (a.data_ptr() != b.data_ptr() || a.sizes() != b.sizes() || a.scalar_type() != b.scalar_type()) return false;
  for (int64_t i = 0; i < a.dim(); i++)
    if (a.size(i) > 1 && a.stride(i) != b.stride(i)) return false;
  return true;
}

// An output overlaps neither itself nor other tensors of the call (those that are not there aside), except
// that it may be the very tensor it is computed from row by row (`own`).  Of tensors with gaps only those
// that begin at the same place are known to overlap: slices of one buffer may lie in each other's gaps.
inline void check_output(const torch::Tensor& out, const char* name, std::initializer_list<OptTensor> others,
                         std::initializer_list<OptTensor> own = {}) {
  TORCH_CHECK(at::has_internal_overlap(out) != at::MemOverlap::Yes, name, " must not overlap itself");
  for (const OptTensor& t : others) {
    if (!t.has_value()) continue;
    const torch::Tensor& x = *t;
    const auto o = at::get_overlap_status(out, x);
    TORCH_CHECK(o != at::MemOverlapStatus::Partial && o != at::MemOverlapStatus::Full &&
                    (out.numel() == 0 || x.numel() == 0 || out.data_ptr() != x.data_ptr()),
                name, " overlaps another tensor of the call");
  }
  for (const OptTensor& t : own) {
    if (!t.has_value()) continue;
    const torch::Tensor& x = *t;
    TORCH_CHECK(out.numel() == 0 || same_place(out, x) ||
                    (at::get_overlap_status(out, x) != at::MemOverlapStatus::Partial && out.data_ptr() != x.data_ptr()),
                name, " partly overlaps another tensor of the call");
  }
}

inline int32_t serve_dtype(const torch::Tensor& t, const char* name) {
  const int dt = elem_dtype(t);
  TORCH_CHECK(dt == SPFA_DTYPE_F32 || dt == SPFA_DTYPE_F16 || dt == SPFA_DTYPE_BF16, name,
              " must be float32, float16 or bfloat16 (got ", t.scalar_type(), ")");
  return dt;
}

// slots, positions: signed integers
inline int signed_index_bytes(const torch::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == torch::kInt32 || t.scalar_type() == torch::kInt64, name, " must be int32 or int64 (got ",
              t.scalar_type(), ")");
  return (int)t.element_size();
}

// The cache of a call: k_cache, v_cache [pages, page_size, heads, d], scales [pages, page_size, heads]
// for the 8-bit types.  dtype: of the keys and values outside it.
inline spfa_cache_t make_cache(const torch::Tensor& k_cache, const torch::Tensor& v_cache, const OptTensor& k_scale,
                               const OptTensor& v_scale, const torch::Tensor& like, const char* like_name) {
  CHECK_ROWS(k_cache);
  CHECK_ROWS(v_cache);
  TORCH_CHECK(k_cache.dim() == 4 && v_cache.dim() == 4, "k_cache and v_cache must be [pages, page_size, heads, d]");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes(), "k_cache and v_cache must have the same shape");
  TORCH_CHECK(k_cache.scalar_type() == v_cache.scalar_type(), "k_cache and v_cache must have the same dtype");
  CHECK_SAME_DEVICE(k_cache, like);
  CHECK_SAME_DEVICE(v_cache, like);
  spfa_cache_t c{};
  c.dtype = serve_dtype(like, like_name);
  switch (k_cache.scalar_type()) {
    case torch::kInt8: c.code = SPFA_CODE_INT8; break;
    case torch::kFloat8_e4m3fn: c.code = SPFA_CODE_E4M3; break;
    default:
      TORCH_CHECK(k_cache.scalar_type() == like.scalar_type(), "k_cache and v_cache must be int8, float8_e4m3fn or of the dtype of ",
                  like_name);
      c.code = SPFA_CODE_NONE;
  }
  c.k = k_cache.data_ptr();
  c.v = v_cache.data_ptr();
  c.pages = k_cache.size(0);
  c.page_size = k_cache.size(1);
  c.heads = k_cache.size(2);
  c.d = k_cache.size(3);
  TORCH_CHECK(c.page_size >= 1, "page_size must be at least 1");
  c.k_stride_page = stride_of(k_cache, 0);
  c.k_stride_slot = stride_of(k_cache, 1);
  c.k_stride_head = stride_of(k_cache, 2);
  c.v_stride_page = stride_of(v_cache, 0);
  c.v_stride_slot = stride_of(v_cache, 1);
  c.v_stride_head = stride_of(v_cache, 2);
  if (c.code == SPFA_CODE_NONE) {
    TORCH_CHECK(!k_scale.has_value() && !v_scale.has_value(), "a cache of the tensors' own dtype has no scales");
    return c;
  }
  TORCH_CHECK(k_scale.has_value() && v_scale.has_value(), "an 8-bit cache needs k_scale and v_scale");
  for (const torch::Tensor& s : {*k_scale, *v_scale}) {
    TORCH_CHECK(s.device().is_cuda(), "k_scale and v_scale must be CUDA tensors");
    CHECK_SAME_DEVICE(s, like);
    TORCH_CHECK(s.scalar_type() == torch::kFloat32, "k_scale and v_scale must be float32");
    TORCH_CHECK(s.dim() == 3 && s.size(0) == c.pages && s.size(1) == c.page_size && s.size(2) == c.heads,
                "k_scale and v_scale must be [pages, page_size, heads]");
  }
  c.k_scale = (float*)k_scale->data_ptr();
  c.v_scale = (float*)v_scale->data_ptr();
  c.ks_stride_page = stride_of(*k_scale, 0);
  c.ks_stride_slot = stride_of(*k_scale, 1);
  c.ks_stride_head = stride_of(*k_scale, 2);
  c.vs_stride_page = stride_of(*v_scale, 0);
  c.vs_stride_slot = stride_of(*v_scale, 1);
  c.vs_stride_head = stride_of(*v_scale, 2);
  return c;
}

}  // namespace spfa_ext
