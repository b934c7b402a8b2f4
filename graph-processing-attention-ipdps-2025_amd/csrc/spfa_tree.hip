// C entry points of the tree attention (spfa_tree.hpp): checks, choice of kernel, workspace.
#include "spfa_tree.hpp"

#include <cfloat>
#include <cmath>
#include <initializer_list>

namespace spfa {
template <> int tree_run<f16, SPFA_CODE_NONE>(const TreeArgs&, const TreeShape&, hipStream_t);
template <> int tree_run<f16, SPFA_CODE_INT8>(const TreeArgs&, const TreeShape&, hipStream_t);
template <> int tree_run<f16, SPFA_CODE_E4M3>(const TreeArgs&, const TreeShape&, hipStream_t);
template <> int tree_run<bf16, SPFA_CODE_NONE>(const TreeArgs&, const TreeShape&, hipStream_t);
template <> int tree_run<bf16, SPFA_CODE_INT8>(const TreeArgs&, const TreeShape&, hipStream_t);
template <> int tree_run<bf16, SPFA_CODE_E4M3>(const TreeArgs&, const TreeShape&, hipStream_t);

namespace {

constexpr int64_t kMaxPositions = INT32_MAX - 1024;

struct TreePlan {
  TreeShape shape;
  int workers;
  size_t part_bytes, state_bytes, acc_bytes;
  size_t bytes() const { return part_bytes + 2 * state_bytes + acc_bytes + 256; }
};

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

int tree_check(const spfa_cache_t* c, const spfa_tree_t* t) {
  if (c == nullptr || t == nullptr) return SPFA_ERR_BAD_ARG;
  if (c->d < 1 || c->d > 256) return SPFA_ERR_EMB_TOO_LARGE;
  if (c->dtype != SPFA_DTYPE_F16 && c->dtype != SPFA_DTYPE_BF16) return SPFA_ERR_UNSUPPORTED;
  if (c->code != SPFA_CODE_NONE && c->code != SPFA_CODE_INT8 && c->code != SPFA_CODE_E4M3) return SPFA_ERR_UNSUPPORTED;
  if (c->pages < 0 || c->pages > INT32_MAX || c->page_size < 1 || c->page_size > INT32_MAX) return SPFA_ERR_BAD_ARG;
  if (c->heads < 1 || c->heads > (1 << 16) || t->heads_q < 1 || t->heads_q > (1 << 20) || t->heads_q % c->heads)
    return SPFA_ERR_BAD_ARG;
  if (t->rows < 0 || t->rows > INT32_MAX || t->n_seqs < 0 || t->n_seqs > (1 << 24)) return SPFA_ERR_BAD_ARG;
  if (t->table_width < 0 || t->mask_words < 0) return SPFA_ERR_BAD_ARG;
  // (a row and a query head of its group make one number of 31 bits)
  if (t->rows > (INT32_MAX - 1024) / (t->heads_q / c->heads)) return SPFA_ERR_UNSUPPORTED;
  // (the kernels multiply page numbers and places by 32-bit strides)
  const int64_t limit = INT32_MAX;
  for (int64_t s : {c->k_stride_page, c->k_stride_slot, c->v_stride_page, c->v_stride_slot, c->ks_stride_page, c->ks_stride_slot,
                    c->vs_stride_page, c->vs_stride_slot})
    if (s < 0 || s > limit) return SPFA_ERR_UNSUPPORTED;
  if ((t->m == nullptr) != (t->l == nullptr)) return SPFA_ERR_BAD_ARG;
  return SPFA_OK;
}

// Which kernel, and how many workgroups, from sizes, types and alignment alone.
TreePlan tree_plan(const spfa_cache_t* c, const spfa_tree_t* t) {
  TreePlan p;
  const int es = c->code == SPFA_CODE_NONE ? 2 : 1;
  const int64_t piece = 16 / es;
  auto whole = [&](int64_t stride, int bytes) { return stride * bytes % 16 == 0; };
  const bool aligned = c->d % piece == 0 && c->d % 8 == 0 && ((uintptr_t)c->k & 15) == 0 && ((uintptr_t)c->v & 15) == 0 &&
                       ((uintptr_t)t->q & 15) == 0 && whole(c->k_stride_page, es) && whole(c->k_stride_slot, es) &&
                       whole(c->k_stride_head, es) && whole(c->v_stride_page, es) && whole(c->v_stride_slot, es) &&
                       whole(c->v_stride_head, es) && whole(t->q_stride_row, 2) && whole(t->q_stride_head, 2);
  TreeShape& s = p.shape;
  s.dp = c->d <= 64 ? 64 : c->d <= 128 ? 128 : 256;
  s.rows_how = !aligned ? kTreeAny : c->d == s.dp ? kTreeWhole : kTreePadded;
  // The rows and keys of an average sequence and head (lengths are not known here: no more keys than the
  // table and the cache have places).
  const int64_t group = t->heads_q / c->heads;
  const int64_t rows = t->n_seqs > 0 ? (t->rows * group + t->n_seqs - 1) / t->n_seqs : 0;
  const int64_t len = t->table_width < kMaxPositions / c->page_size ? t->table_width * c->page_size : kMaxPositions;
  const int64_t blocks = len <= kTreeBlock ? 1 : (len + kTreeBlock - 1) / kTreeBlock;
  double keys = (double)len * (double)t->n_seqs;
  if (keys > (double)c->pages * (double)c->page_size) keys = (double)c->pages * (double)c->page_size;
  // The wide kernel takes a key's way through LDS once for 128 rows, but has to fill, store and join 128:
  // it gains once they are more than two of the narrow kernel's tiles and its workgroups have many blocks.
  // Us, narrow against wide, 8 sequences and 4 heads: 64 elements, 96 rows of 2900 keys f16 26 / 34, bf16 27 / 37,
  // of 20000 85 / 63 and 86 / 74, 512 of 8000 98 / 81 and 103 / 94; 128 bf16 elements, 192 rows of 8000
  // 108 / 117, of 20000 288 / 242, 512 of 20000 660 / 421 (the limit leaves some: 128 of 20000 187 / 164, 512 of 8000
  // 224 / 185); 128 int8 elements, 128 rows of 20000 120 / 121, 192 164 / 180, 256 206 / 183, 512 379 / 323;
  // 256 elements, 128 rows of 20000 bf16 483 / 421, 256 e4m3 598 / 607, 512 1188 / 1107.
  const double per_group = (double)c->heads * (double)((rows + 127) / 128) * keys / kTreeBlock / (256 * wide_groups(s.dp));
  const bool many = rows > (c->code == SPFA_CODE_NONE || s.dp == 64 ? 64 : 192);
  s.wide = s.rows_how != kTreeAny && many && per_group >= (s.dp == 64 ? 4.0 : 16.0);
  s.nr = s.rows_how != kTreeAny && rows > 16 && s.dp < 256 ? 2 : 1;
  const int64_t M = s.rows();
  // as many workgroups as are to run at a time, no more than there can be units of work
  const int64_t most = 256 * (s.wide ? wide_groups(s.dp) : narrow_groups(c->code, s.dp));
  const int64_t tiles = t->rows * group / M + (t->n_seqs < t->rows ? t->n_seqs : t->rows);
  const double units = (double)tiles * (double)c->heads * (double)blocks;
  p.workers = units < (double)most ? (int)units : (int)most;
  if (p.workers < 1) p.workers = 1;
  // (a table of one block cuts no item; the merge has a workgroup per part and row, up to 16: with 32 the many
  // without a row cost 1 us)
  s.merge_rows = blocks <= 1 ? 0 : (int)(rows < 1 ? 1 : rows < 16 ? rows : 16);
  p.part_bytes = round256((size_t)p.workers * sizeof(TreePart));
  p.state_bytes = s.merge_rows ? round256((size_t)2 * p.workers * M * sizeof(float)) : 0;
  p.acc_bytes = s.merge_rows ? round256((size_t)2 * p.workers * M * s.dp * sizeof(float)) : 0;
  return p;
}

}  // namespace
}  // namespace spfa

using namespace spfa;

extern "C" size_t spfa_tree_workspace_bytes(const spfa_cache_t* c, const spfa_tree_t* t) {
  if (tree_check(c, t)) return 256;
  return tree_plan(c, t).bytes();
}

extern "C" int spfa_tree_forward(const spfa_cache_t* c, const spfa_tree_t* t, void* workspace, size_t workspace_bytes,
                                 void* stream) {
  const int rc = tree_check(c, t);
  if (rc) return rc;
  if (t->rows == 0 || t->n_seqs == 0) return SPFA_OK;
  if (t->q == nullptr || t->out == nullptr || t->q_offsets == nullptr || t->ctx_lens == nullptr) return SPFA_ERR_BAD_ARG;
  if (t->mask_words > 0 && t->tree_mask == nullptr) return SPFA_ERR_BAD_ARG;
  const bool keys = c->pages > 0 && t->table_width > 0;
  if (keys && (c->k == nullptr || c->v == nullptr || t->page_table == nullptr)) return SPFA_ERR_BAD_ARG;
  if (keys && c->code != SPFA_CODE_NONE && (c->k_scale == nullptr || c->v_scale == nullptr)) return SPFA_ERR_BAD_ARG;
  const TreePlan p = tree_plan(c, t);
  if (workspace == nullptr || ((uintptr_t)workspace & 255) || workspace_bytes < p.bytes()) return SPFA_ERR_WORKSPACE;

  TreeArgs a{};
  a.q = t->q;
  a.out = t->out;
  a.qs_row = t->q_stride_row;
  a.qs_head = t->q_stride_head;
  a.os_row = t->out_stride_row;
  a.os_head = t->out_stride_head;
  a.m = t->m;
  a.l = t->l;
  a.k = (const char*)c->k;
  a.v = (const char*)c->v;
  a.ks = c->k_scale;
  a.vs = c->v_scale;
  a.k_page = (uint32_t)c->k_stride_page;
  a.k_slot = (uint32_t)c->k_stride_slot;
  a.k_head = c->k_stride_head;
  a.v_page = (uint32_t)c->v_stride_page;
  a.v_slot = (uint32_t)c->v_stride_slot;
  a.v_head = c->v_stride_head;
  a.ks_page = (uint32_t)c->ks_stride_page;
  a.ks_slot = (uint32_t)c->ks_stride_slot;
  a.ks_head = c->ks_stride_head;
  a.vs_page = (uint32_t)c->vs_stride_page;
  a.vs_slot = (uint32_t)c->vs_stride_slot;
  a.vs_head = c->vs_stride_head;
  a.q_offsets = t->q_offsets;
  a.ctx_lens = t->ctx_lens;
  a.page_table = t->page_table;
  a.table_width = t->table_width;
  a.table_stride = t->table_stride;
  a.mask = (const uint64_t*)t->tree_mask;
  a.mask_words = t->mask_words;
  a.rows = t->rows;
  a.pages = c->pages;
  a.heads = (int32_t)c->heads;
  a.group = (int32_t)(t->heads_q / c->heads);
  a.n_seqs = (int32_t)t->n_seqs;
  a.d = (int32_t)c->d;
  a.page_size = (int32_t)c->page_size;
  a.max_len = !keys ? 0 : t->table_width < kMaxPositions / c->page_size ? (int32_t)(t->table_width * c->page_size) : (int32_t)kMaxPositions;
  fast_divider(a.page_size, &a.page_magic, &a.page_shift);
  fast_divider(a.group, &a.group_magic, &a.group_shift);
  fast_divider(p.shape.rows(), &a.tile_magic, &a.tile_shift);
  // the kernels look for the largest score before they scale it: a negative scale becomes the queries'
  // sign, and zero the smallest number there is (masked scores times it stay -infinity)
  a.scale_log2 = fabsf(t->scale) * 1.4426950408889634f;
  if (a.scale_log2 < FLT_MIN) a.scale_log2 = FLT_MIN;
  a.flip = t->scale < 0.f ? 0x80008000u : 0u;
  a.workers = p.workers;
  a.out_vec = c->d % 4 == 0 && ((uintptr_t)t->out & 7) == 0 && t->out_stride_row % 4 == 0 && t->out_stride_head % 4 == 0;
  char* ws = (char*)workspace;
  a.part = (TreePart*)ws;
  a.pm = (float*)(ws + p.part_bytes);
  a.pl = (float*)(ws + p.part_bytes + p.state_bytes);
  a.pacc = (float*)(ws + p.part_bytes + 2 * p.state_bytes);
  const hipStream_t s = (hipStream_t)stream;
  if (c->dtype == SPFA_DTYPE_F16) {
    if (c->code == SPFA_CODE_INT8) return tree_run<f16, SPFA_CODE_INT8>(a, p.shape, s);
    if (c->code == SPFA_CODE_E4M3) return tree_run<f16, SPFA_CODE_E4M3>(a, p.shape, s);
    return tree_run<f16, SPFA_CODE_NONE>(a, p.shape, s);
  }
  if (c->code == SPFA_CODE_INT8) return tree_run<bf16, SPFA_CODE_INT8>(a, p.shape, s);
  if (c->code == SPFA_CODE_E4M3) return tree_run<bf16, SPFA_CODE_E4M3>(a, p.shape, s);
  return tree_run<bf16, SPFA_CODE_NONE>(a, p.shape, s);
}
