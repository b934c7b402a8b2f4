// Attention of drafted tokens (a tree, a chain, a single token) over a paged cache.
//
// Rows are the (node, query head) pairs that share a cache head: n_s * group of them for sequence s
// and cache head h, cut into tiles of M rows.  An item is (sequence, row tile, cache head); its keys
// are cut into blocks of 128 and every item's blocks are laid end to end, sequence by sequence.  Each
// workgroup takes an equal run of that line (lengths differ from sequence to sequence, so any split
// per sequence would leave some of them waiting); where a run begins or ends inside an item, the
// part's softmax state (max, sum, unnormalised result) goes to the workspace and
// tree_merge_kernel joins the parts in order.  No atomics: the result depends on the sizes alone.
//
// A wavefront works on 32 keys at a time for NR * 16 rows, all in registers (16x16x32 products; lane
// c + 16 g, c < 16, g < 4):
//   S^T = K Q^T    A = K: the lane holds 16-byte pieces of the rows of keys c and 16 + c, straight from
//                  memory; which elements stand for which of a product's 32 is free as long as Q's agree
//   softmax        the lane has row c and keys 4 g .. 4 g + 3 and 16 + 4 g .. 16 + 4 g + 3
//   O^T += V^T P^T P^T is S^T's own layout (the order of the keys is free too); V^T: the lane has
//                  elements EB * c .. EB * c + EB - 1 of these eight keys, so one load instruction
//                  takes four whole rows; pairs of keys are put side by side by byte permutes
// 8-bit codes become f16 / bf16 values exactly on the way; their scales multiply the scores (K)
// and the weights (V) in fp32.  Nothing but scales, row offsets and the joined results of the
// wavefronts passes through LDS, so wavefronts run apart until an item ends.
#pragma once

#include <type_traits>

#include "spfa_serve.hpp"

namespace spfa {

constexpr int kTreeBlock = 128;  // keys per unit of work
constexpr int kTreeWaves = 4;
constexpr float kTreeSlack = 8.f;  // weights may grow to 2^8 before the running maximum is moved

typedef float f32x4t __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8t __attribute__((ext_vector_type(8)));
typedef uint32_t uint2t __attribute__((ext_vector_type(2)));

struct TreePart {  // the item whose last part a workgroup holds, for the merge
  int32_t seq, tile, head, first;  // first: the workgroup with its first part; seq < 0: none
};

struct TreeArgs {
  const void* q;
  void* out;
  int64_t qs_row, qs_head, os_row, os_head;
  float* m;
  float* l;
  const char* k;
  const char* v;
  const float* ks;
  const float* vs;
  int64_t k_head, v_head, ks_head, vs_head;
  uint32_t k_page, k_slot, v_page, v_slot, ks_page, ks_slot, vs_page, vs_slot;
  const int32_t* q_offsets;
  const int32_t* ctx_lens;
  const int32_t* page_table;
  int64_t table_width, table_stride;
  const uint64_t* mask;
  int64_t mask_words;
  int64_t rows, pages;
  int32_t heads, group, n_seqs, d, page_size;
  // p / size = (p * magic >> 32) >> shift for p < 2^31; shift < 0: p (host: fast_divider)
  uint32_t page_magic, group_magic, tile_magic;  // of page_size, group, rows of an item
  int32_t page_shift, group_shift, tile_shift;
  int32_t max_len;  // positions the page table covers, cut to 32 bits
  float scale_log2;  // above zero
  uint32_t flip;     // sign bits of a pair where the scale is below
  int32_t workers;
  int32_t out_vec;  // rows of out can be written four elements at a time
  TreePart* part;
  float* pm;  // [2 * workers, M]
  float* pl;
  float* pacc;  // [2 * workers, M, DP]
};

// (64-bit divisions are hundreds of dependent instructions: none on the way of ordinary sizes)
__device__ __forceinline__ int64_t tree_div64(int64_t a, int64_t b) {
  if (((uint64_t)a | (uint64_t)b) >> 32) return a / b;
  return (int64_t)((uint32_t)a / (uint32_t)b);
}

struct TreeSeq {
  int row0, n, ctx, len;
  int tiles, nblk;
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeArgs& g, int s, int M) {
  TreeSeq q;
  int64_t r0 = g.q_offsets[s], r1 = g.q_offsets[s + 1];
  r0 = r0 < 0 ? 0 : r0 > g.rows ? g.rows : r0;
  r1 = r1 < r0 ? r0 : r1 > g.rows ? g.rows : r1;
  q.row0 = (int)r0;
  q.n = (int)(r1 - r0);
  const int ctx = g.ctx_lens[s];
  q.ctx = ctx < 0 ? 0 : ctx;
  const int64_t len = (int64_t)q.ctx + q.n;
  q.len = (int)(len < g.max_len ? len : g.max_len);
  q.tiles = (int)fast_div((uint32_t)(q.n * g.group + M - 1), g.tile_magic, g.tile_shift);  // (host: rows * group stays below 2^31)
  q.nblk = q.len <= kTreeBlock ? 1 : (q.len + kTreeBlock - 1) / kTreeBlock;
  return q;
}
__device__ __forceinline__ int64_t tree_units(const TreeArgs& g, const TreeSeq& q) { return (int64_t)q.tiles * g.heads * q.nblk; }

__device__ __forceinline__ int64_t shfl_i64(int64_t x, int lane) {
  const uint32_t lo = (uint32_t)shfl_i32((int)(uint32_t)x, lane), hi = (uint32_t)shfl_i32((int)(x >> 32), lane);
  return (int64_t)(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t wave_scan_i64(int64_t x) {
#pragma unroll
  for (int m = 1; m < kWave; m *= 2) {
    const int64_t y = shfl_i64(x, lane_id() - m);
    if (lane_id() >= m) x += y;
  }
  return x;
}
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)(x >> 32)) << 32) | (uint32_t)uniform((int)(uint32_t)x));
}
// largest / sum over the four lanes that have a row's keys (16 lanes apart)
__device__ __forceinline__ float row_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  const uint32_t y = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b)));
  const auto t = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  const uint32_t c = t[0], d = t[1];
  return fmaxf(__builtin_bit_cast(float, c), __builtin_bit_cast(float, d));
}
__device__ __forceinline__ float row_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  const uint32_t y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b));
  const auto t = __builtin_amdgcn_permlane16_swap(y, y, false, false);
  const uint32_t c = t[0], d = t[1];
  return __builtin_bit_cast(float, c) + __builtin_bit_cast(float, d);
}

template <typename T>
__device__ __forceinline__ f32x4t tree_mfma(const uint4v& a, const uint4v& b, f32x4t c) {
  if constexpr (__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8t, a), __builtin_bit_cast(bf16x8t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8t, a), __builtin_bit_cast(f16x8t, b), c, 0, 0, 0);
}
template <typename T>
__device__ __forceinline__ uint32_t tree_pack(float lo, float hi) {
  typedef T t2 __attribute__((ext_vector_type(2)));
  const t2 x = {(T)lo, (T)hi};
  return __builtin_bit_cast(uint32_t, x);
}

// The four codes of a word as two words of T pairs, exactly.
template <typename T, int CODE>
__device__ __forceinline__ uint2t decode4(uint32_t w) {
  uint2t r;
  if constexpr (CODE == SPFA_CODE_E4M3) {
    if constexpr (__is_same(T, bf16)) {
      r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
      r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true));
    } else {
      r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
      r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true));
    }
  } else if constexpr (__is_same(T, bf16)) {
    // a small whole number's fp32 form ends in 16 zero bits: its upper half is its bf16 form
    const uint32_t a = __builtin_bit_cast(uint32_t, (float)(int8_t)w), b = __builtin_bit_cast(uint32_t, (float)(int8_t)(w >> 8)),
                   c = __builtin_bit_cast(uint32_t, (float)(int8_t)(w >> 16)), d = __builtin_bit_cast(uint32_t, (float)((int32_t)w >> 24));
    r[0] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    r[1] = __builtin_amdgcn_perm(d, c, 0x07060302u);
  } else {
    // 0x6400 + u is 1024 + u in f16 for a byte u = code + 128
    const uint32_t u = w ^ 0x80808080u;
    const half2v off = {(_Float16)1152.f, (_Float16)1152.f};
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, lo) - off);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, hi) - off);
  }
  return r;
}

// How a row's result leaves: m (log2 units) and l of it, both the same in every lane of the row.
// out = wa * (what it holds) + wb * (the unnormalised result); the state a lane of the row writes
// afterwards, when all have read the old one, is m_out and l_out.
struct TreeWeights {
  float wa, wb, m_out, l_out;
  bool keep;  // nothing to attend and a state to keep
};
__device__ __forceinline__ TreeWeights tree_weights(const TreeArgs& g, int64_t row, int head, float m, float l) {
  TreeWeights r{0.f, 0.f, m * 0.6931471805599453f, l, false};
  if (g.m == nullptr) {
    r.wb = l == 0.f ? 0.f : 1.f / l;
    return r;
  }
  if (l == 0.f) {
    r.keep = true;
    return r;
  }
  const int64_t st = row * ((int64_t)g.heads * g.group) + head;
  const float l_in = g.l[st];
  r.wb = 1.f;
  if (l_in != 0.f) {
    const float m_in = g.m[st], m_nat = r.m_out;
    r.m_out = fmaxf(m_nat, m_in);
    r.wa = l_in * __expf(m_in - r.m_out);
    r.wb = __expf(m_nat - r.m_out);
    r.l_out = r.wa + l * r.wb;
  }
  r.wa /= r.l_out;
  r.wb /= r.l_out;
  return r;
}
// N (2 or 4) elements of the row from e0 on
template <typename T, int N>
__device__ __forceinline__ void tree_store(const TreeArgs& g, int64_t row, int head, int e0, const TreeWeights& w, const float (&x)[N]) {
  T* o = (T*)g.out + row * g.os_row + head * g.os_head + e0;
  if (w.keep || e0 >= g.d) return;
  typedef T tn __attribute__((ext_vector_type(N)));
  if (g.out_vec) {
    tn y, old = {};
    if (w.wa != 0.f) old = *reinterpret_cast<const tn*>(o);
#pragma unroll
    for (int u = 0; u < N; u++) y[u] = (T)((w.wb != 0.f ? x[u] * w.wb : 0.f) + (w.wa != 0.f ? w.wa * (float)old[u] : 0.f));
    *reinterpret_cast<tn*>(o) = y;
  } else {
#pragma unroll
    for (int u = 0; u < N; u++)
      if (e0 + u < g.d) o[u] = (T)((w.wb != 0.f ? x[u] * w.wb : 0.f) + (w.wa != 0.f ? w.wa * (float)o[u] : 0.f));
  }
}
__device__ __forceinline__ void tree_store_state(const TreeArgs& g, int64_t row, int head, const TreeWeights& w) {
  if (g.m == nullptr || w.keep) return;
  const int64_t st = row * ((int64_t)g.heads * g.group) + head;
  g.m[st] = w.m_out;
  g.l[st] = w.l_out;
}

// The factor that takes a state to a larger maximum: never quite zero, so that an infinity among the
// elements stays one.
__device__ __forceinline__ float tree_shrink(float by) { return fmaxf(__builtin_amdgcn_exp2f(by), 1.17549435e-38f); }

// what a wavefront's lanes wrote to LDS is there for its other lanes
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// How rows are loaded: element by element, in whole pieces where d is less than DP, or d == DP.
enum { kTreeAny = 0, kTreePadded = 1, kTreeWhole = 2 };

// Sizes that follow from the element types and the padded head size.
template <typename T, int CODE, int DP>
struct TreeTypes {
  static constexpr bool kCoded = CODE != SPFA_CODE_NONE;
  static constexpr int EB = DP / 16;           // elements per lane of a V row
  static constexpr int ES = kCoded ? 1 : 2;    // bytes of an element in the cache
  static constexpr int NK = DP * ES / 64;      // 16-byte pieces of a K row per lane
  static constexpr int PE = 16 / ES;           // elements of one
  static constexpr int VB = EB * ES;           // bytes of a V row per lane
  static constexpr int VW = VB / 4;
  static constexpr int QF = DP / 32;           // pieces of a query
  using Tv = std::conditional_t<kCoded, bf16, T>;  // (8-bit values times any scale need bf16's range)
  // Weights in two bf16 parts: needed where f16 calls meet 8-bit codes (one part has 8 of their 11 bits),
  // and with bf16 calls what keeps the result to its own rounding (error against 64 bits 0.0017, with one part
  // 0.0023; in the kernel of many rows 124 -> 149 us for 64 elements, 333 -> 288 for 128, 8 x 20000 tokens, 512 rows
  // for each of 4 heads).  f16 calls over f16 have one part, of the result's own 11 bits, in both kernels: 0.00027
  // with many rows where two parts have 0.00021 (f16's rounding), for 76 us instead of 64 at 488 rows of 5000 keys.
  static constexpr bool kTwo = kCoded || __is_same(T, bf16);
};

// This workgroup's run of the line of all items' blocks, item by item.
struct TreeWalk {
  int64_t pos, end;    // what is left of the run
  int64_t per, extra;  // how long runs are
  int64_t in_seq;      // units before pos in its sequence
  TreeSeq sq;
  int seq, w;
  // the item at pos
  int tile, head, blk0, blk1, live_rows, tile0;

  __device__ __forceinline__ bool start(const TreeArgs& g, int M) {
    const int lane = lane_id();
    // workgroups of one XCD (dealt in turn) take neighbouring runs
    w = blockIdx.x;
    if (g.workers % 8 == 0) w = (w % 8) * (g.workers / 8) + w / 8;
    int64_t total = 0, incl = 0, u = 0;
    for (int base = 0; base < g.n_seqs; base += kWave) {
      u = 0;
      if (base + lane < g.n_seqs) u = tree_units(g, tree_seq(g, base + lane, M));
      incl = wave_scan_i64(u);
      total += uniform64(shfl_i64(incl, 63));
    }
    per = tree_div64(total, g.workers);
    extra = total - per * g.workers;
    pos = w * per + (w < extra ? w : extra);
    end = pos + per + (w < extra ? 1 : 0);
    seq = 0;
    in_seq = 0;
    int64_t before = 0;
    for (int base = 0; base < g.n_seqs; base += kWave) {
      if (g.n_seqs > kWave) {  // (else the sums are still here)
        u = 0;
        if (base + lane < g.n_seqs) u = tree_units(g, tree_seq(g, base + lane, M));
        incl = wave_scan_i64(u) + before;
      }
      const uint64_t past = __builtin_amdgcn_ballot_w64(incl > pos);
      if (past) {
        const int at = (int)__builtin_ctzll(past);
        seq = uniform(base + at);
        in_seq = pos - uniform64(shfl_i64(incl - u, at));
        break;
      }
      before = uniform64(shfl_i64(incl, 63));
    }
    if (pos < end) sq = tree_seq(g, seq, M);
    return pos < end;
  }
  // false: the run is done
  __device__ __forceinline__ bool item(const TreeArgs& g, int M) {
    if (pos >= end) return false;
    while (in_seq >= tree_units(g, sq)) {  // (the next sequence with any rows; there is one, pos < end <= total)
      in_seq = 0;
      if (++seq >= g.n_seqs) return false;  // (only if the arrays change under the call)
      sq = tree_seq(g, seq, M);
    }
    const int64_t it = tree_div64(in_seq, sq.nblk);
    blk0 = uniform((int)(in_seq - it * sq.nblk));
    head = uniform((int)tree_div64(it, sq.tiles));
    tile = uniform((int)(it - (int64_t)head * sq.tiles));
    blk1 = uniform((int)(end - pos < sq.nblk - blk0 ? blk0 + (end - pos) : sq.nblk));
    tile0 = tile * M;
    const int n_rows = sq.n * g.group;
    live_rows = n_rows - tile0 < M ? n_rows - tile0 : M;
    return true;
  }
  __device__ __forceinline__ bool whole_item() const { return blk0 == 0 && blk1 == sq.nblk; }
  __device__ __forceinline__ int64_t slot() const { return blk0 == 0 ? 2 * (int64_t)w + 1 : 2 * (int64_t)w; }
  // names the item for the merge when its last part, and not its first, is in this run
  __device__ __forceinline__ void name_part(const TreeArgs& g) const {
    if (blk0 == 0 || blk1 != sq.nblk) return;
    const int64_t first = pos - blk0, cut = extra * (per + 1);  // the item's first unit; who has it:
    g.part[w] = TreePart{seq, tile, head, (int)(first < cut ? tree_div64(first, per + 1) : extra + tree_div64(first - cut, per))};
  }
  __device__ __forceinline__ void next() {
    pos += blk1 - blk0;
    in_seq += blk1 - blk0;
  }
};

// Sixteen rows of a wavefront: lane (c, g) has the pieces of row c that go with its place.
template <typename T, int CODE, int DP, int ROWS>
struct TreeQueries {
  using Ty = TreeTypes<T, CODE, DP>;
  uint4v f[Ty::QF];
  int node;
  const uint64_t* bits;  // of the row's node

  __device__ __forceinline__ void load(const TreeArgs& a, const TreeWalk& it, int first_row) {
    const int c = lane_id() & 15, g = lane_id() >> 4;
    // (lanes without a row work on the tile's last one; what they get is not written)
    const int r = first_row + c < it.live_rows ? first_row + c : it.live_rows - 1;
    const int rr = it.tile0 + r;
    node = (int)fast_div((uint32_t)rr, a.group_magic, a.group_shift);
    const int gi = rr - node * a.group;
    const T* qp = (const T*)a.q + (int64_t)(it.sq.row0 + node) * a.qs_row + (int64_t)(it.head * a.group + gi) * a.qs_head;
    bits = a.mask + (int64_t)(it.sq.row0 + node) * a.mask_words;
#pragma unroll
    for (int s = 0; s < Ty::QF; s++) {
      const int e0 = Ty::ES == 2 ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s % 2);
      f[s] = uint4v{0u, 0u, 0u, 0u};
      if (ROWS != kTreeAny) {
        if (ROWS == kTreeWhole || e0 < a.d) f[s] = *reinterpret_cast<const uint4v*>(qp + e0);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (e0 + i < a.d) f[s][i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, qp[e0 + i]) << (16 * (i % 2));
      }
    }
  }
  // (for a negative scale the queries change sign)
  __device__ __forceinline__ void flip(uint32_t signs) {
#pragma unroll
    for (int s = 0; s < Ty::QF; s++) f[s] ^= signs;
  }
  // The keys the row attends among 32 that begin with draft j0 (negative: cached tokens before the
  // tree), as far as they exist.
  __device__ __forceinline__ uint32_t live(const TreeArgs& a, int j0, uint32_t exist) const {
    uint32_t b = 0xffffffffu;
    if (j0 > -32) {
      if (a.mask == nullptr) {
        const int n = node - j0 + 1;
        b = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
      } else if (j0 < 0) {
        const uint64_t x = a.mask_words > 0 ? bits[0] : 0;
        b = (uint32_t)(x << -j0) | ((1u << -j0) - 1u);
      } else {
        const int word = j0 >> 6, sh = j0 & 63;
        const uint64_t lo = word < a.mask_words ? bits[word] : 0, hi = word + 1 < a.mask_words ? bits[word + 1] : 0;
        b = (uint32_t)(lo >> sh) | (sh > 32 ? (uint32_t)(hi << (64 - sh)) : 0u);
      }
    }
    return b & exist;
  }
};

// Bit number v (of a lane's eight keys) of a word of bits by key that was moved down by 4 g, spread over
// a word.
__device__ __forceinline__ uint32_t spread_bit(uint32_t word, int v) {
  return (uint32_t)((int32_t)(word << (31 - (16 * (v / 4) + v % 4))) >> 31);
}

// A wavefront's way to the rows of 32 keys.  Lane l looks key l % 32 up; the rows' places go round
// through LDS (`off`: 64 words of 64 bits of the wavefront's own).
template <typename T, int CODE, int DP, int ROWS>
struct TreeKeys {
  using Ty = TreeTypes<T, CODE, DP>;
  static constexpr int ES = Ty::ES, EB = Ty::EB, NK = Ty::NK, PE = Ty::PE, VB = Ty::VB, VW = Ty::VW;
  uint4v kr[2][NK];     // of keys c and 16 + c
  uint32_t vr[8][VW];   // of keys 4 g + j, 16 + 4 g + j
  float ks, vs;         // of key l % 32
  int page;             // of the tile looked up last
  uint32_t place;       // in it, kNowhere for a key past the end
  static constexpr uint32_t kNowhere = 0xffffffffu;
  // the same for all lanes
  const char *kb, *vb;
  const float *ksb, *vsb;
  const int32_t* table;
  uint32_t k_page, k_slot, v_page, v_slot, s_page, s_slot, u_page, u_slot;
  uint32_t lim, last, page_size, magic, pages;
  int shift;
  int64_t* off;

  __device__ __forceinline__ void start(const TreeArgs& a, const TreeWalk& it, int t_end, int64_t* off_lds) {
    kb = a.k + uniform64((int64_t)it.head * a.k_head * ES);
    vb = a.v + uniform64((int64_t)it.head * a.v_head * ES);
    if (Ty::kCoded) {
      ksb = a.ks + uniform64((int64_t)it.head * a.ks_head);
      vsb = a.vs + uniform64((int64_t)it.head * a.vs_head);
    }
    table = a.page_table + uniform64((int64_t)it.seq * a.table_stride);
    k_page = uniform(a.k_page), k_slot = uniform(a.k_slot), v_page = uniform(a.v_page), v_slot = uniform(a.v_slot);
    s_page = uniform(a.ks_page), s_slot = uniform(a.ks_slot), u_page = uniform(a.vs_page), u_slot = uniform(a.vs_slot);
    page_size = uniform(a.page_size), magic = uniform(a.page_magic), shift = uniform(a.page_shift), pages = uniform((int)a.pages);
    lim = uniform(it.sq.len < t_end * 32 ? it.sq.len : t_end * 32);
    last = lim > 0 ? fast_div(lim - 1, magic, shift) : 0;
    off = off_lds;
    ks = vs = 0.f;
  }
  // asks for the page of this lane's key of a tile
  __device__ __forceinline__ void look_up(int t) {
    const uint32_t p = (uint32_t)(t * 32 + (lane_id() & 31));
    const uint32_t q = fast_div(p, magic, shift);
    place = p < lim ? p - q * page_size : kNowhere;
    page = table[q < last ? q : last];  // (past the end the last page's entry: no branch around the load)
  }
  // Where the rows of the tile looked up last are (of keys that do not exist: the cache's first row,
  // which does when there are tiles at all); asks for the scales and returns the bits of the keys
  // that exist.
  __device__ __forceinline__ uint32_t locate() {
    const bool ok = (uint32_t)page < pages && place != kNowhere;  // (-1 is no page)
    const uint32_t pg = ok ? (uint32_t)page : 0u, at = ok ? place : 0u;
    const int64_t ko = (int64_t)((uint64_t)pg * k_page + (uint64_t)at * k_slot);
    int64_t vo = ko;
    if (v_page != k_page || v_slot != k_slot) vo = (int64_t)((uint64_t)pg * v_page + (uint64_t)at * v_slot);
    off[lane_id() & 31] = ko;
    off[32 + (lane_id() & 31)] = vo;
    if constexpr (Ty::kCoded) {
      const int64_t so = (int64_t)((uint64_t)pg * s_page + (uint64_t)at * s_slot);
      int64_t uo = so;
      if (u_page != s_page || u_slot != s_slot) uo = (int64_t)((uint64_t)pg * u_page + (uint64_t)at * u_slot);
      ks = ksb[so];
      vs = vsb[uo];
    }
    wave_sync();
    return (uint32_t)__builtin_amdgcn_ballot_w64(ok);
  }
  __device__ __forceinline__ void load_k(int d) {
    const int c = lane_id() & 15, g = lane_id() >> 4;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const char* p = kb + off[16 * u + c] * ES + 16 * g;
#pragma unroll
      for (int s = 0; s < NK; s++) {
        const int e0 = PE * (4 * s + g);
        kr[u][s] = uint4v{0u, 0u, 0u, 0u};
        if (ROWS != kTreeAny) {
          if (ROWS == kTreeWhole || e0 < d) kr[u][s] = *reinterpret_cast<const uint4v*>(p + 64 * s);
        } else {
#pragma unroll
          for (int i = 0; i < PE; i++)
            if (e0 + i < d) {
              const char* x = p + 64 * s + i * ES;
              const uint32_t y = ES == 2 ? *reinterpret_cast<const uint16_t*>(x) : *reinterpret_cast<const uint8_t*>(x);
              kr[u][s][i * ES / 4] |= y << (8 * (i * ES % 4));
            }
        }
      }
    }
  }
  __device__ __forceinline__ void load_v(int d) {
    const int c = lane_id() & 15, g = lane_id() >> 4;
    const char* base = vb + EB * ES * c;
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const char* p = base + off[32 + 16 * (k / 4) + 4 * g + k % 4] * ES;
      uint32_t(&x)[VW] = vr[k];
#pragma unroll
      for (int y = 0; y < VW; y++) x[y] = 0u;
      if (ROWS != kTreeAny) {
        if (ROWS == kTreeWhole || EB * c < d) {
          if constexpr (VB == 4) {
            x[0] = *reinterpret_cast<const uint32_t*>(p);
          } else if constexpr (VB == 8) {
            const uint2t y = *reinterpret_cast<const uint2t*>(p);
            x[0] = y[0];
            x[1] = y[1];
          } else {
#pragma unroll
            for (int y = 0; y < VW; y += 4) {
              // (a piece that begins behind the row's end is not there)
              if (ROWS != kTreeWhole && EB * c + y * 4 / ES >= d) continue;
              const uint4v z = *reinterpret_cast<const uint4v*>(p + 4 * y);
#pragma unroll
              for (int u = 0; u < 4; u++) x[y + u] = z[u];
            }
          }
        }
      } else {
#pragma unroll
        for (int u = 0; u < EB; u++)
          if (EB * c + u < d) {
            const uint32_t y = ES == 2 ? *reinterpret_cast<const uint16_t*>(p + u * 2) : *reinterpret_cast<const uint8_t*>(p + u);
            x[u * ES / 4] |= y << (8 * (u * ES % 4));
          }
      }
    }
    wave_sync();
  }
  // step x of the product's first factor: 32 elements of keys 16 u ..
  __device__ __forceinline__ uint4v key_frag(int u, int x) const {
    if constexpr (!Ty::kCoded) {
      return kr[u][x];
    } else {
      const uint2t a = decode4<T, CODE>(kr[u][x / 2][2 * (x % 2)]), b = decode4<T, CODE>(kr[u][x / 2][2 * (x % 2) + 1]);
      return uint4v{a[0], a[1], b[0], b[1]};
    }
  }
  // word pair `w` (four elements: two of the pairs below) of the lane's eight values, as T pairs
  __device__ __forceinline__ void values(int w, uint32_t (&vq)[8][2]) const {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      if constexpr (!Ty::kCoded) {
        vq[k][0] = vr[k][2 * w];
        vq[k][1] = vr[k][2 * w + 1];
      } else {
        const uint2t a = decode4<bf16, CODE>(vr[k][w]);
        vq[k][0] = a[0];
        vq[k][1] = a[1];
      }
    }
  }
  // For a tile that some rows do not attend as a whole.  Values of keys that do not exist become zeros.
  // An infinity or NaN among the others must reach the rows that attend its key and no other row, which
  // 0 * infinity would not do: it becomes a zero too and is added, row by row, to sums in `tab`, 16 NR
  // rows of `stride` floats in LDS that are this wavefront's until the item ends (seen: they are in use).
  // live: the keys that row c (of each 16) attends.
  template <int NR>
  __device__ __forceinline__ void screen(uint32_t exist, const uint32_t (&live)[NR], float* tab, int stride, bool& seen) {
    const int lane = lane_id(), c = lane & 15, g = lane >> 4;
    const bool there = (exist >> (lane & 31)) & 1;
    const float vs_is = vs;
    bool bad = false;
    if constexpr (Ty::kCoded) {
      bad = there && !(fabsf(vs) <= 3.402823466e38f);  // a scale that is no finite number
      if (bad) vs = 1.f;
      if (!there) ks = vs = 0.f;
    }
    const uint32_t eg = exist >> (4 * g), sick = (uint32_t)__builtin_amdgcn_ballot_w64(bad) >> (4 * g);
    // an exponent of ones (e4m3: all of the code but its sign) runs over into the sign's place
    constexpr bool kB = __is_same(T, bf16);
    constexpr uint32_t kSign = Ty::kCoded ? 0x80808080u : 0x80008000u;
    constexpr uint32_t kAll = CODE == SPFA_CODE_E4M3 ? 0x7f7f7f7fu : Ty::kCoded ? 0u : kB ? 0x7f807f80u : 0x7c007c00u;
    constexpr uint32_t kStep = CODE == SPFA_CODE_E4M3 ? 0x01010101u : Ty::kCoded ? 0u : kB ? 0x00800080u : 0x04000400u;
    uint32_t odd = sick & 0x000f000fu;
#pragma unroll
    for (int k = 0; k < 8; k++)
#pragma unroll
      for (int y = 0; y < VW; y++) {
        vr[k][y] &= spread_bit(eg, k);
        odd |= ((vr[k][y] & kAll) + kStep) & kSign;
      }
    if (__builtin_amdgcn_ballot_w64(odd != 0) == 0) return;
    if (!seen)
      for (int i = lane; i < 16 * NR * stride; i += kWave) tab[i] = 0.f;
    seen = true;
    wave_sync();
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const int at = 16 * (k / 4) + k % 4;
      const bool ill = (sick >> at) & 1;
      uint32_t some = ill;
#pragma unroll
      for (int y = 0; y < VW; y++) some |= ((vr[k][y] & kAll) + kStep) & kSign;
      if (__builtin_amdgcn_ballot_w64(some != 0) == 0) continue;
      float add[EB], scale = 0.f;
      if constexpr (Ty::kCoded) scale = shfl_f32(vs_is, at + 4 * g);
#pragma unroll
      for (int e = 0; e < EB; e++) {
        uint32_t& word = vr[k][e * ES / 4];
        const int sh = 8 * (e * ES % 4);
        if constexpr (!Ty::kCoded) {
          const uint16_t u = (uint16_t)(word >> sh);
          const bool is = (u & (uint16_t)kAll) == (uint16_t)kAll;
          add[e] = is ? (float)__builtin_bit_cast(T, u) : 0.f;
          if (is) word &= ~(0xffffu << sh);
        } else {
          const bool is = ill || (CODE == SPFA_CODE_E4M3 && ((word >> sh) & 0x7fu) == 0x7fu);
          float x;
          if constexpr (CODE == SPFA_CODE_INT8) x = (float)(int8_t)(word >> sh);
          else x = __builtin_amdgcn_cvt_f32_fp8((int)(word >> sh), 0);
          add[e] = is ? x * scale : 0.f;
          if (is) word &= ~(0xffu << sh);
        }
      }
#pragma unroll 1
      for (int turn = 0; turn < 4; turn++) {
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll 1
          for (int r = 0; r < 16; r++) {
            const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)live[n], r);
            if (g == turn && ((row >> (at + 4 * g)) & 1)) {
              float* to = tab + (16 * n + r) * stride + EB * c;
#pragma unroll
              for (int e = 0; e < EB; e++) to[e] += add[e];
            }
          }
        wave_sync();
      }
    }
  }
};

// element 4 w + e (e < 4) of the lane's eight values as a factor of the product
__device__ __forceinline__ uint4v value_frag(const uint32_t (&vq)[8][2], int e) {
  uint4v f;
#pragma unroll
  for (int z = 0; z < 4; z++) f[z] = __builtin_amdgcn_perm(vq[2 * z + 1][e / 2], vq[2 * z][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
  return f;
}

// Words of 16-bit floats: ones in the halves that are an infinity or a NaN.
template <typename Tv>
__device__ __forceinline__ uint32_t odd_halves(uint32_t x) {
  constexpr bool kB = __is_same(Tv, bf16);
  constexpr uint32_t kExp = kB ? 0x7f807f80u : 0x7c007c00u, kUnit = kB ? 0x00800080u : 0x04000400u;
  return ((((x & kExp) + kUnit) >> 15) & 0x00010001u) * 0xffffu;  // (an exponent of ones runs over into the sign's place)
}

// The softmax state of 16 rows and what a tile of 32 keys does to it.
template <typename T, int CODE, int DP, bool TWO>
struct TreeState {
  using Ty = TreeTypes<T, CODE, DP>;
  using Tv = typename Ty::Tv;
  static constexpr int EB = Ty::EB;
  // The reference is taken this much below the largest score.  f16 weights are subnormal below 2^-14 and
  // zero below 2^-25: with 2^7 for the largest one (and 2^15 where the slack is used up, f16 ends at 2^16)
  // a weight keeps its 11 bits down to 2^-21 of it, and is off by 2^-32 of it at most below that.
  static constexpr float kLift = __is_same(Tv, f16) ? 7.f : 0.f;
  f32x4t o[EB];       // element EB * (4 g + v) + e of row c, unnormalised, against ref
  float ref, top, l;  // reference of the scores (log2 units), this lane's largest and its sum of weights
  uint4v pf, pl;

  __device__ __forceinline__ void start() {
    ref = -3.4e38f;  // (below any score, and not infinite: a masked score less it stays one)
    top = kNegInf;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < EB; e++) o[e] = f32x4t{0.f, 0.f, 0.f, 0.f};
  }
  // s: scores of row c, s[u][v] is key 16 u + 4 g + v, still to be multiplied by `scale`
  // (kf: by key, for codes, along with vf for the values).  live: the keys that count, all if whole.
  __device__ __forceinline__ void weigh(f32x4t (&s)[2], float scale, const float* kf, const float* vf, bool whole, uint32_t live) {
    const int g4 = 4 * (lane_id() >> 4);
    float4v vw[2];
    if constexpr (Ty::kCoded) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const float4v a = *reinterpret_cast<const float4v*>(kf + 16 * u + g4);
        vw[u] = *reinterpret_cast<const float4v*>(vf + 16 * u + g4);
#pragma unroll
        for (int v = 0; v < 4; v++) s[u][v] *= a[v];
      }
    }
    if (!whole) {
      const uint32_t bits = live >> g4;
#pragma unroll
      for (int v = 0; v < 8; v++) {
        const uint32_t on = spread_bit(bits, v);
        const float x = s[v / 4][v % 4];
        s[v / 4][v % 4] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & on) | (0xff800000u & ~on));
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int v = 1; v < 8; v++) mx = fmaxf(mx, s[v / 4][v % 4]);
    // (the largest of this lane's keys; the row's four lanes only meet when one of them calls for it)
    if constexpr (!Ty::kCoded) mx *= scale;
    top = fmaxf(top, mx);
    if (__builtin_amdgcn_ballot_w64(mx > ref + (kTreeSlack + kLift)) != 0) {
      const float now = fmaxf(ref, row_max(mx) - kLift);
      const float alpha = tree_shrink(ref - now);
      ref = now;
      l *= alpha;
#pragma unroll
      for (int e = 0; e < EB; e++)
#pragma unroll
        for (int v = 0; v < 4; v++) o[e][v] *= alpha;
    }
    float sum = 0.f;
#pragma unroll
    for (int x = 0; x < 4; x++) {
      float p[2];
#pragma unroll
      for (int z = 0; z < 2; z++) {
        const int u = x / 2, v = 2 * (x % 2) + z;
        p[z] = __builtin_amdgcn_exp2f(Ty::kCoded ? s[u][v] - ref : __builtin_fmaf(s[u][v], scale, -ref));
        sum += p[z];
        if constexpr (Ty::kCoded) p[z] *= vw[u][v];
      }
      const uint32_t hi = tree_pack<Tv>(p[0], p[1]);
      pf[x] = hi;
      if constexpr (TWO)
        pl[x] = tree_pack<Tv>(p[0] - __builtin_bit_cast(float, hi << 16), p[1] - __builtin_bit_cast(float, hi & 0xffff0000u));
    }
    l += sum;
  }
  __device__ __forceinline__ void add(const uint4v& f, int e) {
    o[e] = tree_mfma<Tv>(f, pf, o[e]);
    if constexpr (TWO) o[e] = tree_mfma<Tv>(f, pl, o[e]);
  }
  // Adds the infinities and NaN among the values, and only those, to the rows that attend their keys:
  // how many of each sign a row has comes from products of ones.
  __device__ __forceinline__ void count_odd(const uint4v& f, int e, uint32_t live) {
    constexpr bool kB = __is_same(Tv, bf16);
    constexpr uint32_t kOne = kB ? 0x3f803f80u : 0x3c003c00u, kMan = kB ? 0x007f007fu : 0x03ff03ffu;
    const uint32_t bits = live >> (4 * (lane_id() >> 4));
    uint4v on;
#pragma unroll
    for (int x = 0; x < 4; x++) {
      const int k = 16 * (x / 2) + 2 * (x % 2);
      on[x] = ((((bits >> k) & 1u) | (((bits >> (k + 1)) & 1u) << 16)) * 0xffffu) & kOne;
    }
#pragma unroll
    for (int sign = 0; sign < 2; sign++) {
      uint4v ind;
#pragma unroll
      for (int x = 0; x < 4; x++) {
        const uint32_t w = f[x];
        const uint32_t nan = ((((w & kMan) + kMan) >> (kB ? 7 : 10)) & 0x00010001u) * 0xffffu;
        const uint32_t minus = ((w >> 15) & 0x00010001u) * 0xffffu;
        ind[x] = odd_halves<Tv>(w) & (nan | (sign ? minus : ~minus)) & kOne;
      }
      const f32x4t n = tree_mfma<Tv>(ind, on, f32x4t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
      for (int v = 0; v < 4; v++) o[e][v] += n[v] > 0.f ? (sign ? kNegInf : -kNegInf) : 0.f;
    }
  }
  // The rows' results into LDS: state (max, sum) and unnormalised elements, `stride` floats a row.
  // (odd: the elements' places hold sums that are added)  False if an element of the lane is not finite.
  __device__ __forceinline__ bool leave(float* acc, float2* state, int row, int stride, bool odd) const {
    const int c = lane_id() & 15, g = lane_id() >> 4;
    const float most = row_max(top);
    const float f = most == kNegInf ? 1.f : __builtin_amdgcn_exp2f(ref - most);
    const float lt = row_sum(l) * f;
    if (g == 0) state[row + c] = float2{most, lt};
    float z = 0.f;
#pragma unroll
    for (int v = 0; v < 4; v++) {
      float* to = acc + (row + c) * stride + EB * (4 * g + v);
#pragma unroll
      for (int e = 0; e < EB; e++) {
        z = __builtin_fmaf(o[e][v], 0.f, z);
        to[e] = odd ? o[e][v] * f + to[e] : o[e][v] * f;
      }
    }
    return z == 0.f;
  }
};

// The workgroup's results of an item, `copies` of M rows in LDS (one per share of the keys), joined and
// written: to `out` where the item is whole, else as a part.  Eight lanes a row.
template <typename T, int DP>
__device__ __forceinline__ void tree_join(const TreeArgs& g, const TreeWalk& it, const float* acc, const float2* state, int copies, int M) {
  constexpr int EB = DP / 32, kStride = DP + 4;  // (EB: pieces of four elements per lane)
  const bool whole = it.whole_item();
  const int64_t slot = it.slot();
  const int sub = threadIdx.x & 7;
  for (int r = threadIdx.x >> 3; r < it.live_rows; r += 32) {
    float mx = kNegInf;
    for (int k = 0; k < copies; k++) mx = fmaxf(mx, state[k * M + r].x);
    float x[EB][4] = {};
    float lt = 0.f;
    for (int k = 0; k < copies; k++) {
      const float2 st = state[k * M + r];
      const float f = st.x == kNegInf ? (st.y == 0.f ? 0.f : 1.f) : tree_shrink(st.x - mx);
      if (f == 0.f) continue;
      lt += f * st.y;
#pragma unroll
      for (int e = 0; e < EB; e++) {
        const float4v y = *reinterpret_cast<const float4v*>(acc + (k * M + r) * kStride + 4 * (8 * e + sub));
#pragma unroll
        for (int u = 0; u < 4; u++) x[e][u] += f * y[u];
      }
    }
    if (whole) {
      const int rr = it.tile0 + r;
      const int nd = (int)fast_div((uint32_t)rr, g.group_magic, g.group_shift), gi = rr - nd * g.group;
      const TreeWeights tw = tree_weights(g, it.sq.row0 + nd, it.head * g.group + gi, mx, lt);
#pragma unroll
      for (int e = 0; e < EB; e++) tree_store<T, 4>(g, it.sq.row0 + nd, it.head * g.group + gi, 4 * (8 * e + sub), tw, x[e]);
      if (sub == 0) tree_store_state(g, it.sq.row0 + nd, it.head * g.group + gi, tw);
    } else {
      if (sub == 0) {
        g.pm[slot * M + r] = mx;
        g.pl[slot * M + r] = lt;
      }
#pragma unroll
      for (int e = 0; e < EB; e++)
        *reinterpret_cast<float4v*>(g.pacc + (slot * M + r) * DP + 4 * (8 * e + sub)) = float4v{x[e][0], x[e][1], x[e][2], x[e][3]};
    }
  }
}

// Waits until at most N of the loads issued so far are on their way.
template <int N>
__device__ __forceinline__ void wait_loads() {
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70);
}

// 16 NR rows per item (plain decoding, small trees): the wavefronts deal an item's keys among themselves,
// tile by tile, and run apart until its end.  Bound by the reads of K and V where the rows are few: 64 e4m3
// sequences of up to 8191 tokens, 8 heads of 128, 133 us (5.2 TB/s of the 6.0 to 6.4 that plain reads reach);
// 2 of up to 200001 bf16 tokens 225 us (5.6 TB/s).  With 70 to 90 rows over int8 (16 sequences of up to 12345)
// the softmax and the decoding of codes bound it, 82 us; 32-row tiles there instead of 16 halve the decoding.
// Registers end at two wavefronts per SIMD: 32-row tiles of 128 plain elements spill 17 to 20 of them, 8-bit ones
// of 256 2 to 30.
template <int DP, int NR>
struct NarrowLds {
  static constexpr int kRows = 16 * NR * kTreeWaves, kStride = DP + 4;
  static constexpr int kWaveBytes = 64 * 8 + 2 * 32 * 4;  // a wavefront's row places and scales
  static constexpr int kBytes = kRows * kStride * 4 + kRows * 8 + kTreeWaves * kWaveBytes;
};
// Workgroups per CU: what keeps about 64 KiB of keys and values on the way (more only gets in its own
// way: 2 x 200001 bf16 tokens of 128 elements 225 us with one, 240 with two), as registers allow.
constexpr int narrow_groups(int code, int dp) { return code == SPFA_CODE_NONE ? (dp == 64 ? 2 : 1) : dp == 64 ? 3 : dp == 128 ? 2 : 1; }
constexpr int narrow_waves(int code, int dp, int nr) {
  return narrow_groups(code, dp) == 3 && nr == 1 ? 3 : dp == 256 && code == SPFA_CODE_NONE ? 1 : 2;
}
template <typename T, int CODE, int DP, int NR, int ROWS>
__global__ __launch_bounds__(256, narrow_waves(CODE, DP, NR)) void tree_narrow_kernel(TreeArgs a) {
  using Ty = TreeTypes<T, CODE, DP>;
  using Lds = NarrowLds<DP, NR>;
  constexpr int EB = Ty::EB, M = 16 * NR;
  extern __shared__ __align__(16) char lds[];
  float* acc_lds = reinterpret_cast<float*>(lds);
  float2* state_lds = reinterpret_cast<float2*>(acc_lds + Lds::kRows * Lds::kStride);
  const int wave = uniform(threadIdx.x >> 6);
  char* mine = lds + Lds::kRows * Lds::kStride * 4 + Lds::kRows * 8 + wave * Lds::kWaveBytes;
  float* ks_lds = reinterpret_cast<float*>(mine + 64 * 8);
  float* vs_lds = ks_lds + 32;

  TreeWalk it;
  const bool any = it.start(a, M);
  if (threadIdx.x == 0) a.part[it.w].seq = -1;
  if (!any) return;
  const float scale = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, a.scale_log2)));
  // Tiles that every row attends are not looked through for infinities and NaN among the values.  Such a
  // value shows in the results (as NaN, times a weight that is zero or whose second part is not above zero),
  // and the wavefront works on its tiles once more, now screening all of them.
  bool screened = false;
  while (it.item(a, M)) {
    const int t_all = (it.sq.len + 31) / 32, t_end = it.blk1 * 4 < t_all ? it.blk1 * 4 : t_all;
    int t = it.blk0 * 4 + wave;
    TreeKeys<T, CODE, DP, ROWS> keys;
    TreeQueries<T, CODE, DP, ROWS> q[NR];
    TreeState<T, CODE, DP, Ty::kTwo> st[NR];
    keys.start(a, it, t_end, reinterpret_cast<int64_t*>(mine));
#pragma unroll
    for (int n = 0; n < NR; n++) st[n].start();
    // K and V of a tile are asked for while the tile before is worked on, each as soon as its registers
    // are free, and the page numbers one tile ahead of that.  After the last tile the same one is asked
    // for again: a branch around the loads would make the compiler wait for all of them where its ways
    // meet, and loads of any one place instead would make all workgroups meet there.
    const int t_last = t < t_end ? t + (t_end - 1 - t) / kTreeWaves * kTreeWaves : 0;
    uint32_t exist_next = 0;
    bool odd = false;
    if (t < t_end) {
      keys.look_up(t);
#pragma unroll
      for (int n = 0; n < NR; n++) q[n].load(a, it, 16 * n);
      exist_next = keys.locate();
      keys.look_up(t + kTreeWaves < t_end ? t + kTreeWaves : t_last);
      keys.load_k(a.d);
      keys.load_v(a.d);
      // the queries are here, the others on their way (the loop below need not wait for queries)
      wait_loads<2 * Ty::NK + 8 * (Ty::VW > 4 ? 2 : 1) + 1>();
#pragma unroll
      for (int n = 0; n < NR; n++) q[n].flip(a.flip);
    }
    const int t_full = screened ? 0 : it.sq.ctx / 32;  // tiles below lie before the tree
    for (; t < t_end; t += kTreeWaves) {
      const uint32_t exist = exist_next;
      const bool whole = exist == 0xffffffffu && t < t_full;  // every row attends all 32 keys
      uint32_t live[NR];
#pragma unroll
      for (int n = 0; n < NR; n++) live[n] = 0xffffffffu;
      if (!whole) {
#pragma unroll
        for (int n = 0; n < NR; n++) live[n] = q[n].live(a, t * 32 - it.sq.ctx, exist);
        keys.template screen<NR>(exist, live, acc_lds + wave * M * Lds::kStride, Lds::kStride, odd);
      }
      if constexpr (Ty::kCoded) {
        ks_lds[lane_id() & 31] = keys.ks * scale;
        vs_lds[lane_id() & 31] = keys.vs;
        wave_sync();
      }
      exist_next = keys.locate();
      keys.look_up(t + 2 * kTreeWaves < t_end ? t + 2 * kTreeWaves : t_last);
      f32x4t s[NR][2] = {};
#pragma unroll
      for (int x = 0; x < Ty::QF; x++)
#pragma unroll
        for (int u = 0; u < 2; u++) {
          const uint4v f = keys.key_frag(u, x);
#pragma unroll
          for (int n = 0; n < NR; n++) s[n][u] = tree_mfma<T>(f, q[n].f[x], s[n][u]);
        }
      keys.load_k(a.d);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < NR; n++) st[n].weigh(s[n], scale, ks_lds, vs_lds, whole, live[n]);
#pragma unroll
      for (int w = 0; w < EB / 4; w++) {
        uint32_t vq[8][2];
        keys.values(w, vq);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const uint4v f = value_frag(vq, e);
#pragma unroll
          for (int n = 0; n < NR; n++) st[n].add(f, 4 * w + e);
        }
      }
      keys.load_v(a.d);
    }
    bool fine = true;
#pragma unroll
    for (int n = 0; n < NR; n++) fine &= st[n].leave(acc_lds, state_lds, wave * M + 16 * n, Lds::kStride, odd);
    if (__builtin_expect(!screened && __builtin_amdgcn_ballot_w64(!fine) != 0, 0)) {
      screened = true;
      continue;  // (the same item)
    }
    screened = false;
    __syncthreads();
    tree_join<T, DP>(a, it, acc_lds, state_lds, kTreeWaves, M);
    __syncthreads();  // (all of it has been read: the next item may use the LDS)
    if (threadIdx.x == 0) it.name_part(a);
    it.next();
  }
}

// More rows per item: the workgroup's wavefronts share the keys.  Each brings 32 of a block's 128 keys
// into LDS in the form the products take them (so looking up, decoding and reordering is done once for
// all rows), then works on its own 32 rows.  One buffer: while a workgroup refills it, the CU's other one
// computes.  Bound by the softmax's vector instructions (exponentials, packing, maxima): 6 sequences of up
// to 5000 tokens, 488 rows for each of 8 f16 heads of 64, 56 us and the merge 9 us; 8 of up to 20000, 512 rows for
// each of 4, 114 us (430 TFLOP/s), bf16 138, bf16 heads of 128 288 us (340 TFLOP/s).  Heads of 64 have registers
// enough; with 128 elements 56 to 157 of them spill, with 256 170 to 584, which those sizes pay for.
template <int DP>
struct WideLds {
  static constexpr int kRows = 32 * kTreeWaves;
  static constexpr int kFrags = 2 * (DP / 32) + DP / 16;  // of 1024 bytes, per 32 keys
  static constexpr int kStride = DP + 4;
  static constexpr int kJoin = kRows * kStride * 4;
  static constexpr int kShared = kTreeWaves * kFrags * 1024 > kJoin ? kTreeWaves * kFrags * 1024 : kJoin;
  static constexpr int kState = kRows * 8;
  static constexpr int kTile = 64 * 8 + 2 * 32 * 4 + 16;  // places, scales, existing keys, whether values and results are odd
  static constexpr int kBytes = kShared + kState + kTreeWaves * kTile;
};
constexpr int wide_groups(int dp) { return dp == 256 ? 1 : 2; }  // workgroups per CU
template <typename T, int CODE, int DP, int ROWS>
__global__ __launch_bounds__(256, wide_groups(DP)) void tree_wide_kernel(TreeArgs a) {
  using Ty = TreeTypes<T, CODE, DP>;
  using Lds = WideLds<DP>;
  using Tv = typename Ty::Tv;
  constexpr int EB = Ty::EB, NR = 2, M = Lds::kRows;
  extern __shared__ __align__(16) char lds[];
  uint4v* frags = reinterpret_cast<uint4v*>(lds);
  float* acc_lds = reinterpret_cast<float*>(lds);
  float2* state_lds = reinterpret_cast<float2*>(lds + Lds::kShared);
  char* tiles = lds + Lds::kShared + Lds::kState;
  const int wave = uniform(threadIdx.x >> 6), lane = lane_id();
  char* mine = tiles + wave * Lds::kTile;
  float* ks_mine = reinterpret_cast<float*>(mine + 64 * 8);
  uint32_t* word_mine = reinterpret_cast<uint32_t*>(mine + 64 * 8 + 2 * 32 * 4);

  TreeWalk it;
  const bool any = it.start(a, M);
  if (threadIdx.x == 0) a.part[it.w].seq = -1;
  if (!any) return;
  const float scale = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, a.scale_log2)));
  bool screened = false;  // (as in the narrow kernel, the whole workgroup together)
  while (it.item(a, M)) {
    const int t_all = (it.sq.len + 31) / 32, t_end = it.blk1 * 4 < t_all ? it.blk1 * 4 : t_all;
    int t = it.blk0 * 4;  // first tile of the block
    TreeKeys<T, CODE, DP, ROWS> keys;
    TreeQueries<T, CODE, DP, ROWS> q[NR];
    TreeState<T, CODE, DP, Ty::kTwo> st[NR];
    keys.start(a, it, t_end, reinterpret_cast<int64_t*>(mine));
#pragma unroll
    for (int n = 0; n < NR; n++) st[n].start();
    // (a wavefront without a tile in the last block asks for the last tile's keys; a tile past the end
    // has no existing keys)
    auto tile_of = [&](int first) { return first + wave < t_end ? first + wave : t_end - 1; };
    uint32_t exist_next = 0;
    if (t < t_end) {
      keys.look_up(tile_of(t));
#pragma unroll
      for (int n = 0; n < NR; n++) q[n].load(a, it, 16 * (wave * NR + n));
      exist_next = keys.locate();
      keys.look_up(tile_of(t + kTreeWaves));
      keys.load_k(a.d);
      keys.load_v(a.d);
      wait_loads<2 * Ty::NK + 8 * (Ty::VW > 4 ? 2 : 1) + 1>();
#pragma unroll
      for (int n = 0; n < NR; n++) q[n].flip(a.flip);
    }
    const int t_full = screened ? 0 : it.sq.ctx / 32;  // tiles below lie before the tree
    for (; t < t_end; t += kTreeWaves) {
      // ---- this wavefront's tile into LDS ----
      const int tt = t + wave;
      const uint32_t exist = tt < t_end ? exist_next : 0u;
      float vs = keys.vs;
      uint32_t sick = 0;  // keys whose V scale is no finite number: it goes into the values
      if constexpr (Ty::kCoded) {
        const bool there = (exist >> (lane & 31)) & 1, bad = there && !(fabsf(vs) <= 3.402823466e38f);
        sick = (uint32_t)__builtin_amdgcn_ballot_w64(bad);
        ks_mine[lane & 31] = there ? keys.ks * scale : 0.f;
        ks_mine[32 + (lane & 31)] = !there ? 0.f : bad ? 1.f : vs;
      }
      if (exist != 0xffffffffu) {
        // values of keys that do not exist become zeros
        const uint32_t eg = exist >> (4 * (lane >> 4));
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
          for (int y = 0; y < Ty::VW; y++) keys.vr[k][y] &= spread_bit(eg, k);
      }
      uint4v* to = frags + (wave * Lds::kFrags) * 64 + lane;
      // (clean: infinities and NaN become zeros; whether there are any)
      auto stage_values = [&](auto clean) {
        uint32_t odd = 0;
#pragma unroll
        for (int w = 0; w < EB / 4; w++) {
          uint32_t vq[8][2];
          keys.values(w, vq);
          if (Ty::kCoded && sick != 0) {
#pragma unroll
            for (int k = 0; k < 8; k++) {
              const int key = 16 * (k / 4) + k % 4 + 4 * (lane >> 4);
              const float f = shfl_f32(vs, key);
              if ((sick >> key) & 1) {
#pragma unroll
                for (int y = 0; y < 2; y++)
                  vq[k][y] = tree_pack<Tv>(__builtin_bit_cast(float, vq[k][y] << 16) * f, __builtin_bit_cast(float, vq[k][y] & 0xffff0000u) * f);
              }
            }
          }
          if constexpr (decltype(clean)::value != 0) {
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
              for (int y = 0; y < 2; y++) {
                const uint32_t is = odd_halves<Tv>(vq[k][y]);
                odd |= is;
                if constexpr (decltype(clean)::value == 2) vq[k][y] &= ~is;
              }
          }
#pragma unroll
          for (int e = 0; e < 4; e++) to[(2 * Ty::QF + 4 * w + e) * 64] = value_frag(vq, e);
        }
        return odd;
      };
      if (t + kTreeWaves > t_full) {
        // Tiles that some rows do not attend as a whole: their infinities and NaN must reach the rows that
        // attend their keys and no other row, which 0 * infinity would not do.  They are counted apart
        // and are zeros in the products that follow.
        const uint32_t odd = stage_values(std::integral_constant<int, 1>{});
        word_mine[0] = exist;
        word_mine[1] = __builtin_amdgcn_ballot_w64(odd != 0) != 0;
        __syncthreads();
        for (int j = 0; j < kTreeWaves; j++) {
          const uint32_t* info = reinterpret_cast<const uint32_t*>(tiles + j * Lds::kTile + 64 * 8 + 2 * 32 * 4);
          if (uniform((int)info[1]) == 0) continue;
          const uint32_t ex = (uint32_t)uniform((int)info[0]);
#pragma unroll
          for (int n = 0; n < NR; n++) {
            const uint32_t live = q[n].live(a, (t + j) * 32 - it.sq.ctx, ex);
#pragma unroll
            for (int e = 0; e < EB; e++) {
              __builtin_amdgcn_sched_barrier(0);
              st[n].count_odd(frags[(j * Lds::kFrags + 2 * Ty::QF + e) * 64 + lane], e, live);
            }
          }
        }
        __syncthreads();
        stage_values(std::integral_constant<int, 2>{});
      } else {
        stage_values(std::integral_constant<int, 0>{});
      }
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int x = 0; x < Ty::QF; x++) to[(2 * x + u) * 64] = keys.key_frag(u, x);
      word_mine[0] = exist;
      __syncthreads();
      // ---- the next block is asked for; all of this one's keys for this wavefront's rows ----
      exist_next = keys.locate();
      keys.look_up(tile_of(t + 2 * kTreeWaves));
      keys.load_k(a.d);
      keys.load_v(a.d);
      // Factors come four at a time, asked for well before they are needed: with two wavefronts per SIMD
      // nothing else hides the way through LDS.
      const int j_end = kTreeWaves < t_end - t ? kTreeWaves : t_end - t;
      uint4v kf[4], vf[4];
      auto read4 = [&](int j, int first, uint4v(&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = frags[(j * Lds::kFrags + first + i) * 64 + lane];
      };
      read4(0, 0, kf);
      for (int j = 0; j < j_end; j++) {
        const char* info = tiles + j * Lds::kTile + 64 * 8;
        const uint32_t ex = (uint32_t)uniform((int)*reinterpret_cast<const uint32_t*>(info + 256));
        const bool whole = ex == 0xffffffffu && t + j < t_full;
        f32x4t s[NR][2] = {};
#pragma unroll
        for (int x = 0; x < Ty::QF; x += 2) {
          uint4v now[4];
#pragma unroll
          for (int i = 0; i < 4; i++) now[i] = kf[i];
          if (x + 2 < Ty::QF) read4(j, 2 * (x + 2), kf);
          else read4(j, 2 * Ty::QF, vf);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < NR; n++) s[n][i % 2] = tree_mfma<T>(now[i], q[n].f[x + i / 2], s[n][i % 2]);
          __builtin_amdgcn_sched_barrier(0);
        }
        // (the next tile's first ones; behind the last tile any will do)
        read4(j + 1 < j_end ? j + 1 : j, 0, kf);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NR; n++) {
          uint32_t live = 0xffffffffu;
          if (!whole) live = q[n].live(a, (t + j) * 32 - it.sq.ctx, ex);
          st[n].weigh(s[n], scale, reinterpret_cast<const float*>(info), reinterpret_cast<const float*>(info) + 32, whole, live);
        }
#pragma unroll
        for (int e = 0; e < EB; e += 4) {
          uint4v now[4];
#pragma unroll
          for (int i = 0; i < 4; i++) now[i] = vf[i];
          if (e + 4 < EB) {
            read4(j, 2 * Ty::QF + e + 4, vf);
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < NR; n++) st[n].add(now[i], e + i);
        }
      }
      __syncthreads();
    }
    bool fine = true;
#pragma unroll
    for (int n = 0; n < NR; n++) fine &= st[n].leave(acc_lds, state_lds, 16 * (wave * NR + n), Lds::kStride, false);
    word_mine[2] = __builtin_amdgcn_ballot_w64(!fine) != 0;
    __syncthreads();
    uint32_t bad = 0;
#pragma unroll
    for (int j = 0; j < kTreeWaves; j++) bad |= reinterpret_cast<const uint32_t*>(tiles + j * Lds::kTile + 64 * 8 + 2 * 32 * 4)[2];
    screened = !screened && uniform((int)bad) != 0;
    if (screened) continue;
    tree_join<T, DP>(a, it, acc_lds, state_lds, 1, M);
    __syncthreads();  // (all of it has been read: the next item may use the LDS)
    if (threadIdx.x == 0) it.name_part(a);
    it.next();
  }
}

// Joins the parts of the items that were cut: workgroup (w, y) takes rows of the item whose last part
// workgroup w had.  DP / 4 lanes hold a row's elements; where an item has many parts, S such groups of the
// workgroup share a row's parts and meet in LDS, so that few rows do not wait for long chains of loads (a
// group has kMergeBatch parts on the way at a time).
constexpr int kMergeBatch = 8;
// (CODE only keeps the object files' copies apart.)
template <typename T, int CODE, int DP>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs g, int M) {
  constexpr int kLanes = DP / 4, kGroups = 256 / kLanes;
  __shared__ __align__(16) float4v acc[kGroups][kLanes];
  __shared__ float2 state[kGroups];
  const int w = blockIdx.x;
  const TreePart part = g.part[w];
  if (part.seq < 0) return;
  const TreeSeq sq = tree_seq(g, part.seq, M);
  const int tile0 = part.tile * M, n_rows = sq.n * g.group;
  const int live_rows = n_rows - tile0 < M ? n_rows - tile0 : M;
  const int grp = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int parts = w - part.first + 1;
  const int share = parts <= kMergeBatch ? 1 : parts <= 2 * kMergeBatch ? 2 : parts <= 4 * kMergeBatch ? 4 : 8;
  const int S = share < kGroups ? share : kGroups, per = kGroups / S, sub = grp % S;
  for (int r0 = blockIdx.y * per; r0 < live_rows; r0 += gridDim.y * per) {
    const int r = r0 + grp / S;
    float m = kNegInf, l = 0.f;
    float4v x = {0.f, 0.f, 0.f, 0.f};
    auto join = [&](float m2, float l2, const float4v& x2) {
      const float mn = fmaxf(m, m2);
      const float a = m == kNegInf ? 1.f : tree_shrink(m - mn);
      const float b = m2 == kNegInf ? 1.f : tree_shrink(m2 - mn);
      m = mn;
      l = l * a + l2 * b;
#pragma unroll
      for (int e = 0; e < 4; e++) x[e] = x[e] * a + x2[e] * b;
    };
    if (r < live_rows) {
      for (int p0 = part.first + sub; p0 <= w; p0 += S * kMergeBatch) {
        float pm[kMergeBatch], pl[kMergeBatch];
        float4v px[kMergeBatch];
#pragma unroll
        for (int u = 0; u < kMergeBatch; u++) {
          const int p = p0 + S * u <= w ? p0 + S * u : w;
          const int64_t at = (p == part.first ? 2 * (int64_t)p + 1 : 2 * (int64_t)p) * M + r;
          pm[u] = g.pm[at];
          pl[u] = g.pl[at];
          px[u] = *reinterpret_cast<const float4v*>(g.pacc + at * DP + 4 * c);
        }
#pragma unroll
        for (int u = 0; u < kMergeBatch; u++)
          if (p0 + S * u <= w && pl[u] != 0.f) join(pm[u], pl[u], px[u]);  // (0: nothing attended there)
      }
    }
    if (S > 1) {
      __syncthreads();
      if (c == 0) state[grp] = float2{m, l};
      acc[grp][c] = x;
      __syncthreads();
      if (sub == 0)
        for (int k = grp + 1; k < grp + S; k++)
          if (state[k].y != 0.f) join(state[k].x, state[k].y, acc[k][c]);
    }
    if (sub == 0 && r < live_rows) {
      const int rr = tile0 + r;
      const int nd = (int)fast_div((uint32_t)rr, g.group_magic, g.group_shift), gi = rr - nd * g.group;
      const TreeWeights tw = tree_weights(g, sq.row0 + nd, part.head * g.group + gi, m, l);
      const float y[4] = {x[0], x[1], x[2], x[3]};
      tree_store<T, 4>(g, sq.row0 + nd, part.head * g.group + gi, 4 * c, tw, y);
      if (c == 0) tree_store_state(g, sq.row0 + nd, part.head * g.group + gi, tw);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------

// Which kernel a call takes.
struct TreeShape {
  int rows_how;    // kTreeAny, ...
  int dp;          // padded head size
  int nr;          // 16-row blocks of a wavefront
  bool wide;       // the wide kernel
  int merge_rows;  // workgroups per part in the merge, 0: no item can be cut
  int rows() const { return wide ? WideLds<64>::kRows : 16 * nr; }  // of an item
};

// One element type and code per object file.
template <typename T, int CODE>
int tree_run(const TreeArgs& a, const TreeShape& s, hipStream_t stream);

#ifdef SPFA_TREE_CODE
template <typename T, int CODE, int DP, int NR, int ROWS>
int tree_launch(const TreeArgs& a, int merge_rows, hipStream_t stream) {
  constexpr int kLds = NarrowLds<DP, NR>::kBytes;
  if constexpr (kLds > 65536) {
    static std::atomic<bool> raised[kLdsLimitDevices];
    if (!raise_lds_limit(reinterpret_cast<const void*>(&tree_narrow_kernel<T, CODE, DP, NR, ROWS>), kLds, raised))
      return SPFA_ERR_LAUNCH;
  }
  tree_narrow_kernel<T, CODE, DP, NR, ROWS><<<dim3((unsigned)a.workers), dim3(256), kLds, stream>>>(a);
  if (merge_rows > 0)
    tree_merge_kernel<T, CODE, DP><<<dim3((unsigned)a.workers, (unsigned)merge_rows), dim3(256), 0, stream>>>(a, 16 * NR);
  return launch_status();
}

template <typename T, int CODE, int DP, int ROWS>
int tree_launch_wide(const TreeArgs& a, int merge_rows, hipStream_t stream) {
  constexpr int kLds = WideLds<DP>::kBytes;
  if constexpr (kLds > 65536) {
    static std::atomic<bool> raised[kLdsLimitDevices];
    if (!raise_lds_limit(reinterpret_cast<const void*>(&tree_wide_kernel<T, CODE, DP, ROWS>), kLds, raised))
      return SPFA_ERR_LAUNCH;
  }
  tree_wide_kernel<T, CODE, DP, ROWS><<<dim3((unsigned)a.workers), dim3(256), kLds, stream>>>(a);
  if (merge_rows > 0)
    tree_merge_kernel<T, CODE, DP><<<dim3((unsigned)a.workers, (unsigned)merge_rows), dim3(256), 0, stream>>>(a, WideLds<DP>::kRows);
  return launch_status();
}

template <typename T, int CODE, int DP, int ROWS>
int tree_launch_shape(const TreeArgs& a, const TreeShape& s, hipStream_t stream) {
  if (s.wide) return tree_launch_wide<T, CODE, DP, ROWS>(a, s.merge_rows, stream);
  if constexpr (DP <= 128)
    if (s.nr == 2) return tree_launch<T, CODE, DP, 2, ROWS>(a, s.merge_rows, stream);
  return tree_launch<T, CODE, DP, 1, ROWS>(a, s.merge_rows, stream);
}

template <typename T, int CODE, int DP>
int tree_launch_rows(const TreeArgs& a, const TreeShape& s, hipStream_t stream) {
  if (s.rows_how == kTreeAny) return tree_launch<T, CODE, DP, 1, kTreeAny>(a, s.merge_rows, stream);
  if (s.rows_how == kTreePadded) return tree_launch_shape<T, CODE, DP, kTreePadded>(a, s, stream);
  return tree_launch_shape<T, CODE, DP, kTreeWhole>(a, s, stream);
}

template <>
int tree_run<SPFA_TREE_T, SPFA_TREE_CODE>(const TreeArgs& a, const TreeShape& s, hipStream_t stream) {
  if (s.dp == 64) return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 64>(a, s, stream);
  if (s.dp == 128) return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 128>(a, s, stream);
  return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 256>(a, s, stream);
}
#endif

}  // namespace spfa
