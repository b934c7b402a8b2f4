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
// A wavefront works on 32 keys at a time for RB * 32 rows, all in registers:
//   S^T = K Q^T    A = K: lane (c, h) holds 16-byte pieces of the row of key c, straight from memory;
//                  which elements stand for which of the product's 16 is free as long as Q's agree
//   softmax        a lane owns row c: 16 keys of its own, 16 of the lane of the other half
//   O^T += V^T P^T P^T is S^T's own layout (the order of the keys is free too), V^T: lane (c, h) has
//                  elements EB * c .. + EB - 1 of the 16 keys of its half, so one load instruction
//                  takes two whole rows; pairs of keys are put side by side by byte permutes
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

typedef float f32x16t __attribute__((ext_vector_type(16)));
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
  int64_t k_page, k_slot, k_head, v_page, v_slot, v_head;
  int64_t ks_page, ks_slot, ks_head, vs_page, vs_slot, vs_head;
  const int32_t* q_offsets;
  const int32_t* ctx_lens;
  const int32_t* page_table;
  int64_t table_width, table_stride;
  const uint64_t* mask;
  int64_t mask_words;
  int64_t rows, pages;
  int32_t heads, group, n_seqs, d, page_size;
  int32_t max_len;  // positions the page table covers, cut to 32 bits
  float scale_log2;
  int32_t workers, wave_rows;
  int32_t out_vec;  // rows of out can be written four elements at a time
  TreePart* part;
  float* pm;  // [2 * workers, M]
  float* pl;
  float* pacc;  // [2 * workers, M, DP]
};

struct TreeSeq {
  int row0, n, ctx, len;
  int64_t tiles;
  int nblk;
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
  q.tiles = ((int64_t)q.n * g.group + M - 1) / M;
  q.nblk = q.len <= kTreeBlock ? 1 : (q.len + kTreeBlock - 1) / kTreeBlock;
  return q;
}
__device__ __forceinline__ int64_t tree_units(const TreeArgs& g, const TreeSeq& q) { return q.tiles * g.heads * q.nblk; }

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
// larger / sum of a value and that of the lane of the other half
__device__ __forceinline__ float half_max(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t a = r[0], b = r[1];
  return __builtin_bit_cast(float, a) + __builtin_bit_cast(float, b);
}

template <typename T>
__device__ __forceinline__ f32x16t tree_mfma(const uint4v& a, const uint4v& b, f32x16t c) {
  if constexpr (__is_same(T, bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8t, a), __builtin_bit_cast(bf16x8t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8t, a), __builtin_bit_cast(f16x8t, b), c, 0, 0, 0);
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

// what a wavefront's lanes wrote to LDS is there for its other lanes
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <int DP, int RB>
struct TreeShape {
  static constexpr int kRows = kTreeWaves * 32 * RB;  // rows of all wavefronts
  static constexpr int kStride = DP + 4;              // floats of a row in LDS
  static constexpr int kAccFloats = kRows * kStride;
  static constexpr int kStateFloats = kRows * 2;
  static constexpr int kWaveBytes = 32 * 8 + 2 * 32 * 4;  // a wavefront's row offsets and scales
  static constexpr int kLds = (kAccFloats + kStateFloats) * 4 + kTreeWaves * kWaveBytes;
};

// How rows are loaded: element by element, in whole pieces where d is less than DP, or d == DP.
enum { kTreeAny = 0, kTreePadded = 1, kTreeWhole = 2 };

template <typename T, int CODE, int DP, int RB, int ROWS>
__global__ __launch_bounds__(256, (DP * RB <= 128 ? 2 : 1)) void tree_kernel(TreeArgs g) {
  using Sh = TreeShape<DP, RB>;
  constexpr int EB = DP / 32;                                // blocks of 32 elements, elements per lane of V
  constexpr int ES = CODE == SPFA_CODE_NONE ? 2 : 1;         // bytes of an element in the cache
  constexpr int NK = DP * ES / 32;                           // 16-byte pieces of a K row per lane
  constexpr int PE = 16 / ES;                                // elements of one
  constexpr int VB = EB * ES;                                // bytes of a V row per lane
  constexpr int VW = VB >= 4 ? VB / 4 : 1;
  using Tv = std::conditional_t<CODE == SPFA_CODE_NONE, T, bf16>;  // (8-bit values times any scale need bf16's range)
  constexpr bool kTwoParts = CODE != SPFA_CODE_NONE && __is_same(T, f16);  // weights of f16 calls in two bf16 parts

  extern __shared__ __align__(16) char lds[];
  float* acc_lds = reinterpret_cast<float*>(lds);
  float2* state_lds = reinterpret_cast<float2*>(acc_lds + Sh::kAccFloats);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = uniform(tid >> 6);
  char* mine = lds + (Sh::kAccFloats + Sh::kStateFloats) * 4 + wave * Sh::kWaveBytes;
  int64_t* voff_lds = reinterpret_cast<int64_t*>(mine);
  float* ks_lds = reinterpret_cast<float*>(mine + 32 * 8);
  float* vs_lds = ks_lds + 32;

  const int WR = g.wave_rows, WK = kTreeWaves / WR;
  const int wr = wave % WR, wk = wave / WR;
  const int M = 32 * RB * WR;

  // workgroups of one XCD (dealt in turn) take neighbouring runs
  int w = blockIdx.x;
  if (g.workers % 8 == 0) w = (w % 8) * (g.workers / 8) + w / 8;

  // the line of all items' blocks, and this workgroup's run of it
  int64_t total = 0;
  for (int base = 0; base < g.n_seqs; base += kWave) {
    int64_t u = 0;
    if (base + lane < g.n_seqs) u = tree_units(g, tree_seq(g, base + lane, M));
    total += uniform64(shfl_i64(wave_scan_i64(u), 63));
  }
  const int64_t per = total / g.workers, extra = total - per * g.workers;
  int64_t pos = w * per + (w < extra ? w : extra);
  const int64_t end = pos + per + (w < extra ? 1 : 0);
  if (tid == 0) g.part[w].seq = -1;
  if (pos >= end) return;

  int seq = 0;
  int64_t in_seq = 0;  // units before `pos` in its sequence
  {
    int64_t before = 0;
    for (int base = 0; base < g.n_seqs; base += kWave) {
      int64_t u = 0;
      if (base + lane < g.n_seqs) u = tree_units(g, tree_seq(g, base + lane, M));
      const int64_t incl = wave_scan_i64(u) + before;
      const uint64_t past = __builtin_amdgcn_ballot_w64(incl > pos);
      if (past) {
        const int at = (int)__builtin_ctzll(past);
        seq = base + at;
        in_seq = pos - uniform64(shfl_i64(incl - u, at));
        break;
      }
      before = uniform64(shfl_i64(incl, 63));
    }
  }
  TreeSeq sq = tree_seq(g, seq, M);

  while (pos < end) {
    while (in_seq >= tree_units(g, sq)) {  // (the next sequence with any rows; there is one, pos < end <= total)
      in_seq = 0;
      if (++seq >= g.n_seqs) return;  // (only if the arrays change under the call)
      sq = tree_seq(g, seq, M);
    }
    const int64_t item = in_seq / sq.nblk;
    const int blk0 = uniform((int)(in_seq - item * sq.nblk));
    const int tile = uniform((int)(item / g.heads)), head = uniform((int)(item - (int64_t)tile * g.heads));
    const int blk1 = uniform((int)(end - pos < sq.nblk - blk0 ? blk0 + (end - pos) : sq.nblk));
    const int64_t n_rows = (int64_t)sq.n * g.group;
    const int64_t tile0 = (int64_t)tile * M;
    const int live_rows = (int)(n_rows - tile0 < M ? n_rows - tile0 : M);

    // ---- queries -------------------------------------------------------------------------------
    uint4v qf[RB][DP / 16];
    int node[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const int r = (wr * RB + rb) * 32 + c;
      // (lanes without a row work on the tile's last one; what they get is not written)
      const int64_t rr = tile0 + (r < live_rows ? r : live_rows - 1);
      node[rb] = (int)(rr / g.group);
      const int gi = (int)(rr - (int64_t)node[rb] * g.group);
      const T* qp = (const T*)g.q + (int64_t)(sq.row0 + node[rb]) * g.qs_row + (int64_t)(head * g.group + gi) * g.qs_head;
#pragma unroll
      for (int s = 0; s < DP / 16; s++) {
        const int e0 = ES == 2 ? 8 * (2 * s + h) : 16 * (2 * (s / 2) + h) + 8 * (s % 2);
        qf[rb][s] = uint4v{0u, 0u, 0u, 0u};
        if (ROWS != kTreeAny) {
          if (ROWS == kTreeWhole || e0 < g.d) qf[rb][s] = *reinterpret_cast<const uint4v*>(qp + e0);
        } else {
#pragma unroll
          for (int i = 0; i < 8; i++)
            if (e0 + i < g.d) qf[rb][s][i / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, qp[e0 + i]) << (16 * (i % 2));
        }
      }
    }

    f32x16t o[RB][EB];
    float m_ref[RB], m_top[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      m_ref[rb] = m_top[rb] = kNegInf;
      l[rb] = 0.f;
#pragma unroll
      for (int e = 0; e < EB; e++)
#pragma unroll
        for (int v = 0; v < 16; v++) o[rb][e][v] = 0.f;
    }

    // ---- keys, 32 at a time ----------------------------------------------------------------------
    const int32_t* table = g.page_table + (int64_t)seq * g.table_stride;
    const int t_end = blk1 * 4 < (sq.len + 31) / 32 ? blk1 * 4 : (sq.len + 31) / 32;
    int t = blk0 * 4 + wk;

    uint4v kr[NK];
    uint32_t vr[16][VW];
    float ksr = 0.f, vsr = 0.f;

    // the page of this lane's key of a tile (both halves hold key c)
    auto page_of = [&](int tt) {
      const int p = tt * 32 + c;
      return p < sq.len ? table[(uint32_t)p / (uint32_t)g.page_size] : -1;
    };
    int64_t koff = 0;
    // where the rows of a tile are (of keys that do not exist: the cache's first row, which does when
    // there are tiles at all); returns the bits of the keys that exist
    auto locate = [&](int tt, int page) {
      const uint32_t p = (uint32_t)(tt * 32 + c);
      const bool ok = p < (uint32_t)sq.len && page >= 0 && page < g.pages;
      const int64_t pg = ok ? page : 0, at = ok ? p % (uint32_t)g.page_size : 0;
      koff = pg * g.k_page + at * g.k_slot + head * g.k_head;
      const int64_t voff = pg * g.v_page + at * g.v_slot + head * g.v_head;
      const uint32_t vb = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
      if (h == 0) voff_lds[c] = voff;
      if constexpr (CODE != SPFA_CODE_NONE) {
        ksr = g.ks[pg * g.ks_page + at * g.ks_slot + head * g.ks_head];
        vsr = g.vs[pg * g.vs_page + at * g.vs_slot + head * g.vs_head];
      }
      wave_sync();
      return vb;
    };
    auto load_k = [&]() {
      const char* p = g.k + koff * ES;
#pragma unroll
      for (int s = 0; s < NK; s++) {
        const int e0 = PE * (2 * s + h);
        kr[s] = uint4v{0u, 0u, 0u, 0u};
        if (ROWS != kTreeAny) {
          if (ROWS == kTreeWhole || e0 < g.d) kr[s] = *reinterpret_cast<const uint4v*>(p + e0 * ES);
        } else {
#pragma unroll
          for (int i = 0; i < PE; i++)
            if (e0 + i < g.d) {
              const uint32_t x = ES == 2 ? *reinterpret_cast<const uint16_t*>(p + (e0 + i) * 2) : *reinterpret_cast<const uint8_t*>(p + e0 + i);
              kr[s][i * ES / 4] |= x << (8 * (i * ES % 4));
            }
        }
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
          const char* p = g.v + (voff_lds[8 * i + 4 * h + j] + EB * c) * ES;
          uint32_t(&x)[VW] = vr[4 * i + j];
#pragma unroll
          for (int y = 0; y < VW; y++) x[y] = 0u;
          if (ROWS != kTreeAny) {
            if (ROWS == kTreeWhole || EB * c < g.d) {
              if constexpr (VB == 2) {
                x[0] = *reinterpret_cast<const uint16_t*>(p);
              } else if constexpr (VB == 4) {
                x[0] = *reinterpret_cast<const uint32_t*>(p);
              } else if constexpr (VB == 8) {
                const uint2t y = *reinterpret_cast<const uint2t*>(p);
                x[0] = y[0];
                x[1] = y[1];
              } else {
                const uint4v y = *reinterpret_cast<const uint4v*>(p);
#pragma unroll
                for (int u = 0; u < 4; u++) x[u] = y[u];
              }
            }
          } else {
#pragma unroll
            for (int u = 0; u < EB; u++)
              if (EB * c + u < g.d) {
                const uint32_t y = ES == 2 ? *reinterpret_cast<const uint16_t*>(p + u * 2) : *reinterpret_cast<const uint8_t*>(p + u);
                x[u * ES / 4] |= y << (8 * (u * ES % 4));
              }
          }
        }
    };

    bool odd_seen = false;  // infinities and NaN wait in LDS
    int page = t < t_end ? page_of(t) : -1;
    for (; t < t_end; t += WK) {
      const uint32_t vb = locate(t, page);
      if (t + WK < t_end) page = page_of(t + WK);
      load_k();
      load_v();
      const int j0 = t * 32 - sq.ctx;  // draft index of the tile's first key
      // every row attends all 32 keys: true of all tiles but the last ones and those with lost pages
      const bool whole = vb == 0xffffffffu && j0 + 31 < 0;
      uint32_t live[RB];  // the keys a row attends
      if (!whole) {
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
          uint32_t b = 0xffffffffu;
          if (j0 > -32) {
            if (g.mask == nullptr) {
              const int n = node[rb] - j0 + 1;
              b = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
            } else {
              const uint64_t* row = g.mask + (int64_t)(sq.row0 + node[rb]) * g.mask_words;
              if (j0 < 0) {
                const uint64_t x = g.mask_words > 0 ? row[0] : 0;
                b = (uint32_t)(x << -j0) | ((1u << -j0) - 1u);
              } else {
                const int word = j0 >> 6, sh = j0 & 63;
                const uint64_t lo = word < g.mask_words ? row[word] : 0, hi = word + 1 < g.mask_words ? row[word + 1] : 0;
                b = (uint32_t)(lo >> sh) | (sh > 32 ? (uint32_t)(hi << (64 - sh)) : 0u);
              }
            }
          }
          live[rb] = b & vb;
        }
        // Values of keys that do not exist become zeros.  An infinity or NaN among the others must
        // reach the rows that attend its key and no other row, which 0 * infinity would not do: it
        // becomes a zero too and is added, row by row, to sums in the wavefront's part of the LDS.
        const bool there = (vb >> c) & 1;
        bool bad = false;
        const float vs_is = vsr;
        if constexpr (CODE != SPFA_CODE_NONE) {
          bad = there && !(fabsf(vsr) <= 3.402823466e38f);
          if (bad) vsr = 1.f;
          if (!there) ksr = vsr = 0.f;
        }
        const uint32_t vbh = vb >> (4 * h), sick = (uint32_t)__builtin_amdgcn_ballot_w64(bad) >> (4 * h);
        // an exponent of ones (e4m3: all of the code but its sign) runs over into the sign's place
        constexpr uint32_t kSign = CODE == SPFA_CODE_NONE ? 0x80008000u : 0x80808080u;
        constexpr uint32_t kAll = CODE == SPFA_CODE_E4M3 ? 0x7f7f7f7fu : CODE == SPFA_CODE_INT8 ? 0u : __is_same(T, bf16) ? 0x7f807f80u : 0x7c007c00u;
        constexpr uint32_t kStep = CODE == SPFA_CODE_E4M3 ? 0x01010101u : CODE == SPFA_CODE_INT8 ? 0u : __is_same(T, bf16) ? 0x00800080u : 0x04000400u;
        uint32_t odd = sick;
#pragma unroll
        for (int k = 0; k < 16; k++)
#pragma unroll
          for (int y = 0; y < VW; y++) {
            vr[k][y] &= (uint32_t)((int32_t)(vbh << (31 - (8 * (k / 4) + k % 4))) >> 31);
            odd |= ((vr[k][y] & kAll) + kStep) & kSign;
          }
        if (__builtin_amdgcn_ballot_w64(odd != 0) != 0) {
          float* tab = acc_lds + (wk * M + wr * RB * 32) * Sh::kStride;
          if (!odd_seen)
            for (int i = lane; i < 32 * RB * Sh::kStride; i += kWave) tab[i] = 0.f;
          odd_seen = true;
          wave_sync();
#pragma unroll
          for (int k = 0; k < 16; k++) {
            const int at = 8 * (k / 4) + k % 4;
            const bool ill = (sick >> at) & 1;
            uint32_t some = ill;
#pragma unroll
            for (int y = 0; y < VW; y++) some |= ((vr[k][y] & kAll) + kStep) & kSign;
            if (__builtin_amdgcn_ballot_w64(some != 0) == 0) continue;
            float add[EB], scale = 0.f;
            if constexpr (CODE != SPFA_CODE_NONE) scale = shfl_f32(vs_is, at + 4 * h);
#pragma unroll
            for (int e = 0; e < EB; e++) {
              uint32_t& word = vr[k][e * ES / 4];
              const int sh = 8 * (e * ES % 4);
              if constexpr (CODE == SPFA_CODE_NONE) {
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
            for (int half = 0; half < 2; half++) {
#pragma unroll
              for (int rb = 0; rb < RB; rb++)
#pragma unroll 1
                for (int r = 0; r < 32; r++) {
                  const uint32_t row = (uint32_t)__builtin_amdgcn_readlane((int)live[rb], r);
                  if (h == half && ((row >> (at + 4 * h)) & 1)) {
                    float* to = tab + (rb * 32 + r) * Sh::kStride + EB * c;
#pragma unroll
                    for (int e = 0; e < EB; e++) to[e] += add[e];
                  }
                }
              wave_sync();
            }
          }
        }
      }
      // scales in the order of the scores: number v is key 8 (v / 4) + 4 h + v % 4
      float kf[16], vf[16];
      if constexpr (CODE != SPFA_CODE_NONE) {
        if (h == 0) {
          ks_lds[c] = ksr * g.scale_log2;
          vs_lds[c] = vsr;
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const float4v a = *reinterpret_cast<const float4v*>(ks_lds + 8 * i + 4 * h);
          const float4v b = *reinterpret_cast<const float4v*>(vs_lds + 8 * i + 4 * h);
#pragma unroll
          for (int j = 0; j < 4; j++) {
            kf[4 * i + j] = a[j];
            vf[4 * i + j] = b[j];
          }
        }
        wave_sync();
      }
      // scores
      f32x16t s[RB];
#pragma unroll
      for (int rb = 0; rb < RB; rb++)
#pragma unroll
        for (int v = 0; v < 16; v++) s[rb][v] = 0.f;
#pragma unroll
      for (int x = 0; x < NK; x++) {
        if constexpr (CODE == SPFA_CODE_NONE) {
#pragma unroll
          for (int rb = 0; rb < RB; rb++) s[rb] = tree_mfma<T>(kr[x], qf[rb][x], s[rb]);
        } else {
#pragma unroll
          for (int y = 0; y < 2; y++) {
            const uint2t a = decode4<T, CODE>(kr[x][2 * y]), b = decode4<T, CODE>(kr[x][2 * y + 1]);
            const uint4v f = {a[0], a[1], b[0], b[1]};
#pragma unroll
            for (int rb = 0; rb < RB; rb++) s[rb] = tree_mfma<T>(f, qf[rb][2 * x + y], s[rb]);
          }
        }
      }
      // softmax
#pragma unroll
      for (int rb = 0; rb < RB; rb++)
#pragma unroll
        for (int v = 0; v < 16; v++) s[rb][v] *= CODE == SPFA_CODE_NONE ? g.scale_log2 : kf[v];
      if (!whole) {
#pragma unroll
        for (int rb = 0; rb < RB; rb++) {
          const uint32_t bits = live[rb] >> (4 * h);
#pragma unroll
          for (int v = 0; v < 16; v++) {
            const uint32_t on = (uint32_t)((int32_t)(bits << (31 - (8 * (v / 4) + v % 4))) >> 31);
            const float x = s[rb][v];
            s[rb][v] = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & on) | (0xff800000u & ~on));
          }
        }
      }
      uint4v pf[RB][2], pl[RB][2];
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        float mx = kNegInf;
#pragma unroll
        for (int v = 0; v < 16; v++) mx = fmaxf(mx, s[rb][v]);
        mx = half_max(mx);
        m_top[rb] = fmaxf(m_top[rb], mx);
        if (__builtin_amdgcn_ballot_w64(mx > m_ref[rb] + kTreeSlack) != 0) {
          const float m_new = fmaxf(m_ref[rb], mx);
          const float alpha = m_ref[rb] == kNegInf ? 0.f : __builtin_amdgcn_exp2f(m_ref[rb] - m_new);
          m_ref[rb] = m_new;
          l[rb] *= alpha;
#pragma unroll
          for (int e = 0; e < EB; e++)
#pragma unroll
            for (int v = 0; v < 16; v++) o[rb][e][v] *= alpha;
        }
        const float base = m_ref[rb] == kNegInf ? 0.f : m_ref[rb];
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 2; y++)
#pragma unroll
          for (int x = 0; x < 4; x++) {
            float p[2];
#pragma unroll
            for (int z = 0; z < 2; z++) {
              const int v = 8 * y + 2 * x + z;
              p[z] = __builtin_amdgcn_exp2f(s[rb][v] - base);
              sum += p[z];
              if constexpr (CODE != SPFA_CODE_NONE) p[z] *= vf[v];
            }
            const uint32_t hi = tree_pack<Tv>(p[0], p[1]);
            pf[rb][y][x] = hi;
            if constexpr (kTwoParts)
              pl[rb][y][x] = tree_pack<Tv>(p[0] - __builtin_bit_cast(float, hi << 16), p[1] - __builtin_bit_cast(float, hi & 0xffff0000u));
          }
        l[rb] += sum;
      }
      // values: keys 16 y .. 16 y + 15 of the tile, eight of them of this half
#pragma unroll
      for (int y = 0; y < 2; y++) {
        uint32_t vq[8][EB / 2];  // pairs of elements
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
          for (int x = 0; x < VW; x++) {
            if constexpr (CODE == SPFA_CODE_NONE) {
              vq[k][x] = vr[8 * y + k][x];
            } else {
              const uint2t a = decode4<bf16, CODE>(vr[8 * y + k][x]);
              vq[k][2 * x] = a[0];
              if constexpr (EB / 2 > 1) vq[k][2 * x + 1] = a[1];
            }
          }
#pragma unroll
        for (int e = 0; e < EB; e++) {
          uint4v f;
#pragma unroll
          for (int z = 0; z < 4; z++) f[z] = __builtin_amdgcn_perm(vq[2 * z + 1][e / 2], vq[2 * z][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int rb = 0; rb < RB; rb++) {
            o[rb][e] = tree_mfma<Tv>(f, pf[rb][y], o[rb][e]);
            if constexpr (kTwoParts) o[rb][e] = tree_mfma<Tv>(f, pl[rb][y], o[rb][e]);
          }
        }
      }
    }

    // ---- the wavefronts' results meet -------------------------------------------------------------
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const int r = wk * M + (wr * RB + rb) * 32 + c;
      const float f = m_top[rb] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m_ref[rb] - m_top[rb]);
      const float lt = half_sum(l[rb]) * f;
      if (h == 0) state_lds[r] = float2{m_top[rb], lt};
#pragma unroll
      for (int v = 0; v < 16; v++) {
        float* to = acc_lds + r * Sh::kStride + EB * (8 * (v / 4) + 4 * h + v % 4);
#pragma unroll
        for (int e = 0; e < EB; e++) to[e] = odd_seen ? o[rb][e][v] * f + to[e] : o[rb][e][v] * f;
      }
    }
    __syncthreads();
    const bool final = blk0 == 0 && blk1 == sq.nblk;
    const int64_t slot = blk0 == 0 ? 2 * (int64_t)w + 1 : 2 * (int64_t)w;
    const int sub = tid & 7;
    for (int r = tid >> 3; r < live_rows; r += 32) {
      float mx = kNegInf;
      for (int k = 0; k < WK; k++) mx = fmaxf(mx, state_lds[k * M + r].x);
      float x[EB][4] = {};
      float lt = 0.f;
      for (int k = 0; k < WK; k++) {
        const float2 st = state_lds[k * M + r];
        const float f = st.x == kNegInf ? (st.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(st.x - mx);
        if (f == 0.f) continue;
        lt += f * st.y;
#pragma unroll
        for (int e = 0; e < EB; e++) {
          const float4v y = *reinterpret_cast<const float4v*>(acc_lds + (k * M + r) * Sh::kStride + 4 * (8 * e + sub));
#pragma unroll
          for (int u = 0; u < 4; u++) x[e][u] += f * y[u];
        }
      }
      if (final) {
        const int64_t rr = tile0 + r;
        const int nd = (int)(rr / g.group), gi = (int)(rr - (int64_t)nd * g.group);
        const TreeWeights tw = tree_weights(g, sq.row0 + nd, head * g.group + gi, mx, lt);
#pragma unroll
        for (int e = 0; e < EB; e++) tree_store<T, 4>(g, sq.row0 + nd, head * g.group + gi, 4 * (8 * e + sub), tw, x[e]);
        if (sub == 0) tree_store_state(g, sq.row0 + nd, head * g.group + gi, tw);
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
    __syncthreads();  // (all of it has been read: the next item may use the LDS)
    if (tid == 0 && blk0 > 0 && blk1 == sq.nblk) {
      // the workgroup that has the item's first block
      const int64_t first = pos - blk0, cut = extra * (per + 1);
      g.part[w] = TreePart{seq, tile, head, (int)(first < cut ? first / (per + 1) : extra + (first - cut) / per)};
    }
    pos += blk1 - blk0;
    in_seq += blk1 - blk0;
  }
}

// Joins the parts of the items that were cut: the workgroups of row blockIdx.y, + gridDim.y, ... of
// the item whose last part workgroup blockIdx.x of tree_kernel had.  Eight groups of 32 lanes take
// every eighth part each (all their loads at once for up to 64 parts), then meet in LDS.
// (CODE only keeps the object files' copies apart.)
template <typename T, int CODE, int DP>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs g, int M) {
  constexpr int N = DP / 32, V = N < 4 ? N : 4;  // elements per lane, as pieces of V
  typedef float vec __attribute__((ext_vector_type(V)));
  __shared__ __align__(16) float acc[8][DP];
  __shared__ float2 state[8];
  const int w = blockIdx.x;
  const TreePart part = g.part[w];
  if (part.seq < 0) return;
  const TreeSeq sq = tree_seq(g, part.seq, M);
  const int64_t tile0 = (int64_t)part.tile * M, n_rows = (int64_t)sq.n * g.group;
  const int live_rows = (int)(n_rows - tile0 < M ? n_rows - tile0 : M);
  const int grp = threadIdx.x >> 5, c = threadIdx.x & 31;
  for (int r = blockIdx.y; r < live_rows; r += gridDim.y) {
    float m = kNegInf, l = 0.f, x[N] = {};
    constexpr int U = 4;
    for (int p0 = part.first + grp; p0 <= w; p0 += 8 * U) {
      float pm[U], pl[U];
      vec px[U][N / V];
#pragma unroll
      for (int u = 0; u < U; u++) {
        const int p = p0 + 8 * u <= w ? p0 + 8 * u : w;
        const int64_t at = (p == part.first ? 2 * (int64_t)p + 1 : 2 * (int64_t)p) * M + r;
        pm[u] = g.pm[at];
        pl[u] = p0 + 8 * u <= w ? g.pl[at] : 0.f;
#pragma unroll
        for (int i = 0; i < N / V; i++) px[u][i] = *reinterpret_cast<const vec*>(g.pacc + at * DP + V * (32 * i + c));
      }
#pragma unroll
      for (int u = 0; u < U; u++) {
        if (pl[u] == 0.f) continue;  // (nothing attended there, or past the last part)
        const float mn = fmaxf(m, pm[u]);
        const float a = m == kNegInf ? 1.f : __builtin_amdgcn_exp2f(m - mn);
        const float b = pm[u] == kNegInf ? 1.f : __builtin_amdgcn_exp2f(pm[u] - mn);
        m = mn;
        l = l * a + pl[u] * b;
#pragma unroll
        for (int i = 0; i < N / V; i++)
#pragma unroll
          for (int e = 0; e < V; e++) x[i * V + e] = x[i * V + e] * a + px[u][i][e] * b;
      }
    }
    __syncthreads();
    if (c == 0) state[grp] = float2{m, l};
#pragma unroll
    for (int i = 0; i < N / V; i++)
#pragma unroll
      for (int e = 0; e < V; e++) acc[grp][V * (32 * i + c) + e] = x[i * V + e];
    __syncthreads();
    if (grp == 0) {
      float mx = kNegInf, lt = 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) mx = fmaxf(mx, state[k].x);
#pragma unroll
      for (int e = 0; e < N; e++) x[e] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const float2 st = state[k];
        if (st.y == 0.f) continue;
        const float f = st.x == kNegInf ? 1.f : __builtin_amdgcn_exp2f(st.x - mx);
        lt += f * st.y;
#pragma unroll
        for (int i = 0; i < N / V; i++)
#pragma unroll
          for (int e = 0; e < V; e++) x[i * V + e] += f * acc[k][V * (32 * i + c) + e];
      }
      const int64_t rr = tile0 + r;
      const int nd = (int)(rr / g.group), gi = (int)(rr - (int64_t)nd * g.group);
      const TreeWeights tw = tree_weights(g, sq.row0 + nd, part.head * g.group + gi, mx, lt);
#pragma unroll
      for (int i = 0; i < N / V; i++) {
        float y[V];
#pragma unroll
        for (int e = 0; e < V; e++) y[e] = x[i * V + e];
        tree_store<T, V>(g, sq.row0 + nd, part.head * g.group + gi, V * (32 * i + c), tw, y);
      }
      if (c == 0) tree_store_state(g, sq.row0 + nd, part.head * g.group + gi, tw);
    }
  }
}

// ---- host side ----------------------------------------------------------------------------------

// One element type and code per object file.
template <typename T, int CODE>
int tree_run(const TreeArgs& a, int rows_how, int dp, int rb, bool merge, hipStream_t stream);

#ifdef SPFA_TREE_CODE
template <typename T, int CODE, int DP, int RB, int ROWS>
int tree_launch(const TreeArgs& a, bool merge, hipStream_t stream) {
  constexpr int kLds = TreeShape<DP, RB>::kLds;
  if constexpr (kLds > 65536) {
    static std::atomic<bool> raised[kLdsLimitDevices];
    if (!raise_lds_limit(reinterpret_cast<const void*>(&tree_kernel<T, CODE, DP, RB, ROWS>), kLds, raised))
      return SPFA_ERR_LAUNCH;
  }
  tree_kernel<T, CODE, DP, RB, ROWS><<<dim3((unsigned)a.workers), dim3(256), kLds, stream>>>(a);
  if (merge) {
    const int M = 32 * RB * a.wave_rows;
    tree_merge_kernel<T, CODE, DP><<<dim3((unsigned)a.workers, 8), dim3(256), 0, stream>>>(a, M);
  }
  return launch_status();
}

template <typename T, int CODE, int DP>
int tree_launch_rows(const TreeArgs& a, int rows_how, int rb, bool merge, hipStream_t stream) {
  if (rows_how == kTreeAny) return tree_launch<T, CODE, DP, 1, kTreeAny>(a, merge, stream);
  if (rows_how == kTreePadded) return tree_launch<T, CODE, DP, 1, kTreePadded>(a, merge, stream);
  if constexpr (DP <= 128)
    if (rb == 2) return tree_launch<T, CODE, DP, 2, kTreeWhole>(a, merge, stream);
  return tree_launch<T, CODE, DP, 1, kTreeWhole>(a, merge, stream);
}

template <>
int tree_run<SPFA_TREE_T, SPFA_TREE_CODE>(const TreeArgs& a, int rows_how, int dp, int rb, bool merge, hipStream_t stream) {
  if (dp == 64) return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 64>(a, rows_how, rb, merge, stream);
  if (dp == 128) return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 128>(a, rows_how, rb, merge, stream);
  return tree_launch_rows<SPFA_TREE_T, SPFA_TREE_CODE, 256>(a, rows_how, rb, merge, stream);
}
#endif

}  // namespace spfa
