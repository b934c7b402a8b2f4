// Keys and values written into a paged cache, plain or quantised row by row, and read back.
//
//   code = rne(x * top / amax), scale = amax / top;  value = code * scale
//
// Both directions only move rows: every element is loaded once and stored once, in 16-byte pieces of
// the wider side where the tensors allow it, a row by LPV lanes, the row's largest absolute value
// found among them by DPP.  Rows are dealt to lane groups in the order in which they lie next to
// each other in the tensor outside the cache.  Measured: 32768 e4m3 tokens of 8 heads of 128 to bf16
// 31 us (6.4 TB/s read and written), 2048 bf16 tokens written in 5 us; one token each of four sequences 3 us.
#include <type_traits>

#include "spfa_serve.hpp"

namespace spfa {

constexpr int kCacheThreads = 256;

struct CacheSide {
  void* rows;    // outside the cache: the input of a write, the output of a read
  char* cache;
  float* scale;
  int64_t token, head;                // strides of rows
  int64_t page, slot, chead;          // of the cache
  int64_t spage, sslot, shead;        // of the scales
};

struct CacheArgs {
  CacheSide side[2];
  const void* slots;
  int64_t tokens, heads, page_size, n_slots;
  int32_t d, wide, token_fast;
  int32_t small;  // rows and slots are below 2^31: rows and pages by fast_div
  uint32_t row_magic, page_magic;
  int32_t row_shift, page_shift;
};

// x * top / amax as the code nearest to its exact value, by one division per row.  Against a border
// between two codes, a number of few bits, the exact quotient is either equal or at least 2^-19 of itself
// away for 16-bit floats (2^-34 for fp32, worked on in 64 bits).  x * top is exact and its product with
// the rounded reciprocal is off by less than 2 units of the last place, so dropping the last 2 (12) bits by
// rounding restores what lies on a border and takes nothing across one.
template <typename T, int CODE>
struct Quotient {
  static constexpr float kTop = CODE == SPFA_CODE_INT8 ? 127.f : 448.f;
  using W = std::conditional_t<sizeof(T) == 2, float, double>;
  W by;
  float s;
  __device__ __forceinline__ explicit Quotient(float amax) {
    // (bf16 reaches where x * top would overflow, and the reciprocal: scaled, which changes no quotient)
    s = sizeof(T) == 4 ? 1.f : amax > 0x1p100f ? 0x1p-64f : amax < 0x1p-60f ? 0x1p64f : 1.f;
    by = (W)1 / ((W)amax * (W)s);
  }
  __device__ __forceinline__ float operator()(float x) const {
    if constexpr (sizeof(T) == 2) {
      const float y = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, (x * s) * kTop * by) + 2u) & ~3u);
      return CODE == SPFA_CODE_INT8 ? rintf(y) : y;
    } else {
      const double y = __builtin_bit_cast(double, (__builtin_bit_cast(uint64_t, (double)x * (double)kTop * by) + 0x800u) & ~(uint64_t)0xfff);
      if (CODE == SPFA_CODE_INT8) return (float)rint(y);
      const float f = (float)y;
      if ((double)f == y || y != y) return f;
      // truncated, and its last bit set: still between the same two codes, never on a border
      uint32_t u = __builtin_bit_cast(uint32_t, f);
      if (fabs((double)f) > fabs(y)) u -= 1;
      u |= 1;
      return __builtin_bit_cast(float, u);
    }
  }
};

// Codes of four elements, a byte each.
template <int CODE>
__device__ __forceinline__ uint32_t pack_codes(const float (&y)[4]) {
  if constexpr (CODE == SPFA_CODE_INT8) {
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
      // (a NaN has no code: 0, its row's scale says it all)
      const int q = y[i] == y[i] ? (int)y[i] : 0;
      r |= (uint32_t)(q & 255) << (8 * i);
    }
    return r;
  } else {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
  }
}
template <int CODE>
__device__ __forceinline__ void unpack_codes(uint32_t w, float (&y)[4]) {
  if constexpr (CODE == SPFA_CODE_INT8) {
#pragma unroll
    for (int i = 0; i < 4; i++) y[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    y[0] = lo[0]; y[1] = lo[1]; y[2] = hi[0]; y[3] = hi[1];
  }
}

// largest of the lanes of a group (LPV of them, aligned)
template <int LPV>
__device__ __forceinline__ uint32_t group_max(uint32_t x) {
#pragma unroll
  for (int m = 1; m < LPV; m *= 2) {
    const uint32_t y = (uint32_t)shfl_i32((int)x, lane_id() ^ m);
    x = x > y ? x : y;
  }
  return x;
}

struct CacheRow {
  int64_t outside, inside, scale;  // offsets in elements
  bool ok;
};
__device__ __forceinline__ CacheRow cache_row(const CacheArgs& g, const CacheSide& s, int64_t row) {
  CacheRow r{0, 0, 0, false};
  if (row >= g.tokens * g.heads) return r;
  int64_t t, h;
  // (64-bit divisions are hundreds of instructions)
  if (g.small) {
    const int64_t big = fast_div((uint32_t)row, g.row_magic, g.row_shift), rest = row - big * (g.token_fast ? g.tokens : g.heads);
    t = g.token_fast ? rest : big;
    h = g.token_fast ? big : rest;
  } else if (g.token_fast) {
    h = row / g.tokens;
    t = row - h * g.tokens;
  } else {
    t = row / g.heads;
    h = row - t * g.heads;
  }
  const int64_t slot = load_index(g.slots, t, g.wide);
  if (slot < 0 || slot >= g.n_slots) return r;
  const int64_t page = g.small ? (int64_t)fast_div((uint32_t)slot, g.page_magic, g.page_shift) : slot / g.page_size, place = slot - page * g.page_size;
  r.outside = t * s.token + h * s.head;
  r.inside = page * s.page + place * s.slot + h * s.chead;
  r.scale = page * s.spage + place * s.sslot + h * s.shead;
  r.ok = true;
  return r;
}

// E elements of a lane's piece, a lane's NJ pieces LPV pieces apart.
template <typename T, int CODE, int LPV, int E, int NJ, bool WRITE>
__global__ __launch_bounds__(kCacheThreads) void cache_kernel(CacheArgs g) {
  constexpr int kSlots = kCacheThreads / LPV;
  const int c = threadIdx.x % LPV;
  const CacheSide& s = g.side[blockIdx.y];
  const int64_t rows = g.tokens * g.heads;
  typedef uint32_t Codes __attribute__((ext_vector_type(E < 4 ? 1 : E / 4)));
  constexpr int P = E == 1 ? 1 : 16 / (int)sizeof(T);  // elements of a 16-byte piece of rows
  for (int64_t r0 = (int64_t)blockIdx.x * kSlots; r0 < rows; r0 += (int64_t)gridDim.x * kSlots) {
    const CacheRow r = cache_row(g, s, r0 + threadIdx.x / LPV);
    T* x = (T*)s.rows + r.outside;
    if constexpr (CODE == SPFA_CODE_NONE) {
      T* y = (T*)s.cache + r.inside;
      if (r.ok) {
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          const int i0 = (c + j * LPV) * E;
#pragma unroll
          for (int i = i0; i < i0 + E; i += P) {
            if (i >= g.d) continue;
            if constexpr (E == 1) {
              if (WRITE) y[i] = x[i];
              else x[i] = y[i];
            } else {
              if (WRITE) *reinterpret_cast<uint4v*>(y + i) = *reinterpret_cast<const uint4v*>(x + i);
              else *reinterpret_cast<uint4v*>(x + i) = *reinterpret_cast<const uint4v*>(y + i);
            }
          }
        }
      }
    } else {
      uint8_t* y = (uint8_t*)s.cache + r.inside;
      if constexpr (WRITE) {
        float f[NJ][E];
        uint32_t top = 0;  // of the absolute values' bits: NaN above infinity above the rest
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          const int i0 = (c + j * LPV) * E;
#pragma unroll
          for (int i = 0; i < E; i += P) {
            float p[P] = {};
            if (r.ok && i0 + i < g.d) load_piece<T, P>(x + i0 + i, p);
#pragma unroll
            for (int e = 0; e < P; e++) {
              f[j][i + e] = p[e];
              const uint32_t u = __builtin_bit_cast(uint32_t, p[e]) & 0x7fffffffu;
              top = top > u ? top : u;
            }
          }
        }
        const float amax = __builtin_bit_cast(float, group_max<LPV>(top));
        if (r.ok) {
          const Quotient<T, CODE> code(amax == 0.f ? 1.f : amax);
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            const int i0 = (c + j * LPV) * E;
            if (i0 >= g.d) continue;
            if constexpr (E == 1) {
              const float q[4] = {code(f[j][0]), 0.f, 0.f, 0.f};
              y[i0] = (uint8_t)pack_codes<CODE>(q);
            } else {
              Codes w;
#pragma unroll
              for (int k = 0; k < E / 4; k++) {
                float q[4];
#pragma unroll
                for (int e = 0; e < 4; e++) q[e] = code(f[j][4 * k + e]);
                w[k] = pack_codes<CODE>(q);
              }
              *reinterpret_cast<Codes*>(y + i0) = w;
            }
          }
          if (c == 0) s.scale[r.scale] = amax / (CODE == SPFA_CODE_INT8 ? 127.f : 448.f);
        }
      } else if (r.ok) {
        const float sc = s.scale[r.scale];
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          const int i0 = (c + j * LPV) * E;
          if (i0 >= g.d) continue;
          if constexpr (E == 1) {
            float q[4];
            unpack_codes<CODE>(y[i0], q);
            x[i0] = from_f32<T>(q[0] * sc);
          } else {
            const Codes w = *reinterpret_cast<const Codes*>(y + i0);
            float f[E];
#pragma unroll
            for (int k = 0; k < E / 4; k++) {
              float q[4];
              unpack_codes<CODE>(w[k], q);
#pragma unroll
              for (int e = 0; e < 4; e++) f[4 * k + e] = q[e] * sc;
            }
#pragma unroll
            for (int i = 0; i < E; i += P) {
              float p[P];
#pragma unroll
              for (int e = 0; e < P; e++) p[e] = f[i + e];
              store_piece<T, P>(x + i0 + i, p);
            }
          }
        }
      }
    }
  }
}

namespace {

int cache_check(const spfa_cache_t* c) {
  if (c == nullptr) return SPFA_ERR_BAD_ARG;
  if (c->d < 1 || c->d > 1024) return SPFA_ERR_EMB_TOO_LARGE;
  if (c->dtype != SPFA_DTYPE_F32 && c->dtype != SPFA_DTYPE_F16 && c->dtype != SPFA_DTYPE_BF16) return SPFA_ERR_UNSUPPORTED;
  if (c->code != SPFA_CODE_NONE && c->code != SPFA_CODE_INT8 && c->code != SPFA_CODE_E4M3) return SPFA_ERR_UNSUPPORTED;
  if (c->pages < 0 || c->page_size < 1 || c->heads < 0 || c->heads > (1 << 20)) return SPFA_ERR_BAD_ARG;
  if (c->pages > 0 && c->page_size > INT64_MAX / c->pages) return SPFA_ERR_BAD_ARG;
  if (c->pages > 0 && c->heads > 0) {
    if (c->k == nullptr || c->v == nullptr) return SPFA_ERR_BAD_ARG;
    if (c->code != SPFA_CODE_NONE && (c->k_scale == nullptr || c->v_scale == nullptr)) return SPFA_ERR_BAD_ARG;
  }
  return SPFA_OK;
}

template <typename T, int CODE, bool WRITE>
int cache_launch(const CacheArgs& g, bool aligned, hipStream_t stream) {
  const int64_t rows = g.tokens * g.heads;
  auto grid = [&](int lanes) {
    const int64_t n = (rows + kCacheThreads / lanes - 1) / (kCacheThreads / lanes);
    return dim3((unsigned)(n < (1 << 22) ? n : (1 << 22)), 2);  // (a grid holds fewer than 2^32 work items)
  };
  const dim3 block(kCacheThreads);
  // A lane's piece is 16 bytes of codes, or of the rows where there are no codes (32768 tokens of 8 heads of
  // 128 appended and read back: bf16 89 us, fp32 193, 101 and 489 with 16 elements).  fp32 rows with four
  // elements a lane come back faster by 2 us of 20, but are written in 28 us instead of 16 (15003 tokens of 5
  // heads of 80): each lane has the row's place and reciprocal to work out.
  constexpr int E = CODE == SPFA_CODE_NONE ? 16 / (int)sizeof(T) : 16;
  const int lanes = g.d / E;
  if (aligned && g.d % 16 == 0) {
    if (lanes <= 4) cache_kernel<T, CODE, 4, E, 1, WRITE><<<grid(4), block, 0, stream>>>(g);
    else if (lanes <= 8) cache_kernel<T, CODE, 8, E, 1, WRITE><<<grid(8), block, 0, stream>>>(g);
    else if (lanes <= 16) cache_kernel<T, CODE, 16, E, 1, WRITE><<<grid(16), block, 0, stream>>>(g);
    else if (lanes <= 32) cache_kernel<T, CODE, 32, E, 1, WRITE><<<grid(32), block, 0, stream>>>(g);
    else if (lanes <= 64) cache_kernel<T, CODE, 64, E, 1, WRITE><<<grid(64), block, 0, stream>>>(g);
    else if constexpr (E < 16) cache_kernel<T, CODE, 64, E, 16 / E, WRITE><<<grid(64), block, 0, stream>>>(g);
  } else if (g.d <= 256) {
    cache_kernel<T, CODE, 64, 1, 4, WRITE><<<grid(64), block, 0, stream>>>(g);
  } else {
    cache_kernel<T, CODE, 64, 1, 16, WRITE><<<grid(64), block, 0, stream>>>(g);
  }
  return launch_status();
}

template <typename T, bool WRITE>
int cache_code(const CacheArgs& g, int code, bool aligned, hipStream_t stream) {
  switch (code) {
    case SPFA_CODE_INT8: return cache_launch<T, SPFA_CODE_INT8, WRITE>(g, aligned, stream);
    case SPFA_CODE_E4M3: return cache_launch<T, SPFA_CODE_E4M3, WRITE>(g, aligned, stream);
    default: return cache_launch<T, SPFA_CODE_NONE, WRITE>(g, aligned, stream);
  }
}

template <bool WRITE>
int cache_run(const spfa_cache_t* c, const spfa_heads_t* k, const spfa_heads_t* v, int64_t tokens, const void* slots,
              int slot_bytes, void* stream) {
  const int rc = cache_check(c);
  if (rc) return rc;
  if (tokens < 0 || (slot_bytes != 4 && slot_bytes != 8)) return SPFA_ERR_BAD_ARG;
  if (tokens == 0 || c->heads == 0 || c->pages == 0) return SPFA_OK;
  if (k == nullptr || v == nullptr || k->data == nullptr || v->data == nullptr || slots == nullptr) return SPFA_ERR_BAD_ARG;
  if (tokens > INT64_MAX / 2048 / c->heads) return SPFA_ERR_BAD_ARG;
  CacheArgs g{};
  const spfa_heads_t* x[2] = {k, v};
  void* cache[2] = {c->k, c->v};
  float* scale[2] = {c->k_scale, c->v_scale};
  const int64_t at[2][3] = {{c->k_stride_page, c->k_stride_slot, c->k_stride_head},
                            {c->v_stride_page, c->v_stride_slot, c->v_stride_head}};
  const int64_t sat[2][3] = {{c->ks_stride_page, c->ks_stride_slot, c->ks_stride_head},
                             {c->vs_stride_page, c->vs_stride_slot, c->vs_stride_head}};
  const int size = c->dtype == SPFA_DTYPE_F32 ? 4 : 2, csize = c->code == SPFA_CODE_NONE ? size : 1;
  bool aligned = true;
  for (int i = 0; i < 2; i++) {
    g.side[i] = CacheSide{x[i]->data,  (char*)cache[i], scale[i],  x[i]->stride_token, x[i]->stride_head, at[i][0],
                          at[i][1],    at[i][2],        sat[i][0], sat[i][1],          sat[i][2]};
    aligned = aligned && heads_aligned(*x[i], size, false) && ((uintptr_t)cache[i] & 15) == 0;
    for (int64_t st : at[i]) aligned = aligned && (st * csize) % 16 == 0;
  }
  g.slots = slots;
  g.tokens = tokens;
  g.heads = c->heads;
  g.page_size = c->page_size;
  g.n_slots = c->pages * c->page_size;
  g.d = (int32_t)c->d;
  g.wide = slot_bytes == 8;
  // rows in the order in which they follow each other in the tensor outside the cache
  g.token_fast = k->stride_token < k->stride_head;
  g.small = tokens * c->heads < INT32_MAX && g.n_slots < INT32_MAX;
  if (g.small) {
    fast_divider((int32_t)(g.token_fast ? tokens : c->heads), &g.row_magic, &g.row_shift);
    fast_divider((int32_t)c->page_size, &g.page_magic, &g.page_shift);
  }
  switch (c->dtype) {
    case SPFA_DTYPE_F32: return cache_code<float, WRITE>(g, c->code, aligned, (hipStream_t)stream);
    case SPFA_DTYPE_F16: return cache_code<f16, WRITE>(g, c->code, aligned, (hipStream_t)stream);
    default: return cache_code<bf16, WRITE>(g, c->code, aligned, (hipStream_t)stream);
  }
}

}  // namespace
}  // namespace spfa

extern "C" int spfa_cache_write(const spfa_cache_t* c, const spfa_heads_t* k, const spfa_heads_t* v, int64_t tokens,
                                const void* slots, int slot_bytes, void* stream) {
  return spfa::cache_run<true>(c, k, v, tokens, slots, slot_bytes, stream);
}

extern "C" int spfa_cache_read(const spfa_cache_t* c, const void* slots, int slot_bytes, int64_t tokens,
                               const spfa_heads_t* k_out, const spfa_heads_t* v_out, void* stream) {
  return spfa::cache_run<false>(c, k_out, v_out, tokens, slots, slot_bytes, stream);
}
