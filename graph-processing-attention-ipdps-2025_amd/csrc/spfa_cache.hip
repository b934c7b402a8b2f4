// Keys and values written into a paged cache, plain or quantised row by row, and read back.
//
//   code = rne(x * top / amax), scale = amax / top;  value = code * scale
//
// Both directions only move rows: every element is loaded once and stored once, in 16-byte pieces of
// the wider side where the tensors allow it, a row by LPV lanes, the row's largest absolute value
// found among them by DPP.  Rows are dealt to lane groups in the order in which they lie next to
// each other in the tensor outside the cache.
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
};

// The quotient of two floats, x * top / amax, as the code nearest to its exact value.  In 32 bits
// the quotient of two 16-bit floats is on the right side of every border between two codes (its
// exact value is either on the border, and comes out exactly, or at least 2^-19 of itself away); that of
// two fp32 values needs 64, and for e4m3 a rounding to odd on the way through fp32.
template <typename T, int CODE>
__device__ __forceinline__ float quotient(float x, float amax) {
  constexpr float top = CODE == SPFA_CODE_INT8 ? 127.f : 448.f;
  if constexpr (sizeof(T) == 2) {
    // (bf16 reaches where x * top would overflow: scaled down, which changes no quotient)
    const float s = amax > 0x1p100f ? 0x1p-64f : 1.f;
    const float y = (x * s) * top / (amax * s);
    return CODE == SPFA_CODE_INT8 ? rintf(y) : y;
  } else {
    const double y = (double)x * (double)top / (double)amax;
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
  if (g.token_fast) {
    h = row / g.tokens;
    t = row - h * g.tokens;
  } else {
    t = row / g.heads;
    h = row - t * g.heads;
  }
  const int64_t slot = load_index(g.slots, t, g.wide);
  if (slot < 0 || slot >= g.n_slots) return r;
  const int64_t page = slot / g.page_size, place = slot - page * g.page_size;
  r.outside = t * s.token + h * s.head;
  r.inside = page * s.page + place * s.slot + h * s.chead;
  r.scale = page * s.spage + place * s.sslot + h * s.shead;
  r.ok = true;
  return r;
}

// E elements of a lane's piece (one, or 16: whole 16-byte pieces of codes), a lane's NJ pieces LPV
// pieces apart.
template <typename T, int CODE, int LPV, int E, int NJ, bool WRITE>
__global__ __launch_bounds__(kCacheThreads) void cache_kernel(CacheArgs g) {
  constexpr int kSlots = kCacheThreads / LPV;
  const int c = threadIdx.x % LPV;
  const CacheSide& s = g.side[blockIdx.y];
  const int64_t rows = g.tokens * g.heads;
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
          const float div = amax == 0.f ? 1.f : amax;
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            const int i0 = (c + j * LPV) * E;
            if (i0 >= g.d) continue;
            if constexpr (E == 1) {
              const float q[4] = {quotient<T, CODE>(f[j][0], div), 0.f, 0.f, 0.f};
              y[i0] = (uint8_t)pack_codes<CODE>(q);
            } else {
              uint4v w;
#pragma unroll
              for (int k = 0; k < 4; k++) {
                float q[4];
#pragma unroll
                for (int e = 0; e < 4; e++) q[e] = quotient<T, CODE>(f[j][4 * k + e], div);
                w[k] = pack_codes<CODE>(q);
              }
              *reinterpret_cast<uint4v*>(y + i0) = w;
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
            const uint4v w = *reinterpret_cast<const uint4v*>(y + i0);
            float f[E];
#pragma unroll
            for (int k = 0; k < 4; k++) {
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
  if (aligned && g.d % 16 == 0) {
    if (g.d <= 64) cache_kernel<T, CODE, 4, 16, 1, WRITE><<<grid(4), block, 0, stream>>>(g);
    else if (g.d <= 128) cache_kernel<T, CODE, 8, 16, 1, WRITE><<<grid(8), block, 0, stream>>>(g);
    else if (g.d <= 256) cache_kernel<T, CODE, 16, 16, 1, WRITE><<<grid(16), block, 0, stream>>>(g);
    else cache_kernel<T, CODE, 64, 16, 1, WRITE><<<grid(64), block, 0, stream>>>(g);
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
