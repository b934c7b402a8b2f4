// Shared pieces of the operators around masked attention: pieces of E consecutive elements of a row
// held as floats, and the tensors' strides as the kernels take them.
#pragma once

#include "spfa_common.hpp"
#include "spfa_hip.h"

namespace spfa {

// E consecutive elements at p as floats: one 16-byte piece (E = 16 / sizeof(T)) or a single element.
template <typename T, int E>
__device__ __forceinline__ void load_piece(const T* p, float (&f)[E]) {
  if constexpr (E == 1) {
    f[0] = to_f32(p[0]);
  } else {
    static_assert(E * sizeof(T) == 16, "a piece is 16 bytes or one element");
    VecLay<T, 64>::unpack(*reinterpret_cast<const uint4v*>(p), f);
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_piece(T* p, const float (&f)[E]) {
  if constexpr (E == 1) {
    p[0] = from_f32<T>(f[0]);
  } else {
    static_assert(E * sizeof(T) == 16, "a piece is 16 bytes or one element");
    VecLay<T, 64>::store(p, 0, 0, f);
  }
}

__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, bool wide) {
  return wide ? ((const int64_t*)p)[i] : (int64_t)((const int32_t*)p)[i];
}

// p / d for p < 2^31 as (p * magic >> 32) >> shift (shift < 0: d is 1).  With s the bits of d - 1 and
// magic = ceil(2^(31 + s) / d) < 2^32, p * magic exceeds p * 2^(31 + s) / d by less than
// p / 2^31 * 2^(31 + s) / d, too little to reach the next whole quotient.
inline void fast_divider(int32_t d, uint32_t* magic, int32_t* shift) {
  int s = 0;
  while (((int64_t)1 << s) < d) s++;
  *shift = s - 1;
  *magic = s == 0 ? 0u : (uint32_t)((((uint64_t)1 << (31 + s)) + (uint64_t)d - 1) / (uint64_t)d);
}
__device__ __forceinline__ uint32_t fast_div(uint32_t p, uint32_t magic, int shift) { return shift < 0 ? p : __umulhi(p, magic) >> shift; }

// Can rows of this tensor be read in 16-byte pieces: pointer and every stride that is used are
// multiples of 16 bytes.
inline bool heads_aligned(const spfa_heads_t& h, int elem_bytes, bool batched) {
  const int64_t n = 16 / elem_bytes;
  return ((uintptr_t)h.data & 15) == 0 && h.stride_token % n == 0 && h.stride_head % n == 0 &&
         (!batched || h.stride_batch % n == 0);
}

inline int launch_status() { return hipGetLastError() == hipSuccess ? SPFA_OK : SPFA_ERR_LAUNCH; }

}  // namespace spfa
