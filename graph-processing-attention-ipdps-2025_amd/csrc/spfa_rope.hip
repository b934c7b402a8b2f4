// Head norms with the position rotation, forward and gradients, in one pass over queries and keys.
//
//   n = x r, r = 1 / sqrt(mean(x^2) + eps);  y = n w;  out = Rot(angle) y
//   g = Rot(-angle) d_out;  d_w = sum g n;  d_x = r (g w - n mean(g w n))
//
// Both directions are bound by memory: a vector of d elements is read once (gradients: x and d_out)
// and written once, a handful of operations per element in between.  A vector is held by LPV lanes,
// a lane has two 16-byte pieces of it, half a head apart, chosen so that both elements of every
// pair are in one lane: no element crosses lanes, only the sum of squares (and of g w n) does, over
// LPV lanes by DPP.  The angles of a token are the same for all its heads: a workgroup reduces them
// once in fp64 (position * frequency / 2 pi, less its nearest whole number), takes sine and cosine of
// its fp32 form, adds what that form left of the angle, and keeps them in LDS for the vectors of its tokens.
//
// Measured, 16384 tokens of 32 + 8 bf16 heads of 128: forward 68 us (4.9 TB/s, what a copy reaches),
// gradients 124 us (4.0 TB/s; 191 registers leave two wavefronts per SIMD, fewer registers by one vector
// on the way instead of two: 137 us, by spilling: 171) and 5 us for the weights' sum; one token 4 us.
#include <type_traits>

#include "spfa_serve.hpp"

namespace spfa {

constexpr int kRopeThreads = 256;
constexpr int kRopeBlocks = 1024;   // workgroups of a gradient call over both tensors
constexpr int kRopeBatch = 2;       // vectors of a lane on the way at a time
constexpr int kRopeLds = 32 * 1024; // bytes of cosines and sines a workgroup keeps at most

enum { kNoWeights, kOwnWeights, kFloatWeights };  // of the vectors' type, of fp32
struct RopeSide {
  const void* x;
  void* out;       // forward: the output; gradients: d_x
  const void* dy;  // gradients only
  const void* w;
  int64_t xs[3], os[3], ds[3];  // strides by batch, token, head
  int64_t heads;
  int64_t vectors;  // batch * tokens * heads
  int64_t chunks;   // of args.per_chunk vectors each
  int64_t blocks;   // workgroups that walk them
  int32_t w_how;    // kNoWeights, ...
  uint32_t magic;   // of heads (fast_div)
  int32_t shift;
};

struct RopeArgs {
  RopeSide side[2];
  int64_t tokens;
  int64_t position_stride;
  const void* positions;
  const float* inv_freq;
  float* partial;  // gradients: [blocks of both sides, d]
  float eps;
  int32_t d, rot, per_chunk;
  int32_t wide_pos, interleaved;
  uint32_t half_magic;  // of rot / 2
  int32_t half_shift;
};

// What a lane has of a vector, as loaded.
template <typename T, int E, int NJ>
struct RopeRow {
  using Raw = std::conditional_t<E == 1, T, uint4v>;
  Raw a[NJ], b[NJ];
  __device__ __forceinline__ void load(const T* p, const int (&at_a)[NJ], const int (&at_b)[NJ]) {
#pragma unroll
    for (int j = 0; j < NJ; j++) {  // (pieces that are not there are taken from the vector's start)
      a[j] = *reinterpret_cast<const Raw*>(p + (at_a[j] < 0 ? 0 : at_a[j]));
      b[j] = *reinterpret_cast<const Raw*>(p + (at_b[j] < 0 ? 0 : at_b[j]));
    }
  }
  static __device__ __forceinline__ void piece(const Raw& raw, bool there, float (&f)[E]) {
    if constexpr (E == 1) {
      f[0] = there ? to_f32(raw) : 0.f;
    } else {
      uint4v x = raw;
      const uint32_t mask = there ? 0xffffffffu : 0u;
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] &= mask;
      VecLay<T, 64>::unpack(x, f);
    }
  }
};

// A lane's elements: NJ pairs of pieces, piece j starting at a[j] and b[j] (-1: none).
template <int E, int NJ, int LPV>
__device__ __forceinline__ void piece_starts(const RopeArgs& g, int c, int (&a)[NJ], int (&b)[NJ]) {
#pragma unroll
  for (int j = 0; j < NJ; j++) {
    const int v = (c + j * LPV) * E;
    if constexpr (E == 1) {
      // single elements: a pair each, then the elements behind the rotated ones two by two
      if (v < g.rot / 2) {
        a[j] = g.interleaved ? 2 * v : v;
        b[j] = g.interleaved ? 2 * v + 1 : v + g.rot / 2;
      } else {
        a[j] = g.rot + 2 * (v - g.rot / 2);
        b[j] = a[j] + 1;
      }
    } else if (v >= g.d / 2) {
      a[j] = b[j] = g.d;
    } else if (g.interleaved) {
      a[j] = v;
      b[j] = g.d / 2 + v;
    } else if (v < g.rot / 2) {
      a[j] = v;
      b[j] = g.rot / 2 + v;
    } else {
      a[j] = g.rot + (v - g.rot / 2);
      b[j] = a[j] + (g.d - g.rot) / 2;
    }
    if (a[j] >= g.d) a[j] = -1;
    if (b[j] >= g.d) b[j] = -1;
  }
}

// Turns the pairs among a lane's pieces by their angles (DIR = 1) or back (DIR = -1).
template <int E, int DIR>
__device__ __forceinline__ void turn(const RopeArgs& g, const float2* cs, int a, int b, float (&x)[E], float (&y)[E]) {
  if (E > 1 && g.interleaved) {
    if constexpr (E > 1) {
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        if (a >= 0 && a + e < g.rot) {
          const float2 t = cs[(a + e) >> 1];
          const float u = x[e], v = x[e + 1], s = DIR * t.y;
          x[e] = u * t.x - v * s;
          x[e + 1] = u * s + v * t.x;
        }
        if (b >= 0 && b + e < g.rot) {
          const float2 t = cs[(b + e) >> 1];
          const float u = y[e], v = y[e + 1], s = DIR * t.y;
          y[e] = u * t.x - v * s;
          y[e + 1] = u * s + v * t.x;
        }
      }
    }
  } else if (a >= 0 && a < g.rot) {
    const int p = g.interleaved ? a >> 1 : a;
#pragma unroll
    for (int e = 0; e < E; e++) {
      const float2 t = cs[p + e];
      const float u = x[e], v = y[e], s = DIR * t.y;
      x[e] = u * t.x - v * s;
      y[e] = u * s + v * t.x;
    }
  }
}

// R: vectors a slot of LPV lanes has on the way at a time.  The first of a chunk are asked for before the
// angles are worked out.
template <typename T, int LPV, int E, int NJ, int R, bool GRAD>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs g) {
  constexpr int kSlots = kRopeThreads / LPV;
  using Row = RopeRow<T, E, NJ>;
  extern __shared__ __align__(16) char lds[];
  float2* cs = reinterpret_cast<float2*>(lds);
  const int tid = threadIdx.x, c = tid % LPV, slot = tid / LPV;
  int64_t blk = blockIdx.x;
  const int which = blk >= g.side[0].blocks;
  if (which) blk -= g.side[0].blocks;
  const RopeSide& s = g.side[which];
  const int half = g.rot / 2, H = (int)s.heads;

  int a[NJ], b[NJ];
  piece_starts<E, NJ, LPV>(g, c, a, b);
  // the weights of the lane's elements (single elements, or pieces of 16 bytes: host)
  float wa[NJ][E], wb[NJ][E], da[NJ][E], db[NJ][E];
#pragma unroll
  for (int j = 0; j < NJ; j++) {
#pragma unroll
    for (int e = 0; e < E; e++) {
      wa[j][e] = wb[j][e] = 1.f;
      da[j][e] = db[j][e] = 0.f;
    }
    const int ia = a[j] < 0 ? 0 : a[j], ib = b[j] < 0 ? 0 : b[j];
    if (s.w_how == kOwnWeights) {
      load_piece<T, E>((const T*)s.w + ia, wa[j]);
      load_piece<T, E>((const T*)s.w + ib, wb[j]);
    } else if (s.w_how == kFloatWeights) {
      constexpr int F = E < 4 ? E : 4;
#pragma unroll
      for (int e = 0; e < E; e += F) {
        load_piece<float, F>((const float*)s.w + ia + e, *reinterpret_cast<float(*)[F]>(&wa[j][e]));
        load_piece<float, F>((const float*)s.w + ib + e, *reinterpret_cast<float(*)[F]>(&wb[j][e]));
      }
    }
  }

  for (int64_t ch = blk; ch < s.chunks; ch += s.blocks) {
    const int64_t v0 = ch * g.per_chunk;
    const int n = (int)(s.vectors - v0 < g.per_chunk ? s.vectors - v0 : g.per_chunk);
    // (64-bit divisions are hundreds of instructions)
    const int64_t t0 = s.vectors < INT32_MAX ? (int64_t)fast_div((uint32_t)v0, s.magic, s.shift) : v0 / H;
    const int h0 = (int)(v0 - t0 * H);
    const int64_t b0 = t0 < g.tokens ? 0 : t0 < INT32_MAX ? (int64_t)((uint32_t)t0 / (uint32_t)g.tokens) : t0 / g.tokens;
    const int64_t tok0 = t0 - b0 * g.tokens;
    const int span = (int)fast_div((uint32_t)(h0 + n - 1), s.magic, s.shift) + 1;
    Row x[R], y[GRAD ? R : 1];
    T* to[R];
    const float2* angles[R];
    // the slot's vectors r * kSlots + slot from `first`; behind the chunk's last the last is taken instead
    auto fetch = [&](int first) {
#pragma unroll
      for (int r = 0; r < R; r++) {
        const int vi = first + r * kSlots + slot;
        const int hv = h0 + (vi < n ? vi : n - 1);
        const int k = (int)fast_div((uint32_t)hv, s.magic, s.shift), h = hv - k * H;
        int64_t bb = b0, tok = tok0 + k;
        while (tok >= g.tokens) { tok -= g.tokens; bb++; }
        angles[r] = cs + k * half;
        to[r] = (T*)s.out + bb * s.os[0] + tok * s.os[1] + h * s.os[2];
        x[r].load((const T*)s.x + bb * s.xs[0] + tok * s.xs[1] + h * s.xs[2], a, b);
        if constexpr (GRAD) y[r].load((const T*)s.dy + bb * s.ds[0] + tok * s.ds[1] + h * s.ds[2], a, b);
      }
    };
    // (what the lane's first angle needs is asked for ahead of the vectors)
    auto angle = [&](int i, double& pos, float& freq) {
      const int k = (int)fast_div((uint32_t)i, g.half_magic, g.half_shift), p = i - k * half;
      int64_t bb = b0, tok = tok0 + k;
      while (tok >= g.tokens) { tok -= g.tokens; bb++; }
      pos = (double)load_index(g.positions, bb * g.position_stride + tok, g.wide_pos);
      freq = g.inv_freq[p];
    };
    double pos = 0.0;
    float freq = 0.f;
    if (tid < span * half) angle(tid, pos, freq);
    fetch(0);
    __syncthreads();
    for (int i = tid; i < span * half; i += kRopeThreads) {
      if (i != tid) angle(i, pos, freq);
      const double rev = pos * ((double)freq * 0.15915494309189533577);
      // (half turns as fp32, and what that leaves off, which is as much as sine and cosine's own rounding)
      const double turns = 2.0 * (rev - rint(rev));
      const float half_turns = (float)turns, rest = (float)((turns - (double)half_turns) * 3.14159265358979323846);
      float sn, cn;
      sincospif(half_turns, &sn, &cn);
      cs[i] = float2{__builtin_fmaf(-rest, sn, cn), __builtin_fmaf(rest, cn, sn)};
    }
    __syncthreads();
    for (int first = 0; first < g.per_chunk; first += R * kSlots) {
      if (first > 0) fetch(first);
#pragma unroll
      for (int u = 0; u < R; u++) {
        const bool ok = first + u * kSlots + slot < n;
        float xa[NJ][E], xb[NJ][E];
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; j++) {
          Row::piece(x[u].a[j], ok && a[j] >= 0, xa[j]);
          Row::piece(x[u].b[j], ok && b[j] >= 0, xb[j]);
#pragma unroll
          for (int e = 0; e < E; e++) ss = __builtin_fmaf(xa[j][e], xa[j][e], __builtin_fmaf(xb[j][e], xb[j][e], ss));
        }
        // (with eps = 0 lanes without a vector would add 0 * infinity to the weights' sums)
        const float sq = group_sum<LPV>(ss) / (float)g.d + g.eps, r = ok ? 1.f / sqrtf(sq) : 0.f;
        if constexpr (!GRAD) {
          if (ok) {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
#pragma unroll
              for (int e = 0; e < E; e++) {
                xa[j][e] *= r * wa[j][e];
                xb[j][e] *= r * wb[j][e];
              }
              turn<E, 1>(g, angles[u], a[j], b[j], xa[j], xb[j]);
              if (a[j] >= 0) store_piece<T, E>(to[u] + a[j], xa[j]);
              if (b[j] >= 0) store_piece<T, E>(to[u] + b[j], xb[j]);
            }
          }
        } else {
          float ya[NJ][E], yb[NJ][E], dot = 0.f;
#pragma unroll
          for (int j = 0; j < NJ; j++) {
            Row::piece(y[u].a[j], ok && a[j] >= 0, ya[j]);
            Row::piece(y[u].b[j], ok && b[j] >= 0, yb[j]);
            turn<E, -1>(g, angles[u], a[j], b[j], ya[j], yb[j]);
#pragma unroll
            for (int e = 0; e < E; e++) {
              xa[j][e] *= r;  // n
              xb[j][e] *= r;
              da[j][e] = __builtin_fmaf(ya[j][e], xa[j][e], da[j][e]);
              db[j][e] = __builtin_fmaf(yb[j][e], xb[j][e], db[j][e]);
              ya[j][e] *= wa[j][e];
              yb[j][e] *= wb[j][e];
              dot = __builtin_fmaf(ya[j][e], xa[j][e], __builtin_fmaf(yb[j][e], xb[j][e], dot));
            }
          }
          dot = group_sum<LPV>(dot) / (float)g.d;
          if (ok) {
#pragma unroll
            for (int j = 0; j < NJ; j++) {
#pragma unroll
              for (int e = 0; e < E; e++) {
                ya[j][e] = r * (ya[j][e] - xa[j][e] * dot);
                yb[j][e] = r * (yb[j][e] - xb[j][e] * dot);
              }
              if (a[j] >= 0) store_piece<T, E>(to[u] + a[j], ya[j]);
              if (b[j] >= 0) store_piece<T, E>(to[u] + b[j], yb[j]);
            }
          }
        }
      }
    }
  }

  if constexpr (GRAD) {
    // the workgroup's part of d_w: lanes that hold the same elements of different vectors, then
    // the wavefronts, always in this order
    float* acc = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NJ; j++)
#pragma unroll
      for (int e = 0; e < E; e++) {
#pragma unroll
        for (int m = LPV; m < kWave; m *= 2) {
          da[j][e] += shfl_xor_f32(da[j][e], m);
          db[j][e] += shfl_xor_f32(db[j][e], m);
        }
        if (tid % kWave < LPV) {
          const int wv = tid / kWave;
          if (a[j] >= 0) acc[wv * g.d + a[j] + e] = da[j][e];
          if (b[j] >= 0) acc[wv * g.d + b[j] + e] = db[j][e];
        }
      }
    __syncthreads();
    float* to = g.partial + (int64_t)blockIdx.x * g.d;
    for (int i = tid; i < g.d; i += kRopeThreads) {
      float x = acc[i];
#pragma unroll
      for (int wv = 1; wv < kRopeThreads / kWave; wv++) x += acc[wv * g.d + i];
      to[i] = x;
    }
  }
}

// d_w = the sum of the workgroups' parts: eight columns of a side per workgroup, 32 rows side by side and
// eight of a lane's own on the way at a time.
__global__ __launch_bounds__(256) void rope_weights_kernel(const float* partial, int64_t blocks_q, int64_t blocks_k,
                                                           int d, float* d_w_q, float* d_w_k) {
  __shared__ float acc[32][9];
  float* to = blockIdx.y ? d_w_k : d_w_q;
  if (to == nullptr) return;
  const int64_t first = blockIdx.y ? blocks_q : 0, n = blockIdx.y ? blocks_k : blocks_q;
  const int col = threadIdx.x % 8, row = threadIdx.x / 8, i = blockIdx.x * 8 + col;
  const float* from = partial + first * d + (i < d ? i : 0);
  float x = 0.f;
  for (int64_t r = row; r < n; r += 8 * 32) {
    float y[8];
#pragma unroll
    for (int u = 0; u < 8; u++) y[u] = from[(r + 32 * u < n ? r + 32 * u : r) * d];
#pragma unroll
    for (int u = 0; u < 8; u++) x += r + 32 * u < n ? y[u] : 0.f;
  }
  acc[row][col] = x;
  __syncthreads();
  if (row == 0 && i < d) {
#pragma unroll
    for (int r = 1; r < 32; r++) x += acc[r][col];
    to[i] = x;
  }
}

namespace {

void set_strides(int64_t (&to)[3], const spfa_heads_t& h) {
  to[0] = h.stride_batch;
  to[1] = h.stride_token;
  to[2] = h.stride_head;
}

// Vectors a workgroup takes at a time, and the LDS that needs: four rounds of its lanes, fewer where
// there are too few vectors to fill the device with that or the angles would not fit.
int rope_chunk(const RopeArgs& g, int slots, int64_t min_heads, size_t* lds) {
  const int half = g.rot / 2;
  const int64_t all = g.side[0].vectors + g.side[1].vectors;
  int rounds = 4;
  auto bytes = [&](int r) { return (size_t)(((int64_t)r * slots - 2) / min_heads + 2) * half * sizeof(float2); };
  while (rounds > 1 && (all < (int64_t)1024 * rounds * slots || bytes(rounds) > (size_t)kRopeLds)) rounds /= 2;
  *lds = bytes(rounds);
  return rounds * slots;
}

template <typename T, int LPV, int E, int NJ, bool GRAD>
int rope_launch(RopeArgs& g, hipStream_t stream) {
  constexpr int kSlots = kRopeThreads / LPV;
  int64_t min_heads = INT64_MAX;
  for (const RopeSide& s : g.side)
    if (s.vectors > 0 && s.heads < min_heads) min_heads = s.heads;
  size_t lds = 0;
  g.per_chunk = rope_chunk(g, kSlots, min_heads, &lds);
  const int64_t all = g.side[0].vectors + g.side[1].vectors;
  for (RopeSide& s : g.side) {
    fast_divider((int32_t)s.heads, &s.magic, &s.shift);
    s.chunks = (s.vectors + g.per_chunk - 1) / g.per_chunk;
    s.blocks = s.chunks;
    if (GRAD) {
      // shares of kRopeBlocks by size, at least one
      int64_t share = (int64_t)((double)kRopeBlocks * (double)s.vectors / (double)all);
      if (share < 1) share = 1;
      if (s.blocks > share) s.blocks = share;
    } else if (s.blocks > (1 << 22)) {
      s.blocks = 1 << 22;  // (a grid holds fewer than 2^32 work items)
    }
  }
  const size_t need = GRAD ? (size_t)4 * g.d * sizeof(float) : 0;
  if (lds < need) lds = need;
  const int64_t blocks = g.side[0].blocks + g.side[1].blocks;
  if constexpr (E > 1)
    if (g.per_chunk >= kRopeBatch * kSlots) {
      rope_kernel<T, LPV, E, NJ, kRopeBatch, GRAD><<<dim3((unsigned)blocks), dim3(kRopeThreads), lds, stream>>>(g);
      return launch_status();
    }
  rope_kernel<T, LPV, E, NJ, 1, GRAD><<<dim3((unsigned)blocks), dim3(kRopeThreads), lds, stream>>>(g);
  return launch_status();
}

template <typename T, bool GRAD>
int rope_pick(RopeArgs& g, bool aligned, hipStream_t stream) {
  constexpr int E = 16 / (int)sizeof(T);
  const bool whole = g.d % (2 * E) == 0 && (g.interleaved || g.rot % (2 * E) == 0);
  const int lanes = g.d / (2 * E);
  if (aligned && whole && lanes <= kWave) {
    if (lanes <= 4) return rope_launch<T, 4, E, 1, GRAD>(g, stream);
    if (lanes <= 8) return rope_launch<T, 8, E, 1, GRAD>(g, stream);
    if (lanes <= 16) return rope_launch<T, 16, E, 1, GRAD>(g, stream);
    if (lanes <= 32) return rope_launch<T, 32, E, 1, GRAD>(g, stream);
    return rope_launch<T, 64, E, 1, GRAD>(g, stream);
  }
  if (g.d <= 256) return rope_launch<T, 64, 1, 2, GRAD>(g, stream);
  return rope_launch<T, 64, 1, 8, GRAD>(g, stream);
}

template <bool GRAD>
int rope_run(RopeArgs& g, int dtype, bool aligned, hipStream_t stream) {
  switch (dtype) {
    case SPFA_DTYPE_F32: return rope_pick<float, GRAD>(g, aligned, stream);
    case SPFA_DTYPE_F16: return rope_pick<f16, GRAD>(g, aligned, stream);
    default: return rope_pick<bf16, GRAD>(g, aligned, stream);
  }
}

int rope_check(const spfa_rope_t* p) {
  if (p == nullptr) return SPFA_ERR_BAD_ARG;
  if (p->d < 1 || p->d > 1024) return SPFA_ERR_EMB_TOO_LARGE;
  if (p->dtype != SPFA_DTYPE_F32 && p->dtype != SPFA_DTYPE_F16 && p->dtype != SPFA_DTYPE_BF16) return SPFA_ERR_UNSUPPORTED;
  if (p->w_dtype != p->dtype && p->w_dtype != SPFA_DTYPE_F32) return SPFA_ERR_UNSUPPORTED;
  if (p->batch < 0 || p->tokens < 0 || p->heads_q < 0 || p->heads_k < 0) return SPFA_ERR_BAD_ARG;
  if (p->heads_q > (1 << 20) || p->heads_k > (1 << 20)) return SPFA_ERR_BAD_ARG;
  if (p->rot < 0 || p->rot > p->d || p->rot % 2) return SPFA_ERR_BAD_ARG;
  if (p->position_bytes != 4 && p->position_bytes != 8) return SPFA_ERR_BAD_ARG;
  // (the vectors' number, and that times 2048, fit 64 bits; no product here leaves them)
  const int64_t most = INT64_MAX / 2048 / ((p->heads_q > p->heads_k ? p->heads_q : p->heads_k) + 1);
  if (p->batch > most || (p->batch > 0 && p->tokens > most / p->batch)) return SPFA_ERR_BAD_ARG;
  return SPFA_OK;
}

bool empty(const spfa_rope_t* p) { return p->batch == 0 || p->tokens == 0 || p->heads_q + p->heads_k == 0; }

// The kernel's arguments from the call's; `out` / `dy` by side.  False: a tensor is missing.
bool rope_args(const spfa_rope_t* p, const spfa_heads_t* const (&out)[2], const spfa_heads_t* const (&dy)[2],
               RopeArgs& g, bool* aligned) {
  const spfa_heads_t x[2] = {p->q, p->k};
  const void* w[2] = {p->w_q, p->w_k};
  const int64_t heads[2] = {p->heads_q, p->heads_k};
  const int size = p->dtype == SPFA_DTYPE_F32 ? 4 : 2;
  *aligned = true;
  g = RopeArgs{};
  for (int i = 0; i < 2; i++) {
    RopeSide& s = g.side[i];
    s.heads = heads[i] > 0 ? heads[i] : 1;
    s.vectors = p->batch * p->tokens * heads[i];
    if (s.vectors == 0) continue;
    if (out[i] == nullptr || out[i]->data == nullptr || x[i].data == nullptr) return false;
    s.x = x[i].data;
    s.out = out[i]->data;
    s.w = w[i];
    s.w_how = w[i] == nullptr ? kNoWeights : p->w_dtype == p->dtype ? kOwnWeights : kFloatWeights;
    *aligned = *aligned && ((uintptr_t)w[i] & 15) == 0;
    set_strides(s.xs, x[i]);
    set_strides(s.os, *out[i]);
    *aligned = *aligned && heads_aligned(x[i], size, p->batch > 1) && heads_aligned(*out[i], size, p->batch > 1);
    if (dy[i] != nullptr) {
      if (dy[i]->data == nullptr) return false;
      s.dy = dy[i]->data;
      set_strides(s.ds, *dy[i]);
      *aligned = *aligned && heads_aligned(*dy[i], size, p->batch > 1);
    }
  }
  if (p->positions == nullptr && p->rot > 0) return false;
  if (p->inv_freq == nullptr && p->rot > 0) return false;
  g.tokens = p->tokens;
  g.position_stride = p->position_stride;
  g.positions = p->positions;
  g.inv_freq = p->inv_freq;
  g.eps = p->eps;
  g.d = (int32_t)p->d;
  g.rot = (int32_t)p->rot;
  g.wide_pos = p->position_bytes == 8;
  g.interleaved = p->interleaved != 0;
  if (g.rot > 0) fast_divider(g.rot / 2, &g.half_magic, &g.half_shift);
  return true;
}

}  // namespace
}  // namespace spfa

using namespace spfa;

extern "C" int spfa_qk_norm_rope_forward(const spfa_rope_t* p, const spfa_heads_t* q_out, const spfa_heads_t* k_out,
                                         void* stream) {
  int rc = rope_check(p);
  if (rc) return rc;
  if (empty(p)) return SPFA_OK;
  RopeArgs g;
  bool aligned;
  const spfa_heads_t* const out[2] = {q_out, k_out};
  const spfa_heads_t* const none[2] = {nullptr, nullptr};
  if (!rope_args(p, out, none, g, &aligned)) return SPFA_ERR_BAD_ARG;
  return rope_run<false>(g, p->dtype, aligned, (hipStream_t)stream);
}

extern "C" size_t spfa_qk_norm_rope_backward_workspace_bytes(int64_t batch, int64_t tokens, int64_t heads_q,
                                                             int64_t heads_k, int64_t d) {
  if (batch <= 0 || tokens <= 0 || heads_q < 0 || heads_k < 0 || d < 1 || d > 1024) return 256;
  return (size_t)(kRopeBlocks + 2) * (size_t)d * sizeof(float) + 256;
}

extern "C" int spfa_qk_norm_rope_backward(const spfa_rope_t* p, const spfa_heads_t* d_q_out, const spfa_heads_t* d_k_out,
                                          const spfa_heads_t* d_q, const spfa_heads_t* d_k, float* d_w_q, float* d_w_k,
                                          void* workspace, size_t workspace_bytes, void* stream) {
  int rc = rope_check(p);
  if (rc) return rc;
  RopeArgs g;
  bool aligned = true;
  const spfa_heads_t* const out[2] = {d_q, d_k};
  const spfa_heads_t* const dy[2] = {d_q_out, d_k_out};
  const bool none = empty(p);
  if (!none) {
    if ((p->heads_q > 0 && d_q_out == nullptr) || (p->heads_k > 0 && d_k_out == nullptr)) return SPFA_ERR_BAD_ARG;
    if (!rope_args(p, out, dy, g, &aligned)) return SPFA_ERR_BAD_ARG;
    if (workspace == nullptr || ((uintptr_t)workspace & 255) ||
        workspace_bytes < spfa_qk_norm_rope_backward_workspace_bytes(p->batch, p->tokens, p->heads_q, p->heads_k, p->d))
      return SPFA_ERR_WORKSPACE;
    g.partial = (float*)workspace;
    rc = rope_run<true>(g, p->dtype, aligned, (hipStream_t)stream);
    if (rc) return rc;
  } else {
    g = RopeArgs{};  // no vectors: the weights' gradients are zeros
  }
  if (d_w_q == nullptr && d_w_k == nullptr) return SPFA_OK;
  rope_weights_kernel<<<dim3((unsigned)((p->d + 7) / 8), 2), dim3(256), 0, (hipStream_t)stream>>>(
      g.partial, g.side[0].blocks, g.side[1].blocks, (int)p->d, d_w_q, d_w_k);
  return launch_status();
}
