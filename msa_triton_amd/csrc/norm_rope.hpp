// A row of D elements (one head of one token) held by a run of LPR lanes, for the kernels that norm and
// rotate rows: a lane has VEC elements of the first and VEC of the second half of the rotated part, or of the
// two halves of the rest, so that the pairs the rotation mixes are in one lane.
#pragma once
#include "mfma_util.hpp"

namespace msa {

constexpr int kNormThreads = 256;

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

struct RopeTable {
  const float* table;  // [rows][2 * half]: cosines, then sines
  int64_t rows;
  int half;  // rotated dims / 2
};

// Sum over runs of LPR lanes.
template <int LPR>
__device__ __forceinline__ float run_sum(float v) {
#define MSA_DPP_ADD(CTRL) \
  v += __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(v), CTRL, 0xF, 0xF, false));
  if constexpr (LPR >= 2) MSA_DPP_ADD(0xB1)   // quad_perm [1, 0, 3, 2]
  if constexpr (LPR >= 4) MSA_DPP_ADD(0x4E)   // quad_perm [2, 3, 0, 1]
  if constexpr (LPR >= 8) MSA_DPP_ADD(0x141)  // row_half_mirror
  if constexpr (LPR >= 16) MSA_DPP_ADD(0x140) // row_mirror
#undef MSA_DPP_ADD
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16, kWave);
  if constexpr (LPR >= 64) v += __shfl_xor(v, 32, kWave);
  return v;
}

template <int DT, int VEC>
__device__ __forceinline__ void load_vec(const void* __restrict__ p, int64_t i, float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    v[0] = load_as_f32<DT>(p, i);
  } else if constexpr (DT == kF32) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + i);
    const float4 x = s[0], y = s[1];
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w, v[4] = y.x, v[5] = y.y, v[6] = y.z, v[7] = y.w;
  } else {
    const uint4 x = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + i);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[2 * j] = lo16_f32<DT>(w[j]), v[2 * j + 1] = hi16_f32<DT>(w[j]);
  }
}

template <int DT, int VEC>
__device__ __forceinline__ void store_vec(void* __restrict__ p, int64_t i, const float (&v)[VEC]) {
  if constexpr (VEC == 1) {
    store_from_f32<DT>(p, i, v[0]);
  } else if constexpr (DT == kF32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      w[j] = DT == kF16 ? cvt_pk_f16(v[2 * j], v[2 * j + 1]) : cvt_pk_bf16(v[2 * j], v[2 * j + 1]);
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p) + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// The two element runs [a, a + VEC) and [b, b + VEC) of pair chunk `p` of a row, and whether the
// rotation mixes them. ok: the chunk exists; b_ok: its second run does (the rest may be odd).
struct PairChunk {
  int a, b;
  bool turned, ok, b_ok;
};
template <int VEC>
__device__ __forceinline__ PairChunk pair_chunk(int p, int half, int dim) {
  const int hc = half / VEC;
  if (p < hc) return PairChunk{p * VEC, p * VEC + half, true, true, true};
  const int rest = dim - 2 * half, rc = (rest + 2 * VEC - 1) / (2 * VEC), a = 2 * half + (p - hc) * VEC;
  const bool ok = p - hc < rc;
  return PairChunk{a, a + rc * VEC, false, ok, ok && a + rc * VEC < dim};
}

// One row's rotation factors for a pair chunk: (1, 0) past rot, NaN where the position has no table row.
template <int VEC>
__device__ __forceinline__ void load_turn(const RopeTable& R, const PairChunk& pc, int pos, float (&co)[VEC],
                                          float (&si)[VEC]) {
  const bool known = pos >= 0 && pos < R.rows;
#pragma unroll
  for (int j = 0; j < VEC; ++j) co[j] = pc.turned ? __builtin_nanf("") : 1.f, si[j] = 0.f;
  if (pc.turned && known) {
    const float* row = R.table + static_cast<int64_t>(pos) * (2 * R.half) + pc.a;
    load_vec<kF32, VEC>(row, 0, co);
    load_vec<kF32, VEC>(row, R.half, si);
  }
}

__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, double b, double c) { return fma(a, b, c); }

// A pair chunk rotated in place, or back. Dims past rot stay as they are: a product with a sine of 0 would carry a value
// that is not finite over to the dim beside it. (The multiply-adds are written out: every kernel gives the same bits.)
template <int VEC, typename T>
__device__ __forceinline__ void turn(const PairChunk& pc, const float (&co)[VEC], const float (&si)[VEC], T (&a)[VEC],
                                     T (&b)[VEC]) {
  if (!pc.turned) return;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const T u = a[j], v = b[j];
    a[j] = fused(u, T(co[j]), -(v * si[j]));
    b[j] = fused(u, T(si[j]), v * co[j]);
  }
}
template <int VEC, typename T>
__device__ __forceinline__ void turn_back(const PairChunk& pc, const float (&co)[VEC], const float (&si)[VEC], T (&a)[VEC],
                                          T (&b)[VEC]) {
  if (!pc.turned) return;
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    const T u = a[j], v = b[j];
    a[j] = fused(u, T(co[j]), v * si[j]);
    b[j] = fused(v, T(co[j]), -(u * si[j]));
  }
}

template <int DT, int VEC, int C, int LPR>
struct RowLanes {
  static constexpr int kRows = kNormThreads / LPR;  // rows a workgroup holds at once
  PairChunk pc[C];
  float wa[C][VEC], wb[C][VEC];
  __device__ __forceinline__ RowLanes(const void* w, bool w_f32, int half, int dim) {
    const int l = threadIdx.x % LPR;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      pc[c] = pair_chunk<VEC>(l + c * LPR, half, dim);
#pragma unroll
      for (int j = 0; j < VEC; ++j) wa[c][j] = wb[c][j] = 0.f;
      if (!w) continue;
      if (w_f32) {
        if (pc[c].ok) load_vec<kF32, VEC>(w, pc[c].a, wa[c]);
        if (pc[c].b_ok) load_vec<kF32, VEC>(w, pc[c].b, wb[c]);
      } else {
        if (pc[c].ok) load_vec<DT, VEC>(w, pc[c].a, wa[c]);
        if (pc[c].b_ok) load_vec<DT, VEC>(w, pc[c].b, wb[c]);
      }
    }
  }
  // A row's pieces as they are in memory, and their values.
  static constexpr int kWords = VEC == 8 && DT == kF32 ? 2 : 1;  // 16-byte words of VEC values
  struct Raw {
    uint4 a[C][kWords], b[C][kWords];
  };
  static __device__ __forceinline__ void fetch_vec(const void* p, int64_t i, bool live, uint4 (&w)[kWords]) {
#pragma unroll
    for (int k = 0; k < kWords; ++k) w[k] = make_uint4(0u, 0u, 0u, 0u);
    if (!live) return;
    if constexpr (VEC == 8) {
      const uint4* s = reinterpret_cast<const uint4*>(static_cast<const char*>(p) + i * (DT == kF32 ? 4 : 2));
#pragma unroll
      for (int k = 0; k < kWords; ++k) w[k] = s[k];
    } else if constexpr (DT == kF32) {
      w[0].x = static_cast<const uint32_t*>(p)[i];
    } else {
      w[0].x = static_cast<const uint16_t*>(p)[i];
    }
  }
  __device__ __forceinline__ Raw fetch(const void* p, int64_t at, bool live) const {
    Raw r;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      fetch_vec(p, at + pc[c].a, live && pc[c].ok, r.a[c]);
      fetch_vec(p, at + pc[c].b, live && pc[c].b_ok, r.b[c]);
    }
    return r;
  }
  template <typename T>
  static __device__ __forceinline__ void unpack_vec(const uint4 (&w)[kWords], T (&v)[VEC]) {
    const uint4 x = w[0], y = w[kWords - 1];
    const uint32_t u[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      if constexpr (DT == kF32) v[j] = __uint_as_float(u[j]);
      else v[j] = j & 1 ? hi16_f32<DT>(u[j >> 1]) : lo16_f32<DT>(u[j >> 1]);
    }
  }
  template <typename T>
  static __device__ __forceinline__ void unpack(const Raw& r, T (&a)[C][VEC], T (&b)[C][VEC]) {
#pragma unroll
    for (int c = 0; c < C; ++c) unpack_vec(r.a[c], a[c]), unpack_vec(r.b[c], b[c]);
  }
  // Whether an element is an infinity or a NaN (16-bit types).
  static __device__ __forceinline__ bool not_finite(const Raw& r) {
    u16x2 m = {0, 0};
#pragma unroll
    for (int c = 0; c < C; ++c)
      for (const uint4& x : {r.a[c][0], r.b[c][0]})
        for (uint32_t w : {x.x, x.y, x.z, x.w})
          m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w & 0x7fff7fffu));
    return (m.x > m.y ? m.x : m.y) >= (DT == kF16 ? 0x7c00 : 0x7f80);
  }
  __device__ __forceinline__ void load(const void* p, int64_t at, bool live, float (&a)[C][VEC], float (&b)[C][VEC]) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[c][j] = b[c][j] = 0.f;
      if (live && pc[c].ok) load_vec<DT, VEC>(p, at + pc[c].a, a[c]);
      if (live && pc[c].b_ok) load_vec<DT, VEC>(p, at + pc[c].b, b[c]);
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t at, const float (&a)[C][VEC], const float (&b)[C][VEC]) const {
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (pc[c].ok) store_vec<DT, VEC>(p, at + pc[c].a, a[c]);
      if (pc[c].b_ok) store_vec<DT, VEC>(p, at + pc[c].b, b[c]);
    }
  }
};

template <int C, int VEC>
__device__ __forceinline__ float sum_products(const float (&a)[C][VEC], const float (&b)[C][VEC],
                                              const float (&u)[C][VEC], const float (&v)[C][VEC]) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) s = fmaf(a[c][j], u[c][j], fmaf(b[c][j], v[c][j], s));
  return s;
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace msa
