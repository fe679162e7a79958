// What the window attention kernels share: which keys a token sees, tiles of packed rows, and matrix
// fragments of 16-bit and fp32 values in one layout.
//
// Token i of a sequence sees the keys j <= i with i - j < window (its window) or j < sinks (the first tokens, which
// stay visible). Rows of a key head are its (token, query head) pairs, token by token, so that the heads
// that share keys share a tile of them, and the keys read for a tile of R rows are those of R / ratio tokens.
#pragma once
#include "mfma_util.hpp"
#include "paged.hpp"

namespace msa {

// A packed tensor [T, heads, D] with free strides over tokens and heads. A tile's rows are at 32-bit offsets from an address
// that the whole wave shares, so 33 tokens lie within 2^30 elements, of queries and their gradients with the heads of a key head
// (near_rows); from one key head to the next, offsets are 64 bits.
struct PackedView {
  const void* base;
  int token, head;  // elements
  __device__ __forceinline__ int64_t at(int64_t t, int h) const { return t * token + static_cast<int64_t>(h) * head; }
};
inline PackedView packed_view(const void* base, const int64_t* strides) {
  return PackedView{base, static_cast<int>(strides[0]), static_cast<int>(strides[1])};
}

struct Visible {
  int window;  // 2^31 - 1: none
  int sinks;
  __device__ __forceinline__ bool operator()(int i, int j) const { return j <= i && (i - j < window || j < sinks); }
  // The first key of the window of token i.
  __device__ __forceinline__ int low(int i) const { return max(0, i - window + 1); }
};

// Tile `tile` of a sequence of n tokens that starts at token `start`.
struct TilePlace {
  int seq, start, n, tile;
};

// Tiles of 2^size_log2 units, `per_token` of them a token, sequence by sequence: sequence s has the numbers from
// cu[s] per_token / size + s on, which leaves each of them at least as many as it has tiles (a number behind its last
// tile stands for nothing), so that no prefix sum over the sequences is needed. tile_numbers() of them in all.
__device__ __forceinline__ TilePlace tile_place(const int32_t* __restrict__ cu, int nseq, int64_t number, int per_token,
                                                int size_log2) {
  const auto first = [&](int s) { return (static_cast<int64_t>(cu[s]) * per_token >> size_log2) + s; };
  const int s = __builtin_amdgcn_readfirstlane(nseq == 1 ? 0 : wave_upper_index(nseq, number, first));
  const int start = cu[s];
  return TilePlace{s, start, cu[s + 1] - start, static_cast<int>(number - first(s))};
}
inline int64_t tile_numbers(int64_t tokens, int64_t nseq, int64_t per_token, int size_log2) {
  return (tokens * per_token >> size_log2) + nseq;
}
constexpr int log2_of(int size) { return size <= 1 ? 0 : 1 + log2_of(size / 2); }

// x / d for x < 2^31.
struct Divisor {
  uint32_t mul;
  int shift, d;
  __device__ __forceinline__ int operator()(int x) const {
    return shift < 0 ? x : static_cast<int>(__umulhi(static_cast<uint32_t>(x), mul) >> shift);
  }
};
inline Divisor divisor_of(int64_t d) {
  int bits = 0;  // d <= 2^bits
  while ((int64_t{1} << bits) < d) ++bits;
  if (bits == 0) return Divisor{0, -1, 1};
  return Divisor{static_cast<uint32_t>(((uint64_t{1} << (31 + bits)) + d - 1) / d), bits - 1, static_cast<int>(d)};
}

// The largest (the sum) of a value over the four quarters of a wave (lanes c, c + 16, c + 32, c + 48), by row swaps in the
// vector unit.
__device__ __forceinline__ float quarters_max(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// A running maximum is only raised when a row passes it by this much (log2): weights stay below 2^kSlack, sums and outputs are
// rescaled in few steps. In fp16 weights are held times 2^(15 - kSlack), so that the largest is at most 2^15.
constexpr float kSlack = 8.f;
// The same of raw dots, which are times `factor` in log2; finite, so that a first key raises a maximum of -inf.
__device__ __forceinline__ float raw_slack(float factor) { return fminf(kSlack / factor, 3.402823466e38f); }

// A fragment, times -1 where `turn` says so.
template <int DT, class F>
__device__ __forceinline__ F turned(F f, bool turn) {
  if (!turn) return f;
  if constexpr (DT == kF32) {
    f.a = -f.a, f.b = -f.b;
  } else {
    uint4 w = __builtin_bit_cast(uint4, f.v);
    w.x ^= 0x80008000u, w.y ^= 0x80008000u, w.z ^= 0x80008000u, w.w ^= 0x80008000u;
    f.v = __builtin_bit_cast(bf16x8, w);
  }
  return f;
}

// ---- fragments: eight values of a lane. In 16 bits one 16x16x32 product takes them; in fp32 eight 16x16x4 products do,
// element j of all lanes in the j-th (its four k are those of the lanes' quarters, for both operands alike).

template <int DT>
struct Fragment {
  using Element = uint16_t;
  static constexpr int kPad = 16;  // elements between rows of a tile: transposed reads of 4 rows meet no bank twice
  bf16x8 v;
};
template <>
struct Fragment<kF32> {
  using Element = float;
  static constexpr int kPad = 4;
  f32x4 a, b;
};

template <int DT>
__device__ __forceinline__ f32x4 product(const Fragment<DT>& x, const Fragment<DT>& y, f32x4 c) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.a[j], y.a[j], c, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x.b[j], y.b[j], c, 0, 0, 0);
    return c;
  } else {
    return mfma_t<DT>(x.v, y.v, c);
  }
}

// Eight consecutive values.
template <int DT>
__device__ __forceinline__ Fragment<DT> fragment_at(const typename Fragment<DT>::Element* p) {
  Fragment<DT> f;
  if constexpr (DT == kF32) {
    f.a = *reinterpret_cast<const f32x4*>(p);
    f.b = *reinterpret_cast<const f32x4*>(p + 4);
  } else {
    f.v = __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4*>(p));
  }
  return f;
}
template <int DT>
__device__ __forceinline__ Fragment<DT> no_fragment() {
  Fragment<DT> f;
  if constexpr (DT == kF32) f.a = f.b = f32x4{0.f, 0.f, 0.f, 0.f};
  else f.v = zero_frag();
  return f;
}

// Column n0 + c of a row-major LDS tile, rows k0 + 4 q4 + (0..3) and k0 + 16 + 4 q4 + (0..3): the order in which
// the two 16-row products above it leave their rows in a lane.
template <int DT>
__device__ __forceinline__ Fragment<DT> column_fragment(const typename Fragment<DT>::Element* tile, int stride, int k0, int n0,
                                                        int c, int q4) {
  Fragment<DT> f;
  if constexpr (DT == kF32) {
    const float* p = tile + (k0 + 4 * q4) * stride + n0 + c;
#pragma unroll
    for (int j = 0; j < 4; ++j) f.a[j] = p[j * stride], f.b[j] = p[(16 + j) * stride];
  } else {
    f.v = frag_tr(tile, stride, k0 + 4 * q4, k0 + 16 + 4 * q4, n0, c);
  }
  return f;
}

// Eight fp32 results as an operand, each rounded once to 16 bits.
template <int DT>
__device__ __forceinline__ Fragment<DT> pack_fragment(const float (&x)[8]) {
  Fragment<DT> f;
  if constexpr (DT == kF32) {
    f.a = f32x4{x[0], x[1], x[2], x[3]};
    f.b = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    auto two = [](float a, float b) { return DT == kF16 ? cvt_pk_f16(a, b) : cvt_pk_bf16(a, b); };
    f.v = __builtin_bit_cast(bf16x8, make_uint4(two(x[0], x[1]), two(x[2], x[3]), two(x[4], x[5]), two(x[6], x[7])));
  }
  return f;
}

// What that rounding left out, rounded to 16 bits as well: the second term of each value, to 2^-17 (fp16: 2^-22) of it.
template <int DT>
__device__ __forceinline__ Fragment<DT> second_terms(const Fragment<DT>& first, const float (&x)[8]) {
  static_assert(DT != kF32, "nothing is left out");
  const uint4 w = __builtin_bit_cast(uint4, first.v);
  auto two = [](uint32_t h, float a, float b) {
    return DT == kF16 ? cvt_pk_f16(sub_lo_half_f16(h, a), sub_hi_half_f16(h, b)) : cvt_pk_bf16(sub_lo_half(h, a), sub_hi_half(h, b));
  };
  Fragment<DT> f;
  f.v = __builtin_bit_cast(bf16x8, make_uint4(two(w.x, x[0], x[1]), two(w.y, x[2], x[3]), two(w.z, x[4], x[5]), two(w.w, x[6], x[7])));
  return f;
}

// pack_fragment in two halves: elements 4 half .. 4 half + 3 of f.
template <int DT>
__device__ __forceinline__ void pack_half(Fragment<DT>& f, int half, f32x4 x) {
  if constexpr (DT == kF32) {
    if (half == 0) f.a = x; else f.b = x;
  } else {
    auto two = [](float a, float b) { return DT == kF16 ? cvt_pk_f16(a, b) : cvt_pk_bf16(a, b); };
    uint4 w = __builtin_bit_cast(uint4, f.v);
    if (half == 0) w.x = two(x[0], x[1]), w.y = two(x[2], x[3]);
    else w.z = two(x[0], x[1]), w.w = two(x[2], x[3]);
    f.v = __builtin_bit_cast(bf16x8, w);
  }
}

// Rows [0, ROWS) of a tile by a workgroup of 256: 16-byte pieces through registers, zeros past D.
template <int DT, int DP, int ROWS>
struct TileLoad {
  using E = typename Fragment<DT>::Element;
  static constexpr int kPer = 16 / sizeof(E);   // values of a piece
  static constexpr int kLanes = DP / kPer;      // pieces of a row
  static constexpr int kAll = ROWS * kLanes;
  static constexpr int kPieces = (kAll + 255) / 256;
  uint4 r[kPieces];
  static __device__ __forceinline__ int piece(int p) {
    const int i = p * 256 + static_cast<int>(threadIdx.x);
    return kAll % 256 == 0 ? i : min(i, kAll - 1);
  }
  static __device__ __forceinline__ int row(int p) { return piece(p) / kLanes; }
  static __device__ __forceinline__ int dim(int p) { return piece(p) % kLanes * kPer; }
  // offset(row): elements from base to the row (to any row that exists where it is not wanted)
  template <class Offset>
  __device__ __forceinline__ void load_near(int D, const E* base, Offset offset) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p)
      r[p] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(base) +
                                             static_cast<uint32_t>(offset(row(p)) + (dim(p) < D ? dim(p) : 0)) * uint32_t{sizeof(E)});
  }
  // at(row): address of the row in memory (of any row that exists where it is not wanted)
  template <class At>
  __device__ __forceinline__ void load(int D, At at) {
#pragma unroll
    for (int p = 0; p < kPieces; ++p) r[p] = *reinterpret_cast<const uint4*>(at(row(p)) + (dim(p) < D ? dim(p) : 0));
  }
  __device__ __forceinline__ void store(E* tile, int stride, int D) const {
    if (D == DP) {
#pragma unroll
      for (int p = 0; p < kPieces; ++p) *reinterpret_cast<uint4*>(tile + row(p) * stride + dim(p)) = r[p];
      return;
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p)  // (a last piece that several threads hold is written by all of them alike)
      *reinterpret_cast<uint4*>(tile + row(p) * stride + dim(p)) = dim(p) < D ? r[p] : make_uint4(0u, 0u, 0u, 0u);
  }
};

// One value of a row in memory.
template <int DT>
__device__ __forceinline__ float value_at(const typename Fragment<DT>::Element* p, int64_t i) {
  return load_as_f32<DT>(p, i);
}

// The dot of two rows in memory, 16 bytes at a time.
template <int DT>
__device__ __forceinline__ float row_dot(const typename Fragment<DT>::Element* a, const typename Fragment<DT>::Element* b, int D) {
  float x = 0.f;
  for (int d = 0; d < D; d += DT == kF32 ? 4 : 8) {
    const uint4 u = *reinterpret_cast<const uint4*>(a + d), w = *reinterpret_cast<const uint4*>(b + d);
    const uint32_t us[4] = {u.x, u.y, u.z, u.w}, ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kF32) {
        x = fmaf(__uint_as_float(us[i]), __uint_as_float(ws[i]), x);
      } else {
        x = fmaf(lo16_f32<DT>(us[i]), lo16_f32<DT>(ws[i]), x);
        x = fmaf(hi16_f32<DT>(us[i]), hi16_f32<DT>(ws[i]), x);
      }
    }
  }
  return x;
}

// Four results, rounded once, at p (8 or 16 bytes, aligned).
template <int DT>
__device__ __forceinline__ void store4(typename Fragment<DT>::Element* p, f32x4 x) {
  if constexpr (DT == kF32) *reinterpret_cast<f32x4*>(p) = x;
  else if constexpr (DT == kF16) *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_f16(x[0], x[1]), cvt_pk_f16(x[2], x[3]));
  else *reinterpret_cast<uint2*>(p) = make_uint2(cvt_pk_bf16(x[0], x[1]), cvt_pk_bf16(x[2], x[3]));
}

// What rounding to 16 bits left out of four results: x = its rounding + this, to 2^-17 of x.
template <int DT>
__device__ __forceinline__ f32x4 left_out(f32x4 x) {
  f32x4 y;
  if constexpr (DT == kF16) {
    const uint32_t a = cvt_pk_f16(x[0], x[1]), b = cvt_pk_f16(x[2], x[3]);
    y = f32x4{sub_lo_half_f16(a, x[0]), sub_hi_half_f16(a, x[1]), sub_lo_half_f16(b, x[2]), sub_hi_half_f16(b, x[3])};
  } else {
    const uint32_t a = cvt_pk_bf16(x[0], x[1]), b = cvt_pk_bf16(x[2], x[3]);
    y = f32x4{sub_lo_half(a, x[0]), sub_hi_half(a, x[1]), sub_lo_half(b, x[2]), sub_hi_half(b, x[3])};
  }
  return y;
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < __builtin_inff(); }

constexpr float kLn2Window = 0.69314718055994531f, kLog2e = 1.4426950408889634f;

// heads: those of a tile's rows (0: all rows are of one).
inline bool near_rows(const int64_t* strides, int64_t heads) {
  return strides[0] >= 0 && strides[1] >= 0 && strides[0] < (1 << 25) && strides[1] < (1 << 30) &&
         33 * strides[0] + heads * strides[1] < (1 << 30);
}

// scale * log2(e) is held in fp32
inline bool valid_scale(double scale) { return scale >= -2e38 && scale <= 2e38; }

// What the packed entry points check. strides: token and head strides of q, k, v (elements).
inline bool valid_window_call(const void* q, const void* k, const void* v, int32_t dtype, const int64_t* strides,
                              const int32_t* cu, int64_t num_seqs, int64_t tokens, int64_t q_heads, int64_t groups,
                              int64_t dim, int64_t window, int64_t sinks, double scale) {
  if (!q || !k || !v || !strides || !cu || num_seqs <= 0 || num_seqs > 0x3fffffff || tokens < 0 || tokens > 0x7fffffff ||
      groups <= 0 || q_heads <= 0 || q_heads % groups || q_heads >= (1 << 20) || dim <= 0 || window < 0 || sinks < 0 ||
      !valid_scale(scale) || (dtype != kF32 && dtype != kF16 && dtype != kBF16))
    return false;
  const int unit = dtype == kF32 ? 4 : 8;  // 16 bytes
  for (int i = 0; i < 6; ++i)
    if (strides[i] % unit) return false;
  for (int i = 0; i < 6; i += 2)
    if (!near_rows(strides + i, i == 0 ? q_heads / groups : 0)) return false;
  return reinterpret_cast<uintptr_t>(q) % 16 == 0 && reinterpret_cast<uintptr_t>(k) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(v) % 16 == 0;
}
// (rows of a key head are numbered in 32 bits)
inline bool window_supported(int64_t dim, int64_t tokens, int64_t ratio) {
  return dim % 8 == 0 && dim <= 256 && tokens * ratio < 0x7fff0000;
}

// window 0: none
inline Visible visible_of(int64_t window, int64_t sinks) {
  const auto small = [](int64_t x) { return static_cast<int>(x < 0x7fffffff ? x : 0x7fffffff); };
  return Visible{window == 0 ? 0x7fffffff : small(window), small(sinks)};
}

}  // namespace msa
