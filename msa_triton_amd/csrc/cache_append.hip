// New keys, values and index keys written into a paged cache, keys normed and rotated on the way.
//
// A key row passes y = rotate(x / sqrt(mean x^2 + eps) * w) (qk_norm_rope.hip; either part may be left
// out), a value row is copied. A 16-bit cache takes y rounded once, with the bits that m3_qk_norm_rope
// gives. An 8-bit cache (e4m3) takes y / s rounded once, with one scale s for each page and head: the
// smallest power of two with 448 s >= max |y| over the page's new rows, joined by max with the scale of
// the tokens that the page already holds. Where that makes the scale grow, the held tokens are rounded
// again (exact for a power of two, except where they fall below e4m3's normal range). Values that are
// not finite become NaN and do not enter the scale.
//
// y / s is formed in FP64 and rounded to e4m3 once, so that the stored byte is that of the exact y: a value an
// fp32 step away from a rounding border would be off by a whole e4m3 step (2^-3) otherwise. The scale needs the
// page's maximum only, which fp32 gives except next to a border (append_page).
//
// Work: 16-bit rows go to runs of LPR lanes, as in the norm. An 8-bit page, head and side is one
// workgroup's, because its scale is needed before its first byte: one pass over the page's new rows for the
// maximum, one to write them (from registers where they are few, from the caches otherwise). Pages are
// numbered without a list of them: sequence s gets the numbers from cu[s] / page + 2 s on, which leaves room for the two pages that n tokens can
// touch beyond n / page; numbers without a page end at once.
//
// 16 bits: bound by memory (16 272 tokens, 4 heads of 128 and an index head: 20 us, 4.0 TB/s). 8 bits: by the vector work of
// norm, rotation and two roundings (19 700 tokens: 36 us, 2.3 TB/s), and for single tokens by its chain of loads,
// sequence, page, scale (64 tokens: 11 us).
#include "norm_rope.hpp"
#include "paged.hpp"

namespace msa {
namespace {

struct AppendSide {
  const void* x;
  int64_t stride_t, stride_h;
  const void* w;  // null: not normed
  CacheView cache;
  float* scale;  // [P][heads], 8-bit caches
  int heads, dim;
  bool turned;
};

struct AppendArgs {
  AppendSide side[3];  // keys, values, index keys
  uint32_t launch;       // workgroup of this launch's first one
  uint32_t first[3];     // first workgroup of a side's rows
  uint32_t page_blocks;  // workgroups of 8-bit pages, in front
  bool w_f32;
  RopeTable rope;
  PageMap pages;
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  int64_t tokens;
  float eps;
};

// Sum over runs of LPR lanes.
template <int LPR>
__device__ __forceinline__ double run_sum_f64(double v) {
#define MSA_DPP_ADD64(CTRL)                                                                                    \
  {                                                                                                            \
    const uint64_t u = static_cast<uint64_t>(__double_as_longlong(v));                                         \
    const uint32_t lo = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(u), CTRL, 0xF, 0xF, false);       \
    const uint32_t hi = __builtin_amdgcn_update_dpp(0u, static_cast<uint32_t>(u >> 32), CTRL, 0xF, 0xF, false); \
    v += __longlong_as_double(static_cast<long long>((static_cast<uint64_t>(hi) << 32) | lo));                  \
  }
  if constexpr (LPR >= 2) MSA_DPP_ADD64(0xB1)    // quad_perm [1, 0, 3, 2]
  if constexpr (LPR >= 4) MSA_DPP_ADD64(0x4E)    // quad_perm [2, 3, 0, 1]
  if constexpr (LPR >= 8) MSA_DPP_ADD64(0x141)   // row_half_mirror
  if constexpr (LPR >= 16) MSA_DPP_ADD64(0x140)  // row_mirror
#undef MSA_DPP_ADD64
  if constexpr (LPR >= 32) v += __shfl_xor(v, 16, kWave);
  if constexpr (LPR >= 64) v += __shfl_xor(v, 32, kWave);
  return v;
}

// A loaded row's values y in FP64, in place.
template <int VEC, int C, int LPR, class Lanes>
__device__ __forceinline__ void norm_turn(const AppendArgs& A, const AppendSide& S, const Lanes& lanes,
                                          const float (&co)[C][VEC], const float (&si)[C][VEC], double (&a)[C][VEC],
                                          double (&b)[C][VEC]) {
  if (S.w) {
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss = fma(a[c][j], a[c][j], fma(b[c][j], b[c][j], ss));
    const double r = rsqrt(run_sum_f64<LPR>(ss) / S.dim + static_cast<double>(A.eps));
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[c][j] *= r * lanes.wa[c][j], b[c][j] *= r * lanes.wb[c][j];
  }
#pragma unroll
  for (int c = 0; c < C; ++c) turn<VEC>(lanes.pc[c], co[c], si[c], a[c], b[c]);
}

// An fp32 value whose rounding to e4m3 is that of x, and that is above 448 x 2^k where x is: x cut to 21 significant
// bits with what was cut off folded into the last one (e4m3 has 4, 448 has 3).
__device__ __forceinline__ float for_fp8(double x) {
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x));
  const uint32_t high = static_cast<uint32_t>(u >> 32) | (static_cast<uint32_t>(u) ? 1u : 0u);
  return static_cast<float>(__longlong_as_double(static_cast<long long>(static_cast<uint64_t>(high) << 32)));
}

// The magnitude of a finite value times 2^-16, as for_fp8 (products of 16-bit values may pass fp32's range); 0 otherwise.
__device__ __forceinline__ float finite_size(double x) {
  const float m = fabsf(for_fp8(x * 0x1p-16));
  return m < __builtin_inff() ? m : 0.f;  // (NaN: 0)
}

__device__ __forceinline__ uint32_t pack4_fp8(float x0, float x1, float x2, float x3) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(x0, x1, 0, false);
  return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x2, x3, w, true));
}

// VEC values in e4m3.
template <int VEC>
struct Bytes {
  uint32_t w[VEC == 8 ? 2 : 1];
};
template <int VEC>
__device__ __forceinline__ Bytes<VEC> to_fp8(const float (&x)[VEC]) {
  Bytes<VEC> r;
  if constexpr (VEC == 1) {
    r.w[0] = pack4_fp8(x[0], 0.f, 0.f, 0.f);
  } else {
    r.w[0] = pack4_fp8(x[0], x[1], x[2], x[3]);
    r.w[1] = pack4_fp8(x[4], x[5], x[6], x[7]);
  }
  return r;
}
// v * inv rounded once; NaN for what is not finite, or not held by the largest scale.
template <int VEC>
__device__ __forceinline__ Bytes<VEC> to_fp8(const double (&v)[VEC], double inv) {
  float x[VEC];
#pragma unroll
  for (int j = 0; j < VEC; ++j) {
    x[j] = for_fp8(v[j] * inv);
    x[j] = fabsf(x[j]) <= 449.f ? x[j] : __builtin_nanf("");
  }
  return to_fp8(x);
}
template <int VEC>
__device__ __forceinline__ bool same(const Bytes<VEC>& x, const Bytes<VEC>& y) {
  if constexpr (VEC == 1) return x.w[0] == y.w[0];
  else return x.w[0] == y.w[0] && x.w[1] == y.w[1];
}
template <int VEC>
__device__ __forceinline__ void store_bytes(uint8_t* p, const Bytes<VEC>& x) {
  if constexpr (VEC == 1) *p = static_cast<uint8_t>(x.w[0]);
  else *reinterpret_cast<uint2*>(p) = make_uint2(x.w[0], x.w[1]);
}

// The smallest power of two s in [2^-100, 2^127] with 448 s >= amax 2^shift (448 = 1.75 x 2^8); 0 for 0.
__device__ __forceinline__ float scale_for(float amax, int shift = 0) {
  const uint32_t u = __float_as_uint(amax);
  if (u == 0u) return 0.f;
  int k = static_cast<int>(u >> 23) - 127 - 8 + shift + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  k = k < -100 ? -100 : k > 127 ? 127 : k;
  return __uint_as_float(static_cast<uint32_t>(k + 127) << 23);
}

// The largest of three values over the workgroup (three floats of every wave in `lds`).
__device__ __forceinline__ void block_max3(float& x, float& y, float& z, float* lds) {
  x = wave_max_f32(x);
  y = wave_max_f32(y);
  z = wave_max_f32(z);
  __syncthreads();
  if (threadIdx.x % kWave == 0) {
    float* mine = lds + 3 * (threadIdx.x / kWave);
    mine[0] = x, mine[1] = y, mine[2] = z;
  }
  __syncthreads();
  x = fmaxf(fmaxf(lds[0], lds[3]), fmaxf(lds[6], lds[9]));
  y = fmaxf(fmaxf(lds[1], lds[4]), fmaxf(lds[7], lds[10]));
  z = fmaxf(fmaxf(lds[2], lds[5]), fmaxf(lds[8], lds[11]));
}

// One 8-bit page, head and side.
template <int DT, int VEC, int C, int LPR>
__device__ void append_page(const AppendArgs& A, const AppendSide& S, int64_t unit, int head, float* lds) {
  using Lanes = RowLanes<DT, VEC, C, LPR>;
  // the last sequence whose numbers start at or below `unit`
  const int s = wave_upper_index(A.nseq, unit, [&](int i) { return (A.cu[i] >> A.pages.shift) + 2 * static_cast<int64_t>(i); });
  const int64_t start = A.cu[s], n = A.cu[s + 1] - start, context = A.context[s];
  if (context < 0 || n <= 0) return;
  const int64_t p = (context >> A.pages.shift) + (unit - (start >> A.pages.shift) - 2 * static_cast<int64_t>(s));
  const int64_t page_pos = p << A.pages.shift, page_end = page_pos + (int64_t{1} << A.pages.shift);
  if (page_pos >= context + n) return;
  const int64_t first = context > page_pos ? context : page_pos;
  const int kept = static_cast<int>(first - page_pos);  // tokens that the page holds already
  const int rows = static_cast<int>((context + n < page_end ? context + n : page_end) - first);
  const int64_t t0 = start + (first - context);
  const Lanes lanes(S.w, A.w_f32, S.turned ? A.rope.half : 0, S.dim);
  const int row = threadIdx.x / LPR, last_batch = (rows - 1) / Lanes::kRows;
  const bool exact = S.w || S.turned;  // (otherwise y is the input itself)
  auto fetch = [&](int batch) {
    const int i = batch * Lanes::kRows + row;
    return lanes.fetch(S.x, (t0 + i) * S.stride_t + head * S.stride_h, i < rows);
  };
  // The values y of up to kHeld batches of kRows rows stay in registers, their loads in flight at once; those of more rows
  // are read and formed again for the bytes (19 700 prompt tokens, 4 heads of 128: 38, 36 and 40 us with 1, 2 and 4).
  constexpr int kHeld = 2;
  typename Lanes::Raw raw[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (k <= last_batch) raw[k] = fetch(k);
  const int page = A.pages.page_of(s, page_pos);
  if (page < 0) return;
  float* scale = S.scale + static_cast<int64_t>(page) * S.heads + head;
  const float before = kept ? *scale : 0.f;
  auto factors = [&](int i, float (&co)[C][VEC], float (&si)[C][VEC]) {
#pragma unroll
    for (int c = 0; c < C; ++c) load_turn<VEC>(A.rope, lanes.pc[c], i < rows ? static_cast<int>(first + i) : -1, co[c], si[c]);
  };
  // The values in fp32, and their maximum. They are off by less than 2^-20 (16 steps of 2^-24: half of the 9 levels that
  // the squares pass and of the mean's two, root and reciprocal, two products, the rotation's two, one for what is done with
  // them) of the pair's larger value times |cos| + |sin|, `e`; an input taken as it is is exact. The maximum of e decides
  // below whether the scale is sure. odd: fp32 has no range for the norm, or a value is not finite.
  struct Values {
    float a[C][VEC], b[C][VEC], e[C][VEC];
  };
  float amax = 0.f, most_e = 0.f, odd = 0.f;
  auto values = [&](const typename Lanes::Raw& x, int batch, bool peak) {
    const int i = batch * Lanes::kRows + row;
    Values y;
    Lanes::unpack(x, y.a, y.b);
    if (!exact) {
      if (!peak) return y;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) amax = fmaxf(amax, fmaxf(fabsf(y.a[c][j]), fabsf(y.b[c][j])));
      if (Lanes::not_finite(x)) odd = 1.f;
      return y;
    }
    float co[C][VEC], si[C][VEC];
    factors(i, co, si);
    if (S.w) {
      float ss = 0.f;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float sq[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) sq[j] = fmaf(y.a[c][j], y.a[c][j], y.b[c][j] * y.b[c][j]);
#pragma unroll
        for (int n = VEC / 2; n > 0; n /= 2)
#pragma unroll
          for (int j = 0; j < n; ++j) sq[j] += sq[j + n];
        ss += sq[0];
      }
      const float ms = run_sum<LPR>(ss) / static_cast<float>(S.dim) + A.eps;
      if (peak && i < rows && !(ms < 0x1p100f && ms > 0x1p-60f)) odd = 1.f;
      const float r = 1.f / sqrtf(ms);
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) y.a[c][j] *= r * lanes.wa[c][j], y.b[c][j] *= r * lanes.wb[c][j];
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float u = y.a[c][j], v = y.b[c][j], cs = co[c][j], sn = si[c][j];
        const bool turned = lanes.pc[c].turned;  // (selects: `turn`'s branch costs 2 % of the prompts' time here)
        y.a[c][j] = turned ? fused(u, cs, -(v * sn)) : u;
        y.b[c][j] = turned ? fused(u, sn, v * cs) : v;
        y.e[c][j] = fmaxf(fabsf(u), fabsf(v)) * (fabsf(cs) + fabsf(sn));
        if (peak && i < rows) {
          amax = fmaxf(amax, fmaxf(fabsf(y.a[c][j]), fabsf(y.b[c][j])));
          most_e = fmaxf(most_e, y.e[c][j]);
        }
      }
    return y;
  };
  Values held[kHeld];
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (k <= last_batch) held[k] = values(raw[k], k, true);
  for (int k = kHeld; k <= last_batch; ++k) values(fetch(k), k, true);
  block_max3(amax, most_e, odd, lds);  // (every thread has read the old scale)
  if (amax == __builtin_inff() || odd != 0.f ||
      (exact && scale_for(fmaxf(amax - 0x1p-20f * most_e, 0.f)) != scale_for(amax + 0x1p-20f * most_e))) {
    amax = 0.f;  // again, in FP64 and over the finite values
    odd = 1.f;
    for (int batch = 0; batch <= last_batch; ++batch) {
      const int i = batch * Lanes::kRows + row;
      double ya[C][VEC], yb[C][VEC];
      Lanes::unpack(fetch(batch), ya, yb);
      float co[C][VEC], si[C][VEC];
      factors(i, co, si);
      norm_turn<VEC, C, LPR>(A, S, lanes, co, si, ya, yb);
      if (i < rows) {
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            amax = fmaxf(amax, fmaxf(finite_size(ya[c][j]), finite_size(yb[c][j])));
      }
    }
    block_max3(amax, most_e, odd, lds);
  }
  const float after = fmaxf(before, scale_for(amax, odd != 0.f ? 16 : 0));
  const double inv = after > 0.f ? 1.0 / static_cast<double>(after) : 0.0;
  uint8_t* dst = static_cast<uint8_t*>(S.cache.base) + page * S.cache.stride_page + head * S.cache.stride_head;
  const float inv32 = static_cast<float>(inv);
  // The bytes. An input times a power of two is exact. For other values y - e and y + e: where both round to one byte it is
  // that of the exact value, and a wave with a value where they do not (one in some 2^12) does its rows in FP64.
  auto write = [&](const Values& y, int batch) {
    const int i = batch * Lanes::kRows + row;
    uint8_t* to = dst + (kept + i) * S.cache.stride_slot;
    if (odd == 0.f) {
      bool sure = true;
      Bytes<VEC> wa[C], wb[C];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        float al[VEC], bl[VEC], ah[VEC], bh[VEC];
        if (exact) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            const float e = 0x1p-20f * inv32 * y.e[c][j];
            al[j] = fmaf(y.a[c][j], inv32, -e), ah[j] = fmaf(y.a[c][j], inv32, e);
            bl[j] = fmaf(y.b[c][j], inv32, -e), bh[j] = fmaf(y.b[c][j], inv32, e);
          }
          wa[c] = to_fp8(al), wb[c] = to_fp8(bl);
          sure = sure && same(wa[c], to_fp8(ah)) && same(wb[c], to_fp8(bh));
        } else {
#pragma unroll
          for (int j = 0; j < VEC; ++j) al[j] = y.a[c][j] * inv32, bl[j] = y.b[c][j] * inv32;
          wa[c] = to_fp8(al), wb[c] = to_fp8(bl);
        }
      }
      if (!__any(!sure && i < rows)) {
        if (i >= rows) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
          if (lanes.pc[c].ok) store_bytes(to + lanes.pc[c].a, wa[c]);
          if (lanes.pc[c].b_ok) store_bytes(to + lanes.pc[c].b, wb[c]);
        }
        return;
      }
    }
    double ya[C][VEC], yb[C][VEC];
    Lanes::unpack(fetch(batch), ya, yb);
    float co[C][VEC], si[C][VEC];
    factors(i, co, si);
    norm_turn<VEC, C, LPR>(A, S, lanes, co, si, ya, yb);
    if (i >= rows) return;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      if (lanes.pc[c].ok) store_bytes(to + lanes.pc[c].a, to_fp8(ya[c], inv));
      if (lanes.pc[c].b_ok) store_bytes(to + lanes.pc[c].b, to_fp8(yb[c], inv));
    }
  };
#pragma unroll
  for (int k = 0; k < kHeld; ++k)
    if (k <= last_batch) write(held[k], k);
  for (int k = kHeld; k <= last_batch; ++k) write(values(fetch(k), k, false), k);
  if (kept && after != before) {  // round the held tokens again
    const float ratio = static_cast<float>(static_cast<double>(before) * inv);
    const int words = S.dim / 8;
    for (int i = threadIdx.x; i < kept * words; i += kNormThreads) {
      uint2* at = reinterpret_cast<uint2*>(dst + i / words * S.cache.stride_slot + i % words * 8);
      uint2 w = *at;
      auto again = [&](uint32_t x) {
        const auto l = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), false);
        const auto h = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(x), true);
        return pack4_fp8(l[0] * ratio, l[1] * ratio, h[0] * ratio, h[1] * ratio);
      };
      w.x = again(w.x);
      w.y = again(w.y);
      *at = w;
    }
  }
  if (threadIdx.x == 0) *scale = after;
}

// One batch of 16-bit rows.
template <int DT, int VEC, int C, int LPR>
__device__ void append_rows(const AppendArgs& A, const AppendSide& S, int64_t r0, int2* place) {
  using Lanes = RowLanes<DT, VEC, C, LPR>;
  const int64_t rows = A.tokens * S.heads, t0 = r0 / S.heads;
  const int h0 = static_cast<int>(r0 - t0 * S.heads);
  const int n = static_cast<int>(min(rows - r0, static_cast<int64_t>(Lanes::kRows)));
  const int i = threadIdx.x / LPR;
  const int tok = static_cast<int>(static_cast<uint32_t>(h0 + i) / static_cast<uint32_t>(S.heads));
  const int head = h0 + i - tok * S.heads;
  const Lanes lanes(S.w, A.w_f32, S.turned ? A.rope.half : 0, S.dim);
  float a[C][VEC], b[C][VEC];
  lanes.load(S.x, (t0 + tok) * S.stride_t + head * S.stride_h, i < n, a, b);
  for (int k = threadIdx.x; k < (h0 + n - 1) / S.heads + 1; k += kNormThreads) {
    const TokenPlace at = place_of(A.cu, A.nseq, A.context, t0 + k);
    place[k] = make_int2(static_cast<int>(at.pos), at.pos < 0 ? -1 : A.pages.page_of(at.seq, at.pos));
  }
  __syncthreads();
  float r = 1.f;
  if (S.w) r = 1.f / sqrtf(run_sum<LPR>(sum_products(a, b, a, b)) / static_cast<float>(S.dim) + A.eps);
  if (i >= n || place[tok].y < 0) return;
  const int pos = place[tok].x;
  const int slot = pos & ((1 << A.pages.shift) - 1);
  const int64_t to = place[tok].y * S.cache.stride_page + head * S.cache.stride_head + slot * S.cache.stride_slot;
#pragma unroll
  for (int c = 0; c < C; ++c) {
    if (S.w) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) a[c][j] = a[c][j] * r * lanes.wa[c][j], b[c][j] = b[c][j] * r * lanes.wb[c][j];
    }
    if (S.turned) {
      float co[VEC], si[VEC];
      load_turn<VEC>(A.rope, lanes.pc[c], pos, co, si);
      turn<VEC>(lanes.pc[c], co, si, a[c], b[c]);
    }
  }
  lanes.store(S.cache.base, to, a, b);
}

template <int DT, bool FP8, int VEC, int C, int LPR>
__global__ __launch_bounds__(kNormThreads, FP8 ? 3 : 4) void cache_append_kernel(AppendArgs A) {
  __shared__ int2 place[kNormThreads / LPR + 1];
  const uint32_t block = A.launch + blockIdx.x;
  if constexpr (FP8) {
    __shared__ float lds[3 * kNormThreads / kWave];
    if (block < A.page_blocks) {
      const uint32_t per_unit = A.side[0].heads + A.side[1].heads;
      const uint32_t unit = block / per_unit;
      // (the heads turn with the page: eight in a row go to the eight XCDs, and keys cost more than values)
      const int which = static_cast<int>((block + unit) % per_unit), second = which >= A.side[0].heads;
      append_page<DT, VEC, C, LPR>(A, A.side[second], unit, which - (second ? A.side[0].heads : 0), lds);
      return;
    }
  }
  const int side = block >= A.first[2] ? 2 : block >= A.first[1] ? 1 : 0;
  append_rows<DT, VEC, C, LPR>(A, A.side[side], static_cast<int64_t>(block - A.first[side]) * (kNormThreads / LPR), place);
}

template <int DT, bool FP8>
int append_launch(AppendArgs A, bool vectors, hipStream_t st) {
  int chunks = 0;
  for (const AppendSide& s : A.side)
    if (s.heads && s.dim / 16 > chunks) chunks = s.dim / 16;
  auto go = [&](auto kernel, int rows) -> int {
    int64_t blocks = 0;
    if (FP8) {
      const int64_t units = (A.tokens >> A.pages.shift) + 2 * static_cast<int64_t>(A.nseq);
      blocks = units * (A.side[0].heads + A.side[1].heads);
      A.page_blocks = static_cast<uint32_t>(blocks);
    }
    for (int i = 0; i < 3; ++i) {
      A.first[i] = static_cast<uint32_t>(blocks);
      if (!FP8 || i == 2) blocks += (A.tokens * A.side[i].heads + rows - 1) / rows;
    }
    if (blocks >> 31) return static_cast<int>(kErrUnsupported);  // (inputs or caches of that many pass the memory)
    return launch_parts(blocks, [&](int64_t first, unsigned count) {
      A.launch = static_cast<uint32_t>(first);
      hipLaunchKernelGGL(kernel, dim3(count), dim3(kNormThreads), 0, st, A);
    });
  };
#define MSA_APPEND(VEC, C, LPR) return go(cache_append_kernel<DT, FP8, VEC, C, LPR>, kNormThreads / LPR)
  if (!vectors) MSA_APPEND(1, 2, 64);
  if (chunks <= 4) MSA_APPEND(8, 1, 4);
  if (chunks <= 8) MSA_APPEND(8, 1, 8);
  MSA_APPEND(8, 1, 16);
#undef MSA_APPEND
}

bool rows_fit(const AppendSide& s, int half) {
  return !s.heads || (aligned16(s.x) && aligned16(s.w) && s.stride_t % 8 == 0 && s.stride_h % 8 == 0 &&
                      (!s.turned || half % 8 == 0));
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_cache_append(const void* k, const void* v, const void* index_k, int32_t dtype, int64_t kv_heads,
                                int64_t head_dim, int64_t index_dim, const void* k_weight, const void* index_weight,
                                int32_t weight_dtype, const float* cos_sin, int64_t table_rows, int64_t rotary_dim,
                                double eps, void* k_cache, void* v_cache, void* index_cache, int32_t cache_is_fp8,
                                float* k_scale, float* v_scale, const int64_t* strides, const int32_t* page_table,
                                int64_t table_stride, int64_t pages_per_seq, int64_t num_pages, int64_t page_size,
                                const int32_t* cu_seqlens, int64_t num_seqs, const int32_t* context_lens,
                                int64_t total_tokens, void* stream) {
  const bool with_index = index_k != nullptr;
  if (!strides || !cu_seqlens || !context_lens || num_seqs <= 0 || num_seqs > 0x3fffffff || total_tokens < 0 ||
      total_tokens > 0x7fffffff || !valid_pages(page_table, table_stride, pages_per_seq, num_pages, page_size) ||
      (dtype != kBF16 && dtype != kF16) || (weight_dtype != dtype && weight_dtype != kF32) || !(eps >= 0.0) ||
      rotary_dim < 0 || rotary_dim % 2 || (rotary_dim > 0 && (!cos_sin || table_rows < 0)))
    return kErrInvalidArgument;
  if (!k || !v || kv_heads <= 0 || kv_heads >= (1 << 20) || head_dim <= 0 || rotary_dim > head_dim)
    return kErrInvalidArgument;
  if (num_pages > 0 && (!k_cache || !v_cache || (with_index && !index_cache) || (cache_is_fp8 && (!k_scale || !v_scale))))
    return kErrInvalidArgument;
  if (with_index && (index_dim <= 0 || rotary_dim > index_dim)) return kErrInvalidArgument;
  if (head_dim % 16 || head_dim > 256 || (with_index && (index_dim % 16 || index_dim > 256))) return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  AppendArgs A{};
  const int H = static_cast<int>(kv_heads), D = static_cast<int>(head_dim);
  const bool turned = rotary_dim > 0;
  A.side[0] = AppendSide{k, strides[0], strides[1], k_weight, CacheView{k_cache, strides[5], strides[6], strides[7]},
                         k_scale, H, D, turned};
  A.side[1] = AppendSide{v, strides[2], strides[3], nullptr, CacheView{v_cache, strides[8], strides[9], strides[10]},
                         v_scale, H, D, false};
  A.side[2] = AppendSide{index_k, strides[4], 0, index_weight, CacheView{index_cache, strides[11], 0, strides[12]},
                         nullptr, with_index ? 1 : 0, static_cast<int>(index_dim), turned};
  A.w_f32 = weight_dtype == kF32;
  A.rope = RopeTable{cos_sin, table_rows, static_cast<int>(rotary_dim / 2)};
  A.pages = page_map(page_table, table_stride, pages_per_seq, num_pages, page_size);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.context = context_lens;
  A.tokens = total_tokens;
  A.eps = static_cast<float>(eps);
  // cache rows are written in 16-byte pieces (8-byte ones in 8 bits)
  for (int i = 0; i < 3; ++i) {
    const AppendSide& s = A.side[i];
    const int unit = cache_is_fp8 && i < 2 ? 16 : 8;
    if (s.heads && (!aligned16(s.cache.base) || s.cache.stride_page % unit || s.cache.stride_head % unit ||
                    s.cache.stride_slot % unit))
      return kErrInvalidArgument;
  }
  bool vectors = aligned16(cos_sin);
  for (const AppendSide& s : A.side) vectors = vectors && rows_fit(s, A.rope.half);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == kBF16)
    return cache_is_fp8 ? append_launch<kBF16, true>(A, vectors, st) : append_launch<kBF16, false>(A, vectors, st);
  return cache_is_fp8 ? append_launch<kF16, true>(A, vectors, st) : append_launch<kF16, false>(A, vectors, st);
}
