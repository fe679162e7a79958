// Causal attention with a sliding window and visible first tokens: gradients.
//
//   delta[i, h] = dO . O,  p_ij = exp(scale q_i . k_j - lse_i),  ds_ij = p_ij (dO_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_{i, h} ds_ij q_i,  dv_j = sum_{i, h} p_ij dO_i.
//
// All sums are in fixed orders: delta; dQ by tiles of rows as in the forward (three products a pair); dK and dV by tiles of keys
// (four products), each workgroup over the rows that see its keys, all query heads of the key head among them. The seven
// products are two more than one pass with atomic sums of dQ needs. Rows of a tile of keys are shared by several
// workgroups where the tiles alone would leave the chip idle (split_count), whose sums another launch adds up. The first tokens
// are seen by all later rows: what the rows behind the window give is summed in launches of its own, in chunks of
// rows side by side, before the tiles that hold them add it to their own.
//
// Bound by the matrix products, the vector work between them and the LDS reads that feed them: a wave of 32 rows (or keys)
// reads 8 KB a product and 32 keys (or rows) of 128 dims. 32K tokens, 32 heads of 128 over 4, window 4096, bf16: dQ 3.6 ms, dK
// and dV 6.4. Two waves a SIMD hide the waits (one: dQ 5.5, dK and dV 8.4); for dK and dV that takes the values
// from LDS, the logits of 16 rows after those of the other 16, and 256 registers, of which bf16 at 128 dims spills 4 and at 256 dims
// 14. fp16, whose keys also hold their ranges, spills 77 and 109, in the loop: dK and dV 15.2 ms for the case above where bf16 takes
// 6.8 in the same run, 2.34 for 0.92 at 8192 tokens, 16 heads of 256 over 2, window 2048 (none at 64, 96 dims; one at 192). fp32 spills
// 196 at 96 dims, behind the loop. careful_dkv, which is inlined, goes with 54 to 105 scalar registers spilled (the kernel of the first
// tokens' rows, which has none of it: 0).
//
// Logits, p, ds and all sums are fp32. p enters its product rounded once to the input type; a ds enters as two terms (2^-17 of
// it left out): one would be of the size of the gradients' own rounding and bring dq and dk from 0.0017 to 0.0024 of
// themselves (dQ 3.0 ms, dK and dV 6.1). fp16 has neither range nor small values for a ds: its products take ds times a
// power of two, one a row (dQ) or key (dK) that follows the largest so far, and p times 2^15. delta takes the output with
// what its rounding left out.
#include "window.hpp"

namespace msa {
namespace {

struct WindowBwdArgs {
  PackedView q, k, v, dout;
  const int32_t* cu;
  int nseq, G, D;
  Divisor ratio;
  Visible seen;
  float scale, scale_log2;
  int64_t tokens;
  int64_t first;              // workgroup of this launch's first
  const void *out, *out_lo;   // [T][Hq][D]
  const float* lse;           // [T][Hq]
  float* delta;               // [T][Hq]
  void *dq, *dk, *dv;         // [T][Hq][D], [T][G][D]; null: not wanted
  float* part;                // [chunk numbers][sink tiles][G][2][sink rows][D]
  float* split;               // [splits][2][T][G][D]
  int splits;                 // workgroups that share the rows of a tile of keys
  int sink_tiles, sink_rows;  // of a tile
  bool whole_tiles;           // tiles that hold first tokens go through all rows: there are no chunks
  int chunk_log2;             // tokens of a chunk of the rows that see first tokens from behind the window
};

// ---- delta: the diagonal of a product of 16 rows' outputs and gradients, a wave sixteen rows. By the matrix unit and in the
// order of dP, so that a row that sees one key, whose output is its value, has dp - delta = 0 to the last bit.

template <int DT>
__global__ __launch_bounds__(256) void window_delta_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4, heads = A.G * A.ratio.d;
  const int64_t all = A.tokens * heads, row0 = ((A.first + blockIdx.x) * 4 + (threadIdx.x >> 6)) * 16;
  if (row0 >= all) return;
  const int64_t row = min(row0 + c, all - 1), t = row / heads;
  const E* dout = static_cast<const E*>(A.dout.base) + A.dout.at(t, static_cast<int>(row - t * heads));
  const E* out = static_cast<const E*>(A.out) + row * A.D;
  const E* lo = static_cast<const E*>(A.out_lo) + row * A.D;
  f32x4 sum = f32x4{0.f, 0.f, 0.f, 0.f}, left = sum;
  for (int d0 = 0; d0 < A.D; d0 += 32) {
    const int d = d0 + 8 * q4;
    const Fragment<DT> g = d < A.D ? fragment_at<DT>(dout + d) : no_fragment<DT>();
    sum = product<DT>(d < A.D ? fragment_at<DT>(out + d) : no_fragment<DT>(), g, sum);
    if (DT != kF32 && A.out_lo) left = product<DT>(d < A.D ? fragment_at<DT>(lo + d) : no_fragment<DT>(), g, left);
  }
  if (c >> 2 == q4 && row0 + c < all) {  // row c of the product is in the quarter c / 4
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((c & 3) == i) A.delta[row0 + c] = finite(sum[i]) ? sum[i] + left[i] : sum[i];  // (an infinity times what is left out: any sign, or NaN)
  }
}

// ---- fp16: the power of two that ds of a lane's row (or key) is multiplied by, so that the largest one so far stays below 2^15

struct Range {
  float cap = 0.f, up = 0.f;  // values stay below cap; up = 2^15 / cap (0: none yet)
  // A new largest value: the factor for what was summed so far.
  __device__ __forceinline__ float widen(float big) {
    if (!(big >= cap) || big == 0.f) return 1.f;
    // eight times the power of two below it: room to grow, and 27 bits below it are kept
    const int e = static_cast<int>(__float_as_uint(fmaxf(big, 0x1p-90f)) >> 23) - 127 + 3;
    cap = e > 120 ? __builtin_inff() : __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
    const float next = e > 120 ? 0.f : __uint_as_float(static_cast<uint32_t>(15 - e + 127) << 23);
    const float factor = up == 0.f ? 0.f : next / up;
    up = next;
    return factor;
  }
  __device__ __forceinline__ float down() const { return up == 0.f ? 0.f : cap * 0x1p-15f; }
};

// The first four fp16 elements of f times a power of two (downwards).
__device__ __forceinline__ void rescale_half(Fragment<kF16>& f, float factor) {
  uint4 w = __builtin_bit_cast(uint4, f.v);
  w.x = cvt_pk_f16(lo16_f32<kF16>(w.x) * factor, hi16_f32<kF16>(w.x) * factor);
  w.y = cvt_pk_f16(lo16_f32<kF16>(w.y) * factor, hi16_f32<kF16>(w.y) * factor);
  f.v = __builtin_bit_cast(bf16x8, w);
}

// ---- dQ

// The gradient of one row, key by key, by a wave: where a value that is not finite met the products of a tile, which
// multiply the keys that a row does not see by 0.
template <int DT>
__device__ __forceinline__ void careful_dq(const WindowBwdArgs& A, int start, int g, int tok, int head) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63;
  const int64_t t = start + static_cast<int64_t>(tok), row = t * (A.G * A.ratio.d) + head;
  const E* q = static_cast<const E*>(A.q.base) + A.q.at(t, head);
  const E* dout = static_cast<const E*>(A.dout.base) + A.dout.at(t, head);
  const E* k = static_cast<const E*>(A.k.base) + A.k.at(start, g);
  const E* v = static_cast<const E*>(A.v.base) + A.v.at(start, g);
  const float lse = A.lse[row], delta = A.delta[row];
  const float shift = lse == -__builtin_inff() ? lse : lse * -kLog2e;  // (all logits -inf: no weights)
  const int low = A.seen.low(tok);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  bool lost = lse != lse || delta != delta;  // a ds of NaN: no dim is left
  auto keys = [&](int from, int to) {
    for (int base = from; base < to && !lost; base += kWave) {
      const int j = min(base + lane, to - 1), count = min(kWave, to - base);
      const float x = row_dot<DT>(q, k + static_cast<int64_t>(j) * A.k.token, A.D);
      const float dp = row_dot<DT>(dout, v + static_cast<int64_t>(j) * A.v.token, A.D);
      const float ds = __builtin_amdgcn_exp2f(fmaf(x, A.scale_log2, shift)) * (dp - delta);
      lost = __any(ds != ds);
      for (int i = 0; i < count && !lost; ++i) {
        const float ds_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ds), i));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + u * kWave;
          if (d < A.D) o[u] = fmaf(ds_i, value_at<DT>(k + static_cast<int64_t>(base + i) * A.k.token, d), o[u]);
        }
      }
    }
  };
  keys(0, min(A.seen.sinks, low));
  keys(low, tok + 1);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + u * kWave;
    if (d < A.D) store_from_f32<DT>(A.dq, row * A.D + d, lost ? __builtin_nanf("") : o[u] * A.scale);
  }
}

template <int DT, int NK, int MT, int KS>
__global__ __launch_bounds__(256, DT == kF32 && NK > 4 ? 1 : 2) void window_dq_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int DP = 32 * NK, RS = DP + Fragment<DT>::kPad, ND = DP / 16, KT = KS / 16, R = 64 * MT;
  constexpr bool kTwo = DT != kF32;  // terms of a ds
  __shared__ alignas(16) E kbuf[2][KS * RS], vbuf[2][KS * RS];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = A.first + blockIdx.x;
  const int g = static_cast<int>(item % A.G), ratio = A.ratio.d;
  const TilePlace at = tile_place(A.cu, A.nseq, item / A.G, ratio, log2_of(R));
  const int64_t rows = static_cast<int64_t>(at.n) * ratio, r0 = static_cast<int64_t>(at.tile) * R;
  if (r0 >= rows) return;
  const int live = static_cast<int>(min(rows - r0, int64_t{R}));
  auto token_of = [&](int r) { return A.ratio(static_cast<int>(r0) + r); };
  const int t0 = token_of(0), t1 = token_of(live - 1);

  const E* kbase = static_cast<const E*>(A.k.base) + A.k.at(at.start, g);
  const E* vbase = static_cast<const E*>(A.v.base) + A.v.at(at.start, g);
  int tok[MT], head[MT];
  float shift[MT], delta[MT];
  Fragment<DT> qf[MT][NK], gf[MT][NK];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(16 * (MT * wave + m) + c, live - 1);
    tok[m] = token_of(r);
    head[m] = g * ratio + static_cast<int>(r0) + r - tok[m] * ratio;
    const int64_t t = at.start + static_cast<int64_t>(tok[m]);
    const E* q = static_cast<const E*>(A.q.base) + A.q.at(t, head[m]);
    const E* dout = static_cast<const E*>(A.dout.base) + A.dout.at(t, head[m]);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = 32 * kk + 8 * q4;
      qf[m][kk] = d < A.D ? fragment_at<DT>(q + d) : no_fragment<DT>();
      gf[m][kk] = d < A.D ? fragment_at<DT>(dout + d) : no_fragment<DT>();
    }
    shift[m] = A.lse[t * (A.G * ratio) + head[m]] * -kLog2e;
    delta[m] = A.delta[t * (A.G * ratio) + head[m]];
    if (shift[m] == __builtin_inff()) shift[m] = -__builtin_inff();  // (no weights)
  }
  const int low = A.seen.low(t0), sinks = min(A.seen.sinks, low);
  const int sink_steps = (sinks + KS - 1) / KS, steps = sink_steps + (t1 - low) / KS + 1;
  auto first_key = [&](int e) { return e < sink_steps ? e * KS : low + (e - sink_steps) * KS; };
  const bool has_rows = 16 * MT * wave < live;
  const int w0 = token_of(min(16 * MT * wave, live - 1)), w1 = token_of(min(16 * MT * (wave + 1), live) - 1);

  TileLoad<DT, DP, KS> kload, vload;
  auto load_step = [&](int e) {
    const int j0 = first_key(e);
    const E *k = kbase + static_cast<int64_t>(j0) * A.k.token, *v = vbase + static_cast<int64_t>(j0) * A.v.token;
    if (j0 + KS - 1 <= t1) {
      kload.load_near(A.D, k, [&](int r) { return r * A.k.token; });
      vload.load_near(A.D, v, [&](int r) { return r * A.v.token; });
    } else {
      kload.load_near(A.D, k, [&](int r) { return min(r, t1 - j0) * A.k.token; });
      vload.load_near(A.D, v, [&](int r) { return min(r, t1 - j0) * A.v.token; });
    }
  };
  auto store_step = [&](int e) {
    kload.store(kbuf[e & 1], RS, A.D);
    vload.store(vbuf[e & 1], RS, A.D);
  };
  f32x4 acc[MT][ND];
  Range range[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  load_step(0);
  store_step(0);
  for (int e = 0; e < steps; ++e) {
    __syncthreads();
    if (e + 1 < steps) load_step(e + 1);
    const int j0 = first_key(e);
    const bool of_sinks = e < sink_steps;
    const E *kt_ = kbuf[e & 1], *vt_ = vbuf[e & 1];
    if (has_rows && (of_sinks || (j0 <= w1 && (j0 + KS > A.seen.low(w0) || j0 < A.seen.sinks)))) {
      f32x4 s[MT][KT], dp[MT][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m][kt] = dp[m][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const Fragment<DT> kf = fragment_at<DT>(kt_ + (16 * kt + c) * RS + 32 * kk + 8 * q4);
          const Fragment<DT> vf = fragment_at<DT>(vt_ + (16 * kt + c) * RS + 32 * kk + 8 * q4);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            s[m][kt] = product<DT>(kf, qf[m][kk], s[m][kt]);
            dp[m][kt] = product<DT>(vf, gf[m][kk], dp[m][kt]);
          }
        }
      }
      const bool whole = of_sinks ? j0 + KS <= sinks : j0 + KS - 1 <= w0 && (w1 - j0 < A.seen.window || j0 + KS <= A.seen.sinks);
      Fragment<DT> df[MT][KT / 2], dl[MT][KT / 2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float ds[KT][4];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            ds[kt][i] = __builtin_amdgcn_exp2f(fmaf(s[m][kt][i], A.scale_log2, shift[m])) * (dp[m][kt][i] - delta[m]);
        if (!whole) {
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = j0 + 16 * kt + 4 * q4 + i;
              const bool seen = of_sinks ? j < sinks : A.seen(tok[m], j);
              ds[kt][i] = seen ? ds[kt][i] : 0.f;
            }
        }
        if constexpr (DT == kF16) {
          float big = 0.f;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) big = fmaxf(big, fabsf(ds[kt][i]));
          big = quarters_max(big);
          if (__any(big >= range[m].cap && big != 0.f)) {
            const float factor = range[m].widen(big);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[m][d] *= factor;
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) ds[kt][i] *= range[m].up;
        }
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
          float x[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = ds[2 * u + (i >> 2)][i & 3];
          df[m][u] = pack_fragment<DT>(x);
          if constexpr (kTwo) dl[m][u] = second_terms<DT>(df[m][u], x);
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
          const Fragment<DT> kf = column_fragment<DT>(kt_, RS, 32 * u, 16 * d, c, q4);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            acc[m][d] = product<DT>(kf, df[m][u], acc[m][d]);
            if constexpr (kTwo) acc[m][d] = product<DT>(kf, dl[m][u], acc[m][d]);
          }
        }
    }
    if (e + 1 < steps) store_step(e + 1);
  }

#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const bool mine = 16 * (MT * wave + m) + c < live;
    const float factor = DT == kF16 ? A.scale * range[m].down() : A.scale;
    E* dq = static_cast<E*>(A.dq) + ((at.start + static_cast<int64_t>(tok[m])) * (A.G * ratio) + head[m]) * A.D;
    float all = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const f32x4 o = acc[m][d] * factor;
      all += (acc[m][d][0] + acc[m][d][1]) + (acc[m][d][2] + acc[m][d][3]);
      if (mine && 16 * d + 4 * q4 < A.D) store4<DT>(dq + 16 * d + 4 * q4, o);
    }
    uint64_t odd = __ballot(mine && !finite(all));
    odd |= odd >> 32, odd |= odd >> 16;
    for (uint32_t left = odd & 0xffffu; left; left &= left - 1) {
      const int from = __builtin_ctz(left);
      careful_dq<DT>(A, at.start, g, __builtin_amdgcn_readlane(tok[m], from), __builtin_amdgcn_readlane(head[m], from));
    }
  }
}

// ---- dK and dV

// The gradients of one key that came out not finite, by a wave: where a value that is not finite met the products of a tile,
// which multiply the rows that do not see a key by 0. A row whose log sum is NaN leaves no dim of either, one whose delta is
// none of dK; a dim in which a row's dO is not finite is these values' sum in dV. What is left is formed again row by row.
template <int DT>
__device__ __forceinline__ void careful_dkv(const WindowBwdArgs& A, int start, int n, int g, int j, bool need_k, bool need_v) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63, ratio = A.ratio.d;
  const int64_t t = start + static_cast<int64_t>(j), at = (t * A.G + g) * A.D;
  const E* k = static_cast<const E*>(A.k.base) + A.k.at(t, g);
  const E* v = static_cast<const E*>(A.v.base) + A.v.at(t, g);
  const int begin = j * ratio, end = (j < A.seen.sinks || A.seen.window >= n - j ? n : j + A.seen.window) * ratio;
  need_k &= A.dk != nullptr, need_v &= A.dv != nullptr;
  auto token_of = [&](int r) { return start + static_cast<int64_t>(A.ratio(r)); };
  auto head_of = [&](int r) { return g * ratio + r - A.ratio(r) * ratio; };
  auto state_of = [&](int r) { return token_of(r) * (A.G * ratio) + head_of(r); };
  bool lost_k = false, lost_v = false;
  for (int base = begin; base < end && !(lost_v || (lost_k && !need_v)); base += kWave) {
    const int64_t row = state_of(min(base + lane, end - 1));
    const float lse = A.lse[row], delta = A.delta[row];
    lost_v |= __any(lse != lse) != 0;
    lost_k |= __any(lse != lse || delta != delta) != 0;
  }
  float ok[4] = {0.f, 0.f, 0.f, 0.f}, ov[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad[4], again = false;
  if (need_v && !lost_v) {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // (what this wave's other lanes stored)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
#pragma unroll
    for (int u = 0; u < 4; ++u) bad[u] = lane + u * kWave < A.D && !finite(load_as_f32<DT>(A.dv, at + lane + u * kWave));
    for (int base = begin; base < end; base += kWave) {
      bool open = false;
#pragma unroll
      for (int u = 0; u < 4; ++u) open |= bad[u] && odd[u] == odd[u];
      if (!__any(open)) break;
      uint64_t dead = 0;  // rows of a logit of -inf, looked for when a value is infinite
      bool known = false;
      for (int r = base; r < min(end, base + kWave); ++r) {
        const E* y = static_cast<const E*>(A.dout.base) + A.dout.at(token_of(r), head_of(r));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float x = bad[u] ? value_at<DT>(y, lane + u * kWave) : 0.f;
          if (!known && __any(!finite(x) && x == x)) {
            const int i = min(base + lane, end - 1);
            dead = __ballot(row_dot<DT>(static_cast<const E*>(A.q.base) + A.q.at(token_of(i), head_of(i)), k, A.D) * A.scale_log2 ==
                            -__builtin_inff());
            known = true;
          }
          if (!finite(x)) odd[u] += dead >> (r - base) & 1 ? __builtin_nanf("") : x;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) again |= bad[u] && odd[u] == 0.f;
  }
  const bool sum_k = need_k && !lost_k, sum_v = need_v && !lost_v && __any(again);
  for (int base = begin; base < end && ((sum_k && !lost_k) || sum_v); base += kWave) {
    const int r = min(base + lane, end - 1), count = min(kWave, end - base);
    const E* q = static_cast<const E*>(A.q.base) + A.q.at(token_of(r), head_of(r));
    const E* dout = static_cast<const E*>(A.dout.base) + A.dout.at(token_of(r), head_of(r));
    const float lse = A.lse[state_of(r)];
    const float x = row_dot<DT>(q, k, A.D), dp = row_dot<DT>(dout, v, A.D);
    const float p = lse == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(fmaf(x, A.scale_log2, lse * -kLog2e));
    const float ds = p * (dp - A.delta[state_of(r)]);
    lost_k |= __any(ds != ds) != 0;
    for (int i = 0; i < count; ++i) {
      const float p_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
      const float ds_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ds), i));
      const E* qi = static_cast<const E*>(A.q.base) + A.q.at(token_of(base + i), head_of(base + i));
      const E* gi = static_cast<const E*>(A.dout.base) + A.dout.at(token_of(base + i), head_of(base + i));
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + u * kWave;
        if (d >= A.D) break;
        if (sum_k && !lost_k) ok[u] = fmaf(ds_i, value_at<DT>(qi, d), ok[u]);
        if (sum_v) ov[u] = fmaf(p_i, value_at<DT>(gi, d), ov[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + u * kWave;
    if (d >= A.D) break;
    if (need_k) store_from_f32<DT>(A.dk, at + d, lost_k ? __builtin_nanf("") : ok[u] * A.scale);
    if (need_v && lost_v) store_from_f32<DT>(A.dv, at + d, __builtin_nanf(""));
    else if (need_v && bad[u]) store_from_f32<DT>(A.dv, at + d, odd[u] != 0.f ? odd[u] : ov[u]);
  }
}

// What the rows behind the window give for first tokens: floats of one chunk, and the part of a chunk, tile and key head.
__device__ __forceinline__ int64_t sink_chunk_floats(const WindowBwdArgs& A) {
  return int64_t{2} * A.sink_rows * A.D * A.G * A.sink_tiles;
}
__device__ __forceinline__ float* sink_part(const WindowBwdArgs& A, int start, int seq, int chunk, int tile, int g) {
  const int64_t number = (static_cast<int64_t>(start) >> A.chunk_log2) + seq + chunk;
  return A.part + ((number * A.sink_tiles + tile) * A.G + g) * 2 * A.sink_rows * A.D;
}

// SINKS: the rows of one chunk that see the first tokens from behind the window; their sums go to A.part.
template <int DT, int NK, int KT, bool SINKS>
__global__ __launch_bounds__(256, DT == kF32 && NK > 4 ? 1 : 2) void window_dkv_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int DP = 32 * NK, RS = DP + Fragment<DT>::kPad, ND = DP / 16, BK = 64 * KT, QS = 32;
  constexpr float kUp = DT == kF16 ? 15.f : 0.f;
  constexpr int kBuffers = NK <= 4 || DT == kF32 ? 2 : 1;  // (of LDS for two workgroups a CU)
  constexpr bool kTwo = DT != kF32;        // terms of a ds
  constexpr bool kValuesInLds = DT != kF32;  // (in registers with the keys they would leave room for one wave a SIMD)
  __shared__ alignas(16) E qbuf[kBuffers][QS * RS], gbuf[kBuffers][QS * RS], values[kValuesInLds ? BK * RS : 8];
  __shared__ alignas(16) float shift_of[kBuffers][QS], delta_of[kBuffers][QS];
  __shared__ alignas(16) int token_at[kBuffers][QS];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t item = A.first + blockIdx.x;
  const int g = static_cast<int>(item % A.G), ratio = A.ratio.d;
  item /= A.G;
  TilePlace at;
  int j0, from, to;  // first key; tokens of the rows
  int64_t number = item;
  int z = 0;  // which split of them
  if constexpr (SINKS) {
    number = item / A.sink_tiles;
    at = tile_place(A.cu, A.nseq, number, 1, A.chunk_log2);
    j0 = static_cast<int>(item - number * A.sink_tiles) * BK;
    const int64_t behind = static_cast<int64_t>(j0) + BK - 1 + A.seen.window, start = static_cast<int64_t>(at.tile) << A.chunk_log2;
    if (max(behind, start) >= at.n) return;
    from = static_cast<int>(max(behind, start));
    to = static_cast<int>(min(start + (1 << A.chunk_log2), static_cast<int64_t>(at.n)));
    if (from >= to) return;
  } else {
    number = item / A.splits;
    z = static_cast<int>(item - number * A.splits);
    at = tile_place(A.cu, A.nseq, number, 1, log2_of(BK));
    if (static_cast<int64_t>(at.tile) * BK >= at.n) return;
    j0 = at.tile * BK;
    from = j0;
    to = A.whole_tiles && j0 < A.seen.sinks ? at.n
                                            : static_cast<int>(min(static_cast<int64_t>(at.n), static_cast<int64_t>(j0) + BK - 1 + A.seen.window));
  }
  int rb = from * ratio, re = to * ratio;
  if (!SINKS && A.splits > 1) {
    const int share = ((re - rb + A.splits - 1) / A.splits + QS - 1) / QS * QS;
    rb = min(re, rb + z * share);
    re = min(re, rb + share);
  }

  // keys of this wave: [ka, kb], lane c one of each 16
  const int ka = j0 + 16 * KT * wave, last = SINKS ? min(at.n, A.seen.sinks) - 1 : at.n - 1;
  const int kb = min(ka + 16 * KT - 1, last);
  const bool has_keys = ka <= last;
  Fragment<DT> kf[KT][NK], vf[kValuesInLds ? 1 : KT][kValuesInLds ? 1 : NK];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int64_t t = at.start + static_cast<int64_t>(min(ka + 16 * kt + c, at.n - 1));
    const E* k = static_cast<const E*>(A.k.base) + A.k.at(t, g);
    const E* v = static_cast<const E*>(A.v.base) + A.v.at(t, g);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = 32 * kk + 8 * q4;
      kf[kt][kk] = d < A.D ? fragment_at<DT>(k + d) : no_fragment<DT>();
      if constexpr (!kValuesInLds) vf[kt][kk] = d < A.D ? fragment_at<DT>(v + d) : no_fragment<DT>();
    }
  }
  if constexpr (kValuesInLds) {
    TileLoad<DT, DP, BK> load;
    load.load(A.D, [&](int r) {
      return static_cast<const E*>(A.v.base) + A.v.at(at.start + static_cast<int64_t>(min(j0 + r, at.n - 1)), g);
    });
    load.store(values, RS, A.D);
  }
  auto value_fragment = [&](int kt, int kk) {
    if constexpr (kValuesInLds) return fragment_at<DT>(values + (16 * (KT * wave + kt) + c) * RS + 32 * kk + 8 * q4);
    else return vf[kt][kk];
  };
  f32x4 dk[KT][ND], dv[KT][ND];
  Range range[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[kt][d] = dv[kt][d] = f32x4{0.f, 0.f, 0.f, 0.f};

  TileLoad<DT, DP, QS> qload, gload;
  float own_shift = 0.f, own_delta = 0.f;
  int own_token = -1;
  auto load_step = [&](int r0) {
    // (tokens and heads from those of the step's first row on)
    const int t0 = A.ratio(r0), h0 = r0 - t0 * ratio, end = re - 1 - t0 * ratio;
    auto token_of = [&](int r) { return A.ratio(min(h0 + r, end)); };
    auto offset = [&](const PackedView& x, int r) {
      const int t = token_of(r);
      return t * x.token + (min(h0 + r, end) - t * ratio) * x.head;
    };
    const int64_t first = at.start + static_cast<int64_t>(t0);
    qload.load_near(A.D, static_cast<const E*>(A.q.base) + A.q.at(first, g * ratio), [&](int r) { return offset(A.q, r); });
    gload.load_near(A.D, static_cast<const E*>(A.dout.base) + A.dout.at(first, g * ratio), [&](int r) { return offset(A.dout, r); });
    if (threadIdx.x < QS) {
      const int r = min(h0 + static_cast<int>(threadIdx.x), end), t = A.ratio(r);
      const int64_t row = first * (A.G * ratio) + g * ratio;
      const uint32_t own = t * (A.G * ratio) + r - t * ratio;
      const float lse = A.lse[row + own];
      own_shift = lse == -__builtin_inff() ? -__builtin_inff() : lse * -kLog2e;
      own_delta = A.delta[row + own];
      own_token = h0 + static_cast<int>(threadIdx.x) <= end ? t0 + t : -1;  // (no row: sees nothing)
    }
  };
  auto store_step = [&](int b) {
    qload.store(qbuf[b], RS, A.D);
    gload.store(gbuf[b], RS, A.D);
    if (threadIdx.x < QS)
      shift_of[b][threadIdx.x] = own_shift, delta_of[b][threadIdx.x] = own_delta, token_at[b][threadIdx.x] = own_token;
  };

  if (rb < re) {
    load_step(rb);
    store_step(0);
  }
  int b = 0;
  for (int r0 = rb; r0 < re; r0 += QS, b ^= kBuffers - 1) {
    __syncthreads();
    const bool more = r0 + QS < re;
    if (more) load_step(r0 + QS);
    const int ta = A.ratio(r0), tb = A.ratio(min(r0 + QS, re) - 1);
    if (has_keys && tb >= ka && (ta - kb < A.seen.window || ka < A.seen.sinks)) {
      const E *qt = qbuf[b], *gt = gbuf[b];
      const bool whole = r0 + QS <= re && ta >= kb && (tb - ka < A.seen.window || kb < A.seen.sinks);
      Fragment<DT> pf[KT], df[KT], dl[KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) pf[kt] = df[kt] = dl[kt] = no_fragment<DT>();
      // (16 rows after the other: both at once take more registers than two waves a SIMD have)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        f32x4 s[KT], dp[KT];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[kt] = dp[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const Fragment<DT> qf = fragment_at<DT>(qt + (16 * h + c) * RS + 32 * kk + 8 * q4);
          const Fragment<DT> gf = fragment_at<DT>(gt + (16 * h + c) * RS + 32 * kk + 8 * q4);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            s[kt] = product<DT>(qf, kf[kt][kk], s[kt]);
            dp[kt] = product<DT>(gf, value_fragment(kt, kk), dp[kt]);
          }
        }
        const f32x4 shift = *reinterpret_cast<const f32x4*>(&shift_of[b][16 * h + 4 * q4]);
        const f32x4 delta = *reinterpret_cast<const f32x4*>(&delta_of[b][16 * h + 4 * q4]);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          f32x4 p, ds;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[i] = __builtin_amdgcn_exp2f(fmaf(s[kt][i], A.scale_log2, shift[i]));
            ds[i] = p[i] * (dp[kt][i] - delta[i]);
          }
          if (!whole) {
            const int j = ka + 16 * kt + c;
            const int4 tok = *reinterpret_cast<const int4*>(&token_at[b][16 * h + 4 * q4]);
            const int toks[4] = {tok.x, tok.y, tok.z, tok.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bool seen = A.seen(toks[i], j);
              p[i] = seen ? p[i] : 0.f;
              ds[i] = seen ? ds[i] : 0.f;
            }
          }
          if constexpr (DT == kF16) {
            const float big = quarters_max(fmaxf(fmaxf(fabsf(ds[0]), fabsf(ds[1])), fmaxf(fabsf(ds[2]), fabsf(ds[3]))));
            if (__any(big >= range[kt].cap && big != 0.f)) {
              const float factor = range[kt].widen(big);
#pragma unroll
              for (int d = 0; d < ND; ++d) dk[kt][d] *= factor;
              if (h == 1) rescale_half(df[kt], factor), rescale_half(dl[kt], factor);
            }
            ds *= range[kt].up, p *= 0x1p15f;
          }
          pack_half<DT>(pf[kt], h, p);
          pack_half<DT>(df[kt], h, ds);
          if constexpr (kTwo) pack_half<DT>(dl[kt], h, left_out<DT>(ds));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const Fragment<DT> gf = column_fragment<DT>(gt, RS, 0, 16 * d, c, q4);
        const Fragment<DT> qf = column_fragment<DT>(qt, RS, 0, 16 * d, c, q4);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          dv[kt][d] = product<DT>(gf, pf[kt], dv[kt][d]);
          dk[kt][d] = product<DT>(qf, df[kt], dk[kt][d]);
          if constexpr (kTwo) dk[kt][d] = product<DT>(qf, dl[kt], dk[kt][d]);
        }
      }
    }
    if (kBuffers == 1) __syncthreads();
    if (more) store_step(b ^ (kBuffers - 1));
  }

#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int j = ka + 16 * kt + c;
    const bool mine = j <= last;
    const float down_k = DT == kF16 ? A.scale * range[kt].down() : A.scale, down_v = kUp == 0.f ? 1.f : 0x1p-15f;
    const int64_t row = (at.start + static_cast<int64_t>(mine ? j : 0)) * A.G + g;
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[kt][d] *= down_k, dv[kt][d] *= down_v;
    if (SINKS || A.splits > 1) {  // parts of a sum
      float* part = SINKS ? A.part + ((item * A.G + g) * 2 * A.sink_rows + j - j0) * A.D : A.split + (z * 2 * A.tokens * A.G + row) * A.D;
      float* part_v = part + (SINKS ? A.sink_rows : A.tokens * A.G) * A.D;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (mine && 16 * d + 4 * q4 < A.D) {
          *reinterpret_cast<f32x4*>(part + 16 * d + 4 * q4) = dk[kt][d];
          *reinterpret_cast<f32x4*>(part_v + 16 * d + 4 * q4) = dv[kt][d];
        }
    } else {
      if (mine && j < A.seen.sinks && to < at.n) {
        const float* part = sink_part(A, at.start, at.seq, to >> A.chunk_log2, at.tile, g) + static_cast<int64_t>(j - j0) * A.D + 4 * q4;
#pragma unroll
        for (int d = 0; d < ND; ++d)
          if (16 * d + 4 * q4 < A.D) {
            dk[kt][d] += *reinterpret_cast<const f32x4*>(part + 16 * d);
            dv[kt][d] += *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(A.sink_rows) * A.D + 16 * d);
          }
      }
      float all_k = 0.f, all_v = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        all_k += (dk[kt][d][0] + dk[kt][d][1]) + (dk[kt][d][2] + dk[kt][d][3]);
        all_v += (dv[kt][d][0] + dv[kt][d][1]) + (dv[kt][d][2] + dv[kt][d][3]);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (mine && 16 * d + 4 * q4 < A.D) {
          if (A.dk) store4<DT>(static_cast<E*>(A.dk) + row * A.D + 16 * d + 4 * q4, dk[kt][d]);
          if (A.dv) store4<DT>(static_cast<E*>(A.dv) + row * A.D + 16 * d + 4 * q4, dv[kt][d]);
        }
      uint64_t odd_k = __ballot(mine && !finite(all_k)), odd_v = __ballot(mine && !finite(all_v));
      odd_k |= odd_k >> 32, odd_k |= odd_k >> 16, odd_v |= odd_v >> 32, odd_v |= odd_v >> 16;
      for (uint32_t left = (odd_k | odd_v) & 0xffffu; left; left &= left - 1) {
        const int i = __builtin_ctz(left);
        careful_dkv<DT>(A, at.start, at.n, g, ka + 16 * kt + i, odd_k >> i & 1, odd_v >> i & 1);
      }
    }
  }
}

// The chunks' sums for first tokens added up in order, in the place of the first chunk: four values a thread, a workgroup 1024 of
// a sequence, tile and key head.
template <int BK>
__global__ __launch_bounds__(256) void window_sink_sum(WindowBwdArgs A) {
  const int64_t floats = int64_t{2} * A.sink_rows * A.D, blocks = (floats + 1023) / 1024;
  const int64_t item = (A.first + blockIdx.x) / blocks, block = A.first + blockIdx.x - item * blocks;
  const int64_t at = block * 1024 + threadIdx.x * 4, tiles = static_cast<int64_t>(A.sink_tiles) * A.G;
  const int s = static_cast<int>(item / tiles), rest = static_cast<int>(item - s * tiles), tile = rest / A.G, g = rest - tile * A.G;
  const int start = A.cu[s], n = A.cu[s + 1] - start;
  const int64_t behind = static_cast<int64_t>(tile) * BK + BK - 1 + A.seen.window;
  // (rows of the tile past the first tokens hold nothing and are not read)
  const int row = static_cast<int>(at / A.D) % A.sink_rows;
  if (behind >= n || at >= floats || tile * BK + row >= min(n, A.seen.sinks)) return;
  const int first = static_cast<int>(behind) >> A.chunk_log2, end = (n - 1) >> A.chunk_log2;
  float* part = sink_part(A, start, s, first, tile, g) + at;
  const int64_t step = sink_chunk_floats(A);
  f32x4 sum = *reinterpret_cast<const f32x4*>(part);
#pragma unroll 8
  for (int ch = 1; ch <= end - first; ++ch) sum += *reinterpret_cast<const f32x4*>(part + ch * step);
  *reinterpret_cast<f32x4*>(part) = sum;
}

// The parts of a key's sums added up in order, a wave a key: those of its tile's splits, then that of the rows behind the
// window, if it is a first token.
template <int DT, int BK>
__global__ __launch_bounds__(256) void window_dkv_join(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63;
  const int64_t row = (A.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= A.tokens * A.G) return;
  const int64_t t = row / A.G, plane = A.tokens * A.G * A.D;
  const int g = static_cast<int>(row - t * A.G), d = 4 * lane;
  const bool mine = d < A.D;
  f32x4 dk = f32x4{0.f, 0.f, 0.f, 0.f}, dv = dk;
  const float* part = A.split + row * A.D + (mine ? d : 0);
#pragma unroll 4
  for (int z = 0; z < A.splits; ++z, part += 2 * plane) {
    dk += *reinterpret_cast<const f32x4*>(part);
    dv += *reinterpret_cast<const f32x4*>(part + plane);
  }
  const int s = A.nseq == 1 ? 0 : wave_upper_index(A.nseq, t, [&](int i) { return static_cast<int64_t>(A.cu[i]); });
  const int start = A.cu[s], n = A.cu[s + 1] - start, j = static_cast<int>(t - start), tile = j / BK;
  const int64_t behind = static_cast<int64_t>(tile) * BK + BK - 1 + A.seen.window;  // tokens of the chunks: from here on
  if (j < A.seen.sinks && behind < n && !A.whole_tiles) {
    part = sink_part(A, start, s, static_cast<int>(behind) >> A.chunk_log2, tile, g) + static_cast<int64_t>(j - tile * BK) * A.D +
           (mine ? d : 0);
    dk += *reinterpret_cast<const f32x4*>(part);
    dv += *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(A.sink_rows) * A.D);
  }
  if (mine) {
    if (A.dk) store4<DT>(static_cast<E*>(A.dk) + row * A.D + d, dk);
    if (A.dv) store4<DT>(static_cast<E*>(A.dv) + row * A.D + d, dv);
  }
  const bool odd_k = __any(mine && !finite((dk[0] + dk[1]) + (dk[2] + dk[3])));
  const bool odd_v = __any(mine && !finite((dv[0] + dv[1]) + (dv[2] + dv[3])));
  if (odd_k || odd_v) careful_dkv<DT>(A, start, n, g, j, odd_k, odd_v);
}

// Keys of a workgroup of the dK / dV kernels.
int keys_per_tile(int32_t dtype, int64_t dim) { return dtype != kF32 && dim <= 128 ? 128 : 64; }

// Tiles that hold first tokens, their rows in one, and the chunks of the rows behind the window; no tiles where no sequence has
// such rows, or where the chunks' sums would take more than 256 MiB (many first tokens, or many short sequences: their tiles
// go through all rows then).
struct SinkShape {
  int64_t tiles, rows;
  int chunk_log2;
  bool whole;  // tiles that hold first tokens go through all rows
};
int64_t sink_floats(const SinkShape& shape, int64_t tokens, int64_t nseq, int64_t groups, int64_t dim) {
  return tile_numbers(tokens, nseq, 1, shape.chunk_log2) * shape.tiles * groups * 2 * shape.rows * dim;
}
SinkShape sink_shape(int32_t dtype, int64_t dim, int64_t tokens, int64_t nseq, int64_t longest, int64_t ratio, int64_t groups,
                     int64_t window, int64_t sinks) {
  if (window == 0 || sinks == 0 || longest <= window) return SinkShape{0, 0, 0, false};
  // 256 rows a chunk at least, and no more than 256 chunks in all
  int chunk_log2 = 4;
  while (ratio << chunk_log2 < 256 || tokens >> chunk_log2 > 256) ++chunk_log2;
  const int64_t keys = keys_per_tile(dtype, dim), most = sinks < longest ? sinks : longest;
  const SinkShape shape{(most + keys - 1) / keys, most < keys ? (most + 15) / 16 * 16 : keys, chunk_log2, false};
  return sink_floats(shape, tokens, nseq, groups, dim) <= int64_t{1} << 26 ? shape : SinkShape{0, 0, 0, true};
}

// Workgroups that share the rows of a tile of keys: the number next to the quotient of the largest tile's work and what each of the
// workgroups that run at once (512, or 256 of more than 128 fp32 dims) gets of all the work, which is at least that of the longest
// sequence and of sequences of equal length; no more than give a share 128 rows, nor than fill 256 MiB with parts. Rounding down leaves
// a largest share of up to 1.5 times the even one, and rounds of workgroups that run at once are not counted: six fp16 sequences of
// 1 to 6151 tokens, 16 heads of 96 over 4, window 1024 have a quotient of 1.39, one workgroup a tile, 524 in all, 12 of them in a second
// round (414 us); two fp32 ones of 701 and 1347, 16 heads of 128 over 2, window 500 have 792 in 1.5 rounds (151 us).
int64_t split_count(int32_t dtype, int64_t tokens, int64_t nseq, int64_t longest, int64_t q_heads, int64_t groups, int64_t dim,
                    int64_t window, bool whole) {
  const double keys = keys_per_tile(dtype, dim), w = window == 0 ? 1e18 : static_cast<double>(window);
  const auto pairs = [&](double n) { return n <= w ? n * n / 2 : w * (n - w / 2); };
  const double all = static_cast<double>(nseq) * pairs(static_cast<double>(tokens) / nseq), one = pairs(static_cast<double>(longest));
  const double work = groups * (all > one ? all : one) / keys;  // tokens of rows that tiles go through
  const double most = whole || longest < w + keys ? longest : w + keys;
  const int64_t even = static_cast<int64_t>(most * (dtype == kF32 && dim > 128 ? 256 : 512) / (work < 1 ? 1 : work) + 0.5);
  const int64_t by_rows = static_cast<int64_t>(most * (q_heads / groups) / 128), by_size = (int64_t{1} << 25) / (tokens * groups * dim);
  int64_t n = even < by_rows ? even : by_rows;
  n = n < by_size ? n : by_size;
  return n < 1 ? 1 : n < 64 ? n : 64;
}

int64_t delta_floats(int64_t tokens, int64_t q_heads) { return (tokens * q_heads + 3) / 4 * 4; }

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int64_t msa_window_attn_bwd_workspace_bytes(int32_t dtype, int64_t total_tokens, int64_t num_seqs,
                                                       int64_t longest, int64_t q_heads, int64_t kv_groups,
                                                       int64_t head_dim, int64_t window, int64_t sinks) {
  if (total_tokens <= 0 || num_seqs <= 0 || q_heads <= 0 || kv_groups <= 0 || q_heads % kv_groups || head_dim <= 0 || window < 0 ||
      sinks < 0)
    return 0;
  const SinkShape shape = sink_shape(dtype, head_dim, total_tokens, num_seqs, longest, q_heads / kv_groups, kv_groups, window, sinks);
  const int64_t splits = split_count(dtype, total_tokens, num_seqs, longest, q_heads, kv_groups, head_dim, window,
                                     shape.whole);
  return 4 * (delta_floats(total_tokens, q_heads) + sink_floats(shape, total_tokens, num_seqs, kv_groups, head_dim) +
              (splits > 1 ? splits * 2 * total_tokens * kv_groups * head_dim : 0));
}

extern "C" int msa_window_attn_bwd(const void* q, const void* k, const void* v, int32_t dtype, const int64_t* strides,
                                   const int32_t* cu_seqlens, int64_t num_seqs, int64_t longest, int64_t total_tokens,
                                   int64_t q_heads, int64_t kv_groups, int64_t head_dim, int64_t window, int64_t sinks,
                                   double scale, const void* out, const void* out_lo, const float* lse,
                                   const void* grad_out, void* grad_q, void* grad_k, void* grad_v, void* workspace,
                                   int64_t workspace_bytes, void* stream) {
  if (!valid_window_call(q, k, v, dtype, strides, cu_seqlens, num_seqs, total_tokens, q_heads, kv_groups, head_dim, window,
                         sinks, scale) ||
      !out || !lse || !grad_out || reinterpret_cast<uintptr_t>(grad_out) % 16 || longest < 0 || longest > total_tokens)
    return kErrInvalidArgument;
  const int unit = dtype == kF32 ? 4 : 8;
  if (strides[6] % unit || strides[7] % unit || !near_rows(strides + 6, q_heads / kv_groups)) return kErrInvalidArgument;
  if (!window_supported(head_dim, total_tokens, q_heads / kv_groups)) return kErrUnsupported;
  if (total_tokens == 0 || !(grad_q || grad_k || grad_v)) return kOk;
  if (!workspace || workspace_bytes < msa_window_attn_bwd_workspace_bytes(dtype, total_tokens, num_seqs, longest, q_heads,
                                                                          kv_groups, head_dim, window, sinks))
    return kErrInvalidArgument;
  const SinkShape shape = sink_shape(dtype, head_dim, total_tokens, num_seqs, longest, q_heads / kv_groups, kv_groups, window, sinks);
  WindowBwdArgs A{};
  A.q = packed_view(q, strides);
  A.k = packed_view(k, strides + 2);
  A.v = packed_view(v, strides + 4);
  A.dout = packed_view(grad_out, strides + 6);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.ratio = divisor_of(q_heads / kv_groups);
  A.G = static_cast<int>(kv_groups);
  A.D = static_cast<int>(head_dim);
  A.seen = visible_of(window, sinks);
  A.scale = static_cast<float>(scale);
  A.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  A.tokens = total_tokens;
  A.out = out;
  A.out_lo = out_lo;
  A.lse = lse;
  A.delta = static_cast<float*>(workspace);
  A.part = A.delta + delta_floats(total_tokens, q_heads);
  A.split = A.part + sink_floats(shape, total_tokens, num_seqs, kv_groups, head_dim);
  A.splits = static_cast<int>(split_count(dtype, total_tokens, num_seqs, longest, q_heads, kv_groups, head_dim, window, shape.whole));
  A.whole_tiles = shape.whole;
  A.sink_tiles = static_cast<int>(shape.tiles);
  A.sink_rows = static_cast<int>(shape.rows);
  A.chunk_log2 = shape.chunk_log2;
  A.dq = grad_q;
  A.dk = grad_k;
  A.dv = grad_v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  int rc = launch_parts((total_tokens * q_heads + 63) / 64, [&](int64_t first, unsigned count) {
    A.first = first;
    if (dtype == kBF16) hipLaunchKernelGGL(window_delta_kernel<kBF16>, dim3(count), block, 0, st, A);
    else if (dtype == kF16) hipLaunchKernelGGL(window_delta_kernel<kF16>, dim3(count), block, 0, st, A);
    else hipLaunchKernelGGL(window_delta_kernel<kF32>, dim3(count), block, 0, st, A);
  });
#define MSA_WINDOW_LAUNCH(KERNEL, ITEMS)                                       \
  rc = launch_parts(ITEMS, [&](int64_t first, unsigned count) {                \
    A.first = first;                                                           \
    hipLaunchKernelGGL(KERNEL, dim3(count), block, 0, st, A);                  \
  })
#define MSA_WINDOW_BWD(DT, NK, MT, KS, KT)                                                                                       \
  {                                                                                                                              \
    if (rc == kOk && grad_q)                                                                                                     \
      MSA_WINDOW_LAUNCH((window_dq_kernel<DT, NK, MT, KS>), tile_numbers(total_tokens, num_seqs, A.ratio.d, log2_of(64 * MT)) * kv_groups); \
    if (rc == kOk && (grad_k || grad_v) && shape.tiles)                                                                          \
      MSA_WINDOW_LAUNCH((window_dkv_kernel<DT, NK, KT, true>),                                                                   \
                        tile_numbers(total_tokens, num_seqs, 1, shape.chunk_log2) * shape.tiles * kv_groups);                    \
    if (rc == kOk && (grad_k || grad_v) && shape.tiles)                                                                          \
      MSA_WINDOW_LAUNCH((window_sink_sum<64 * KT>),                                                                              \
                        num_seqs * shape.tiles * kv_groups * ((2 * shape.rows * head_dim + 1023) / 1024));                       \
    if (rc == kOk && (grad_k || grad_v))                                                                                         \
      MSA_WINDOW_LAUNCH((window_dkv_kernel<DT, NK, KT, false>),                                                                  \
                        tile_numbers(total_tokens, num_seqs, 1, log2_of(64 * KT)) * A.splits * kv_groups);                                \
    if (rc == kOk && (grad_k || grad_v) && A.splits > 1)                                                                         \
      MSA_WINDOW_LAUNCH((window_dkv_join<DT, 64 * KT>), (total_tokens * kv_groups + 3) / 4);                                     \
    return rc;                                                                                                                   \
  }
  if (dtype == kF32) {
    if (head_dim <= 64) MSA_WINDOW_BWD(kF32, 2, 1, 32, 1)
    if (head_dim <= 96) MSA_WINDOW_BWD(kF32, 3, 1, 32, 1)
    if (head_dim <= 128) MSA_WINDOW_BWD(kF32, 4, 1, 32, 1)
    if (head_dim <= 192) MSA_WINDOW_BWD(kF32, 6, 1, 32, 1)
    MSA_WINDOW_BWD(kF32, 8, 1, 32, 1)
  }
#define MSA_WINDOW_BWD_DIM(DT)                         \
  if (head_dim <= 64) MSA_WINDOW_BWD(DT, 2, 2, 32, 2)  \
  if (head_dim <= 96) MSA_WINDOW_BWD(DT, 3, 2, 32, 2)  \
  if (head_dim <= 128) MSA_WINDOW_BWD(DT, 4, 2, 32, 2) \
  if (head_dim <= 192) MSA_WINDOW_BWD(DT, 6, 1, 32, 1) \
  MSA_WINDOW_BWD(DT, 8, 1, 32, 1)
  if (dtype == kBF16) { MSA_WINDOW_BWD_DIM(kBF16) }
  MSA_WINDOW_BWD_DIM(kF16)
#undef MSA_WINDOW_BWD_DIM
#undef MSA_WINDOW_BWD
#undef MSA_WINDOW_LAUNCH
}
