// Causal attention with a sliding window and visible first tokens: gradients.
//
//   delta[i, h] = dO . O,  p_ij = exp(scale q_i . k_j - lse_i),  ds_ij = p_ij (dO_i . v_j - delta_i),
//   dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_{i, h} ds_ij q_i,  dv_j = sum_{i, h} p_ij dO_i.
//
// Three launches, all sums in fixed orders: delta; dQ by tiles of rows as in the forward (three products a pair); dK and dV by
// tiles of keys (four products), each workgroup over the rows that see its keys, all query heads of the key head among
// them. The seven products are two more than one pass with atomic sums of dQ needs. The first tokens are seen by
// all later rows: what their rows behind the window give is summed in a launch of its own, in chunks of rows
// side by side, before the tiles that hold them add those sums to their own.
//
// Bound by the matrix products, which wait for LDS: a wave of 32 rows (or keys) reads 8 KB a product and 32 keys
// (or rows) of 128 dims.
//
// Logits, p, ds and all sums are fp32; p and ds enter their products rounded once to the input type. fp16 has neither
// range nor small values for a ds: its products take ds times a power of two, one a row (dQ) or key (dK) that
// follows the largest so far, and p times 2^15. delta takes the output with what its rounding left out.
#include "window.hpp"

namespace msa {
namespace {

constexpr int kChunk = 1024;  // tokens of a chunk of the rows that see first tokens from behind the window

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
  int sink_tiles, sink_rows;  // of a tile
};

// ---- delta: 16 lanes a row

template <int DT>
__global__ __launch_bounds__(256) void window_delta_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int kPer = DT == kF32 ? 4 : 8;
  const int heads = A.G * A.ratio.d;
  const int64_t row = (A.first + blockIdx.x) * 16 + threadIdx.x / 16;
  if (row >= A.tokens * heads) return;
  const int64_t t = row / heads;
  const E* dout = static_cast<const E*>(A.dout.base) + t * A.dout.token + (row - t * heads) * A.dout.head;
  const E* out = static_cast<const E*>(A.out) + row * A.D;
  const E* lo = static_cast<const E*>(A.out_lo) + row * A.D;
  float sum = 0.f;
  for (int d = threadIdx.x % 16 * kPer; d < A.D; d += 16 * kPer) {
    const uint4 x = *reinterpret_cast<const uint4*>(dout + d), y = *reinterpret_cast<const uint4*>(out + d);
    const uint4 z = A.out_lo ? *reinterpret_cast<const uint4*>(lo + d) : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w}, zs[4] = {z.x, z.y, z.z, z.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == kF32) {
        sum = fmaf(__uint_as_float(xs[i]), __uint_as_float(ys[i]), sum);
      } else {
        sum = fmaf(lo16_f32<DT>(xs[i]), lo16_f32<DT>(ys[i]) + lo16_f32<DT>(zs[i]), sum);
        sum = fmaf(hi16_f32<DT>(xs[i]), hi16_f32<DT>(ys[i]) + hi16_f32<DT>(zs[i]), sum);
      }
    }
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  if (threadIdx.x % 16 == 0) A.delta[row] = sum;
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

// ---- dQ

// The gradient of one row, key by key, by a wave: where a value that is not finite met the products of a tile, which
// multiply the keys that a row does not see by 0.
template <int DT>
__device__ __forceinline__ void careful_dq(const WindowBwdArgs& A, int start, int g, int tok, int head) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63;
  const int64_t t = start + static_cast<int64_t>(tok), row = t * (A.G * A.ratio.d) + head;
  const E* q = static_cast<const E*>(A.q.base) + t * A.q.token + head * A.q.head;
  const E* dout = static_cast<const E*>(A.dout.base) + t * A.dout.token + head * A.dout.head;
  const E* k = static_cast<const E*>(A.k.base) + start * A.k.token + g * A.k.head;
  const E* v = static_cast<const E*>(A.v.base) + start * A.v.token + g * A.v.head;
  const float lse = A.lse[row], shift = -lse / kLn2Window, delta = A.delta[row];
  const int low = A.seen.low(tok);
  float o[4] = {0.f, 0.f, 0.f, 0.f};
  bool lost = false;  // a ds of NaN: no dim is left
  auto keys = [&](int from, int to) {
    for (int base = from; base < to && !lost; base += kWave) {
      const int j = min(base + lane, to - 1), count = min(kWave, to - base);
      float x = 0.f, dp = 0.f;
      for (int d = 0; d < A.D; ++d) {
        x = fmaf(value_at<DT>(q, d), value_at<DT>(k + j * A.k.token, d), x);
        dp = fmaf(value_at<DT>(dout, d), value_at<DT>(v + j * A.v.token, d), dp);
      }
      const float ds = __builtin_amdgcn_exp2f(fmaf(x, A.scale_log2, shift)) * (dp - delta);
      lost = __any(ds != ds);
      for (int i = 0; i < count && !lost; ++i) {
        const float ds_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ds), i));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int d = lane + u * kWave;
          if (d < A.D) o[u] = fmaf(ds_i, value_at<DT>(k + (base + i) * A.k.token, d), o[u]);
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
__global__ __launch_bounds__(256, 1) void window_dq_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int DP = 32 * NK, RS = DP + Fragment<DT>::kPad, ND = DP / 16, KT = KS / 16, R = 64 * MT;
  __shared__ alignas(16) E kbuf[2][KS * RS], vbuf[2][KS * RS];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = A.first + blockIdx.x;
  const int g = static_cast<int>(item % A.G), ratio = A.ratio.d;
  const TilePlace at = tile_place<R>(A.cu, A.nseq, item / A.G, ratio);
  const int64_t rows = static_cast<int64_t>(at.n) * ratio, r0 = static_cast<int64_t>(at.tile) * R;
  if (r0 >= rows) return;
  const int live = static_cast<int>(min(rows - r0, int64_t{R}));
  auto token_of = [&](int r) { return A.ratio(static_cast<int>(r0) + r); };
  const int t0 = token_of(0), t1 = token_of(live - 1);

  const E* kbase = static_cast<const E*>(A.k.base) + at.start * A.k.token + g * A.k.head;
  const E* vbase = static_cast<const E*>(A.v.base) + at.start * A.v.token + g * A.v.head;
  int tok[MT], head[MT];
  float shift[MT], delta[MT];
  Fragment<DT> qf[MT][NK], gf[MT][NK];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(16 * (MT * wave + m) + c, live - 1);
    tok[m] = token_of(r);
    head[m] = g * ratio + static_cast<int>(r0) + r - tok[m] * ratio;
    const int64_t t = at.start + static_cast<int64_t>(tok[m]);
    const E* q = static_cast<const E*>(A.q.base) + t * A.q.token + head[m] * A.q.head;
    const E* dout = static_cast<const E*>(A.dout.base) + t * A.dout.token + head[m] * A.dout.head;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = 32 * kk + 8 * q4;
      qf[m][kk] = d < A.D ? fragment_at<DT>(q + d) : no_fragment<DT>();
      gf[m][kk] = d < A.D ? fragment_at<DT>(dout + d) : no_fragment<DT>();
    }
    shift[m] = -A.lse[t * (A.G * ratio) + head[m]] / kLn2Window;
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
    kload.load(A.D, [&](int r) { return kbase + min(j0 + r, t1) * A.k.token; });
    vload.load(A.D, [&](int r) { return vbase + min(j0 + r, t1) * A.v.token; });
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
      Fragment<DT> df[MT][KT / 2];
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
          big = quad_max(big);
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
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
          const Fragment<DT> kf = column_fragment<DT>(kt_, RS, 32 * u, 16 * d, c, q4);
#pragma unroll
          for (int m = 0; m < MT; ++m) acc[m][d] = product<DT>(kf, df[m][u], acc[m][d]);
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

// The gradients of one key, row by row, by a wave: where a value that is not finite met the products of a tile, which
// multiply the rows that do not see a key by 0.
template <int DT>
__device__ __forceinline__ void careful_dkv(const WindowBwdArgs& A, int start, int n, int g, int j) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63, ratio = A.ratio.d;
  const int64_t t = start + static_cast<int64_t>(j);
  const E* k = static_cast<const E*>(A.k.base) + t * A.k.token + g * A.k.head;
  const E* v = static_cast<const E*>(A.v.base) + t * A.v.token + g * A.v.head;
  const int end = (j < A.seen.sinks || A.seen.window >= n - j ? n : j + A.seen.window) * ratio;
  float ok[4] = {0.f, 0.f, 0.f, 0.f}, ov[4] = {0.f, 0.f, 0.f, 0.f};
  bool lost_k = false, lost_v = false;  // a ds (a p) of NaN: no dim is left
  for (int base = j * ratio; base < end && !(lost_k && lost_v); base += kWave) {
    const int r = min(base + lane, end - 1), count = min(kWave, end - base);
    const int64_t tr = start + static_cast<int64_t>(A.ratio(r));
    const int head = g * ratio + r - A.ratio(r) * ratio;
    const E* q = static_cast<const E*>(A.q.base) + tr * A.q.token + head * A.q.head;
    const E* dout = static_cast<const E*>(A.dout.base) + tr * A.dout.token + head * A.dout.head;
    const float lse = A.lse[tr * (A.G * ratio) + head];
    float x = 0.f, dp = 0.f;
    for (int d = 0; d < A.D; ++d) {
      x = fmaf(value_at<DT>(q, d), value_at<DT>(k, d), x);
      dp = fmaf(value_at<DT>(dout, d), value_at<DT>(v, d), dp);
    }
    const float p = lse == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(fmaf(x, A.scale_log2, -lse / kLn2Window));
    const float ds = p * (dp - A.delta[tr * (A.G * ratio) + head]);
    lost_k |= __any(ds != ds) != 0;
    lost_v |= __any(p != p) != 0;
    for (int i = 0; i < count; ++i) {
      const float p_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
      const float ds_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(ds), i));
      const int ti = A.ratio(base + i), hi = g * ratio + base + i - ti * ratio;
      const E* qi = static_cast<const E*>(A.q.base) + (start + static_cast<int64_t>(ti)) * A.q.token + hi * A.q.head;
      const E* gi = static_cast<const E*>(A.dout.base) + (start + static_cast<int64_t>(ti)) * A.dout.token + hi * A.dout.head;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int d = lane + u * kWave;
        if (d >= A.D) break;
        ok[u] = fmaf(ds_i, value_at<DT>(qi, d), ok[u]);
        ov[u] = fmaf(p_i, value_at<DT>(gi, d), ov[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int d = lane + u * kWave;
    if (d >= A.D) break;
    if (A.dk) store_from_f32<DT>(A.dk, (t * A.G + g) * A.D + d, lost_k ? __builtin_nanf("") : ok[u] * A.scale);
    if (A.dv) store_from_f32<DT>(A.dv, (t * A.G + g) * A.D + d, lost_v ? __builtin_nanf("") : ov[u]);
  }
}

// SINKS: the rows of one chunk that see the first tokens from behind the window; their sums go to A.part.
template <int DT, int NK, int KT, bool SINKS>
__global__ __launch_bounds__(256, 1) void window_dkv_kernel(WindowBwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int DP = 32 * NK, RS = DP + Fragment<DT>::kPad, ND = DP / 16, BK = 64 * KT, QS = 32;
  constexpr float kUp = DT == kF16 ? 15.f : 0.f;
  __shared__ alignas(16) E qbuf[2][QS * RS], gbuf[2][QS * RS];
  __shared__ alignas(16) float shift_of[2][QS], delta_of[2][QS];
  __shared__ alignas(16) int token_at[2][QS];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t item = A.first + blockIdx.x;
  const int g = static_cast<int>(item % A.G), ratio = A.ratio.d;
  item /= A.G;
  TilePlace at;
  int j0, from, to;  // first key; tokens of the rows
  int64_t number = item;
  if constexpr (SINKS) {
    number = item / A.sink_tiles;
    at = tile_place<kChunk>(A.cu, A.nseq, number, 1);
    j0 = static_cast<int>(item - number * A.sink_tiles) * BK;
    const int64_t behind = static_cast<int64_t>(j0) + BK - 1 + A.seen.window, start = static_cast<int64_t>(at.tile) * kChunk;
    if (max(behind, start) >= at.n) return;
    from = static_cast<int>(max(behind, start));
    to = static_cast<int>(min(start + kChunk, static_cast<int64_t>(at.n)));
    if (from >= to) return;
  } else {
    at = tile_place<BK>(A.cu, A.nseq, item, 1);
    if (static_cast<int64_t>(at.tile) * BK >= at.n) return;
    j0 = at.tile * BK;
    from = j0;
    to = static_cast<int>(min(static_cast<int64_t>(at.n), static_cast<int64_t>(j0) + BK - 1 + A.seen.window));
  }
  const int rb = from * ratio, re = to * ratio;

  // keys of this wave: [ka, kb], lane c one of each 16
  const int ka = j0 + 16 * KT * wave, last = SINKS ? min(at.n, A.seen.sinks) - 1 : at.n - 1;
  const int kb = min(ka + 16 * KT - 1, last);
  const bool has_keys = ka <= last;
  Fragment<DT> kf[KT][NK], vf[KT][NK];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int64_t t = at.start + static_cast<int64_t>(min(ka + 16 * kt + c, at.n - 1));
    const E* k = static_cast<const E*>(A.k.base) + t * A.k.token + g * A.k.head;
    const E* v = static_cast<const E*>(A.v.base) + t * A.v.token + g * A.v.head;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = 32 * kk + 8 * q4;
      kf[kt][kk] = d < A.D ? fragment_at<DT>(k + d) : no_fragment<DT>();
      vf[kt][kk] = d < A.D ? fragment_at<DT>(v + d) : no_fragment<DT>();
    }
  }
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
    auto row_of = [&](const PackedView& x, int r) {
      r = min(r, re - 1);
      const int t = A.ratio(r);
      return static_cast<const E*>(x.base) + (at.start + static_cast<int64_t>(t)) * x.token +
             (g * ratio + r - t * ratio) * x.head;
    };
    qload.load(A.D, [&](int r) { return row_of(A.q, r0 + r); });
    gload.load(A.D, [&](int r) { return row_of(A.dout, r0 + r); });
    if (threadIdx.x < QS) {
      const int r = min(r0 + static_cast<int>(threadIdx.x), re - 1), t = A.ratio(r);
      const int64_t row = (at.start + static_cast<int64_t>(t)) * (A.G * ratio) + g * ratio + r - t * ratio;
      const float lse = A.lse[row];
      own_shift = lse == -__builtin_inff() ? -__builtin_inff() : -lse / kLn2Window;
      own_delta = A.delta[row];
      own_token = r0 + static_cast<int>(threadIdx.x) < re ? t : -1;  // (no row: sees nothing)
    }
  };
  auto store_step = [&](int b) {
    qload.store(qbuf[b], RS, A.D);
    gload.store(gbuf[b], RS, A.D);
    if (threadIdx.x < QS)
      shift_of[b][threadIdx.x] = own_shift, delta_of[b][threadIdx.x] = own_delta, token_at[b][threadIdx.x] = own_token;
  };

  load_step(rb);
  store_step(0);
  int b = 0;
  for (int r0 = rb; r0 < re; r0 += QS, b ^= 1) {
    __syncthreads();
    const bool more = r0 + QS < re;
    if (more) load_step(r0 + QS);
    const int ta = A.ratio(r0), tb = A.ratio(min(r0 + QS, re) - 1);
    if (has_keys && tb >= ka && (ta - kb < A.seen.window || ka < A.seen.sinks)) {
      const E *qt = qbuf[b], *gt = gbuf[b];
      f32x4 s[2][KT], dp[2][KT];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) s[h][kt] = dp[h][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const Fragment<DT> qf = fragment_at<DT>(qt + (16 * h + c) * RS + 32 * kk + 8 * q4);
          const Fragment<DT> gf = fragment_at<DT>(gt + (16 * h + c) * RS + 32 * kk + 8 * q4);
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            s[h][kt] = product<DT>(qf, kf[kt][kk], s[h][kt]);
            dp[h][kt] = product<DT>(gf, vf[kt][kk], dp[h][kt]);
          }
        }
      }
      const bool whole = r0 + QS <= re && ta >= kb && (tb - ka < A.seen.window || kb < A.seen.sinks);
      Fragment<DT> pf[KT], df[KT];
      f32x4 shift[2], delta[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        shift[h] = *reinterpret_cast<const f32x4*>(&shift_of[b][16 * h + 4 * q4]);
        delta[h] = *reinterpret_cast<const f32x4*>(&delta_of[b][16 * h + 4 * q4]);
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        float p[8], ds[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          p[i] = __builtin_amdgcn_exp2f(fmaf(s[i >> 2][kt][i & 3], A.scale_log2, shift[i >> 2][i & 3]));
          ds[i] = p[i] * (dp[i >> 2][kt][i & 3] - delta[i >> 2][i & 3]);
        }
        if (!whole) {
          const int j = ka + 16 * kt + c;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const bool seen = A.seen(token_at[b][16 * (i >> 2) + 4 * q4 + (i & 3)], j);
            p[i] = seen ? p[i] : 0.f;
            ds[i] = seen ? ds[i] : 0.f;
          }
        }
        if constexpr (DT == kF16) {
          float big = 0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(ds[i]));
          big = quad_max(big);
          if (__any(big >= range[kt].cap && big != 0.f)) {
            const float factor = range[kt].widen(big);
#pragma unroll
            for (int d = 0; d < ND; ++d) dk[kt][d] *= factor;
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) ds[i] *= range[kt].up, p[i] *= 0x1p15f;
        }
        pf[kt] = pack_fragment<DT>(p);
        df[kt] = pack_fragment<DT>(ds);
      }
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const Fragment<DT> gf = column_fragment<DT>(gt, RS, 0, 16 * d, c, q4);
        const Fragment<DT> qf = column_fragment<DT>(qt, RS, 0, 16 * d, c, q4);
#pragma unroll
        for (int kt = 0; kt < KT; ++kt) {
          dv[kt][d] = product<DT>(gf, pf[kt], dv[kt][d]);
          dk[kt][d] = product<DT>(qf, df[kt], dk[kt][d]);
        }
      }
    }
    if (more) store_step(b ^ 1);
  }

  const int64_t tile_floats = int64_t{2} * A.sink_rows * A.D;  // of one chunk, tile of first tokens and key head
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    const int j = ka + 16 * kt + c, local = j - j0;
    const float down_k = DT == kF16 ? A.scale * range[kt].down() : A.scale, down_v = kUp == 0.f ? 1.f : 0x1p-15f;
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[kt][d] *= down_k, dv[kt][d] *= down_v;
    if constexpr (SINKS) {
      if (j > last) continue;
      float* part = A.part + (item * A.G + g) * tile_floats + static_cast<int64_t>(local) * A.D;
#pragma unroll
      for (int d = 0; d < ND; ++d)
        if (16 * d + 4 * q4 < A.D) {
          *reinterpret_cast<f32x4*>(part + 16 * d + 4 * q4) = dk[kt][d];
          *reinterpret_cast<f32x4*>(part + static_cast<int64_t>(A.sink_rows) * A.D + 16 * d + 4 * q4) = dv[kt][d];
        }
    } else {
      const bool mine = j < at.n;
      if (mine && j < A.seen.sinks && to < at.n) {  // what the chunks of later rows gave
        const int64_t chunk0 = static_cast<int64_t>(at.start) / kChunk + at.seq;
        for (int ch = to / kChunk; ch <= (at.n - 1) / kChunk; ++ch) {
          const float* part = A.part + (((chunk0 + ch) * A.sink_tiles + at.tile) * A.G + g) * tile_floats +
                              static_cast<int64_t>(local) * A.D;
#pragma unroll
          for (int d = 0; d < ND; ++d)
            if (16 * d + 4 * q4 < A.D) {
              dk[kt][d] += *reinterpret_cast<const f32x4*>(part + 16 * d + 4 * q4);
              dv[kt][d] += *reinterpret_cast<const f32x4*>(part + static_cast<int64_t>(A.sink_rows) * A.D + 16 * d + 4 * q4);
            }
        }
      }
      const int64_t row = (at.start + static_cast<int64_t>(mine ? j : 0)) * A.G + g;
      float all = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        all += ((dk[kt][d][0] + dk[kt][d][1]) + (dk[kt][d][2] + dk[kt][d][3])) +
               ((dv[kt][d][0] + dv[kt][d][1]) + (dv[kt][d][2] + dv[kt][d][3]));
        if (mine && 16 * d + 4 * q4 < A.D) {
          if (A.dk) store4<DT>(static_cast<E*>(A.dk) + row * A.D + 16 * d + 4 * q4, dk[kt][d]);
          if (A.dv) store4<DT>(static_cast<E*>(A.dv) + row * A.D + 16 * d + 4 * q4, dv[kt][d]);
        }
      }
      uint64_t odd = __ballot(mine && !finite(all));
      odd |= odd >> 32, odd |= odd >> 16;
      for (uint32_t left = odd & 0xffffu; left; left &= left - 1)
        careful_dkv<DT>(A, at.start, at.n, g, ka + 16 * kt + __builtin_ctz(left));
    }
  }
}

// Keys of a workgroup of the dK / dV kernels.
int keys_per_tile(int32_t dtype, int64_t dim) { return dtype != kF32 && dim <= 128 ? 128 : 64; }

// Tiles that hold first tokens, and their rows in one; 0 where no sequence has rows behind the window.
struct SinkShape {
  int64_t tiles, rows;
};
SinkShape sink_shape(int32_t dtype, int64_t dim, int64_t longest, int64_t window, int64_t sinks) {
  if (window == 0 || sinks == 0 || longest <= window) return SinkShape{0, 0};
  const int64_t keys = keys_per_tile(dtype, dim), most = sinks < longest ? sinks : longest;
  return SinkShape{(most + keys - 1) / keys, most < keys ? (most + 15) / 16 * 16 : keys};
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int64_t msa_window_attn_bwd_workspace_bytes(int32_t dtype, int64_t total_tokens, int64_t num_seqs,
                                                       int64_t longest, int64_t q_heads, int64_t kv_groups,
                                                       int64_t head_dim, int64_t window, int64_t sinks) {
  if (total_tokens <= 0 || num_seqs <= 0 || q_heads <= 0 || kv_groups <= 0 || head_dim <= 0 || window < 0 || sinks < 0) return 0;
  const SinkShape shape = sink_shape(dtype, head_dim, longest, window, sinks);
  const int64_t rows = (total_tokens * q_heads + 3) / 4 * 4;
  return 4 * (rows + tile_numbers(total_tokens, num_seqs, 1, kChunk) * shape.tiles * kv_groups * 2 * shape.rows * head_dim);
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
  if (strides[6] % unit || strides[7] % unit) return kErrInvalidArgument;
  if (!window_supported(dtype, head_dim, total_tokens, q_heads / kv_groups)) return kErrUnsupported;
  if (total_tokens == 0 || !(grad_q || grad_k || grad_v)) return kOk;
  if (!workspace || workspace_bytes < msa_window_attn_bwd_workspace_bytes(dtype, total_tokens, num_seqs, longest, q_heads,
                                                                          kv_groups, head_dim, window, sinks))
    return kErrInvalidArgument;
  const SinkShape shape = sink_shape(dtype, head_dim, longest, window, sinks);
  WindowBwdArgs A{};
  A.q = PackedView{q, strides[0], strides[1]};
  A.k = PackedView{k, strides[2], strides[3]};
  A.v = PackedView{v, strides[4], strides[5]};
  A.dout = PackedView{grad_out, strides[6], strides[7]};
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
  A.part = A.delta + (total_tokens * q_heads + 3) / 4 * 4;
  A.sink_tiles = static_cast<int>(shape.tiles);
  A.sink_rows = static_cast<int>(shape.rows);
  A.dq = grad_q;
  A.dk = grad_k;
  A.dv = grad_v;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  int rc = launch_parts((total_tokens * q_heads + 15) / 16, [&](int64_t first, unsigned count) {
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
      MSA_WINDOW_LAUNCH((window_dq_kernel<DT, NK, MT, KS>), tile_numbers(total_tokens, num_seqs, A.ratio.d, 64 * MT) * kv_groups); \
    if (rc == kOk && (grad_k || grad_v) && shape.tiles)                                                                          \
      MSA_WINDOW_LAUNCH((window_dkv_kernel<DT, NK, KT, true>),                                                                   \
                        tile_numbers(total_tokens, num_seqs, 1, kChunk) * shape.tiles * kv_groups);                              \
    if (rc == kOk && (grad_k || grad_v))                                                                                         \
      MSA_WINDOW_LAUNCH((window_dkv_kernel<DT, NK, KT, false>), tile_numbers(total_tokens, num_seqs, 1, 64 * KT) * kv_groups);   \
    return rc;                                                                                                                   \
  }
  if (dtype == kF32) {
    if (head_dim <= 64) MSA_WINDOW_BWD(kF32, 2, 1, 32, 1)
    if (head_dim <= 128) MSA_WINDOW_BWD(kF32, 4, 1, 32, 1)
    MSA_WINDOW_BWD(kF32, 8, 1, 32, 1)
  }
#define MSA_WINDOW_BWD_DIM(DT)                        \
  if (head_dim <= 64) MSA_WINDOW_BWD(DT, 2, 2, 32, 2) \
  if (head_dim <= 128) MSA_WINDOW_BWD(DT, 4, 2, 32, 2) \
  MSA_WINDOW_BWD(DT, 8, 1, 32, 1)
  if (dtype == kBF16) { MSA_WINDOW_BWD_DIM(kBF16) }
  MSA_WINDOW_BWD_DIM(kF16)
#undef MSA_WINDOW_BWD_DIM
#undef MSA_WINDOW_BWD
#undef MSA_WINDOW_LAUNCH
}
