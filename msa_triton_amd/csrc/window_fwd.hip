// Causal attention of packed sequences with a sliding window and a few first tokens that stay visible: forward.
//
//   out[i, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[i, h] . k_j - max),
// over the keys that token i sees (window.hpp), one pass over them with the running maximum and sum of each row.
//
// Bound by the matrix products (4 D flops a pair, against 2 R bytes of keys and values from L2 for R rows). A
// workgroup has R = 64 MT rows of one key head, 16 MT a wave; keys and values of a step go to LDS, two steps'
// worth, the next one's loads in flight during this one's products. S^T = K Q^T puts a row into a lane's column, so that
// maximum and sum need two exchanges, and the weights P^T leave that product in the operand layout of
// O^T = V^T P^T (values by transposed reads with the keys in that same order).
//
// Logits, statistics and outputs are fp32. The weights enter the second product rounded once to the input type (half a step
// of 2^-8 in bf16, of the size of the output's own rounding and averaged over the keys: 0.0021 of the output where its own
// is 0.0017; in fp16 times 2^7, so that weights down to 2^-21 keep their bits). For a backward pass they are two terms: its
// delta = dO . out goes into every ds of a row, and dq and dk would be off by 0.0005 of themselves more. The
// sum of the weights is that of the unrounded ones. 32K tokens, 32 heads of 128 over 4, window 4096, bf16: 2.25 ms
// (920 TFLOP/s), for a backward pass 2.87.
#include "window.hpp"

namespace msa {
namespace {

struct WindowFwdArgs {
  PackedView q, k, v;
  const int32_t* cu;
  int nseq, ratio, G, D;
  Visible seen;
  float scale_log2;  // scale * log2(e)
  int64_t first;     // workgroup of this launch's first
  void* out;         // [T][Hq][D]
  void* out_lo;      // what the rounding of out left out, or null
  float* lse;        // [T][Hq], or null
};

// The dims of a row that came out not finite, by a wave: where a value that is not finite met the products of a tile, which
// multiply the keys that a row does not see by 0. Such values count whatever their weight above 0; a weight of 0 under
// a logit of -inf makes NaN of them. Dims in which the row sees one are these values' sum, which takes a look at their
// column; the others are formed again key by key, from weights whose sum is 1 (values next to the end of fp32's range, of
// which a tile's sums are infinities, have a finite mean). The weight is exp2(logit * log2(e) + shift) inv.
template <int DT>
__device__ __forceinline__ void careful_row(const WindowFwdArgs& A, int start, int g, int tok, int head, float shift,
                                            float inv) {
  using E = typename Fragment<DT>::Element;
  const int lane = threadIdx.x & 63;
  const E* q = static_cast<const E*>(A.q.base) + A.q.at(start + static_cast<int64_t>(tok), head);
  const E* k = static_cast<const E*>(A.k.base) + A.k.at(start, g);
  const E* v = static_cast<const E*>(A.v.base) + A.v.at(start, g);
  const int low = A.seen.low(tok), sinks = min(A.seen.sinks, low);
  const int64_t at = ((start + static_cast<int64_t>(tok)) * (A.G * A.ratio) + head) * A.D;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // (what this wave's other lanes stored)
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  float o[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) bad[u] = lane + u * kWave < A.D && !finite(load_as_f32<DT>(A.out, at + lane + u * kWave));
  auto open = [&]() {  // dims whose value may still change
    bool any = false;
#pragma unroll
    for (int u = 0; u < 4; ++u) any |= bad[u] && odd[u] == odd[u];
    return __any(any);
  };
  auto column = [&](int from, int to) {
    for (int base = from; base < to && open(); base += kWave) {
      uint64_t dead = 0;  // keys of a logit of -inf, looked for when a value is infinite
      bool known = false;
      for (int j = base; j < min(to, base + kWave); ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float y = bad[u] ? value_at<DT>(v + static_cast<int64_t>(j) * A.v.token, lane + u * kWave) : 0.f;
          if (!known && __any(!finite(y) && y == y)) {
            dead = __ballot(row_dot<DT>(q, k + static_cast<int64_t>(min(base + lane, to - 1)) * A.k.token, A.D) * A.scale_log2 ==
                            -__builtin_inff());
            known = true;
          }
          if (!finite(y)) odd[u] += dead >> (j - base) & 1 ? __builtin_nanf("") : y;
        }
    }
  };
  column(0, sinks);
  column(low, tok + 1);
  bool again = false;
#pragma unroll
  for (int u = 0; u < 4; ++u) again |= bad[u] && odd[u] == 0.f;
  auto keys = [&](int from, int to) {
    for (int base = from; base < to; base += kWave) {
      const int j = min(base + lane, to - 1), count = min(kWave, to - base);
      const float x = row_dot<DT>(q, k + static_cast<int64_t>(j) * A.k.token, A.D) * A.scale_log2;
      const float p = __builtin_amdgcn_exp2f(x + shift) * inv;
      for (int i = 0; i < count; ++i) {
        const float p_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (bad[u] && odd[u] == 0.f) o[u] = fmaf(p_i, value_at<DT>(v + static_cast<int64_t>(base + i) * A.v.token, lane + u * kWave), o[u]);
      }
    }
  };
  if (__any(again)) {
    keys(0, sinks);
    keys(low, tok + 1);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (!bad[u]) continue;
    const int d = lane + u * kWave;
    const float y = odd[u] != 0.f ? odd[u] : o[u];
    store_from_f32<DT>(A.out, at + d, y);
    if (DT != kF32 && A.out_lo) {
      uint16_t high;
      store_from_f32<DT>(&high, 0, y);
      const float lo = y - load_as_f32<DT>(&high, 0);
      store_from_f32<DT>(A.out_lo, at + d, lo == lo ? lo : 0.f);
    }
  }
}

// TWO: weights as two terms.
template <int DT, int NK, int MT, int KS, bool TWO>
__global__ __launch_bounds__(256, NK > 4 ? (DT == kF32 ? 1 : 2) : DT == kF32 ? 2 : 3) void window_fwd_kernel(WindowFwdArgs A) {
  using E = typename Fragment<DT>::Element;
  constexpr int DP = 32 * NK, RS = DP + Fragment<DT>::kPad, ND = DP / 16, KT = KS / 16, R = 64 * MT;
  constexpr float kUp = DT == kF16 ? 15.f - kSlack : 0.f;
  // The weight of a row's only key is 1 to the last bit, and its output the value (what delta relies on); one operation more.
  constexpr bool kExact = TWO || DT == kF32;
  __shared__ alignas(16) E kbuf[2][KS * RS], vbuf[2][KS * RS];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = A.first + blockIdx.x;
  const int g = static_cast<int>(item % A.G);
  const TilePlace at = tile_place(A.cu, A.nseq, item / A.G, A.ratio, log2_of(R));
  const int64_t rows = static_cast<int64_t>(at.n) * A.ratio, r0 = static_cast<int64_t>(at.tile) * R;
  if (r0 >= rows) return;
  const int live = static_cast<int>(min(rows - r0, int64_t{R}));
  const int t0 = static_cast<int>(r0 / A.ratio), t1 = static_cast<int>((r0 + live - 1) / A.ratio);
  const int off = static_cast<int>(r0 - static_cast<int64_t>(t0) * A.ratio);  // head of the first row
  auto token_of = [&](int r) { return t0 + (off + r) / A.ratio; };

  const E* kbase = static_cast<const E*>(A.k.base) + A.k.at(at.start, g);
  const E* vbase = static_cast<const E*>(A.v.base) + A.v.at(at.start, g);
  int tok[MT];
  Fragment<DT> qf[MT][NK];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = min(16 * (MT * wave + m) + c, live - 1);
    tok[m] = token_of(r);
    const E* row = static_cast<const E*>(A.q.base) +
                   A.q.at(at.start + static_cast<int64_t>(tok[m]), g * A.ratio + (off + r) % A.ratio);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
      qf[m][kk] = 32 * kk + 8 * q4 < A.D && A.scale_log2 != 0.f
                      ? turned<DT>(fragment_at<DT>(row + 32 * kk + 8 * q4), A.scale_log2 < 0.f)
                      : no_fragment<DT>();
  }
  // keys of this workgroup: sinks in front of the first row's window, then from there to the last row
  const int low = A.seen.low(t0), sinks = min(A.seen.sinks, low);
  const int sink_steps = (sinks + KS - 1) / KS, steps = sink_steps + (t1 - low) / KS + 1;
  auto first_key = [&](int e) { return e < sink_steps ? e * KS : low + (e - sink_steps) * KS; };
  // tokens of this wave's rows (none: first above last)
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

  // A maximum is kept of the raw dots (queries are turned where the scale is negative, and zero with a factor of 1 where it is 0).
  const float factor = A.scale_log2 == 0.f ? 1.f : fabsf(A.scale_log2), slack = raw_slack(factor);
  float top[MT], l[MT];
  f32x4 acc[MT][ND];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    top[m] = -__builtin_inff(), l[m] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  load_step(0);
  store_step(0);
  for (int e = 0; e < steps; ++e) {
    __syncthreads();
    if (e + 1 < steps) load_step(e + 1);
    const int j0 = first_key(e);
    const bool of_sinks = e < sink_steps;
    const E *kt_ = kbuf[e & 1], *vt_ = vbuf[e & 1];
    if (has_rows && (of_sinks || (j0 <= w1 && (j0 + KS > A.seen.low(w0) || j0 < A.seen.sinks)))) {
      f32x4 s[MT][KT];
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
        for (int m = 0; m < MT; ++m) s[m][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const Fragment<DT> kf = fragment_at<DT>(kt_ + (16 * kt + c) * RS + 32 * kk + 8 * q4);
#pragma unroll
          for (int m = 0; m < MT; ++m) s[m][kt] = product<DT>(kf, qf[m][kk], s[m][kt]);
        }
      }
      const bool whole = of_sinks ? j0 + KS <= sinks : j0 + KS - 1 <= w0 && (w1 - j0 < A.seen.window || j0 + KS <= A.seen.sinks);
      if (!whole) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int j = j0 + 16 * kt + 4 * q4 + i;
              const bool seen = of_sinks ? j < sinks : A.seen(tok[m], j);
              s[m][kt][i] = seen ? s[m][kt][i] : -__builtin_inff();
            }
      }
      Fragment<DT> pf[MT][KT / 2], pl[MT][KT / 2];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float high = s[m][0][0];
#pragma unroll
        for (int kt = 0; kt < KT; ++kt)
#pragma unroll
          for (int i = 0; i < 4; ++i) high = fmaxf(high, s[m][kt][i]);
        if (__any(high > top[m] + slack)) {
          const float next = fmaxf(top[m], quarters_max(high));
          const float keep = top[m] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((top[m] - next) * factor);
          top[m] = next;
          l[m] *= keep;
#pragma unroll
          for (int d = 0; d < ND; ++d) acc[m][d] *= keep;
        }
        const float base = top[m] == -__builtin_inff() ? 0.f : top[m], shift = kUp - base * factor;
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
          float p[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = s[m][2 * u + (i >> 2)][i & 3];
            p[i] = __builtin_amdgcn_exp2f(kExact ? fmaf(x - base, factor, kUp) : fmaf(x, factor, shift));
            l[m] += p[i];
          }
          pf[m][u] = pack_fragment<DT>(p);
          if constexpr (TWO) pl[m][u] = second_terms<DT>(pf[m][u], p);
        }
      }
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int u = 0; u < KT / 2; ++u) {
          const Fragment<DT> vf = column_fragment<DT>(vt_, RS, 32 * u, 16 * d, c, q4);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            acc[m][d] = product<DT>(vf, pf[m][u], acc[m][d]);
            if constexpr (TWO) acc[m][d] = product<DT>(vf, pl[m][u], acc[m][d]);
          }
        }
    }
    if (e + 1 < steps) store_step(e + 1);
  }

#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int r = 16 * (MT * wave + m) + c;
    const bool mine = r < live;
    l[m] += __shfl_xor(l[m], 16, kWave);
    l[m] += __shfl_xor(l[m], 32, kWave);
    const float inv = l[m] == 0.f ? 0.f : 1.f / l[m];
    const int head = g * A.ratio + (off + (mine ? r : 0)) % A.ratio;
    const int64_t at_row = (at.start + static_cast<int64_t>(tok[m])) * (A.G * A.ratio) + head;
    E* out = static_cast<E*>(A.out) + at_row * A.D;
    E* lo = static_cast<E*>(A.out_lo) + at_row * A.D;
    float all = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const f32x4 o = acc[m][d] * inv;
      all += (o[0] + o[1]) + (o[2] + o[3]);
      if (mine && 16 * d + 4 * q4 < A.D) {
        store4<DT>(out + 16 * d + 4 * q4, o);
        if constexpr (DT != kF32)
          if (A.out_lo) store4<DT>(lo + 16 * d + 4 * q4, left_out<DT>(o));
      }
    }
    const float level = top[m] == -__builtin_inff() ? 0.f : top[m] * factor;
    if (mine && q4 == 0 && A.lse)
      A.lse[at_row] = l[m] == 0.f ? -__builtin_inff() : (level - kUp + __log2f(l[m])) * kLn2Window;
    // (a sum of NaN makes the row NaN)
    uint64_t odd = __ballot(mine && !finite(all) && l[m] == l[m]);
    if constexpr (DT != kF32)
      if (odd && A.out_lo) {  // (the two terms above come from pairs of values: one that is not finite spoils its neighbour's)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = acc[m][d][i] * inv;
            uint16_t high;
            store_from_f32<DT>(&high, 0, x);
            if (mine && 16 * d + 4 * q4 < A.D) store_from_f32<DT>(lo, 16 * d + 4 * q4 + i, x - load_as_f32<DT>(&high, 0));
          }
      }
    odd |= odd >> 32, odd |= odd >> 16;
    for (uint32_t left = odd & 0xffffu; left; left &= left - 1) {
      const int from = __builtin_ctz(left);
      careful_row<DT>(A, at.start, g, __builtin_amdgcn_readlane(tok[m], from), __builtin_amdgcn_readlane(head, from),
                      kUp - __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(level), from)),
                      __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inv), from)));
    }
  }
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_window_attn_fwd(const void* q, const void* k, const void* v, int32_t dtype, const int64_t* strides,
                                   const int32_t* cu_seqlens, int64_t num_seqs, int64_t total_tokens, int64_t q_heads,
                                   int64_t kv_groups, int64_t head_dim, int64_t window, int64_t sinks, double scale, void* out,
                                   void* out_lo, float* lse, void* stream) {
  if (!valid_window_call(q, k, v, dtype, strides, cu_seqlens, num_seqs, total_tokens, q_heads, kv_groups, head_dim, window,
                         sinks, scale) ||
      !out)
    return kErrInvalidArgument;
  if (!window_supported(head_dim, total_tokens, q_heads / kv_groups)) return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  WindowFwdArgs A{};
  A.q = packed_view(q, strides);
  A.k = packed_view(k, strides + 2);
  A.v = packed_view(v, strides + 4);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.ratio = static_cast<int>(q_heads / kv_groups);
  A.G = static_cast<int>(kv_groups);
  A.D = static_cast<int>(head_dim);
  A.seen = visible_of(window, sinks);
  A.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  A.out = out;
  A.out_lo = out_lo;
  A.lse = lse;
  hipStream_t st = static_cast<hipStream_t>(stream);
#define MSA_WINDOW_FWD(DT, NK, MT, TWO)                                                                                 \
  return launch_parts(tile_numbers(total_tokens, num_seqs, A.ratio, log2_of(64 * MT)) * kv_groups, [&](int64_t first, unsigned count) { \
    A.first = first;                                                                                                    \
    hipLaunchKernelGGL((window_fwd_kernel<DT, NK, MT, 32, TWO>), dim3(count), dim3(256), 0, st, A);                     \
  })
#define MSA_WINDOW_FWD_DIM(DT, MT, TWO)                  \
  {                                                      \
    if (head_dim <= 64) MSA_WINDOW_FWD(DT, 2, MT, TWO);  \
    if (head_dim <= 96) MSA_WINDOW_FWD(DT, 3, MT, TWO);  \
    if (head_dim <= 128) MSA_WINDOW_FWD(DT, 4, MT, TWO); \
    if (head_dim <= 192) MSA_WINDOW_FWD(DT, 6, 1, TWO);  \
    MSA_WINDOW_FWD(DT, 8, 1, TWO);                       \
  }
  // (out_lo is asked for where a backward pass takes the output)
  if (dtype == kBF16 && out_lo) MSA_WINDOW_FWD_DIM(kBF16, 2, true)
  if (dtype == kBF16) MSA_WINDOW_FWD_DIM(kBF16, 2, false)
  if (dtype == kF16 && out_lo) MSA_WINDOW_FWD_DIM(kF16, 2, true)
  if (dtype == kF16) MSA_WINDOW_FWD_DIM(kF16, 2, false)
  MSA_WINDOW_FWD_DIM(kF32, 1, false)
#undef MSA_WINDOW_FWD_DIM
#undef MSA_WINDOW_FWD
}
