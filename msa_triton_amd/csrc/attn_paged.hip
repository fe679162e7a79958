// Sparse attention of new tokens over the selected blocks of a paged cache (16-bit or e4m3 with a scale
// for each page and head).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),
// over the keys j <= position(t) of the blocks that (t, group of h) selected, each once. Keys and values of
// an 8-bit page are its bytes times its scales: the key scale goes into the logits and the value scale into the
// weights, so the bytes enter the matrix products as they are (e4m3 is exact in bf16 and fp16).
//
// Bound by reading the selected keys and values from HBM once (a decoding step has ratio x 4 flops a
// byte in bf16). A workgroup has one token, group and tile of 16 query heads; its four waves take
// steps of 32 keys from a list of the steps that hold visible keys, made in LDS first. A wave works on
// its own: key fragments straight from memory (lane c a key), logits S^T = K Q^T, running maximum and
// sum of its head (the lane's column), weights P^T as they come out of the product (the keys of a
// lane's four quarters), values through its LDS tile and transposed reads with the keys in that same order. The
// next step's loads are in flight during the softmax and the second product. Few rows: the steps of one row are
// split over several workgroups (split_count), whose maxima, sums and fp32 outputs a second launch joins in
// a fixed order.
//
// Logits, statistics and outputs are fp32. A weight enters the second product as two 16-bit terms
// (hi + lo, 2^-17 of it left out), so that the output's error stays that of its own rounding: one term would add 2^-9 of a
// weight. In fp16 they are the terms of the weight times 2^15 (fp16 ends at 2^-24; so weights down to 2^-22 keep that bound).
// Values of keys that are not visible are zeroed on their way to LDS: 0 x NaN is NaN.
#include "mfma_util.hpp"
#include "paged.hpp"

namespace msa {
namespace {

constexpr int kList = 256;       // steps listed at once: one a thread
constexpr int kIds = 1024;       // ids kept in LDS where there are more than 64, to find repeated ones
constexpr int kMostSplits = 64;  // of one row: a lane of the joining wave each

struct PagedAttnArgs {
  const uint16_t* q;  // [T][Hq][D]
  CacheView k, v;
  const float *k_scale, *v_scale;  // [P][G]
  PageMap pages;
  const int32_t* indices;  // [T][G][K]
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  int64_t tokens;
  int Hq, G, D, K, B;
  int head_tiles, splits;
  int64_t first;     // item (joining launch: workgroup) of this launch's first workgroup
  float scale_log2;  // scale * log2(e)
  uint16_t* out;     // [T][Hq][D]
  float* lse;        // [T][Hq], or null
  float* part;       // [items][splits][16][D]
  float* stats;      // [items][splits][2][16]: maximum (log2), sum
};

constexpr float kLn2 = 0.69314718055994531f;
// The least maximum of keys that exist (all of their logits may be -inf); -inf stands for no key.
constexpr float kLeastMax = -3.402823466e38f;

template <int DT, bool FP8, int NK>
__global__ __launch_bounds__(256, NK == 8 && !FP8 ? 1 : 2) void attn_paged_kernel(PagedAttnArgs A) {
  constexpr int DP = 32 * NK, RS = DP + 16, ND = DP / 16;
  constexpr int PT = FP8 ? kBF16 : DT;          // type of the second product
  constexpr int VL = FP8 ? DP / 16 : DP / 8;    // lanes of one value row
  constexpr int NV = VL / 2, VR = 64 / VL;      // 16-byte pieces of 32 rows, rows of a piece
  constexpr int VD = FP8 ? 16 : 8;              // values of a piece
  constexpr float kUp = PT == kF16 ? 0x1p15f : 1.f;  // of the weights in the second product
  constexpr int NKR = FP8 ? NK / 2 : NK;        // 16-byte pieces of a key row and lane
  __shared__ alignas(16) uint16_t vbuf[4][32 * RS];
  __shared__ int list_key[kList], list_p0[kList], list_p1[kList], listed[4];
  __shared__ float wave_max[4][16], wave_sum[4][16];
  __shared__ int early_ids[kIds];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t item = A.first + blockIdx.x / static_cast<unsigned>(A.splits);
  const int split = static_cast<int>(blockIdx.x % static_cast<unsigned>(A.splits));
  const int ht = static_cast<int>(item % A.head_tiles);
  const int64_t tg = item / A.head_tiles, t = tg / A.G;
  const int g = static_cast<int>(tg % A.G);
  const int ratio = A.Hq / A.G, head = 16 * ht + c;
  const int32_t* ids = A.indices + tg * A.K;
  const int32_t wave_id = lane < A.K ? ids[lane] : -1;  // the first 64 ids, one a lane
  if (A.K > 64) {
    for (int i = threadIdx.x; i < min(A.K, kIds); i += 256) early_ids[i] = ids[i];
    __syncthreads();
  }
  const bool full = A.D == DP;

  // dims of a lane in step kk of the first product (any order, the same for keys and queries)
  auto dim_of = [&](int kk) { return FP8 ? 64 * (kk >> 1) + 16 * q4 + 8 * (kk & 1) : 32 * kk + 8 * q4; };
  bf16x8 qf[NK];
  {
    const uint16_t* row = A.q + (t * A.Hq + g * ratio + (head < ratio ? head : 0)) * A.D;
#pragma unroll
    for (int kk = 0; kk < NK; ++kk)
      qf[kk] = head < ratio && dim_of(kk) < A.D ? load_frag(row + dim_of(kk)) : zero_frag();
  }

  const TokenPlace at = wave_place_of(A.cu, A.nseq, A.context, t);
  const int pos = static_cast<int>(min(at.pos, A.pages.last_position()));
  const int per_block = min((A.B - 1) / 32, pos / 32) + 1;  // steps of a block, of those up to the token
  // this workgroup's steps: every splits-th (the blocks that exist come first in a selection)
  const int64_t steps = pos < 0 ? 0 : static_cast<int64_t>(A.K) * per_block;

  float m = -__builtin_inff(), l = 0.f;  // of head c: the maximum over all quarters, the sum over this one
  bool had_keys = false;                 // this wave
  f32x4 acc[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};

  const char* kbase = static_cast<const char*>(A.k.base) + g * A.k.stride_head * (FP8 ? 1 : 2);
  const char* vbase = static_cast<const char*>(A.v.base) + g * A.v.stride_head * (FP8 ? 1 : 2);
  constexpr int ES = FP8 ? 1 : 2;
  const int slot_mask = (1 << A.pages.shift) - 1;
  uint4 kr[2][NKR], vr[NV];
  int key0 = 0, p0 = -1, p1 = -1;
  float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;
  auto load_step = [&](int e) {
    key0 = __builtin_amdgcn_readfirstlane(list_key[e]);
    p0 = __builtin_amdgcn_readfirstlane(list_p0[e]);
    p1 = __builtin_amdgcn_readfirstlane(list_p1[e]);
    const int64_t s0 = p0 < 0 ? 0 : p0, s1 = p1 < 0 ? 0 : p1;  // (page 0 exists; its rows are masked)
    const int slot0 = key0 & slot_mask, slot1 = (key0 + 16) & slot_mask;
    const char* kp[2] = {kbase + (s0 * A.k.stride_page + (slot0 + c) * A.k.stride_slot) * ES,
                         kbase + (s1 * A.k.stride_page + (slot1 + c) * A.k.stride_slot) * ES};
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < NKR; ++i) {
        const int d = FP8 ? 64 * i + 16 * q4 : 32 * i + 8 * q4;
        kr[h][i] = *reinterpret_cast<const uint4*>(kp[h] + (d < A.D ? d : 0) * ES);
      }
    const int d = lane % VL * VD;
    const char* v0 = vbase + (s0 * A.v.stride_page + (d < A.D ? d : 0)) * ES;
    const char* v1 = vbase + (s1 * A.v.stride_page + (d < A.D ? d : 0)) * ES;
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      const int r = p * VR + lane / VL;
      vr[p] = *reinterpret_cast<const uint4*>(
          p < NV / 2 ? v0 + (slot0 + r) * A.v.stride_slot * ES : v1 + (slot1 + r - 16) * A.v.stride_slot * ES);
    }
    if constexpr (FP8) {
      // (a page that is not there has weights of 0: its factor must be finite)
      ks0 = p0 < 0 ? 0.f : A.k_scale[s0 * A.G + g], ks1 = p1 < 0 ? 0.f : A.k_scale[s1 * A.G + g];
      vs0 = p0 < 0 ? 0.f : A.v_scale[s0 * A.G + g], vs1 = p1 < 0 ? 0.f : A.v_scale[s1 * A.G + g];
    }
  };

  for (int64_t base = split; base < steps; base += static_cast<int64_t>(kList) * A.splits) {
    // ---- the steps of this stretch that hold visible keys, in order
    const int64_t n = base + static_cast<int64_t>(threadIdx.x) * A.splits;
    int key = -1, a = -1, b = -1;
    const int slot = static_cast<int>(min(n, steps - 1) / per_block);
    const int id = A.K <= 64 ? __shfl(wave_id, slot, kWave) : ids[slot];
    bool again = false;  // an id that an earlier slot holds
    for (int i = 0; i < min(A.K, 64); ++i) again |= i < slot && __builtin_amdgcn_readlane(wave_id, i) == id;
    for (int i = 64; i < min(slot, kIds); ++i) again |= early_ids[i] == id;
    for (int i = kIds; i < slot; ++i) again |= ids[i] == id;
    if (n < steps) {
      const int step = static_cast<int>(n - static_cast<int64_t>(slot) * per_block);
      const int64_t first = static_cast<int64_t>(id) * A.B + 32 * step;
      if (id >= 0 && first <= pos) {
        if (!again) {
          a = A.pages.page_of(at.seq, first);
          b = 32 * step + 16 < A.B && first + 16 <= pos ? A.pages.page_of(at.seq, first + 16) : -1;
          if (a >= 0 || b >= 0) key = static_cast<int>(first);
        }
      }
    }
    const uint64_t mask = __ballot(key >= 0);
    if (lane == 0) listed[wave] = __popcll(mask);
    __syncthreads();
    int place = __popcll(mask & ((uint64_t{1} << lane) - 1)), count = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      place += w < wave ? listed[w] : 0;
      count += listed[w];
    }
    if (key >= 0) list_key[place] = key, list_p0[place] = a, list_p1[place] = b;
    __syncthreads();
    count = __builtin_amdgcn_readfirstlane(count);

    // ---- this wave's steps
    if (wave < count) load_step(wave), had_keys = true;
    for (int e = wave; e < count; e += 4) {
      const int k_now = key0, a_now = p0, b_now = p1;
      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          uint4 w;
          if constexpr (FP8) {
            const uint4 x = kr[h][kk >> 1];
            w = kk & 1 ? widen_fp8<DT == kF16>(x.z, x.w) : widen_fp8<DT == kF16>(x.x, x.y);
          } else {
            w = kr[h][kk];
          }
          if (!full && dim_of(kk) >= A.D) w = make_uint4(0u, 0u, 0u, 0u);
          s[h] = mfma_t<DT>(__builtin_bit_cast(bf16x8, w), qf[kk], s[h]);
        }
      }
      uint16_t* vt = vbuf[wave];
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        const int r = p * VR + lane / VL;
        const bool seen = (p < NV / 2 ? a_now : b_now) >= 0 && k_now + r <= pos;
        const uint4 x = seen ? vr[p] : make_uint4(0u, 0u, 0u, 0u);
        uint4* to = reinterpret_cast<uint4*>(vt + r * RS + lane % VL * VD);
        if constexpr (FP8) {
          to[0] = widen_fp8<false>(x.x, x.y);
          to[1] = widen_fp8<false>(x.z, x.w);
        } else {
          to[0] = x;
        }
      }
      const float kf0 = A.scale_log2 * ks0, kf1 = A.scale_log2 * ks1, vf0 = vs0, vf1 = vs1;
      if (e + 4 < count) load_step(e + 4);
      float x[8], top = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int h = j >> 2;
        const bool seen = (h ? b_now : a_now) >= 0 && k_now + 16 * h + 4 * q4 + (j & 3) <= pos;
        x[j] = seen ? s[h][j & 3] * (h ? kf1 : kf0) : -__builtin_inff();
        top = fmaxf(top, x[j]);
      }
      top = quad_max(top);
      if (__any(top > m)) {
        const float next = fmaxf(m, top);
        const float keep = m == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= keep;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= keep;
      }
      const float shift = m == -__builtin_inff() ? 0.f : m;  // (all logits -inf: weights 0)
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float y0 = __builtin_amdgcn_exp2f(x[j] - shift), y1 = __builtin_amdgcn_exp2f(x[j + 1] - shift);
        l += y0 + y1;
        if constexpr (PT == kF16) y0 *= kUp, y1 *= kUp;
        if constexpr (FP8) y0 *= j < 4 ? vf0 : vf1, y1 *= j < 4 ? vf0 : vf1;
        if constexpr (PT == kF16) {
          hi[j >> 1] = cvt_pk_f16(y0, y1);
          lo[j >> 1] = cvt_pk_f16(sub_lo_half_f16(hi[j >> 1], y0), sub_hi_half_f16(hi[j >> 1], y1));
        } else {
          hi[j >> 1] = cvt_pk_bf16(y0, y1);
          lo[j >> 1] = cvt_pk_bf16(sub_lo_half(hi[j >> 1], y0), sub_hi_half(hi[j >> 1], y1));
        }
      }
      const bf16x8 ph = __builtin_bit_cast(bf16x8, make_uint4(hi[0], hi[1], hi[2], hi[3]));
      const bf16x8 pl = __builtin_bit_cast(bf16x8, make_uint4(lo[0], lo[1], lo[2], lo[3]));
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const bf16x8 f = frag_tr(vt, RS, 4 * q4, 16 + 4 * q4, 16 * d, c);
        acc[d] = mfma_t<PT>(f, ph, acc[d]);
        acc[d] = mfma_t<PT>(f, pl, acc[d]);
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
    __syncthreads();  // the list and the tiles are free again
  }

  // ---- the four waves joined: maxima and sums, then the outputs through LDS. A part with keys enters also with a factor of
  // 0, and a dim that is not finite in any part is looked at again (odd_values).
  if (had_keys) m = fmaxf(m, kLeastMax);
  l += __shfl_xor(l, 16, kWave);
  l += __shfl_xor(l, 32, kWave);
  if (q4 == 0) wave_max[wave][c] = m, wave_sum[wave][c] = l;
  constexpr int OS = DP + 4;  // floats from one head's row to the next
  static_assert(16 * OS * 4 <= 32 * RS * 2, "a wave's output fits its value tile");
  float* mine = reinterpret_cast<float*>(vbuf[wave]);
#pragma unroll
  for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(mine + c * OS + 16 * d + 4 * q4) = acc[d];
  __syncthreads();
  const int row = threadIdx.x >> 4, col = threadIdx.x & 15;  // 16 threads a head
  float top = fmaxf(fmaxf(wave_max[0][row], wave_max[1][row]), fmaxf(wave_max[2][row], wave_max[3][row]));
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    f[w] = wave_max[w][row] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(wave_max[w][row] - top);
    sum += f[w] * wave_sum[w][row];
  }
  const int h = 16 * ht + row;
  if (h >= ratio) return;
  const int64_t out_row = t * A.Hq + g * ratio + h;
  // The values of dims d .. d + 3 that are not finite, added up over this workgroup's keys; 0 where there are none. A weight is
  // positive, so an infinity stays itself whatever its weight and NaN comes of both signs; under a logit of -inf (weight 0) it
  // is NaN. The matrix product cannot tell: a weight's two terms are 0 or negative as well. Rare, so a thread reads all keys.
  auto odd_values = [&](int d) {
    f32x4 odd = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int64_t n = split; n < steps; n += A.splits) {
      const int64_t slot = n / per_block;  // (repeated ids add nothing new)
      const int id = ids[slot], step = static_cast<int>(n - slot * per_block);
      for (int half = 0; half < 2; ++half) {
        const int64_t first = static_cast<int64_t>(id) * A.B + 32 * step + 16 * half;
        if (id < 0 || first > pos || 32 * step + 16 * half >= A.B) break;
        const int64_t page = A.pages.page_of(at.seq, first);
        if (page < 0) continue;
        const int64_t slot0 = first & slot_mask;
        const char* vp = vbase + (page * A.v.stride_page + slot0 * A.v.stride_slot + d) * ES;
        const char* kp = kbase + (page * A.k.stride_page + slot0 * A.k.stride_slot) * ES;
        const float vs = FP8 ? A.v_scale[page * A.G + g] : 1.f, ks = FP8 ? A.k_scale[page * A.G + g] : 1.f;
        const int keys = static_cast<int>(min(pos - first, int64_t{15})) + 1;
#pragma unroll 4
        for (int r = 0; r < keys; ++r) {
          float x[4];
          load4<DT, FP8>(vp + r * A.v.stride_slot * ES, x);
          bool some = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] *= vs, some |= !(fabsf(x[i]) < __builtin_inff());
          if (!some) continue;
          const uint16_t* qrow = A.q + (t * A.Hq + g * ratio + h) * A.D;
          float dot = 0.f;
          for (int e = 0; e < A.D; e += 4) {
            float y[4], z[4];
            load4<DT, false>(reinterpret_cast<const char*>(qrow + e), y);
            load4<DT, FP8>(kp + (r * A.k.stride_slot + e) * ES, z);
#pragma unroll
            for (int i = 0; i < 4; ++i) dot = fmaf(y[i], z[i], dot);
          }
          const bool none = dot * (A.scale_log2 * ks) == -__builtin_inff();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(fabsf(x[i]) < __builtin_inff())) odd[i] += none ? __builtin_nanf("") : x[i];
        }
      }
    }
    return odd;
  };
  const bool whole = A.splits == 1;
  const float inv = (whole ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f) / kUp;
  float* part = whole ? nullptr : A.part + ((item * A.splits + split) * 16 + row) * A.D;
  const bool none = !whole && top == -__builtin_inff();  // no keys: the joining launch does not look at it
  auto store = [&](int d, f32x4 o) {
    o *= inv;
    if (whole) {
      const uint2 r = DT == kF16 ? make_uint2(cvt_pk_f16(o[0], o[1]), cvt_pk_f16(o[2], o[3]))
                                 : make_uint2(cvt_pk_bf16(o[0], o[1]), cvt_pk_bf16(o[2], o[3]));
      *reinterpret_cast<uint2*>(A.out + out_row * A.D + d) = r;
    } else {
      *reinterpret_cast<f32x4*>(part + d) = o;
    }
  };
  float all = 0.f;  // not finite if an output is not, or a part with a factor of 0
  for (int d = 4 * col; d < A.D && !none; d += 64) {
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vbuf[w]) + row * OS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = fmaf(f[w], x[i], o[i]);
    }
    all += (o[0] + o[1]) + (o[2] + o[3]);
    store(d, o);
  }
  if (col == 0) {
    if (whole) {
      if (A.lse) A.lse[out_row] = sum == 0.f ? -__builtin_inff() : (top + __log2f(sum)) * kLn2;
    } else {
      float* st = A.stats + (item * A.splits + split) * 32;
      st[row] = top;
      st[16 + row] = sum;
    }
  }
  if (__builtin_expect(fabsf(all) < __builtin_inff() || sum != sum, 1)) return;  // (a sum of NaN makes the row NaN)
  for (int d = 4 * col; d < A.D && !none; d += 64) {
    const f32x4 odd = odd_values(d);
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int w = 0; w < 4; ++w) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vbuf[w]) + row * OS + d);
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = f[w] == 0.f ? o[i] : fmaf(f[w], x[i], o[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = odd[i] != 0.f ? odd[i] : o[i];  // (a sum past fp32's range stays one)
    store(d, o);
  }
}

// o + f x, with x itself where it is not finite: such a value counts whatever its weight, also 0.
__device__ __forceinline__ float add_part(float f, float x, float o) {
  return fabsf(x) < __builtin_inff() ? fmaf(f, x, o) : o + x;
}

// The splits of a row joined, a wave for each head's row: lane z weighs split z (at most kMostSplits = 64), and
// the lanes take two dims each of all of them, eight splits' loads in flight at a time (4 us: a launch and two loads' latency).
template <int DT>
__global__ __launch_bounds__(256) void attn_paged_join(PagedAttnArgs A) {
  const int lane = threadIdx.x & 63;
  const int64_t out_row = (A.first + blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (out_row >= A.tokens * A.Hq) return;
  const int64_t t = out_row / A.Hq;
  const int ratio = A.Hq / A.G, hq = static_cast<int>(out_row - t * A.Hq), g = hq / ratio, h = hq - g * ratio;
  const int64_t item = (t * A.G + g) * A.head_tiles + (h >> 4);
  const int row = h & 15;
  const float* st = A.stats + (item * A.splits + lane) * 32 + row;
  const bool live = lane < A.splits;
  const float top_z = live ? st[0] : -__builtin_inff(), sum_z = live ? st[16] : 0.f;
  const float top = wave_max_f32(top_z);
  const float weight = top_z == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(top_z - top);
  const float sum = wave_sum_f32(weight * sum_z);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const uint64_t written = __ballot(top_z != -__builtin_inff());  // (a split without keys wrote nothing)
  const float* part = A.part + (item * A.splits * 16 + row) * A.D;
  for (int d = 2 * lane; d < A.D; d += 128) {
    float o0 = 0.f, o1 = 0.f;
    for (int z0 = 0; z0 < A.splits; z0 += 8) {
      float2 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)  // (past the last split: that one again, as a split that wrote nothing)
        x[i] = *reinterpret_cast<const float2*>(part + static_cast<int64_t>(min(z0 + i, A.splits - 1)) * 16 * A.D + d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), z0 + i));
        const bool there = written >> (z0 + i) & 1u;
        o0 = there ? fmaf(f, x[i].x, o0) : o0;
        o1 = there ? fmaf(f, x[i].y, o1) : o1;
      }
    }
    if (__builtin_expect(!(fabsf(o0 + o1) < __builtin_inff()), 0)) {
      o0 = o1 = 0.f;
      for (int z = 0; z < A.splits; ++z) {
        if (!(written >> z & 1u)) continue;
        const float2 x = *reinterpret_cast<const float2*>(part + static_cast<int64_t>(z) * 16 * A.D + d);
        const float f = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(weight), z));
        o0 = add_part(f, x.x, o0);
        o1 = add_part(f, x.y, o1);
      }
    }
    reinterpret_cast<uint32_t*>(A.out)[(out_row * A.D + d) >> 1] =
        DT == kF16 ? cvt_pk_f16(o0 * inv, o1 * inv) : cvt_pk_bf16(o0 * inv, o1 * inv);
  }
  if (lane == 0 && A.lse) A.lse[out_row] = sum == 0.f ? -__builtin_inff() : (top + __log2f(sum)) * kLn2;
}

int64_t head_tiles_of(int64_t heads, int64_t groups) { return (heads / groups + 15) / 16; }

// Workgroups that share one row's steps. 512 of them (two a CU) run at once and draw what HBM gives (64 rows of 16
// blocks over 4 groups: 256 items of 128 dims in bf16 take 52 us, 5.1 TB/s, as 512 workgroups, 58 as 768 and 55 as 1024;
// e4m3 33, 34 and 38); a workgroup costs about four steps of its waves before the first and after the last one. So:
// the number with the fewest steps, rounds of 512 times the steps of a wave and those four. 328 items of 128 steps as
// 328, 656 and 984 workgroups: 112, 115 and 98 us; 4 items of 64 steps: one step a wave, 64 workgroups, 13 us.
int64_t split_count(int64_t items, int64_t slots, int64_t block_size) {
  const int64_t steps = slots * ((block_size - 1) / 32 + 1);
  int64_t best = 1, cost = -1;
  for (int64_t n = 1; n == 1 || (n <= (steps + 3) / 4 && n <= kMostSplits); ++n) {
    const int64_t x = ((items * n + 511) / 512) * ((steps + 4 * n - 1) / (4 * n) + 4);
    if (cost < 0 || x < cost) best = n, cost = x;
  }
  return best;
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int64_t msa_attn_paged_workspace_bytes(int64_t total_tokens, int64_t q_heads, int64_t kv_groups,
                                                  int64_t head_dim, int64_t topk_slots, int64_t block_size) {
  if (total_tokens <= 0 || q_heads <= 0 || kv_groups <= 0 || q_heads % kv_groups || head_dim <= 0 || topk_slots < 0 ||
      block_size <= 0)
    return 0;
  const int64_t items = total_tokens * kv_groups * head_tiles_of(q_heads, kv_groups);
  const int64_t splits = split_count(items, topk_slots, block_size);
  return splits == 1 ? 0 : items * splits * (16 * head_dim + 32) * static_cast<int64_t>(sizeof(float));
}

extern "C" int msa_attn_paged(const void* q, const void* k_cache, const void* v_cache, int32_t dtype,
                              int32_t cache_is_fp8, const float* k_scale, const float* v_scale, const int64_t* strides,
                              const int32_t* indices, const int32_t* page_table, int64_t table_stride,
                              int64_t pages_per_seq, int64_t num_pages, int64_t page_size, const int32_t* cu_seqlens,
                              int64_t num_seqs, const int32_t* context_lens, int64_t total_tokens, int64_t q_heads,
                              int64_t kv_groups, int64_t head_dim, int64_t topk_slots, int64_t block_size, double scale,
                              void* workspace, int64_t workspace_bytes, void* out, float* lse, void* stream) {
  if (!q || !out || !strides || !cu_seqlens || !context_lens || num_seqs <= 0 || num_seqs > 0x3fffffff ||
      total_tokens < 0 || total_tokens > 0x7fffffff || q_heads <= 0 || kv_groups <= 0 || q_heads % kv_groups ||
      q_heads >= (1 << 20) || head_dim <= 0 || topk_slots < 0 || topk_slots > 0x7fffffff || (topk_slots > 0 && !indices) ||
      block_size <= 0 || block_size > 0x7fffffff || !__builtin_isfinite(scale) || (dtype != kBF16 && dtype != kF16) ||
      !valid_pages(page_table, table_stride, pages_per_seq, num_pages, page_size) ||
      (num_pages > 0 && (!k_cache || !v_cache || (cache_is_fp8 && (!k_scale || !v_scale)))))
    return kErrInvalidArgument;
  const int unit = cache_is_fp8 ? 16 : 8;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % unit) return kErrInvalidArgument;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(k_cache) % 16 ||
      reinterpret_cast<uintptr_t>(v_cache) % 16)
    return kErrInvalidArgument;
  if (head_dim % 16 || head_dim > 256 || block_size % 16) return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  PagedAttnArgs A{};
  A.q = static_cast<const uint16_t*>(q);
  A.k = CacheView{const_cast<void*>(k_cache), strides[0], strides[1], strides[2]};
  A.v = CacheView{const_cast<void*>(v_cache), strides[3], strides[4], strides[5]};
  A.k_scale = k_scale;
  A.v_scale = v_scale;
  A.pages = page_map(page_table, table_stride, pages_per_seq, num_pages, page_size);
  A.indices = indices;
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.context = context_lens;
  A.tokens = total_tokens;
  A.Hq = static_cast<int>(q_heads);
  A.G = static_cast<int>(kv_groups);
  A.D = static_cast<int>(head_dim);
  A.K = static_cast<int>(topk_slots);
  A.B = static_cast<int>(block_size);
  A.head_tiles = static_cast<int>(head_tiles_of(q_heads, kv_groups));
  const int64_t items = total_tokens * kv_groups * A.head_tiles;
  A.splits = static_cast<int>(split_count(items, topk_slots, block_size));
  A.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  A.out = static_cast<uint16_t*>(out);
  A.lse = lse;
  if (A.splits > 1) {
    if (!workspace || workspace_bytes < msa_attn_paged_workspace_bytes(total_tokens, q_heads, kv_groups, head_dim,
                                                                       topk_slots, block_size))
      return kErrInvalidArgument;
    A.part = static_cast<float*>(workspace);
    A.stats = A.part + items * A.splits * 16 * head_dim;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 block(256);
  int rc = kOk;
#define MSA_ATTN_PAGED(DT, F8, NK)                                                                              \
  rc = launch_parts(                                                                                            \
      items,                                                                                                    \
      [&](int64_t first, unsigned count) {                                                                      \
        A.first = first;                                                                                        \
        hipLaunchKernelGGL((attn_paged_kernel<DT, F8, NK>), dim3(count * A.splits), block, 0, st, A);           \
      },                                                                                                        \
      A.splits)
#define MSA_ATTN_PAGED_DIM(DT, F8)                \
  if (head_dim <= 64) MSA_ATTN_PAGED(DT, F8, 2);  \
  else if (head_dim <= 128) MSA_ATTN_PAGED(DT, F8, 4); \
  else MSA_ATTN_PAGED(DT, F8, 8)
  if (dtype == kBF16) {
    if (cache_is_fp8) { MSA_ATTN_PAGED_DIM(kBF16, true); }
    else { MSA_ATTN_PAGED_DIM(kBF16, false); }
  } else {
    if (cache_is_fp8) { MSA_ATTN_PAGED_DIM(kF16, true); }
    else { MSA_ATTN_PAGED_DIM(kF16, false); }
  }
#undef MSA_ATTN_PAGED_DIM
#undef MSA_ATTN_PAGED
  if (rc != kOk || A.splits == 1) return rc;
  return launch_parts((total_tokens * q_heads + 3) / 4, [&](int64_t first, unsigned count) {
    A.first = first;
    if (dtype == kBF16) hipLaunchKernelGGL(attn_paged_join<kBF16>, dim3(count), block, 0, st, A);
    else hipLaunchKernelGGL(attn_paged_join<kF16>, dim3(count), block, 0, st, A);
  });
}
