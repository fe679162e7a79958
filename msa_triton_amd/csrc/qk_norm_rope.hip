// RMS norm of every query and key head with the position rotation, forward and backward.
//
// A head x of D values, its token's position p and the weight w of its side (queries or keys):
//   r = 1 / sqrt(mean x^2 + eps),  n = x r,  m = n w,
//   y_i = m_i cos_i - m_{i+h} sin_i,  y_{i+h} = m_{i+h} cos_i + m_i sin_i   (i < h = rot / 2),
//   y_i = m_i   (i >= rot),
// with (cos, sin) row p of a table. Backward, from g = dL/dy: the inverse rotation gives dm, then
//   dw = sum over heads of dm n,   dx = r (dm w - n mean(dm w n)).
// Sums and products are fp32; outputs are rounded once.
//
// Both passes are bound by memory: 2 (forward) and 3 (backward) bytes moved per byte of x, nothing else
// touches HBM (the table rows of a token serve all its heads from the caches). So x is read once,
// with the row in registers: a lane holds the element pairs that the rotation mixes, VEC of them from
// each half (and, past rot, VEC from each half of the rest), so that one 16-byte load per half, one
// reduction over LPR lanes and no exchange of elements are needed. Workgroups take a contiguous run
// of rows of one side; the positions of its tokens are looked up once, into LDS.
//
// dw: a lane adds its rows' terms in registers, a workgroup its lanes' in a fixed order, and a second
// launch the workgroups' partial sums (in FP64): the same bits on every run, no atomics.
#include "norm_rope.hpp"

namespace msa {
namespace {

constexpr int kMostTokens = 1024;    // tokens of one workgroup: positions in LDS
constexpr int kMostDim = 512;
constexpr int kBwdBlocks = 1022;     // workgroups of the backward, both sides, unless rows need more

struct NormSide {
  const void* x;
  int64_t stride_t, stride_h;  // elements
  const void* w;
  void* y;            // forward: output; backward: dx (or null)
  const void* g;      // backward: dL/dy, contiguous
  float* dw_part;     // backward: [blocks][D]
  int heads;
};

struct NormArgs {
  NormSide side[2];
  int64_t first;       // workgroup of this launch's first one
  int64_t q_blocks;    // workgroups of side 0
  int rows_per_block;
  bool w_f32;
  RopeTable rope;
  const int32_t* cu;
  int nseq;
  const int32_t* context;  // or null: 0
  int64_t tokens;
  int dim;
  float eps;
};

// Positions of the tokens [t0, t0 + n) into LDS; the largest int32 below 0 stands for "none".
__device__ __forceinline__ void load_positions(const NormArgs& A, int64_t t0, int n, int32_t* pos) {
  for (int i = threadIdx.x; i < n; i += kNormThreads) {
    const int64_t t = t0 + i;
    const int s = find_seq(A.cu, A.nseq, t);
    const int64_t p = t - A.cu[s] + (A.context ? A.context[s] : 0);
    pos[i] = p < 0 || p > 0x7fffffff ? -1 : static_cast<int32_t>(p);
  }
  __syncthreads();
}

// One row a lane run: with many workgroups a CU more rows in flight each only cost registers (32K tokens x 36 heads of 128,
// bf16: 132 us, 4.6 TB/s; two and four rows took 11 and 25 % longer).
template <int DT, int VEC, int C, int LPR>
__global__ __launch_bounds__(kNormThreads) void norm_rope_fwd_kernel(NormArgs A) {
  using Lanes = RowLanes<DT, VEC, C, LPR>;
  __shared__ int32_t pos[Lanes::kRows + 1];
  const int64_t at = A.first + blockIdx.x;
  const bool second = at >= A.q_blocks;
  const NormSide& S = A.side[second];
  const int64_t r0 = (at - (second ? A.q_blocks : 0)) * Lanes::kRows;
  const int64_t rows = A.tokens * S.heads, t0 = r0 / S.heads;
  const int h0 = static_cast<int>(r0 - t0 * S.heads);
  const int n = static_cast<int>(min(rows - r0, static_cast<int64_t>(Lanes::kRows)));
  const Lanes lanes(S.w, A.w_f32, A.rope.half, A.dim);
  const int i = threadIdx.x / LPR;
  const int tok = static_cast<int>(static_cast<uint32_t>(h0 + i) / static_cast<uint32_t>(S.heads));
  const int head = h0 + i - tok * S.heads;
  float a[C][VEC], b[C][VEC];
  lanes.load(S.x, (t0 + tok) * S.stride_t + head * S.stride_h, i < n, a, b);
  load_positions(A, t0, (h0 + n - 1) / S.heads + 1, pos);
  const float ss = run_sum<LPR>(sum_products(a, b, a, b));
  if (i >= n) return;
  const float r = 1.f / sqrtf(ss / static_cast<float>(A.dim) + A.eps);
  const int p = pos[tok];
#pragma unroll
  for (int c = 0; c < C; ++c) {
    float co[VEC], si[VEC];
    load_turn<VEC>(A.rope, lanes.pc[c], p, co, si);
#pragma unroll
    for (int j = 0; j < VEC; ++j) a[c][j] = a[c][j] * r * lanes.wa[c][j], b[c][j] = b[c][j] * r * lanes.wb[c][j];
    turn<VEC>(lanes.pc[c], co, si, a[c], b[c]);
  }
  lanes.store(S.y, ((t0 + tok) * S.heads + head) * A.dim, a, b);
}

// The row after this one is on its way while it is worked on (32K tokens x 36 heads of 128, bf16: 194 us, 4.7 TB/s; 211
// without).
template <int DT, int VEC, int C, int LPR>
__global__ __launch_bounds__(kNormThreads, DT == kF32 ? 3 : 4) void norm_rope_bwd_kernel(NormArgs A) {
  using Lanes = RowLanes<DT, VEC, C, LPR>;
  __shared__ int32_t pos[kMostTokens + 1];
  __shared__ float sums[kNormThreads / kWave][kMostDim];
  const int64_t at = A.first + blockIdx.x;
  const bool second = at >= A.q_blocks;
  const NormSide& S = A.side[second];
  const int64_t block = at - (second ? A.q_blocks : 0);
  const int64_t r0 = block * A.rows_per_block;
  const int64_t rows = A.tokens * S.heads, t0 = r0 / S.heads;
  const int h0 = static_cast<int>(r0 - t0 * S.heads);
  const int n = static_cast<int>(min(rows - r0, static_cast<int64_t>(A.rows_per_block)));
  const Lanes lanes(S.w, A.w_f32, A.rope.half, A.dim);
  struct Row {
    typename Lanes::Raw x, g;
    int tok;
    int64_t at;
  };
  auto fetch = [&](int i) {
    Row r;
    r.tok = static_cast<int>(static_cast<uint32_t>(h0 + i) / static_cast<uint32_t>(S.heads));
    const int head = h0 + i - r.tok * S.heads;
    r.at = ((t0 + r.tok) * S.heads + head) * A.dim;
    r.x = lanes.fetch(S.x, (t0 + r.tok) * S.stride_t + head * S.stride_h, i < n);
    r.g = lanes.fetch(S.g, r.at, i < n);
    return r;
  };
  const int own = threadIdx.x / LPR;
  Row next = fetch(own);
  load_positions(A, t0, (h0 + n - 1) / S.heads + 1, pos);
  float da[C][VEC], db[C][VEC];
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) da[c][j] = db[c][j] = 0.f;
  for (int base = 0; base < n; base += Lanes::kRows) {  // (uniform: every lane takes part in the sums)
    const Row now = next;
    const int i = base + own;
    if (base + Lanes::kRows < n) next = fetch(i + Lanes::kRows);
    float a[C][VEC], b[C][VEC], ga[C][VEC], gb[C][VEC];
    Lanes::unpack(now.x, a, b);
    Lanes::unpack(now.g, ga, gb);
    const float ss = run_sum<LPR>(sum_products(a, b, a, b));
    const float r = 1.f / sqrtf(ss / static_cast<float>(A.dim) + A.eps);
    const int p = i < n ? pos[now.tok] : 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      float co[VEC], si[VEC];
      load_turn<VEC>(A.rope, lanes.pc[c], p, co, si);
      turn_back<VEC>(lanes.pc[c], co, si, ga[c], gb[c]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float dma = ga[c][j], dmb = gb[c][j];
        a[c][j] *= r;  // n
        b[c][j] *= r;
        if (i < n) {
          da[c][j] = fmaf(dma, a[c][j], da[c][j]);
          db[c][j] = fmaf(dmb, b[c][j], db[c][j]);
        }
        ga[c][j] = dma * lanes.wa[c][j];
        gb[c][j] = dmb * lanes.wb[c][j];
      }
    }
    const float mean = run_sum<LPR>(sum_products(ga, gb, a, b)) / static_cast<float>(A.dim);
    if (S.y && i < n) {
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          ga[c][j] = r * (ga[c][j] - a[c][j] * mean);
          gb[c][j] = r * (gb[c][j] - b[c][j] * mean);
        }
      lanes.store(S.y, now.at, ga, gb);
    }
  }
  if (!S.dw_part) return;
  // the lanes of a wave that hold the same elements, then the waves
#pragma unroll
  for (int c = 0; c < C; ++c)
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
#pragma unroll
      for (int o = LPR; o < kWave; o <<= 1) {
        da[c][j] += __shfl_xor(da[c][j], o, kWave);
        db[c][j] += __shfl_xor(db[c][j], o, kWave);
      }
      const int wave = threadIdx.x / kWave;
      if (threadIdx.x % kWave < LPR) {
        if (lanes.pc[c].ok) sums[wave][lanes.pc[c].a + j] = da[c][j];
        if (lanes.pc[c].b_ok) sums[wave][lanes.pc[c].b + j] = db[c][j];
      }
    }
  __syncthreads();
  for (int d = threadIdx.x; d < A.dim; d += kNormThreads) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kNormThreads / kWave; ++w) s += sums[w][d];
    S.dw_part[block * A.dim + d] = s;
  }
}

// The partial sums of `blocks` workgroups added up: 16 columns per workgroup, 16 runs of partial
// sums each (64-byte rows of the partial array per load).
template <int WDT>
__global__ __launch_bounds__(256) void norm_weight_grad_kernel(const float* __restrict__ q_part, int q_blocks,
                                                               void* __restrict__ q_dw, const float* __restrict__ k_part,
                                                               int k_blocks, void* __restrict__ k_dw, int dim) {
  __shared__ double sums[16][17];
  const int tiles = (dim + 15) / 16;
  const bool second = static_cast<int>(blockIdx.x) >= (q_dw ? tiles : 0);
  const int tile = blockIdx.x - (second && q_dw ? tiles : 0);
  const float* part = second ? k_part : q_part;
  const int n = second ? k_blocks : q_blocks;
  const int col = threadIdx.x & 15, run = threadIdx.x >> 4, d = tile * 16 + col;
  double s = 0.0;
  if (d < dim)
#pragma unroll 8
    for (int i = run; i < n; i += 16) s += static_cast<double>(part[static_cast<int64_t>(i) * dim + d]);
  sums[run][col] = s;
  __syncthreads();
  if (run == 0 && d < dim) {
    s = 0.0;
    for (int i = 0; i < 16; ++i) s += sums[i][col];
    store_from_f64<WDT>(second ? k_dw : q_dw, d, s);
  }
}

// Rows of one backward workgroup, the same on both sides: as many workgroups as run at once (four a CU; one each side is
// the last, partly filled one), at least 64 rows, and no more tokens than the LDS positions hold (n rows touch
// at most n / heads + 2 tokens). 32K tokens x 36 heads of 128, bf16, backward and weights' sums: 193 + 5 us, with twice as
// many workgroups 195 + 10; before the next row was fetched ahead 211 + 5, with 1152 workgroups 279 + 5.
int64_t bwd_rows(int64_t tokens, int64_t hq, int64_t hk) {
  const int64_t more = hq > hk ? hq : hk, fewer = hq > hk ? hk : hq, least = fewer ? fewer : more;
  int64_t n = (tokens * (hq + hk) + kBwdBlocks - 1) / kBwdBlocks;
  n = n < 64 ? 64 : n;
  const int64_t most = (kMostTokens - 1) * least;
  return n < most ? n : most;
}

// Whether every row of a side can be read and written 16 bytes at a time.
bool side_fits_vectors(const NormSide& s, int esize, bool w_f32, int dim) {
  return aligned16(s.x) && aligned16(s.w) && aligned16(s.y) && aligned16(s.g) && s.stride_t * esize % 16 == 0 &&
         s.stride_h * esize % 16 == 0 && dim * esize % 16 == 0;
}

template <int DT, bool BWD>
int norm_launch(NormArgs A, bool vectors, int64_t q_rows, int64_t k_rows, hipStream_t st) {
  const int chunks = A.rope.half / 8 + (A.dim - 2 * A.rope.half) / 16;
  auto go = [&](auto kernel, int rows) -> int {
    if (BWD) rows = A.rows_per_block;
    const int64_t nq = (q_rows + rows - 1) / rows, nk = (k_rows + rows - 1) / rows;
    A.q_blocks = nq;
    return launch_parts(nq + nk, [&](int64_t first, unsigned count) {
      A.first = first;
      hipLaunchKernelGGL(kernel, dim3(count), dim3(kNormThreads), 0, st, A);
    });
  };
#define MSA_NORM(VEC, C, LPR)                                                 \
  if constexpr (BWD) return go(norm_rope_bwd_kernel<DT, VEC, C, LPR>, 0);     \
  else return go(norm_rope_fwd_kernel<DT, VEC, C, LPR>, kNormThreads / LPR)
  if (!vectors) { MSA_NORM(1, 4, 64); }
  if (chunks <= 4) { MSA_NORM(8, 1, 4); }
  if (chunks <= 8) { MSA_NORM(8, 1, 8); }
  if (chunks <= 16) { MSA_NORM(8, 1, 16); }
  MSA_NORM(8, 1, 32);
#undef MSA_NORM
}

template <bool BWD>
int norm_dispatch(int32_t dtype, const NormArgs& A, bool vectors, int64_t q_rows, int64_t k_rows, hipStream_t st) {
  switch (dtype) {
    case kF32: return norm_launch<kF32, BWD>(A, vectors, q_rows, k_rows, st);
    case kF16: return norm_launch<kF16, BWD>(A, vectors, q_rows, k_rows, st);
    case kBF16: return norm_launch<kBF16, BWD>(A, vectors, q_rows, k_rows, st);
    default: return kErrInvalidArgument;
  }
}

bool valid_norm(int64_t q_heads, int64_t k_heads, int64_t D, int64_t rot, const float* table, int64_t table_rows,
                const int32_t* cu, int64_t nseq, int64_t T, double eps) {
  return q_heads >= 0 && k_heads >= 0 && q_heads + k_heads > 0 && q_heads < (1 << 20) && k_heads < (1 << 20) && D > 0 &&
         rot >= 0 && rot <= D && rot % 2 == 0 && (rot == 0 || (table && table_rows >= 0)) && cu && nseq > 0 &&
         nseq < 0x7fffffff && T >= 0 && T <= 0x7fffffff && eps >= 0.0;
}

NormArgs norm_args(const void* q, int64_t q_st, int64_t q_sh, int64_t Hq, const void* k, int64_t k_st, int64_t k_sh,
                   int64_t Hk, const void* wq, const void* wk, int32_t dtype, int32_t wdtype, const float* table,
                   int64_t table_rows, int64_t rot, const int32_t* cu, int64_t nseq, const int32_t* context, int64_t T,
                   int64_t D, double eps) {
  NormArgs A{};
  A.side[0] = NormSide{q, q_st, q_sh, wq, nullptr, nullptr, nullptr, static_cast<int>(Hq)};
  A.side[1] = NormSide{k, k_st, k_sh, wk, nullptr, nullptr, nullptr, static_cast<int>(Hk)};
  A.w_f32 = wdtype == kF32;
  A.rope = RopeTable{table, table_rows, static_cast<int>(rot / 2)};
  A.cu = cu;
  A.nseq = static_cast<int>(nseq);
  A.context = context;
  A.tokens = T;
  A.dim = static_cast<int>(D);
  A.eps = static_cast<float>(eps);
  return A;
}

// 16-byte accesses: runs of 8 elements in both halves of the rotated part and of the rest.
bool fits_vectors(const NormArgs& A, int32_t dtype) {
  const int esize = dtype == kF32 ? 4 : 2;
  if (A.rope.half % 8 || (A.dim - 2 * A.rope.half) % 16 || !aligned16(A.rope.table)) return false;
  for (const NormSide& s : A.side)
    if (s.heads && !side_fits_vectors(s, esize, A.w_f32, A.dim)) return false;
  return true;
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_qk_norm_rope(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t q_heads, const void* k,
                                int64_t k_stride_t, int64_t k_stride_h, int64_t k_heads, int32_t dtype,
                                const void* q_weight, const void* k_weight, int32_t weight_dtype, const float* cos_sin,
                                int64_t table_rows, int64_t rotary_dim, const int32_t* cu_seqlens, int64_t num_seqs,
                                const int32_t* context_lens, int64_t total_tokens, int64_t head_dim, double eps,
                                void* q_out, void* k_out, void* stream) {
  if (!valid_norm(q_heads, k_heads, head_dim, rotary_dim, cos_sin, table_rows, cu_seqlens, num_seqs, total_tokens, eps) ||
      (weight_dtype != dtype && weight_dtype != kF32))
    return kErrInvalidArgument;
  if ((q_heads && (!q || !q_weight || !q_out)) || (k_heads && (!k || !k_weight || !k_out))) return kErrInvalidArgument;
  if (head_dim > kMostDim) return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  NormArgs A = norm_args(q, q_stride_t, q_stride_h, q_heads, k, k_stride_t, k_stride_h, k_heads, q_weight, k_weight, dtype,
                         weight_dtype, cos_sin, table_rows, rotary_dim, cu_seqlens, num_seqs, context_lens, total_tokens,
                         head_dim, eps);
  A.side[0].y = q_out;
  A.side[1].y = k_out;
  return norm_dispatch<false>(dtype, A, fits_vectors(A, dtype), total_tokens * q_heads, total_tokens * k_heads,
                              static_cast<hipStream_t>(stream));
}

extern "C" int64_t msa_qk_norm_rope_bwd_workspace_bytes(int64_t total_tokens, int64_t q_heads, int64_t k_heads,
                                                        int64_t head_dim) {
  if (total_tokens <= 0 || q_heads < 0 || k_heads < 0 || head_dim <= 0 || head_dim > kMostDim) return 0;
  if (q_heads + k_heads == 0) return 0;
  const int64_t rows = bwd_rows(total_tokens, q_heads, k_heads);
  return ((total_tokens * q_heads + rows - 1) / rows + (total_tokens * k_heads + rows - 1) / rows) * head_dim *
         static_cast<int64_t>(sizeof(float));
}

extern "C" int msa_qk_norm_rope_bwd(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t q_heads,
                                    const void* k, int64_t k_stride_t, int64_t k_stride_h, int64_t k_heads,
                                    int32_t dtype, const void* q_weight, const void* k_weight, int32_t weight_dtype,
                                    const float* cos_sin, int64_t table_rows, int64_t rotary_dim,
                                    const int32_t* cu_seqlens, int64_t num_seqs, const int32_t* context_lens,
                                    int64_t total_tokens, int64_t head_dim, double eps, const void* grad_q_out,
                                    const void* grad_k_out, void* grad_q, void* grad_k, void* grad_q_weight,
                                    void* grad_k_weight, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!valid_norm(q_heads, k_heads, head_dim, rotary_dim, cos_sin, table_rows, cu_seqlens, num_seqs, total_tokens, eps) ||
      (weight_dtype != dtype && weight_dtype != kF32) || total_tokens == 0)
    return kErrInvalidArgument;
  if (head_dim > kMostDim) return kErrUnsupported;
  // a side without any gradient to compute is left out
  const int64_t hq = grad_q || grad_q_weight ? q_heads : 0, hk = grad_k || grad_k_weight ? k_heads : 0;
  if (hq + hk == 0) return kOk;
  if ((hq && (!q || !q_weight || !grad_q_out)) || (hk && (!k || !k_weight || !grad_k_out))) return kErrInvalidArgument;
  if ((grad_q_weight || grad_k_weight) &&
      (!workspace || workspace_bytes < msa_qk_norm_rope_bwd_workspace_bytes(total_tokens, hq, hk, head_dim)))
    return kErrInvalidArgument;
  hipStream_t st = static_cast<hipStream_t>(stream);
  NormArgs A = norm_args(q, q_stride_t, q_stride_h, hq, k, k_stride_t, k_stride_h, hk, q_weight, k_weight, dtype,
                         weight_dtype, cos_sin, table_rows, rotary_dim, cu_seqlens, num_seqs, context_lens, total_tokens,
                         head_dim, eps);
  const int64_t rows = bwd_rows(total_tokens, hq, hk);
  const int64_t nq = (total_tokens * hq + rows - 1) / rows, nk = (total_tokens * hk + rows - 1) / rows;
  A.rows_per_block = static_cast<int>(rows);
  A.side[0].g = grad_q_out;
  A.side[1].g = grad_k_out;
  A.side[0].y = grad_q;
  A.side[1].y = grad_k;
  float* part = static_cast<float*>(workspace);
  A.side[0].dw_part = grad_q_weight ? part : nullptr;
  A.side[1].dw_part = grad_k_weight ? part + nq * head_dim : nullptr;
  const int rc = norm_dispatch<true>(dtype, A, fits_vectors(A, dtype), total_tokens * hq, total_tokens * hk, st);
  if (rc != kOk || (!grad_q_weight && !grad_k_weight)) return rc;
  const int D = static_cast<int>(head_dim), tiles = (D + 15) / 16;
  const dim3 grid((grad_q_weight ? tiles : 0) + (grad_k_weight ? tiles : 0));
#define MSA_WGRAD(W)                                                                                                 \
  hipLaunchKernelGGL(norm_weight_grad_kernel<W>, grid, dim3(256), 0, st, A.side[0].dw_part, static_cast<int>(nq),      \
                     grad_q_weight, A.side[1].dw_part, static_cast<int>(nk), grad_k_weight, D)
  if (weight_dtype == kF32) MSA_WGRAD(kF32);
  else if (weight_dtype == kF16) MSA_WGRAD(kF16);
  else MSA_WGRAD(kBF16);
#undef MSA_WGRAD
  return status_from(hipGetLastError());
}
