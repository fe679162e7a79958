// Indexer scores of new tokens against the index keys of a paged cache, and their top-k selection.
//
// score[t, g, b] = max over the keys j of block b with j <= position(t) of scale * index_q[t, g] . key[j],
// with the public rounding of the packed score (public_score of the exact winning dot), so that a sequence scored
// from a cache selects the same blocks as one scored in a pack.
//
// Exactness. The maximum has to be that of the exact dots (equal scores tie by block number, and a score an
// ulp off would reorder near ties). A 16x16x32 matrix product gives every dot in fp32, s, and a second one of
// the magnitudes gives S = sum |q||k|, which bounds its error: the products of 16-bit values are exact in
// fp32, and DP additions of partial sums below S are off by at most a step of 2^-23 S each (also if the unit
// truncates), plus what falls below fp32's range: below 2^-126 for a product, and below 2^-126 |q| for a bf16 key
// value that the unit may take as zero (a query with such values is settled in FP64 throughout). A key can hold the
// maximum only if s + e >= max (s - e), e = (DP + 16) (2^-23 S + 2^-126 (1 + max |q|)); usually one key of a block does. Those keys' dots are formed in FP64 (four lanes a
// row, each with the dims of its query fragment, two exchanges), and their maximum is the score. Rows with an
// infinity or a NaN somewhere fail the comparison and are settled in FP64 as well.
//
// Bound by reading the index keys once from HBM (256 bytes a key for 128 dims): a wave takes one key
// block for 16 query rows (tokens x groups of a sequence), its key fragments straight from memory in the
// operand layout (lane c a key, 64 contiguous bytes of it for each 32 dims and four lanes). Query rows are
// numbered without a list of tiles: sequence s gets the tiles from cu[s] G / 16 + s on, which leaves room
// for its partly filled last one.
#include "mfma_util.hpp"
#include "paged.hpp"
#include "score_mfma.hpp"
#include "topk_row.hpp"

namespace msa {
namespace {

constexpr int kChunkTiles = 8;  // key tiles of 16 whose logits a wave holds at once

struct PagedScoreArgs {
  const uint16_t* iq;  // [T][G][Di]
  CacheView keys;      // one head
  PageMap pages;
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  int64_t tokens;
  int G, Di, NB, B;
  int block_groups;  // workgroups of four blocks a tile
  float sign, scale; // of the logits: direction and magnitude
  float* scores;     // [T][G][NB]
};

template <int NK>
struct QueryFrags {
  bf16x8 q[NK], mag[NK];
  bool plain;  // no bf16 value below the normal range
};

__device__ __forceinline__ bf16x8 magnitudes(bf16x8 f) {
  uint4 w = __builtin_bit_cast(uint4, f);
  w.x &= 0x7fff7fffu, w.y &= 0x7fff7fffu, w.z &= 0x7fff7fffu, w.w &= 0x7fff7fffu;
  return __builtin_bit_cast(bf16x8, w);
}

template <int DT>
__device__ __forceinline__ double fma_words(bf16x8 a, bf16x8 b, double acc) {
  const uint4 x = __builtin_bit_cast(uint4, a), y = __builtin_bit_cast(uint4, b);
  const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    acc = fma(static_cast<double>(lo16_f32<DT>(u[i])), static_cast<double>(lo16_f32<DT>(v[i])), acc);
    acc = fma(static_cast<double>(hi16_f32<DT>(u[i])), static_cast<double>(hi16_f32<DT>(v[i])), acc);
  }
  return acc;
}

template <int DT, int NK>
__global__ __launch_bounds__(256) void score_paged_kernel(PagedScoreArgs A) {
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x / A.block_groups;
  const int block = static_cast<int>(blockIdx.x % A.block_groups) * 4 + wave;
  if (block >= A.NB) return;
  int lo = 0, hi = A.nseq;  // the last sequence whose tiles start at or below `tile`
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (((A.cu[mid] * static_cast<int64_t>(A.G)) >> 4) + mid <= tile) lo = mid; else hi = mid;
  }
  const int s = lo;
  const int64_t start = A.cu[s], rows = (A.cu[s + 1] - start) * A.G;
  const int64_t r0 = (tile - ((start * A.G) >> 4) - s) * 16;
  if (r0 >= rows) return;
  const int32_t context = A.context[s];
  const int64_t row = r0 + c;
  const bool live = row < rows;
  const int32_t i = static_cast<int32_t>((live ? row : rows - 1) / A.G);  // token of the sequence
  const int64_t pos = context < 0 ? -1 : static_cast<int64_t>(context) + i;
  const int64_t last = context < 0 ? -1 : static_cast<int64_t>(context) + (min(r0 + 16, rows) - 1) / A.G;
  const int64_t k0 = static_cast<int64_t>(block) * A.B, k1 = min(k0 + A.B, last + 1);
  double best = -__builtin_inf();
  bool any = false;
  if (k0 < k1 && A.pages.num_pages > 0) {
    const uint16_t* qrow = A.iq + (start * A.G + (live ? row : rows - 1)) * A.Di;
    QueryFrags<NK> Q;
    float most = 0.f, tiny = 0.f;
    int dim[NK];  // this lane's dims of a key row (past Di: any, against a zero query)
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) {
      const int d = 32 * kk + 8 * q4;
      dim[kk] = d < A.Di ? d : 0;
      uint4 w = d < A.Di && live ? *reinterpret_cast<const uint4*>(qrow + d) : make_uint4(0u, 0u, 0u, 0u);
      if (A.sign < 0.f) w.x ^= 0x80008000u, w.y ^= 0x80008000u, w.z ^= 0x80008000u, w.w ^= 0x80008000u;
      if (A.sign == 0.f) w = make_uint4(0u, 0u, 0u, 0u);
      Q.q[kk] = __builtin_bit_cast(bf16x8, w);
      Q.mag[kk] = magnitudes(Q.q[kk]);
      const uint4 m = __builtin_bit_cast(uint4, Q.mag[kk]);
      for (uint32_t u : {m.x, m.y, m.z, m.w}) {
        most = fmaxf(most, fmaxf(lo16_f32<DT>(u), hi16_f32<DT>(u)));
        if (DT == kBF16)
          tiny = fmaxf(tiny, ((u & 0xffffu) - 1u < 0x7fu || (u >> 16) - 1u < 0x7fu) ? 1.f : 0.f);
      }
    }
    Q.plain = quad_max(tiny) == 0.f;
    const float e0 = static_cast<float>(32 * NK + 16) * 0x1p-126f * (1.f + quad_max(most));
    const uint16_t* keys = static_cast<const uint16_t*>(A.keys.base);
    const int slot_mask = (1 << A.pages.shift) - 1;
    auto key_at = [&](int64_t j, int page) {  // row of key j, in page `page`
      return keys + page * A.keys.stride_page + (j & slot_mask) * A.keys.stride_slot;
    };
    for (int64_t kc = k0; kc < k1; kc += 16 * kChunkTiles) {
      f32x4 dot[kChunkTiles], mag[kChunkTiles];
      int page[kChunkTiles];
#pragma unroll
      for (int kt = 0; kt < kChunkTiles; ++kt) {
        dot[kt] = mag[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
        const int64_t j = kc + 16 * kt;
        page[kt] = j < k1 ? A.pages.page_of(s, j) : -1;
        const uint16_t* krow = key_at(j + c, page[kt] < 0 ? 0 : page[kt]);  // (a page that exists; masked below)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          const bf16x8 f = load_frag(krow + dim[kk]);
          dot[kt] = mfma_t<DT>(f, Q.q[kk], dot[kt]);
          mag[kt] = mfma_t<DT>(magnitudes(f), Q.mag[kk], mag[kt]);
        }
      }
      constexpr float kErr = static_cast<float>(32 * NK + 16) * 0x1p-23f;
      float floor_ = -__builtin_inff();  // below the block's maximum
#pragma unroll
      for (int kt = 0; kt < kChunkTiles; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = page[kt] >= 0 && kc + 16 * kt + 4 * q4 + r <= pos && live;
          const float e = fmaf(kErr, mag[kt][r], e0);
          if (seen) floor_ = fmaxf(floor_, dot[kt][r] - e);
          mag[kt][r] = e;
        }
      floor_ = quad_max(floor_);
      uint32_t open = 0;  // keys that may hold the maximum: bit 4 kt + r
#pragma unroll
      for (int kt = 0; kt < kChunkTiles; ++kt)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool seen = page[kt] >= 0 && kc + 16 * kt + 4 * q4 + r <= pos && live;
          if (seen && !(dot[kt][r] + mag[kt][r] < floor_ && Q.plain)) open |= 1u << (4 * kt + r);
        }
      while (__ballot(open != 0u)) {  // one key of every row at a time (each round takes a bit from each row that has one)
        int key = 0x7fffffff;
        if (open) {
          const int bit = __builtin_ctz(open);
          key = 16 * (bit >> 2) + 4 * q4 + (bit & 3);
        }
        int first = min(key, __shfl_xor(key, 16, kWave));
        first = min(first, __shfl_xor(first, 32, kWave));
        const bool mine = first == key && open;
        if (mine) open &= open - 1;
        double part = 0.0;
        if (first != 0x7fffffff) {
          const int64_t j = kc + first;
          const uint16_t* krow = key_at(j, A.pages.page_of(s, j));
#pragma unroll
          for (int kk = 0; kk < NK; ++kk)
            if (32 * kk + 8 * q4 < A.Di) part = fma_words<DT>(load_frag(krow + dim[kk]), Q.q[kk], part);
        }
        part += __shfl_xor(part, 16, kWave);
        part += __shfl_xor(part, 32, kWave);
        if (first != 0x7fffffff) {
          any = true;
          if (part > best) best = part;
        }
      }
    }
  }
  if (live && q4 == 0)
    A.scores[((start + i) * A.G + (row - static_cast<int64_t>(i) * A.G)) * A.NB + block] =
        any ? public_score(best, A.scale) : -__builtin_inff();
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int msa_index_score_topk_paged(const void* index_q, const void* index_cache, int32_t dtype,
                                          int64_t cache_stride_page, int64_t cache_stride_slot,
                                          const int32_t* page_table, int64_t table_stride, int64_t pages_per_seq,
                                          int64_t num_pages, int64_t page_size, const int32_t* cu_seqlens,
                                          int64_t num_seqs, const int32_t* context_lens, int64_t total_tokens,
                                          int64_t groups, int64_t index_dim, int64_t num_blocks, int64_t block_size,
                                          double scale, int64_t topk_blocks, int64_t local_blocks, float* scores,
                                          int32_t* indices, void* stream) {
  if (!index_q || !scores || !cu_seqlens || !context_lens || num_seqs <= 0 || num_seqs > 0x3fffffff || total_tokens < 0 ||
      total_tokens > 0x7fffffff || groups <= 0 || groups >= (1 << 20) || index_dim <= 0 || num_blocks <= 0 ||
      num_blocks > 0x7fffffff || block_size <= 0 || block_size > 0x7fffffff || topk_blocks < 0 || topk_blocks > 0x7fffffff ||
      local_blocks < 0 || local_blocks > topk_blocks || (topk_blocks > 0 && !indices) || !__builtin_isfinite(scale) ||
      !valid_pages(page_table, table_stride, pages_per_seq, num_pages, page_size) || (num_pages > 0 && !index_cache) ||
      (dtype != kBF16 && dtype != kF16))
    return kErrInvalidArgument;
  if (reinterpret_cast<uintptr_t>(index_cache) % 16 || reinterpret_cast<uintptr_t>(index_q) % 16 ||
      cache_stride_page % 8 || cache_stride_slot % 8)
    return kErrInvalidArgument;
  if (index_dim % 8 || index_dim > 256 || block_size % 16) return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  PagedScoreArgs A{};
  A.iq = static_cast<const uint16_t*>(index_q);
  A.keys = CacheView{const_cast<void*>(index_cache), cache_stride_page, 0, cache_stride_slot};
  A.pages = page_map(page_table, table_stride, pages_per_seq, num_pages, page_size);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.context = context_lens;
  A.tokens = total_tokens;
  A.G = static_cast<int>(groups);
  A.Di = static_cast<int>(index_dim);
  A.NB = static_cast<int>(num_blocks);
  A.B = static_cast<int>(block_size);
  A.block_groups = (A.NB + 3) / 4;
  A.sign = scale > 0.0 ? 1.f : scale < 0.0 ? -1.f : 0.f;
  A.scale = static_cast<float>(scale < 0.0 ? -scale : scale);
  A.scores = scores;
  const int64_t tiles = total_tokens * groups / 16 + num_seqs;
  if (tiles >= (int64_t{1} << 24) / A.block_groups) return kErrUnsupported;  // 2^32 threads of a launch
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(tiles * A.block_groups)), block(256);
#define MSA_SCORE_PAGED(NK)                                                                               \
  if (dtype == kBF16) hipLaunchKernelGGL((score_paged_kernel<kBF16, NK>), grid, block, 0, st, A);         \
  else hipLaunchKernelGGL((score_paged_kernel<kF16, NK>), grid, block, 0, st, A)
  if (index_dim <= 64) { MSA_SCORE_PAGED(2); }
  else if (index_dim <= 128) { MSA_SCORE_PAGED(4); }
  else { MSA_SCORE_PAGED(8); }
#undef MSA_SCORE_PAGED
  const int rc = status_from(hipGetLastError());
  if (rc != kOk || topk_blocks == 0) return rc;
  return topk_launch(scores, cu_seqlens, A.nseq, total_tokens * groups, A.G, A.NB, A.B, static_cast<int>(topk_blocks),
                     static_cast<int>(local_blocks), indices, st, context_lens);
}
