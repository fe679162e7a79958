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
// maximum only if s >= max s - 2 e, e = (DP + 16) (2^-23 max S + 2^-126 (1 + max |q|)); usually one key of a block does. Those keys' dots are formed in FP64 (four lanes a
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
#include <stdlib.h>

namespace msa {
namespace {

struct PagedScoreArgs {
  const uint16_t* iq;  // [T][G][Di]
  CacheView keys;      // one head
  PageMap pages;
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  int64_t tokens;
  int G, Di, NB, B;
  int parts;         // workgroups of a tile: four blocks each at a time
  float sign, scale; // of the logits: direction and magnitude
  float* scores;     // [T][G][NB]
};

template <int NK>
struct QueryFrags {
  bf16x8 q[NK], mag[NK];
};

__device__ __forceinline__ bf16x8 magnitudes(bf16x8 f) {
  uint4 w = __builtin_bit_cast(uint4, f);
  w.x &= 0x7fff7fffu, w.y &= 0x7fff7fffu, w.z &= 0x7fff7fffu, w.w &= 0x7fff7fffu;
  return __builtin_bit_cast(bf16x8, w);
}

// f, from here on: keeps what is made of it (its values in FP64, 64 registers for 128 dims) inside the round.
__device__ __forceinline__ bf16x8 in_this_round(bf16x8 f) {
  uint4 w = __builtin_bit_cast(uint4, f);
  asm volatile("" : "+v"(w.x), "+v"(w.y), "+v"(w.z), "+v"(w.w));
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

// FULL: Di is 32 NK, and a lane's pieces of a key row are at constant offsets.
template <int DT, int NK, bool FULL>
__global__ __launch_bounds__(256, NK == 8 ? 1 : 2) void score_paged_kernel(PagedScoreArgs A) {
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t tile = blockIdx.x / A.parts;
  const int part = static_cast<int>(blockIdx.x % A.parts);
  // the last sequence whose tiles start at or below `tile`
  const int s = wave_upper_index(A.nseq, tile, [&](int i) { return ((A.cu[i] * static_cast<int64_t>(A.G)) >> 4) + i; });
  const int64_t start = A.cu[s], rows = (A.cu[s + 1] - start) * A.G;
  const int32_t context = A.context[s];
  const int64_t r0 = (tile - ((start * A.G) >> 4) - s) * 16;
  if (r0 >= rows) return;
  const int64_t row = r0 + c;
  const bool live = row < rows;
  const int32_t i = static_cast<int32_t>((live ? row : rows - 1) / A.G);  // token of the sequence
  const int64_t pos = context < 0 ? -1 : static_cast<int64_t>(context) + i;
  const int64_t last = context < 0 ? -1 : static_cast<int64_t>(context) + (min(r0 + 16, rows) - 1) / A.G;
  float* out = A.scores + (start * A.G + (live ? row : rows - 1)) * A.NB;
  const int seen_blocks = A.pages.num_pages > 0 ? static_cast<int>(min((last + A.B) / A.B, static_cast<int64_t>(A.NB))) : 0;

  // blocks behind the tile's tokens: four lanes a row, this workgroup's share
  for (int b = seen_blocks + 16 * part + 4 * wave + q4; b < A.NB; b += 16 * A.parts)
    if (live) out[b] = -__builtin_inff();

  if (4 * part + wave >= seen_blocks) return;
  const uint16_t* qrow = A.iq + (start * A.G + (live ? row : rows - 1)) * A.Di;
  QueryFrags<NK> Q;
  float most = 0.f, tiny = 0.f;
  int dim[NK];  // this lane's dims of a key row (past Di: any, against a zero query)
#pragma unroll
  for (int kk = 0; kk < NK; ++kk) {
    const int d = 32 * kk + 8 * q4;
    dim[kk] = FULL || d < A.Di ? d : 0;
    uint4 w = (FULL || d < A.Di) && live ? *reinterpret_cast<const uint4*>(qrow + d) : make_uint4(0u, 0u, 0u, 0u);
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
  const bool plain = quad_max(tiny) == 0.f;  // no bf16 value below the normal range
  const float e0 = static_cast<float>(32 * NK + 16) * 0x1p-126f * (1.f + quad_max(most));
  constexpr float kErr = static_cast<float>(32 * NK + 16) * 0x1p-23f;
  constexpr int GT = NK == 8 ? 2 : 4, kTiles = 2 * GT;  // tiles of a group and of a chunk
  const uint16_t* keys = static_cast<const uint16_t*>(A.keys.base);
  const int slot_mask = (1 << A.pages.shift) - 1;
  auto key_at = [&](int64_t j, int page) {  // row of key j, in page `page`
    return keys + page * A.keys.stride_page + (j & slot_mask) * A.keys.stride_slot;
  };
  // pages of a chunk's tiles, one a lane; -1 past the end
  auto pages_of = [&](int64_t kc, int64_t end) {
    const int64_t j = kc + 16 * (lane & (kTiles - 1));
    return j < end ? A.pages.page_of(s, j) : -1;
  };
  // The key fragments of a group of tiles. All loads are issued here: left to itself, the compiler puts each load
  // in front of its product and waits for it.
  auto load_group = [&](bf16x8 (&f)[GT][NK], int64_t kc, int own_page, int group) {
#pragma unroll
    for (int kt = 0; kt < GT; ++kt) {
      const int page = __builtin_amdgcn_readlane(own_page, group * GT + kt);
      const uint16_t* krow = key_at(kc + 16 * (group * GT + kt) + c, page < 0 ? 0 : page);  // (page 0 exists; not seen)
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) f[kt][kk] = load_frag(krow + dim[kk]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };

  int block = 4 * part + wave;
  int64_t kc = static_cast<int64_t>(block) * A.B, k1 = min(kc + A.B, last + 1);
  int own_page = pages_of(kc, k1);
  bf16x8 f0[GT][NK], f1[GT][NK];
  load_group(f0, kc, own_page, 0);
  double best = -__builtin_inf();
  bool any = false;
  while (true) {
    // the chunk behind this one: of this block, or the first of this wave's next one
    const bool block_ends = kc + 16 * kTiles >= k1;
    const int next_block = block_ends ? block + 4 * A.parts : block;
    const bool more = next_block < seen_blocks;
    const int64_t next_kc = block_ends ? static_cast<int64_t>(next_block) * A.B : kc + 16 * kTiles;
    const int64_t next_k1 = block_ends ? min(next_kc + A.B, last + 1) : k1;
    const int next_page = more ? pages_of(next_kc, next_k1) : -1;
    load_group(f1, kc, own_page, 1);
    f32x4 dot[kTiles];
    int seen[kTiles];  // this lane's keys of the tile up to the row's position
    const int limit = live ? static_cast<int>(min(pos - kc - 4 * q4, int64_t{16 * kTiles})) : -1;
#pragma unroll
    for (int kt = 0; kt < kTiles; ++kt)
      seen[kt] = __builtin_amdgcn_readlane(own_page, kt) < 0 ? 0 : limit - 16 * kt + 1;
    float most_mag = 0.f, top = -__builtin_inff();
    auto products = [&](const bf16x8 (&f)[GT][NK], int group) {
#pragma unroll
      for (int i = 0; i < GT; ++i) {
        const int kt = group * GT + i;
        f32x4 mag = f32x4{0.f, 0.f, 0.f, 0.f};
        dot[kt] = mag;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
          dot[kt] = mfma_t<DT>(f[i][kk], Q.q[kk], dot[kt]);
          mag = mfma_t<DT>(magnitudes(f[i][kk]), Q.mag[kk], mag);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (r < seen[kt]) {
            top = fmaxf(top, dot[kt][r]);
            most_mag = fmaxf(most_mag, mag[r]);
          }
      }
    };
    products(f0, 0);
    if (more) load_group(f0, next_kc, next_page, 0);
    products(f1, 1);
    // (an infinite bound, from an infinity or an overflow, leaves every key in)
    const float bound = quad_max(top) - 2.f * fmaf(kErr, quad_max(most_mag), e0);
    uint32_t open = 0;  // keys that may hold the maximum: bit 4 kt + r
#pragma unroll
    for (int kt = 0; kt < kTiles; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (r < seen[kt] && !(dot[kt][r] < bound && plain)) open |= 1u << (4 * kt + r);
    while (__ballot(open != 0u)) {  // one key of every row at a time
      int key = 0x7fffffff;
      if (open) {
        const int bit = __builtin_ctz(open);
        key = 16 * (bit >> 2) + 4 * q4 + (bit & 3);
      }
      int first = min(key, __shfl_xor(key, 16, kWave));
      first = min(first, __shfl_xor(first, 32, kWave));
      if (first == key && open) open &= open - 1;
      const int page = __shfl(own_page, (first >> 4) & (kTiles - 1), kWave);
      double part_dot = 0.0;
      if (first != 0x7fffffff) {
        const uint16_t* krow = key_at(kc + first, page);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
          if (FULL || 32 * kk + 8 * q4 < A.Di)
            part_dot = fma_words<DT>(load_frag(krow + dim[kk]), in_this_round(Q.q[kk]), part_dot);
      }
      part_dot += __shfl_xor(part_dot, 16, kWave);
      part_dot += __shfl_xor(part_dot, 32, kWave);
      if (first != 0x7fffffff) {
        any = true;
        if (part_dot > best) best = part_dot;
      }
    }
    if (block_ends) {
      if (live && q4 == 0) out[block] = any ? public_score(best, A.scale) : -__builtin_inff();
      best = -__builtin_inf();
      any = false;
    }
    if (!more) return;
    block = next_block;
    kc = next_kc;
    k1 = next_k1;
    own_page = next_page;
  }
}

int part_count(int64_t tiles, int64_t blocks) {
  const char* e = getenv("MSA_PARTS");
  int64_t n = ((e ? atoi(e) : 1024) + tiles - 1) / tiles;
  const int64_t most = (blocks + 3) / 4;
  n = n < most ? n : most;
  return static_cast<int>(n < 1 ? 1 : n);
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
  A.sign = scale > 0.0 ? 1.f : scale < 0.0 ? -1.f : 0.f;
  A.scale = static_cast<float>(scale < 0.0 ? -scale : scale);
  A.scores = scores;
  const int64_t tiles = total_tokens * groups / 16 + num_seqs;
  A.parts = part_count(tiles, A.NB);
  if (tiles >= (int64_t{1} << 24) / A.parts) return kErrUnsupported;  // 2^32 threads of a launch
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(tiles * A.parts)), block(256);
#define MSA_SCORE_PAGED(NK)                                                                               \
  if (dtype == kBF16 && index_dim == 32 * NK)                                                             \
    hipLaunchKernelGGL((score_paged_kernel<kBF16, NK, true>), grid, block, 0, st, A);                     \
  else if (dtype == kBF16)                                                                                \
    hipLaunchKernelGGL((score_paged_kernel<kBF16, NK, false>), grid, block, 0, st, A);                    \
  else if (index_dim == 32 * NK)                                                                          \
    hipLaunchKernelGGL((score_paged_kernel<kF16, NK, true>), grid, block, 0, st, A);                      \
  else                                                                                                    \
    hipLaunchKernelGGL((score_paged_kernel<kF16, NK, false>), grid, block, 0, st, A)
  if (index_dim <= 64) { MSA_SCORE_PAGED(2); }
  else if (index_dim <= 128) { MSA_SCORE_PAGED(4); }
  else { MSA_SCORE_PAGED(8); }
#undef MSA_SCORE_PAGED
  const int rc = status_from(hipGetLastError());
  if (rc != kOk || topk_blocks == 0) return rc;
  return topk_launch(scores, cu_seqlens, A.nseq, total_tokens * groups, A.G, A.NB, A.B, static_cast<int>(topk_blocks),
                     static_cast<int>(local_blocks), indices, st, context_lens);
}
