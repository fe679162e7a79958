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
// maximum only if s >= max s - 2 e, e = (DP + 16) (2^-23 max S + 2^-126 (1 + max |q|)); usually one
// key of a block does. Those keys' dots are formed in FP64 (four lanes a row, each with the dims of its query fragment, two
// exchanges), and their maximum is the score. Rows with an infinity or a NaN somewhere fail the comparison and are
// settled in FP64 as well.
//
// Bound by reading the index keys once from HBM (256 bytes a key for 128 dims): a wave takes one key
// block for 16 query rows (tokens x groups of a sequence), its key fragments straight from memory in the
// operand layout (lane c a key, 64 contiguous bytes of it for each 32 dims and four lanes), the next group of
// them in flight during the products of one. Sequences of a batch differ in length by orders, so the (tile,
// block) pairs of all of them are counted in front and shared out evenly over the waves.
#include "mfma_util.hpp"
#include "paged.hpp"
#include "score_mfma.hpp"
#include "topk_row.hpp"

namespace msa {
namespace {

// Workgroups of a call: two a CU, as many as run at once (us with 256 / 512 / 768, top-k included: 32 requests of
// 0.5 to 30K tokens 27.6 / 25.7 / 30.0, 64 of 16K 58.0 / 58.5 / 61.9, that is 4.6 TB/s, 256 of 4K 63.9 / 62.2 / 64.9). Their
// stretches go block by block through one tile: all tiles of a few blocks first, for the keys to come from the L2 the second
// time, gives 25.6 -> 24.4 us for 5 tokens of 4 groups behind 130 000, but 30.2 -> 36.7 for 16 requests of 16K with 5 each.
constexpr int64_t kBlocks = 512;

struct PagedScoreArgs {
  const uint16_t* iq;  // [T][G][Di]
  CacheView keys;      // one head
  PageMap pages;
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  int G, Di, NB, B;
  float sign, scale; // of the logits: direction and magnitude
  float* scores;     // [T][G][NB]
};

// A sequence of the call: its first token and its tokens, the cached ones in front, its tiles of 16 query rows and the key
// blocks they go through (one for a sequence that is not there).
struct SeqWork {
  int32_t start, count, context;
  int tiles, blocks;
  __device__ __forceinline__ int64_t items() const { return static_cast<int64_t>(tiles) * blocks; }
};
__device__ __forceinline__ SeqWork seq_work(const PagedScoreArgs& A, int32_t start, int32_t end, int32_t context) {
  // (unsigned: a context that no page table holds may bring the sum past 2^31)
  const uint32_t n = end - start, blocks = context < 0 || n == 0 ? 1u : (context + n - 1) / static_cast<uint32_t>(A.B) + 1;
  return SeqWork{start, end - start, context, static_cast<int>((n * A.G + 15) / 16),
                 static_cast<int>(min(blocks, static_cast<uint32_t>(A.NB)))};
}

// a / b, in 32 bits where a fits (a 64-bit division is some 100 instructions)
__device__ __forceinline__ int64_t quotient(int64_t a, uint32_t b) {
  return a >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / b);
}

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

// Blocks [block0, block1) of one tile of a sequence, by a wave; what its tokens do not see, up to block `fill`, gets -inf.
// FULL: Di is 32 NK, and a lane's pieces of a key row are at constant offsets.
template <int DT, int NK, bool FULL>
__device__ __forceinline__ void score_run(const PagedScoreArgs& A, const SeqWork& W, int s, int tile, int block0,
                                          int block1, int fill) {
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int64_t start = W.start, rows = static_cast<int64_t>(W.count) * A.G, r0 = static_cast<int64_t>(tile) * 16;
  const int32_t context = W.context;
  const int64_t row = r0 + c;
  const bool live = row < rows;
  const int32_t i = static_cast<uint32_t>(live ? row : rows - 1) / static_cast<uint32_t>(A.G);  // token of the sequence
  const int64_t end = A.pages.last_position();
  const int64_t pos = context < 0 ? -1 : min(end, static_cast<int64_t>(context) + i);
  const int64_t last = context < 0 ? -1 : min(end, static_cast<int64_t>(context) +
                                                       static_cast<uint32_t>(min(r0 + 16, rows) - 1) / static_cast<uint32_t>(A.G));
  float* out = A.scores + (start * A.G + (live ? row : rows - 1)) * A.NB;
  const int seen_blocks = A.pages.num_pages == 0 || last < 0
                              ? 0
                              : static_cast<int>(min(static_cast<uint32_t>(last) / A.B + 1, static_cast<uint32_t>(A.NB)));
  const int stop = min(block1, seen_blocks);
  for (int b = max(block0, seen_blocks) + q4; b < fill; b += 4)
    if (live) out[b] = -__builtin_inff();
  if (block0 >= stop) return;
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

  int block = block0;
  int64_t kc = static_cast<int64_t>(block) * A.B, k1 = min(kc + A.B, last + 1);
  int own_page = pages_of(kc, k1);
  bf16x8 f0[GT][NK], f1[GT][NK];
  load_group(f0, kc, own_page, 0);
  double best = -__builtin_inf();
  bool any = false;
  while (true) {
    // the chunk behind this one: of this block, or the first of this wave's next one
    const bool block_ends = kc + 16 * kTiles >= k1;
    const int next_block = block_ends ? block + 1 : block;
    const bool more = next_block < stop;
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

template <int DT, int NK, bool FULL>
__global__ __launch_bounds__(256, 2) void score_paged_kernel(PagedScoreArgs A) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // The batch's work is its (tile, block) pairs, numbered sequence by sequence: counted here, a sequence a lane where
  // there are up to 64 (no LDS, no barrier: 2 us of the 10 us of one long sequence's call), otherwise `per` a thread.
  __shared__ int64_t first_item[257];  // of the sequences that thread i counts
  __shared__ int64_t wave_items[4];
  const bool few = A.nseq <= 64;
  const int per = (A.nseq + 255) / 256;
  SeqWork mine{};
  int64_t upto = 0, items;
  if (few) {
    if (lane < A.nseq) mine = seq_work(A, A.cu[lane], A.cu[lane + 1], A.context[lane]);
    upto = mine.items();
  } else {
    for (int s = threadIdx.x * per; s < min(A.nseq, (static_cast<int>(threadIdx.x) + 1) * per); ++s)
      upto += seq_work(A, A.cu[s], A.cu[s + 1], A.context[s]).items();
  }
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int64_t x = __shfl_up(upto, o, kWave);
    if (lane >= o) upto += x;
  }
  if (few) {
    items = __shfl(upto, 63, kWave);
  } else {
    if (lane == 63) wave_items[wave] = upto;
    __syncthreads();
    for (int w = 0; w < wave; ++w) upto += wave_items[w];
    first_item[threadIdx.x + 1] = upto;
    if (threadIdx.x == 0) first_item[0] = 0;
    __syncthreads();
    items = first_item[256];
  }
  // a wave takes a stretch of them as long as the others', to one
  const uint32_t waves = gridDim.x * 4, own = blockIdx.x * 4 + wave;
  const int64_t share = quotient(items, waves), extra = items - share * waves;
  int64_t item = own * share + min(static_cast<int64_t>(own), extra);
  const int64_t end_item = item + share + (own < extra ? 1 : 0);
  while (item < end_item) {
    int s;
    int64_t rest;
    SeqWork work;
    if (few) {
      s = __builtin_ctzll(__ballot(upto > item));
      work.start = __builtin_amdgcn_readlane(mine.start, s);
      work.count = __builtin_amdgcn_readlane(mine.count, s);
      work.context = __builtin_amdgcn_readlane(mine.context, s);
      work.tiles = __builtin_amdgcn_readlane(mine.tiles, s);
      work.blocks = __builtin_amdgcn_readlane(mine.blocks, s);
      rest = item - (__shfl(upto, s, kWave) - work.items());
    } else {
      int lo = 0, hi = 256;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first_item[mid] <= item) lo = mid; else hi = mid;
      }
      s = __builtin_amdgcn_readfirstlane(lo * per);
      rest = item - first_item[lo];
      work = seq_work(A, A.cu[s], A.cu[s + 1], A.context[s]);
      while (rest >= work.items()) {
        rest -= work.items();
        ++s;
        work = seq_work(A, A.cu[s], A.cu[s + 1], A.context[s]);
      }
    }
    const int tile = static_cast<int>(quotient(rest, work.blocks));
    const int block0 = static_cast<int>(rest - static_cast<int64_t>(tile) * work.blocks);
    const int block1 = static_cast<int>(min(static_cast<int64_t>(work.blocks), block0 + (end_item - item)));
    item += block1 - block0;
    score_run<DT, NK, FULL>(A, work, s, tile, block0, block1, block1 == work.blocks ? A.NB : block1);
  }
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
  // (a selection's launch takes 16 rows a workgroup, of fewer than 2^24)
  if (index_dim % 8 || index_dim > 256 || block_size % 16 || total_tokens * groups > 0x7fffffff ||
      (topk_blocks > 0 && total_tokens * groups >= int64_t{1} << 28))
    return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  PagedScoreArgs A{};
  A.iq = static_cast<const uint16_t*>(index_q);
  A.keys = CacheView{const_cast<void*>(index_cache), cache_stride_page, 0, cache_stride_slot};
  A.pages = page_map(page_table, table_stride, pages_per_seq, num_pages, page_size);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.context = context_lens;
  A.G = static_cast<int>(groups);
  A.Di = static_cast<int>(index_dim);
  A.NB = static_cast<int>(num_blocks);
  A.B = static_cast<int>(block_size);
  A.sign = scale > 0.0 ? 1.f : scale < 0.0 ? -1.f : 0.f;
  A.scale = static_cast<float>(scale < 0.0 ? -scale : scale);
  A.scores = scores;
  const int64_t items = (total_tokens * groups / 16 + num_seqs) * num_blocks;  // at most
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(items < 4 * kBlocks ? (items + 3) / 4 : kBlocks)), block(256);
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
