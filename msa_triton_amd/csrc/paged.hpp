// A cache in pages, and where a sequence's tokens lie in it.
//
// A cache tensor is [P, H, page, D] with free strides over pages, heads and slots and unit stride
// along D. Position j of sequence s (below 2^31) is slot j % page of page table[s][j / page]. Entries outside
// [0, P) stand for pages that do not exist: nothing is read or written there. New tokens are packed by cu_seqlens; a
// sequence holds context[s] tokens in front of them, so that new token t has position
// context[s] + t - cu[s]. A negative context marks a sequence that is not there (padding of a fixed batch).
#pragma once
#include "common.hpp"

namespace msa {

struct CacheView {
  void* base;
  int64_t stride_page, stride_head, stride_slot;  // elements
};

struct PageMap {
  const int32_t* table;
  int64_t stride;        // entries from one sequence to the next
  int pages_per_seq;
  int num_pages;
  int shift;             // log2(page size)

  // The last position that the table has an entry for (-1: none). Keys behind it do not exist, whatever a sequence's
  // length says, and no loop goes there.
  __device__ __forceinline__ int64_t last_position() const { return (static_cast<int64_t>(pages_per_seq) << shift) - 1; }

  // The page that holds position j of sequence s, or -1.
  __device__ __forceinline__ int page_of(int s, int64_t j) const {
    const int64_t m = j >> shift;
    if (m >= pages_per_seq) return -1;
    const int p = table[s * stride + m];
    return p >= 0 && p < num_pages ? p : -1;
  }
};

// Sequence and position of a new token; position -1 where the sequence is not there.
struct TokenPlace {
  int seq;
  int64_t pos;
};

// The last s in [0, n) with first(s) <= x, for nondecreasing first with first(0) <= x; x the same in all lanes of the
// wave, which all call it. 64 entries are compared at a time, so that a batch of up to 64 sequences costs one load's
// latency (a bisection: one for every halving) and one of 4096 two.
template <class First>
__device__ __forceinline__ int wave_upper_index(int n, int64_t x, First first) {
  const int lane = threadIdx.x & 63;
  int lo = 0;
  for (int64_t step = 1;; step = 1) {
    while (n - lo > 64 * step) step *= 64;
    const int64_t i = lo + lane * step;
    const uint64_t at_most = __ballot(i < n && first(static_cast<int>(i)) <= x);
    lo += static_cast<int>((__popcll(at_most) - 1) * step);
    if (step == 1) return lo;
    n = static_cast<int>(min(static_cast<int64_t>(n), lo + step));
  }
}
__device__ __forceinline__ TokenPlace place_of(const int32_t* __restrict__ cu, int nseq,
                                               const int32_t* __restrict__ context, int64_t t) {
  const int s = find_seq(cu, nseq, t);
  const int32_t c = context[s];
  return TokenPlace{s, c < 0 ? -1 : c + (t - cu[s])};
}

// place_of for a token that is the same in all lanes of a wave, which all call it.
__device__ __forceinline__ TokenPlace wave_place_of(const int32_t* __restrict__ cu, int nseq,
                                                    const int32_t* __restrict__ context, int64_t t) {
  const auto start_of = [&](int i) { return static_cast<int64_t>(cu[i]); };
  if (nseq <= 64) {  // both loads at once
    const int lane = threadIdx.x & 63, i = lane < nseq ? lane : nseq - 1;
    const int32_t start = cu[i], c_own = context[i];
    const int s = __popcll(__ballot(lane < nseq && start <= t)) - 1;
    const int32_t c = __builtin_amdgcn_readlane(c_own, s);
    return TokenPlace{s, c < 0 ? -1 : c + (t - __builtin_amdgcn_readlane(start, s))};
  }
  const int s = wave_upper_index(nseq, t, start_of);
  const int32_t c = context[s];
  return TokenPlace{s, c < 0 ? -1 : c + (t - cu[s])};
}

// What every paged entry point checks about its page map.
inline bool valid_pages(const int32_t* table, int64_t stride, int64_t pages_per_seq, int64_t num_pages,
                        int64_t page_size) {
  return (table || pages_per_seq == 0) && stride >= 0 && num_pages >= 0 && num_pages <= 0x7fffffff && page_size >= 16 &&
         page_size <= 256 && (page_size & (page_size - 1)) == 0 && pages_per_seq >= 0 && pages_per_seq <= 0x7fffffff / page_size;
}

inline PageMap page_map(const int32_t* table, int64_t stride, int64_t pages_per_seq, int64_t num_pages,
                        int64_t page_size) {
  return PageMap{table, stride, static_cast<int>(pages_per_seq), static_cast<int>(num_pages),
                 __builtin_ctz(static_cast<unsigned>(page_size))};
}

}  // namespace msa
