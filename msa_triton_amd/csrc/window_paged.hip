// Window and tree attention of new tokens over a paged cache (16-bit or e4m3 with a scale for each page and head).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale q[t, h] . k_j - max),
// over the keys that token t sees: those up to its own slot in its window, the first `sinks` ones, and in a tree of
// drafted tokens, of the new ones, itself and its ancestors. Node i of a tree lies in slot context + i and has position
// context + depth(i); windows and sinks go by positions.
//
// Bound by reading the visible keys and values once from HBM for few rows, by the matrix products for many. Rows of a key head
// are (token, query head) pairs in tiles of R; a tile goes through its keys in steps of 32. All steps of the batch
// are counted in front and shared out evenly over the workgroups, whatever the lengths (a request of 30 000 tokens next to
// one of 60): a workgroup takes a stretch of them, its four waves every fourth step of a tile each on their own, as in
// the block-sparse form: key fragments straight from memory, S^T = K Q^T, weights as they come out of it, values through
// the wave's LDS tile. A tile that lies in one stretch is finished there; the parts of the others, maxima, sums and fp32
// outputs, are joined by a second launch in a fixed order. 64 requests of 60 to 30 000 tokens, 4 key heads of 128, 16 bits, no
// window: 131 + 11 us, 4.8 TB/s; 512, 300 and 1 new tokens behind 8192, 1000 and 5000, window 2048, 32 heads: 60 + 16 us.
// The attention kernels spill 102 to 179 scalar registers into lanes of vector registers (careful_row is inlined in them); of vector
// registers e4m3 at 256 dims spills 38 a lane, and 16 bits at 256 dims with 16 rows a tile takes 430, one wave a SIMD.
//
// Logits, statistics and outputs are fp32. With one tile of 16 rows, where the products are not the bound, a weight
// enters the second product as two 16-bit terms (2^-17 of it left out); with more it is rounded once, as in the packed
// form (fp16 queries over an 8-bit cache, whose products are bf16's, take two terms). In fp16 both are of the weight times
// 2^7. Bytes of an 8-bit page are exact in bf16; its scales go into logits and weights.
#include "window.hpp"

namespace msa {
namespace {

constexpr int kMostParts = 128;     // workgroups that share a tile
constexpr int kTreeNodes = 512;     // most new tokens of a tree
constexpr float kLowest = -3.402823466e38f;  // the least maximum of keys that exist

struct PagedPlan {
  int64_t items, share;  // steps of the batch, of a workgroup
};

struct PagedWindowArgs {
  const uint16_t* q;  // [T][Hq][D]
  CacheView k, v;
  const float *k_scale, *v_scale;  // [P][G]
  PageMap pages;
  const int32_t* cu;
  int nseq;
  const int32_t* context;
  const int32_t* parents;  // [T], or null: no tree
  Divisor ratio;
  int G, D;
  Visible seen;
  float scale_log2;  // scale * log2(e)
  uint16_t* out;  // [T][Hq][D]
  float* lse;     // [T][Hq], or null
  PagedPlan* plan;
  int64_t* first_item;  // [N]
  float* part;    // [workgroups][2][R][D]: of a tile that it does not begin, of one that it does not end
  float* stats;   // [workgroups][2][2][R]: maximum (log2), sum
};

// The keys that a tile of rows goes through: [0, sinks) in steps of 32, then [low, hi] in steps of 32, low a multiple of it.
struct TileKeys {
  int a, b;  // first and last token
  int low, hi, sinks, sink_steps, steps;
  __device__ __forceinline__ int first(int e) const { return e < sink_steps ? 32 * e : low + 32 * (e - sink_steps); }
  // The same in all lanes, said to the compiler (64-bit minima are formed in the vector unit).
  __device__ __forceinline__ TileKeys in_scalars() const {
    auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return TileKeys{one(a), one(b), one(low), one(hi), one(sinks), one(sink_steps), one(steps)};
  }
};
__device__ __forceinline__ int64_t scalar(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(x)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(x >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}
__device__ __forceinline__ int scalar_int(int64_t x) {
  return __builtin_amdgcn_readfirstlane(static_cast<int>(min(max(x, int64_t{-0x7fffffff}), int64_t{0x7fffffff})));
}

// A sequence of the call: its tiles, and the steps that each of them is given (those behind a tile's last do nothing).
struct SeqPlan {
  int n, context, tiles, steps;
  __device__ __forceinline__ int64_t items(int groups) const { return static_cast<int64_t>(tiles) * groups * steps; }
};

template <int R>
__device__ __forceinline__ TileKeys tile_keys(const PagedWindowArgs& A, int n, int context, int tile) {
  TileKeys K;
  const int r0 = tile * R;
  K.a = A.ratio(r0);
  K.b = A.ratio(min(r0 + R, n * A.ratio.d) - 1);
  const int64_t last = A.pages.last_position(), c = context;
  K.hi = context < 0 ? -1 : static_cast<int>(min(c + K.b, last));
  const int64_t low = max(int64_t{0}, c + (A.parents ? 0 : K.a) - A.seen.window + 1);
  // (past hi: none; a table may reach up to 2^31 - 17)
  K.low = static_cast<int>(min(low, min(static_cast<int64_t>(K.hi) + 32, int64_t{0x7fffffff}))) & ~31;
  if (context < 0) K.low = 0;
  K.sinks = min(A.seen.sinks, min(K.low, K.hi + 1));
  K.sink_steps = (K.sinks >> 5) + ((K.sinks & 31) != 0);
  K.steps = K.sink_steps + (K.hi >= K.low ? (K.hi >> 5) - (K.low >> 5) + 1 : 0);
  return K;
}

template <int R>
__device__ __forceinline__ SeqPlan seq_plan(const PagedWindowArgs& A, int start, int end, int context) {
  SeqPlan P;
  P.n = end - start;
  P.context = context;
  P.tiles = (P.n * A.ratio.d + R - 1) / R;
  P.steps = 1;
  if (P.tiles == 0 || context < 0) return P;
  const TileKeys K = tile_keys<R>(A, P.n, context, P.tiles - 1);
  if (P.tiles == 1) {
    P.steps = max(1, K.steps);
  } else {  // at least those of any tile
    const int64_t span = static_cast<int64_t>(A.seen.window) + (A.parents ? P.n : R / A.ratio.d + 1);
    const int64_t by_window = (static_cast<int64_t>(A.seen.sinks) + 31) / 32 + span / 32 + 2;
    P.steps = static_cast<int>(max(int64_t{1}, min(by_window, static_cast<int64_t>(K.hi >= 0 ? (K.hi >> 5) + 1 : 1))));
  }
  return P;
}

// a / b, in 32 bits where a fits
__device__ __forceinline__ int64_t quotient(int64_t a, uint32_t b) {
  return a >> 32 ? a / b : static_cast<int64_t>(static_cast<uint32_t>(a) / b);
}

// The parent of node i among its sequence's new tokens, or -1: anything that is not in front of it is none.
__device__ __forceinline__ int parent_of(int p, int i) { return p >= 0 && p < i ? p : -1; }

// The dims of a row that came out not finite, by a wave: where a value that is not finite met the products of a tile, which
// multiply the keys that a row does not see by 0. Such values count whatever their weight above 0; a weight of 0 under
// a logit of -inf makes NaN of them. Dims in which the row sees one are these values' sum, which takes a look at their
// column; the others are formed again key by key, from weights whose sum is 1 (values next to the end of fp32's range, of
// which a tile's sums are infinities, have a finite mean). The weight is exp2(logit * log2(e) - top) inv.
template <int DT, bool FP8>
__device__ __forceinline__ void careful_row(const PagedWindowArgs& A, int s, int start, int context, int tok, int g, int head,
                                            float top, float inv) {
  constexpr int ES = FP8 ? 1 : 2;
  if (top == -__builtin_inff()) top = 0.f;  // (all logits -inf: weights 0)
  const int lane = threadIdx.x & 63, slot_mask = (1 << A.pages.shift) - 1;
  const int64_t row = (start + static_cast<int64_t>(tok)) * (A.G * A.ratio.d) + head;
  const uint16_t* q = A.q + row * A.D;
  const char* kbase = static_cast<const char*>(A.k.base) + g * A.k.stride_head * ES;
  const char* vbase = static_cast<const char*>(A.v.base) + g * A.v.stride_head * ES;
  const int32_t* parents = A.parents ? A.parents + start : nullptr;
  int64_t pos = context + static_cast<int64_t>(tok);
  if (parents) {
    pos = context;
    for (int i = parent_of(parents[tok], tok); i >= 0; i = parent_of(parents[i], i)) ++pos;
  }
  const int64_t hi = min(context + static_cast<int64_t>(tok), A.pages.last_position()), low = max(int64_t{0}, pos - A.seen.window + 1);
  const int d = 4 * lane;  // (at most 256 dims)
  float o[4] = {0.f, 0.f, 0.f, 0.f}, odd[4] = {0.f, 0.f, 0.f, 0.f};
  bool bad[4] = {false, false, false, false}, look = true;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // (what this wave's other lanes stored)
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
  if (d < A.D) {
    float y[4];
    load4<DT, false>(reinterpret_cast<const char*>(A.out + row * A.D + d), y);
#pragma unroll
    for (int u = 0; u < 4; ++u) bad[u] = !finite(y[u]);
  }
  auto wanted = [&](int u) { return bad[u] && (look ? odd[u] == odd[u] : odd[u] == 0.f); };
  auto keys = [&](int64_t from, int64_t to) {  // both below 2^31; cached tokens and new ones never in one go
    for (int64_t base = from; base < to; base += kWave) {
      const bool mine = wanted(0) || wanted(1) || wanted(2) || wanted(3);
      if (!__any(mine)) return;
      const int64_t j = min(base + lane, to - 1);
      bool seen = base + lane < to;
      if (parents && base >= context) {  // new tokens on the way up
        const int own = static_cast<int>(j - context);
        bool on_path = false;
        int64_t place = pos;
        for (int i = tok; i >= 0; i = parent_of(parents[i], i), --place)
          on_path |= i == own && (pos - place < A.seen.window || place < A.seen.sinks);
        seen &= on_path;
      }
      const int page = A.pages.page_of(s, j);
      seen &= page >= 0;
      auto logit = [&]() {
        const int64_t p0 = page < 0 ? 0 : page;
        const char* kp = kbase + (p0 * A.k.stride_page + (j & slot_mask) * A.k.stride_slot) * ES;
        float x = 0.f;
        for (int e = 0; e < A.D; e += 4) {
          float y[4], z[4];
          load4<DT, false>(reinterpret_cast<const char*>(q + e), y);
          load4<DT, FP8>(kp + e * ES, z);
#pragma unroll
          for (int i = 0; i < 4; ++i) x = fmaf(y[i], z[i], x);
        }
        return x * (A.scale_log2 * (FP8 ? A.k_scale[p0 * A.G + g] : 1.f));
      };
      const float p = look ? 0.f : __builtin_amdgcn_exp2f(logit() - top) * inv;
      uint64_t dead = 0;  // keys of a logit of -inf, looked for when a value is infinite
      bool known = false;
      for (uint64_t left = __ballot(seen); left; left &= left - 1) {
        const int i = __builtin_ctzll(left);
        const float p_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
        const int64_t page_i = __builtin_amdgcn_readlane(page, i);
        const char* vp = vbase + (page_i * A.v.stride_page + ((base + i) & slot_mask) * A.v.stride_slot) * ES;
        const float vs = FP8 ? A.v_scale[page_i * A.G + g] : 1.f;
        float y[4] = {0.f, 0.f, 0.f, 0.f};
        if (mine) load4<DT, FP8>(vp + d * ES, y);
        if (look) {
          bool infinite = false;
#pragma unroll
          for (int u = 0; u < 4; ++u) y[u] = bad[u] ? y[u] * vs : 0.f, infinite |= !finite(y[u]) && y[u] == y[u];
          if (!known && __any(infinite)) dead = __ballot(logit() == -__builtin_inff()), known = true;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (!finite(y[u])) odd[u] += dead >> i & 1 ? __builtin_nanf("") : y[u];
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u)
            if (wanted(u)) o[u] = fmaf(p_i, y[u] * vs, o[u]);
        }
      }
    }
  };
  if (context >= 0 && A.pages.num_pages > 0) {
    const int64_t cached = parents ? min(static_cast<int64_t>(context), hi + 1) : hi + 1;
    for (int pass = 0; pass < 2; ++pass, look = false) {
      keys(0, min(static_cast<int64_t>(A.seen.sinks), min(low, cached)));
      keys(min(low, cached), cached);
      if (parents) keys(context, hi + 1);
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (bad[u]) store_from_f32<DT>(A.out, row * A.D + d + u, odd[u] != 0.f ? odd[u] : o[u]);
}

// Which keys a row sees: `low` the first of its window, `slot` its own.
struct RowKeys {
  int low, slot;
  RowKeys() = default;
  // place: of the token's position behind the context
  __device__ __forceinline__ RowKeys(const PagedWindowArgs& A, const TileKeys& K, int context, int tok, int place)
      : low(static_cast<int>(min(max(int64_t{0}, static_cast<int64_t>(context) + place - A.seen.window + 1), int64_t{0x7fffffff}))),
        slot(static_cast<int>(min(static_cast<int64_t>(context) + tok, static_cast<int64_t>(K.hi)))) {}
  // on_path(node): of a tree's new tokens, whether the row sees this one
  template <class OnPath>
  __device__ __forceinline__ bool sees(const PagedWindowArgs& A, int context, int key, OnPath on_path) const {
    if (A.parents && key >= context) return on_path(key - context);
    return key <= slot && (key >= low || key < A.seen.sinks);
  }
};

// The batch's steps, sequence by sequence, and the stretch of them that is this workgroup's: a sequence a lane where there are
// up to 64, otherwise `per` a thread. The first workgroup leaves the plan for the join.
template <int R>
struct Batch {
  struct Shared {
    int64_t first_item[257], wave_items[4];  // of the sequences that thread i counts
    int wave_most[4];
  };
  bool few;
  int per;
  SeqPlan mine;
  int64_t upto, item, end;

  __device__ __forceinline__ void open(const PagedWindowArgs& A, Shared& S) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    few = A.nseq <= 64;
    per = (A.nseq + 255) / 256;
    mine = SeqPlan{};
    upto = 0;
    int64_t items;
    int most = 1;
    if (few) {
      if (lane < A.nseq) {
        mine = seq_plan<R>(A, A.cu[lane], A.cu[lane + 1], A.context[lane]);
        upto = mine.items(A.G), most = mine.steps;
      }
    } else {
      for (int s = threadIdx.x * per; s < min(A.nseq, (static_cast<int>(threadIdx.x) + 1) * per); ++s) {
        const SeqPlan P = seq_plan<R>(A, A.cu[s], A.cu[s + 1], A.context[s]);
        upto += P.items(A.G), most = max(most, P.steps);
      }
    }
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int64_t x = __shfl_up(upto, o, kWave);
      if (lane >= o) upto += x;
      most = max(most, __shfl_xor(most, o, kWave));
    }
    if (few) {
      items = __shfl(upto, 63, kWave);
    } else {
      if (lane == 63) S.wave_items[wave] = upto, S.wave_most[wave] = most;
      __syncthreads();
      for (int w = 0; w < wave; ++w) upto += S.wave_items[w];
      for (int w = 0; w < 4; ++w) most = max(most, S.wave_most[w]);
      S.first_item[threadIdx.x + 1] = upto;
      if (threadIdx.x == 0) S.first_item[0] = 0;
      __syncthreads();
      items = S.first_item[256];
    }
    most = __builtin_amdgcn_readfirstlane(most);
    // four steps at least (one a wave of the kernel of 16 rows; the one of many rows takes them one after the other: 15 nodes behind
    // 1999 tokens, 4 key heads, in 64 workgroups 24 us), and no tile in more than kMostParts stretches
    items = scalar(items);
    const int64_t share = scalar(max(max(int64_t{4}, quotient(items + gridDim.x - 1, gridDim.x)),
                                     static_cast<int64_t>((most + kMostParts - 2) / (kMostParts - 1))));
    if (blockIdx.x == 0) {
      if (threadIdx.x == 0) *A.plan = PagedPlan{items, share};
      if (few) {
        if (wave == 0 && lane < A.nseq) A.first_item[lane] = upto - mine.items(A.G);
      } else {
        int64_t at = S.first_item[threadIdx.x];
        for (int s = threadIdx.x * per; s < min(A.nseq, (static_cast<int>(threadIdx.x) + 1) * per); ++s) {
          A.first_item[s] = at;
          at += seq_plan<R>(A, A.cu[s], A.cu[s + 1], A.context[s]).items(A.G);
        }
      }
    }
    item = blockIdx.x * share;
    end = scalar(min(item + share, items));
  }

  // The next tile of the stretch and which of its steps are this workgroup's; false: none left.
  struct Piece {
    int s, g, tile, e0, e1;
    SeqPlan P;
  };
  __device__ __forceinline__ bool next(const PagedWindowArgs& A, const Shared& S, Piece& X) {
    if (item >= end) return false;
    int64_t rest;
    if (few) {
      X.s = __builtin_ctzll(__ballot(upto > item));
      X.P.n = __builtin_amdgcn_readlane(mine.n, X.s);
      X.P.context = __builtin_amdgcn_readlane(mine.context, X.s);
      X.P.tiles = __builtin_amdgcn_readlane(mine.tiles, X.s);
      X.P.steps = __builtin_amdgcn_readlane(mine.steps, X.s);
      rest = item - (__shfl(upto, X.s, kWave) - X.P.items(A.G));
    } else {
      int lo = 0, hi = 256;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (S.first_item[mid] <= item) lo = mid; else hi = mid;
      }
      X.s = __builtin_amdgcn_readfirstlane(lo * per);
      rest = item - S.first_item[lo];
      X.P = seq_plan<R>(A, A.cu[X.s], A.cu[X.s + 1], A.context[X.s]);
      while (rest >= X.P.items(A.G)) {
        rest -= X.P.items(A.G);
        ++X.s;
        X.P = seq_plan<R>(A, A.cu[X.s], A.cu[X.s + 1], A.context[X.s]);
      }
    }
    // (the same in all lanes)
    X.s = __builtin_amdgcn_readfirstlane(X.s);
    X.P.n = __builtin_amdgcn_readfirstlane(X.P.n), X.P.context = __builtin_amdgcn_readfirstlane(X.P.context);
    X.P.tiles = __builtin_amdgcn_readfirstlane(X.P.tiles), X.P.steps = __builtin_amdgcn_readfirstlane(X.P.steps);
    const int64_t tile_no = scalar(quotient(scalar(rest), X.P.steps));  // group by group
    X.e0 = static_cast<int>(rest - tile_no * X.P.steps);
    X.e1 = static_cast<int>(min(static_cast<int64_t>(X.P.steps), X.e0 + (end - item)));
    item += X.e1 - X.e0;
    X.g = __builtin_amdgcn_readfirstlane(static_cast<int>(quotient(tile_no, X.P.tiles)));
    X.tile = __builtin_amdgcn_readfirstlane(static_cast<int>(tile_no - static_cast<int64_t>(X.g) * X.P.tiles));
    X.e0 = __builtin_amdgcn_readfirstlane(X.e0), X.e1 = __builtin_amdgcn_readfirstlane(X.e1);
    return true;
  }
};

// Which new tokens each token of a tile sees, a bit each, and its depth. (All threads call it.)
template <int R>
struct TreeRows {
  static constexpr int kWords = kTreeNodes / 32;
  int parent[kTreeNodes], depth[R + 1];
  uint32_t path[(R + 1) * kWords];
  __device__ __forceinline__ void fill(const PagedWindowArgs& A, int start, int context, const TileKeys& K) {
    for (int i = threadIdx.x; i <= K.b; i += 256) parent[i] = parent_of(A.parents[start + i], i);
    __syncthreads();
    const int t = threadIdx.x;
    if (t <= K.b - K.a) {
      uint32_t* bits = path + t * kWords;
      for (int w = 0; w <= K.b >> 5; ++w) bits[w] = 0;
      int deep = 0;
      for (int i = parent[K.a + t]; i >= 0; i = parent[i]) ++deep;
      depth[t] = deep;
      int up = 0;
      for (int i = K.a + t; i >= 0; i = parent[i], ++up)
        if (up < A.seen.window || static_cast<int64_t>(context) + deep - up < A.seen.sinks) bits[i >> 5] |= 1u << (i & 31);
    }
    __syncthreads();
  }
  __device__ __forceinline__ bool sees(int token, int node) const {
    return path[token * kWords + (node >> 5)] >> (node & 31) & 1u;
  }
};

template <int DT, bool FP8, int NK>
__global__ __launch_bounds__(256, NK == 8 && !FP8 ? 1 : 2) void window_paged_kernel(PagedWindowArgs A) {
  constexpr int R = 16, DP = 32 * NK, RS = DP + 16, ND = DP / 16, ES = FP8 ? 1 : 2;
  constexpr int PT = FP8 ? kBF16 : DT;          // type of the second product
  constexpr float kUp = PT == kF16 ? 15.f - kSlack : 0.f;
  constexpr int VL = FP8 ? DP / 16 : DP / 8, NV = VL / 2, VR = 64 / VL, VD = FP8 ? 16 : 8;
  constexpr int NKR = FP8 ? NK / 2 : NK;
  constexpr int OS = DP + 4;
  static_assert(16 * OS * 4 <= 32 * RS * 2, "a wave's output fits its value tile");
  __shared__ alignas(16) uint16_t vbuf[4][32 * RS];
  __shared__ float wave_max[4][R], wave_sum[4][R];
  __shared__ typename Batch<R>::Shared shared;
  __shared__ TreeRows<R> tree;
  __shared__ uint32_t odd_rows;
  __shared__ float row_top[R], row_inv[R];
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ratio = A.ratio.d;
  Batch<R> batch_;
  batch_.open(A, shared);

  auto dim_of = [&](int kk) { return FP8 ? 64 * (kk >> 1) + 16 * q4 + 8 * (kk & 1) : 32 * kk + 8 * q4; };
  const bool full = A.D == DP;
  const int slot_mask = (1 << A.pages.shift) - 1;
  typename Batch<R>::Piece X;
  while (batch_.next(A, shared, X)) {
    auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int s = one(X.s), g = one(X.g), e0 = one(X.e0), e1 = one(X.e1);
    const SeqPlan P{one(X.P.n), one(X.P.context), one(X.P.tiles), one(X.P.steps)};
    const TileKeys K = tile_keys<R>(A, P.n, P.context, X.tile).in_scalars();
    const int start = A.cu[s], r0 = X.tile * R, live = min(R, P.n * ratio - r0);
    if (A.parents) tree.fill(A, start, P.context, K);
    const int own_tok = A.ratio(r0 + min(c, live - 1));
    bf16x8 qf[NK];
    {
      const int r = r0 + min(c, live - 1);
      const uint16_t* row = A.q + ((start + static_cast<int64_t>(own_tok)) * (A.G * ratio) + g * ratio + r - own_tok * ratio) * A.D;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) qf[kk] = dim_of(kk) < A.D ? load_frag(row + dim_of(kk)) : zero_frag();
    }
    const RowKeys row_keys(A, K, P.context, own_tok, A.parents ? tree.depth[own_tok - K.a] : own_tok);
    const int common = scalar_int(A.parents ? P.context : min(static_cast<int64_t>(P.context) + K.a, static_cast<int64_t>(K.hi)) + 1);
    const int low_most = scalar_int(static_cast<int64_t>(P.context) + K.b - A.seen.window + 1);

    float top = -__builtin_inff(), l = 0.f;
    bool had_keys = false;
    f32x4 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* kbase = static_cast<const char*>(A.k.base) + g * A.k.stride_head * ES;
    const char* vbase = static_cast<const char*>(A.v.base) + g * A.v.stride_head * ES;
    uint4 kr[2][NKR], vr[NV];
    int key0 = 0, p0 = -1, p1 = -1;
    float ks0 = 1.f, ks1 = 1.f, vs0 = 1.f, vs1 = 1.f;

    // this wave's steps: pages of 32 at a time, a half step a lane; those with a page that exists are gone through
    int batch = e0 + wave, own_page = -1;
    uint64_t open = 0;
    const int stop = __builtin_amdgcn_readfirstlane(min(e1, K.steps));
    auto key_of = [&](int i) { return K.first(batch - 128 + 4 * (i >> 1)) + 16 * (i & 1); };
    auto next_step = [&]() {  // false: none left
      while (open == 0) {
        if (batch >= stop) return false;
        const int e = batch + 4 * (lane >> 1);
        const int j = K.first(e) + 16 * (lane & 1);
        own_page = e < stop && j <= (e < K.sink_steps ? K.sinks - 1 : K.hi) ? A.pages.page_of(s, j) : -1;
        const uint64_t there = __ballot(own_page >= 0);
        open = (there | there >> 1) & 0x5555555555555555ull;
        batch += 128;
      }
      const int i = __builtin_ctzll(open);
      open &= open - 1;
      key0 = __builtin_amdgcn_readfirstlane(key_of(i));
      p0 = __builtin_amdgcn_readlane(own_page, i);
      p1 = __builtin_amdgcn_readlane(own_page, i + 1);
      return true;
    };
    auto load_step = [&]() {
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

    bool more = next_step();
    if (more) load_step();
    while (more) {
      had_keys = true;
      const int k_now = key0, a_now = p0, b_now = p1;
      const bool of_sinks = k_now < K.low;
      const int upto_key = of_sinks ? K.sinks - 1 : K.hi;  // of the tile
      f32x4 sc[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sc[h] = f32x4{0.f, 0.f, 0.f, 0.f};
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
          sc[h] = mfma_t<DT>(__builtin_bit_cast(bf16x8, w), qf[kk], sc[h]);
        }
      }
      uint16_t* vt = vbuf[wave];
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        const int r = p * VR + lane / VL;
        const bool there = (p < NV / 2 ? a_now : b_now) >= 0 && k_now + r <= upto_key;  // (unwritten slots hold anything)
        const uint4 x = there ? vr[p] : make_uint4(0u, 0u, 0u, 0u);
        uint4* to = reinterpret_cast<uint4*>(vt + r * RS + lane % VL * VD);
        if constexpr (FP8) {
          to[0] = widen_fp8<false>(x.x, x.y);
          to[1] = widen_fp8<false>(x.z, x.w);
        } else {
          to[0] = x;
        }
      }
      const float kf0 = A.scale_log2 * ks0, kf1 = A.scale_log2 * ks1, vf0 = vs0, vf1 = vs1;
      more = next_step();
      if (more) load_step();
      const bool whole = a_now >= 0 && b_now >= 0 && k_now + 31 < common && k_now + 31 <= upto_key &&
                         (of_sinks || k_now >= low_most || k_now + 31 < A.seen.sinks);
      float x[8], high = -__builtin_inff();
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = sc[j >> 2][j & 3] * (j >> 2 ? kf1 : kf0);
      if (!whole) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int h = j >> 2, key = k_now + 16 * h + 4 * q4 + (j & 3);
          const bool seen = (h ? b_now : a_now) >= 0 && key <= upto_key && row_keys.sees(A, P.context, key, [&](int node) {
            return tree.sees(own_tok - K.a, node);
          });
          x[j] = seen ? x[j] : -__builtin_inff();
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) high = fmaxf(high, x[j]);
      if (__any(high > top + kSlack)) {
        const float next = fmaxf(top, quarters_max(high));
        const float keep = top == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(top - next);
        top = next;
        l *= keep;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= keep;
      }
      const float shift = kUp - (top == -__builtin_inff() ? 0.f : top);  // (all logits -inf: weights 0)
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        float y0 = __builtin_amdgcn_exp2f(x[j] + shift), y1 = __builtin_amdgcn_exp2f(x[j + 1] + shift);
        l += y0 + y1;
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

    // ---- the four waves joined: maxima and sums, then the outputs through LDS
    if (had_keys) top = fmaxf(top, kLowest);
    l += __shfl_xor(l, 16, kWave);
    l += __shfl_xor(l, 32, kWave);
    if (q4 == 0) wave_max[wave][c] = top, wave_sum[wave][c] = l;
    if (threadIdx.x == 0) odd_rows = 0;
    const bool done = e0 == 0 && e1 == P.steps;
    const int64_t place = static_cast<int64_t>(blockIdx.x) * 2 + (e0 > 0 ? 0 : 1);
    float* own = reinterpret_cast<float*>(vbuf[wave]);
#pragma unroll
    for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4*>(own + c * OS + 16 * d + 4 * q4) = acc[d];
    __syncthreads();
    const int r = threadIdx.x >> 4, col = threadIdx.x & 15;  // 16 threads a row
    const float high = fmaxf(fmaxf(wave_max[0][r], wave_max[1][r]), fmaxf(wave_max[2][r], wave_max[3][r]));
    float f[4], sum = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      f[w] = wave_max[w][r] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(wave_max[w][r] - high);
      sum += f[w] * wave_sum[w][r];
    }
    if (r < live) {
      const int tok = A.ratio(r0 + r);
      const int64_t out_row = (start + static_cast<int64_t>(tok)) * (A.G * ratio) + g * ratio + r0 + r - tok * ratio;
      const float inv = done ? (sum == 0.f ? 0.f : 1.f / sum) : 1.f;
      float all = 0.f;
      for (int d = 4 * col; d < A.D; d += 64) {
        f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const f32x4 x = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(vbuf[w]) + r * OS + d);
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = fmaf(f[w], x[i], o[i]);
        }
        o *= inv;
        all += (o[0] + o[1]) + (o[2] + o[3]);
        if (done) store4<DT>(A.out + out_row * A.D + d, o);
        else *reinterpret_cast<f32x4*>(A.part + (place * R + r) * A.D + d) = o;
      }
      if (col == 0) {
        if (!done) {
          A.stats[(place * 2) * R + r] = high;
          A.stats[(place * 2 + 1) * R + r] = sum;
        } else if (A.lse) {
          A.lse[out_row] = sum == 0.f ? -__builtin_inff() : (high - kUp + __log2f(sum)) * kLn2Window;
        }
        row_top[r] = high - kUp, row_inv[r] = inv;
      }
      // (a sum of NaN makes the row NaN)
      if (done && !finite(all) && sum == sum) atomicOr(&odd_rows, 1u << r);
    }
    __syncthreads();
    uint32_t left = __builtin_amdgcn_readfirstlane(odd_rows);
    for (int turn = 0; left; left &= left - 1, ++turn) {
      if ((turn & 3) != wave) continue;
      const int i = __builtin_ctz(left), tok = A.ratio(r0 + i);
      careful_row<DT, FP8>(A, s, start, P.context, tok, g, g * ratio + r0 + i - tok * ratio, row_top[i], row_inv[i]);
    }
    __syncthreads();
  }
}

// The same for many rows a key head (drafted runs and trees, a prompt's next part): tiles of R = 64 MT rows, 16 MT a wave,
// and the keys and values of a step in LDS for all four waves, as in the packed form (an 8-bit page's bytes widened on
// their way there).
template <int DT, bool FP8, int NK, int MT>
__global__ __launch_bounds__(256, 2) void window_paged_rows_kernel(PagedWindowArgs A) {
  constexpr int R = 64 * MT, DP = 32 * NK, RS = DP + 16, ND = DP / 16, ES = FP8 ? 1 : 2;
  constexpr int PT = FP8 ? kBF16 : DT;          // type of the second product
  constexpr bool kTwo = DT != PT;               // terms of a weight: fp16 results from bf16 products
  constexpr float kUp = PT == kF16 ? 15.f - kSlack : 0.f;
  constexpr int VD = 16 / ES, VL = DP / VD, kAll = 32 * VL, NV = (kAll + 255) / 256;  // values and lanes of a row's pieces
  __shared__ alignas(16) uint16_t kbuf[2][32 * RS], vbuf[2][32 * RS];
  __shared__ typename Batch<R>::Shared shared;
  __shared__ TreeRows<R> tree;
  const int lane = threadIdx.x & 63, c = lane & 15, q4 = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int ratio = A.ratio.d, slot_mask = (1 << A.pages.shift) - 1;
  // (past the last piece: that wave's again)
  auto piece_of = [&](int p) { return min(p * 256 + 64 * wave, kAll - 64) + lane; };
  Batch<R> batch_;
  batch_.open(A, shared);
  uint32_t k_off[NV], v_off[NV];  // bytes of this thread's pieces from their half step's first row on
#pragma unroll
  for (int p = 0; p < NV; ++p) {
    const int i = piece_of(p), d = i % VL * VD < A.D ? i % VL * VD : 0;
    k_off[p] = (i / VL % 16 * static_cast<uint32_t>(A.k.stride_slot) + d) * ES;
    v_off[p] = (i / VL % 16 * static_cast<uint32_t>(A.v.stride_slot) + d) * ES;
  }

  typename Batch<R>::Piece X;
  while (batch_.next(A, shared, X)) {
    auto one = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    const int s = one(X.s), g = one(X.g), e0 = one(X.e0), e1 = one(X.e1);
    const SeqPlan P{one(X.P.n), one(X.P.context), one(X.P.tiles), one(X.P.steps)};
    const TileKeys K = tile_keys<R>(A, P.n, P.context, X.tile).in_scalars();
    const int start = A.cu[s], r0 = X.tile * R, live = min(R, P.n * ratio - r0);
    if (A.parents) tree.fill(A, start, P.context, K);
    int tok[MT];
    bf16x8 qf[MT][NK];
    RowKeys row_keys[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int r = r0 + min(16 * (MT * wave + m) + c, live - 1);
      tok[m] = A.ratio(r);
      const uint16_t* row = A.q + ((start + static_cast<int64_t>(tok[m])) * (A.G * ratio) + g * ratio + r - tok[m] * ratio) * A.D;
#pragma unroll
      for (int kk = 0; kk < NK; ++kk) {
        const Fragment<DT> f = 32 * kk + 8 * q4 < A.D && A.scale_log2 != 0.f ? fragment_at<DT>(row + 32 * kk + 8 * q4) : no_fragment<DT>();
        qf[m][kk] = turned<DT>(f, A.scale_log2 < 0.f).v;
      }
      row_keys[m] = RowKeys(A, K, P.context, tok[m], A.parents ? tree.depth[tok[m] - K.a] : tok[m]);
    }
    const bool has_rows = 16 * MT * wave < live;
    // (of this wave's rows where there is no tree)
    const int first_tok = A.ratio(r0 + min(16 * MT * wave, live - 1)), last_tok = A.ratio(r0 + min(16 * MT * (wave + 1), live) - 1);
    const int64_t c64 = P.context;
    const int common = scalar_int(A.parents ? c64 : min(c64 + first_tok, static_cast<int64_t>(K.hi)) + 1);
    const int low_most = scalar_int(c64 + (A.parents ? K.b : last_tok) - A.seen.window + 1);
    const int low_least = scalar_int(max(c64 + (A.parents ? 0 : first_tok) - A.seen.window + 1, int64_t{0}));
    const int last_slot = scalar_int(min(c64 + last_tok, static_cast<int64_t>(K.hi)));

    // a maximum is kept of the raw dots (queries are turned where the scale is negative, and zero with a factor of 1 where it is 0)
    const float factor = A.scale_log2 == 0.f ? 1.f : fabsf(A.scale_log2), slack = raw_slack(factor);
    float top[MT], l[MT];
    f32x4 acc[MT][ND];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] = -__builtin_inff(), l[m] = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const char* kbase = static_cast<const char*>(A.k.base) + g * A.k.stride_head * ES;
    const char* vbase = static_cast<const char*>(A.v.base) + g * A.v.stride_head * ES;
    const int stop = __builtin_amdgcn_readfirstlane(min(e1, K.steps));
    // pages and scales of the steps' halves, of 32 steps at a time, a half a lane; -1: none, nothing of it is seen
    int listed = e0 - 32, own_page = -1;
    float own_ks = 0.f, own_vs = 0.f;
    struct Step {
      int key, p0, p1, upto;
      float ks0, ks1, vs0, vs1;
    };
    uint4 kr[NV], vr[NV];
    Step in_flight;
    // a piece's half step is the same for the whole wave
    auto half_of = [&](int p) { return __builtin_amdgcn_readfirstlane(min(p * 256 + 64 * wave, kAll - 64) / (16 * VL)); };
    auto load_step = [&](int e) {
      if (e - listed == 32) {
        listed = e;
        const int own = e + (lane >> 1), j = K.first(own) + 16 * (lane & 1);
        own_page = own < stop && j <= (own < K.sink_steps ? K.sinks - 1 : K.hi) ? A.pages.page_of(s, j) : -1;
        if constexpr (FP8) {  // (a page that is not there has weights of 0: its factor must be finite)
          own_ks = own_page >= 0 ? A.k_scale[static_cast<int64_t>(own_page) * A.G + g] : 0.f;
          own_vs = own_page >= 0 ? A.v_scale[static_cast<int64_t>(own_page) * A.G + g] : 0.f;
        }
      }
      const int at = __builtin_amdgcn_readfirstlane(2 * (e - listed));
      const int p0 = __builtin_amdgcn_readlane(own_page, at), p1 = __builtin_amdgcn_readlane(own_page, at + 1);
      in_flight.key = __builtin_amdgcn_readfirstlane(K.first(e)), in_flight.p0 = p0, in_flight.p1 = p1;
      in_flight.upto = e < K.sink_steps ? K.sinks - 1 : K.hi;
      const int64_t s0 = p0 < 0 ? 0 : p0, s1 = p1 < 0 ? 0 : p1;  // (page 0 exists; its rows are masked)
      const int slot0 = in_flight.key & slot_mask, slot1 = (in_flight.key + 16) & slot_mask;
      const int64_t k0 = (s0 * A.k.stride_page + slot0 * A.k.stride_slot) * ES, k1 = (s1 * A.k.stride_page + slot1 * A.k.stride_slot) * ES;
      const int64_t v0 = (s0 * A.v.stride_page + slot0 * A.v.stride_slot) * ES, v1 = (s1 * A.v.stride_page + slot1 * A.v.stride_slot) * ES;
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        const bool second = half_of(p) != 0;
        const char *k = kbase + scalar(second ? k1 : k0), *v = vbase + scalar(second ? v1 : v0);
        kr[p] = *reinterpret_cast<const uint4*>(k + k_off[p]);
        vr[p] = *reinterpret_cast<const uint4*>(v + v_off[p]);
      }
      in_flight.ks0 = in_flight.ks1 = in_flight.vs0 = in_flight.vs1 = 1.f;
      if constexpr (FP8) {
        auto of = [&](float x, int i) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), i)); };
        in_flight.ks0 = of(own_ks, at), in_flight.ks1 = of(own_ks, at + 1);
        in_flight.vs0 = of(own_vs, at), in_flight.vs1 = of(own_vs, at + 1);
      }
    };
    auto store_step = [&](int b) {
      const bool all = A.D == DP && in_flight.p0 >= 0 && in_flight.p1 >= 0 && in_flight.key + 31 <= in_flight.upto;
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        const int i = piece_of(p), r = i / VL, d = i % VL * VD;
        uint4 k = kr[p], v = vr[p];
        if (!all) {
          const bool there = (half_of(p) ? in_flight.p1 : in_flight.p0) >= 0 && in_flight.key + r <= in_flight.upto;
          if (d >= A.D) k = make_uint4(0u, 0u, 0u, 0u);
          if (d >= A.D || !there) v = make_uint4(0u, 0u, 0u, 0u);  // (unwritten slots hold anything)
        }
        uint4* kt = reinterpret_cast<uint4*>(&kbuf[b][r * RS + d]);
        uint4* vt = reinterpret_cast<uint4*>(&vbuf[b][r * RS + d]);
        if constexpr (FP8) {
          kt[0] = widen_fp8<DT == kF16>(k.x, k.y), kt[1] = widen_fp8<DT == kF16>(k.z, k.w);
          vt[0] = widen_fp8<false>(v.x, v.y), vt[1] = widen_fp8<false>(v.z, v.w);
        } else {
          kt[0] = k, vt[0] = v;
        }
      }
    };

    if (e0 < stop && A.pages.num_pages > 0) {
      load_step(e0);
      store_step(0);
      for (int e = e0, b = 0; e < stop; ++e, b ^= 1) {
        __syncthreads();
        const Step now = in_flight;
        if (e + 1 < stop) load_step(e + 1);
        const bool of_sinks = e < K.sink_steps;
        if (has_rows && (now.p0 >= 0 || now.p1 >= 0) &&
            (of_sinks || (now.key <= last_slot && (now.key > low_least - 32 || now.key < A.seen.sinks)))) {
          const uint16_t *kt = kbuf[b], *vt = vbuf[b];
          f32x4 sc[MT][2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int m = 0; m < MT; ++m) sc[m][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
              const bf16x8 kf = load_frag(kt + (16 * h + c) * RS + 32 * kk + 8 * q4);
#pragma unroll
              for (int m = 0; m < MT; ++m) sc[m][h] = mfma_t<DT>(kf, qf[m][kk], sc[m][h]);
            }
          }
          const bool whole = now.p0 >= 0 && now.p1 >= 0 && now.key + 31 < common && now.key + 31 <= now.upto &&
                             (of_sinks || now.key >= low_most || now.key + 31 < A.seen.sinks);
          Fragment<PT> pf[MT], pl[MT];
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            // raw dots; of an 8-bit page times its scale
            float x[8], high = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = FP8 ? sc[m][j >> 2][j & 3] * (j >> 2 ? now.ks1 : now.ks0) : sc[m][j >> 2][j & 3];
            if (!whole) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const int h = j >> 2, key = now.key + 16 * h + 4 * q4 + (j & 3);
                const bool seen = (h ? now.p1 : now.p0) >= 0 && key <= now.upto &&
                                  row_keys[m].sees(A, P.context, key, [&](int node) { return tree.sees(tok[m] - K.a, node); });
                x[j] = seen ? x[j] : -__builtin_inff();
              }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) high = fmaxf(high, x[j]);
            if (__any(high > top[m] + slack)) {
              const float next = fmaxf(top[m], quarters_max(high));
              const float keep = top[m] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f((top[m] - next) * factor);
              top[m] = next;
              l[m] *= keep;
#pragma unroll
              for (int d = 0; d < ND; ++d) acc[m][d] *= keep;
            }
            const float shift = kUp - (top[m] == -__builtin_inff() ? 0.f : top[m] * factor);  // (all logits -inf: weights 0)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], factor, shift));
              l[m] += x[j];
              if constexpr (FP8) x[j] *= j < 4 ? now.vs0 : now.vs1;
            }
            pf[m] = pack_fragment<PT>(x);
            if constexpr (kTwo) pl[m] = second_terms<PT>(pf[m], x);
          }
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            const Fragment<PT> vf = column_fragment<PT>(vt, RS, 0, 16 * d, c, q4);
#pragma unroll
            for (int m = 0; m < MT; ++m) {
              acc[m][d] = product<PT>(vf, pf[m], acc[m][d]);
              if constexpr (kTwo) acc[m][d] = product<PT>(vf, pl[m], acc[m][d]);
            }
          }
        }
        if (e + 1 < stop) store_step(b ^ 1);
      }
    }

    const bool done = e0 == 0 && e1 == P.steps;
    const int64_t place = static_cast<int64_t>(blockIdx.x) * 2 + (e0 > 0 ? 0 : 1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      top[m] *= factor;
      const int r = 16 * (MT * wave + m) + c, head = g * ratio + r0 + min(r, live - 1) - tok[m] * ratio;
      const bool mine = r < live;
      l[m] += __shfl_xor(l[m], 16, kWave);
      l[m] += __shfl_xor(l[m], 32, kWave);
      const float inv = done ? (l[m] == 0.f ? 0.f : 1.f / l[m]) : 1.f;
      const int64_t out_row = (start + static_cast<int64_t>(tok[m])) * (A.G * ratio) + head;
      float all = 0.f;
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        const f32x4 o = acc[m][d] * inv;
        all += (o[0] + o[1]) + (o[2] + o[3]);
        if (mine && 16 * d + 4 * q4 < A.D) {
          if (done) store4<DT>(A.out + out_row * A.D + 16 * d + 4 * q4, o);
          else *reinterpret_cast<f32x4*>(A.part + (place * R + r) * A.D + 16 * d + 4 * q4) = o;
        }
      }
      if (mine && q4 == 0) {
        if (!done) {
          A.stats[(place * 2) * R + r] = top[m];
          A.stats[(place * 2 + 1) * R + r] = l[m];
        } else if (A.lse) {
          A.lse[out_row] = l[m] == 0.f ? -__builtin_inff() : (top[m] - kUp + __log2f(l[m])) * kLn2Window;
        }
      }
      // (a sum of NaN makes the row NaN)
      uint64_t odd = __ballot(done && mine && !finite(all) && l[m] == l[m]);
      odd |= odd >> 32, odd |= odd >> 16;
      for (uint32_t left = odd & 0xffffu; left; left &= left - 1) {
        const int from = __builtin_ctz(left);
        careful_row<DT, FP8>(A, s, start, P.context, __builtin_amdgcn_readlane(tok[m], from), g,
                             __builtin_amdgcn_readlane(head, from),
                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top[m]), from)) - kUp,
                             __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inv), from)));
      }
    }
    __syncthreads();
  }
}

// The parts of rows that several workgroups share, of many rows: a workgroup sixteen rows of a tile, a wave four of them, their
// maxima and sums sixteen parts at a time, then the outputs with four parts of each row in flight, two dims a lane and pass.
template <int DT, bool FP8, int R>
__global__ __launch_bounds__(256) void window_paged_join_rows(PagedWindowArgs A, int64_t first) {
  constexpr float kUp = !FP8 && DT == kF16 ? 15.f - kSlack : 0.f;
  __shared__ float weights[4][4][kMostParts];
  const int lane = threadIdx.x & 63, ratio = A.ratio.d;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int64_t item = first + blockIdx.x;
  const int row0 = static_cast<int>(item % (R / 16)) * 16 + 4 * wave;
  item /= R / 16;
  const int g = static_cast<int>(item % A.G);
  const TilePlace at = tile_place(A.cu, A.nseq, item / A.G, ratio, log2_of(R));
  const PagedPlan plan = *A.plan;
  const int context = A.context[at.seq], live = min(R, at.n * ratio - at.tile * R);
  if (row0 >= live) return;
  const SeqPlan P = seq_plan<R>(A, at.start, at.start + at.n, context);
  const int64_t begin = A.first_item[at.seq] + (static_cast<int64_t>(g) * P.tiles + at.tile) * P.steps;
  const int64_t w0 = scalar(begin / plan.share);
  const int parts = __builtin_amdgcn_readfirstlane(static_cast<int>((begin + P.steps - 1) / plan.share - w0) + 1);
  if (parts == 1) return;
  auto place_of = [&](int z) { return (w0 + z) * 2 + (z == 0 ? 1 : 0); };

  const int i_own = lane >> 4, r_own = min(row0 + i_own, live - 1);  // the row that this lane weighs parts of
  float top = -__builtin_inff(), sum = 0.f;
  for (int z = lane & 15; z < parts; z += 16) {
    const float high = A.stats[place_of(z) * 2 * R + r_own];
    weights[wave][i_own][z] = high;
    top = fmaxf(top, high);
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, kWave));
  for (int z = lane & 15; z < parts; z += 16) {
    const float high = weights[wave][i_own][z];
    const float w = high == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(high - top);
    weights[wave][i_own][z] = w;
    sum += w * A.stats[(place_of(z) * 2 + 1) * R + r_own];
  }
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, kWave);
  const float inv_own = sum == 0.f ? 0.f : 1.f / sum;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float inv[4], all[4] = {0.f, 0.f, 0.f, 0.f};
  int64_t out_row[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int in_group = at.tile * R + min(row0 + i, live - 1), tok = A.ratio(in_group);
    inv[i] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(inv_own), 16 * i));
    out_row[i] = (at.start + static_cast<int64_t>(tok)) * (A.G * ratio) + g * ratio + in_group - tok * ratio;
  }
  for (int d0 = 0; d0 < A.D; d0 += 128) {
    const int d = min(d0 + 2 * lane, A.D - 2);
    float2 o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = make_float2(0.f, 0.f);
    for (int z0 = 0; z0 < parts; z0 += 4) {
      float2 x[4][4];
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[z][i] = z0 + z < parts ? *reinterpret_cast<const float2*>(
                                         A.part + (place_of(z0 + z) * R + min(row0 + i, live - 1)) * A.D + d)
                                   : make_float2(0.f, 0.f);
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float f = z0 + z < parts ? weights[wave][i][z0 + z] : 0.f;
          o[i].x = fmaf(f, x[z][i].x, o[i].x);
          o[i].y = fmaf(f, x[z][i].y, o[i].y);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i].x *= inv[i], o[i].y *= inv[i];
      all[i] += o[i].x + o[i].y;
      if (row0 + i < live && d0 + 2 * lane < A.D)
        *reinterpret_cast<uint32_t*>(A.out + out_row[i] * A.D + d) = DT == kF16 ? cvt_pk_f16(o[i].x, o[i].y) : cvt_pk_bf16(o[i].x, o[i].y);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float top_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(top), 16 * i));
    const float sum_i = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(sum), 16 * i));
    if (row0 + i >= live) break;
    if (lane == 0 && A.lse) A.lse[out_row[i]] = sum_i == 0.f ? -__builtin_inff() : (top_i - kUp + __log2f(sum_i)) * kLn2Window;
    if (__any(!finite(all[i])) && sum_i == sum_i) {
      const int in_group = at.tile * R + row0 + i, tok = A.ratio(in_group);
      careful_row<DT, FP8>(A, at.seq, at.start, context, tok, g, g * ratio + in_group - tok * ratio, top_i - kUp, inv[i]);
    }
  }
}

// The same of few rows: four waves a row, every fourth part each, eight of them in flight.
template <int DT, bool FP8, int R>
__global__ __launch_bounds__(256) void window_paged_join(PagedWindowArgs A, int64_t first) {
  constexpr float kUp = !FP8 && DT == kF16 ? 15.f - kSlack : 0.f;
  __shared__ float weights[4][kMostParts], sums[4][128];
  const int lane = threadIdx.x & 63, ratio = A.ratio.d;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t out_row = first + blockIdx.x;
  const int heads = A.G * ratio;
  const int64_t t = out_row / heads;
  const int head = static_cast<int>(out_row - t * heads), g = A.ratio(head);
  const PagedPlan plan = *A.plan;
  const int s = A.nseq == 1 ? 0 : wave_upper_index(A.nseq, t, [&](int i) { return static_cast<int64_t>(A.cu[i]); });
  const int start = A.cu[s], context = A.context[s];
  const int64_t first_item = A.first_item[s];
  const SeqPlan P = seq_plan<R>(A, start, A.cu[s + 1], context);
  const int tok = static_cast<int>(t - start), in_group = tok * ratio + head - g * ratio, tile = in_group / R, r = in_group - tile * R;
  const int64_t begin = first_item + (static_cast<int64_t>(g) * P.tiles + tile) * P.steps;
  const int64_t w0 = begin / plan.share;
  const int parts = static_cast<int>((begin + P.steps - 1) / plan.share - w0) + 1;
  if (parts == 1) return;
  auto place_of = [&](int z) { return (w0 + z) * 2 + (z == 0 ? 1 : 0); };
  float* weight = weights[wave];
  // every wave weighs all of the row's (at most kMostParts = 128: two a lane)
  float high[2], sum_z[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int z = lane + 64 * i;
    const int64_t p = place_of(min(z, parts - 1)) * 2 * R + r;
    high[i] = z < parts ? A.stats[p] : -__builtin_inff();
    sum_z[i] = z < parts ? A.stats[p + R] : 0.f;
  }
  const float top = wave_max_f32(fmaxf(high[0], high[1]));
  float w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = high[i] == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(high[i] - top);
    weight[lane + 64 * i] = w[i];
  }
  const float sum = wave_sum_f32(w[0] * sum_z[0] + w[1] * sum_z[1]);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  float all = 0.f;
  for (int d0 = 0; d0 < A.D; d0 += 128) {
    const int d = min(d0 + 2 * lane, A.D - 2);
    float o0 = 0.f, o1 = 0.f;
    for (int z0 = wave; z0 < parts; z0 += 32) {
      float2 x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        x[i] = z0 + 4 * i < parts ? *reinterpret_cast<const float2*>(A.part + (place_of(z0 + 4 * i) * R + r) * A.D + d)
                                      : make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float f = z0 + 4 * i < parts ? weight[z0 + 4 * i] : 0.f;
        o0 = fmaf(f, x[i].x, o0);
        o1 = fmaf(f, x[i].y, o1);
      }
    }
    sums[wave][2 * lane] = o0, sums[wave][2 * lane + 1] = o1;
    __syncthreads();
    o0 = ((sums[0][2 * lane] + sums[1][2 * lane]) + (sums[2][2 * lane] + sums[3][2 * lane]));
    o1 = ((sums[0][2 * lane + 1] + sums[1][2 * lane + 1]) + (sums[2][2 * lane + 1] + sums[3][2 * lane + 1]));
    __syncthreads();
    o0 *= inv, o1 *= inv;
    all += o0 + o1;
    if (wave == 0 && d0 + 2 * lane < A.D)
      *reinterpret_cast<uint32_t*>(A.out + out_row * A.D + d) = DT == kF16 ? cvt_pk_f16(o0, o1) : cvt_pk_bf16(o0, o1);
  }
  if (wave != 0) return;
  if (lane == 0 && A.lse) A.lse[out_row] = sum == 0.f ? -__builtin_inff() : (top - kUp + __log2f(sum)) * kLn2Window;
  if (__any(!finite(all)) && sum == sum)
    careful_row<DT, FP8>(A, s, start, context, tok, g, head, top - kUp, inv);
}

// Rows of a tile: 16, gone through by the waves of a workgroup key by key, where no sequence has more of them a key head;
// otherwise 64, or 128 (of more than 128 dims a wave's registers hold 16). One size for all sequences of a call: a long one among
// single tokens takes those to its own tiles and to weights that are rounded once.
int tile_rows(int64_t longest, int64_t ratio, int64_t dim) { return longest * ratio <= 16 ? 16 : longest * ratio <= 64 || dim > 128 ? 64 : 128; }

// Workgroups of a call at most. 512 run at once; with 16 rows twice as many, whose waves' waits differ, draw more of HBM (64 requests
// of 60 to 30 000 tokens, us as 512 / 768 / 1024: 16 bits 153 / 147 / 143, e4m3 in a window 66 / 67 / 64), with more rows each costs
// its outputs' way to memory and back (a prompt's part 101 / 122 / 110, a tree of 127 nodes 203 / 259 / 226).
int64_t most_workgroups(int rows) { return rows == 16 ? 1024 : 512; }

struct PagedShape {
  int rows;  // of a tile
  int64_t workgroups;
};
// keys: most that a sequence may have (its page table's entries)
PagedShape paged_shape(int64_t tokens, int64_t nseq, int64_t longest, int64_t ratio, int64_t groups, int64_t dim, int64_t keys,
                       int64_t window, int64_t sinks) {
  PagedShape S{tile_rows(longest, ratio, dim), 0};
  const int64_t tiles = (tokens * ratio / S.rows + nseq) * groups;
  int64_t steps = (keys + 31) / 32;
  if (window) {
    const int64_t seen = (window + longest) / 32 + 2 + (sinks + 31) / 32;
    steps = steps < seen ? steps : seen;
  }
  const int64_t most = (tiles * (steps < 1 ? 1 : steps) + 3) / 4;
  S.workgroups = most < most_workgroups(S.rows) ? most : most_workgroups(S.rows);
  return S;
}

}  // namespace
}  // namespace msa

using namespace msa;

extern "C" int64_t msa_window_attn_paged_workspace_bytes(int64_t total_tokens, int64_t num_seqs, int64_t longest,
                                                         int64_t q_heads, int64_t kv_groups, int64_t head_dim,
                                                         int64_t pages_per_seq, int64_t page_size, int64_t window,
                                                         int64_t sinks) {
  if (total_tokens <= 0 || num_seqs <= 0 || longest <= 0 || q_heads <= 0 || kv_groups <= 0 || q_heads % kv_groups ||
      head_dim <= 0 || pages_per_seq < 0 || page_size <= 0 || window < 0 || sinks < 0)
    return 0;
  const PagedShape S = paged_shape(total_tokens, num_seqs, longest, q_heads / kv_groups, kv_groups, head_dim,
                                   pages_per_seq * page_size, window, sinks);
  const int64_t rows = 2 * S.workgroups * S.rows;
  return static_cast<int64_t>(sizeof(PagedPlan)) + 8 * num_seqs + 4 * rows * (head_dim + 2);
}

extern "C" int msa_window_attn_paged(const void* q, const void* k_cache, const void* v_cache, int32_t dtype,
                                     int32_t cache_is_fp8, const float* k_scale, const float* v_scale, const int64_t* strides,
                                     const int32_t* parents, const int32_t* page_table, int64_t table_stride,
                                     int64_t pages_per_seq, int64_t num_pages, int64_t page_size, const int32_t* cu_seqlens,
                                     int64_t num_seqs, int64_t longest, const int32_t* context_lens, int64_t total_tokens,
                                     int64_t q_heads, int64_t kv_groups, int64_t head_dim, int64_t window, int64_t sinks,
                                     double scale, void* workspace, int64_t workspace_bytes, void* out, float* lse,
                                     void* stream) {
  if (!q || !out || !strides || !cu_seqlens || !context_lens || num_seqs <= 0 || num_seqs > 0x3fffffff || total_tokens < 0 ||
      total_tokens > 0x7fffffff || longest < 0 || longest > total_tokens || q_heads <= 0 || kv_groups <= 0 ||
      q_heads % kv_groups || q_heads >= (1 << 20) || head_dim <= 0 || window < 0 || sinks < 0 || !valid_scale(scale) ||
      (dtype != kBF16 && dtype != kF16) || !valid_pages(page_table, table_stride, pages_per_seq, num_pages, page_size) ||
      (num_pages > 0 && (!k_cache || !v_cache || (cache_is_fp8 && (!k_scale || !v_scale)))))
    return kErrInvalidArgument;
  const int unit = cache_is_fp8 ? 16 : 8;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % unit) return kErrInvalidArgument;
  if (reinterpret_cast<uintptr_t>(q) % 16 || reinterpret_cast<uintptr_t>(k_cache) % 16 ||
      reinterpret_cast<uintptr_t>(v_cache) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
    return kErrInvalidArgument;
  const int64_t ratio = q_heads / kv_groups;
  for (int i : {2, 5})  // (16 slots within 32 bits of bytes)
    if (strides[i] < 0 || strides[i] >= (1 << 27)) return kErrUnsupported;
  if (head_dim % 16 || head_dim > 256 || total_tokens * ratio >= 0x7fff0000 || (parents && longest > kTreeNodes))
    return kErrUnsupported;
  if (total_tokens == 0) return kOk;
  if (longest == 0 || !workspace ||
      workspace_bytes < msa_window_attn_paged_workspace_bytes(total_tokens, num_seqs, longest, q_heads, kv_groups, head_dim,
                                                              pages_per_seq, page_size, window, sinks))
    return kErrInvalidArgument;
  const PagedShape S = paged_shape(total_tokens, num_seqs, longest, ratio, kv_groups, head_dim, pages_per_seq * page_size,
                                   window, sinks);
  PagedWindowArgs A{};
  A.q = static_cast<const uint16_t*>(q);
  A.k = CacheView{const_cast<void*>(k_cache), strides[0], strides[1], strides[2]};
  A.v = CacheView{const_cast<void*>(v_cache), strides[3], strides[4], strides[5]};
  A.k_scale = k_scale;
  A.v_scale = v_scale;
  A.pages = page_map(page_table, table_stride, pages_per_seq, num_pages, page_size);
  A.cu = cu_seqlens;
  A.nseq = static_cast<int>(num_seqs);
  A.context = context_lens;
  A.parents = parents;
  A.ratio = divisor_of(ratio);
  A.G = static_cast<int>(kv_groups);
  A.D = static_cast<int>(head_dim);
  A.seen = visible_of(window, sinks);
  A.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  A.out = static_cast<uint16_t*>(out);
  A.lse = lse;
  A.plan = static_cast<PagedPlan*>(workspace);
  A.part = reinterpret_cast<float*>(A.plan + 1);
  A.stats = A.part + 2 * S.workgroups * S.rows * head_dim;
  A.first_item = reinterpret_cast<int64_t*>(A.stats + 4 * S.workgroups * S.rows);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(S.workgroups)), block(256);
  // rows that four waves each add up (480 rows of 16 parts 5.5 us, four rows a wave 9.5), or one wave four (26 000 rows of 2 or 3 16
  // us, a wave each 26)
  const bool few = total_tokens * q_heads <= 2048;
#define MSA_WINDOW_PAGED(KERNEL, JOIN, PARTS)                                                           \
  {                                                                                                     \
    hipLaunchKernelGGL(KERNEL, grid, block, 0, st, A);                                                  \
    const int rc = status_from(hipGetLastError());                                                      \
    if (rc != kOk) return rc;                                                                           \
    return launch_parts(PARTS, [&](int64_t first, unsigned count) {                                     \
      hipLaunchKernelGGL(JOIN, dim3(count), block, 0, st, A, first);                                    \
    });                                                                                                 \
  }
#define MSA_WINDOW_PAGED_ROWS(DT, F8, NK, MT)                                                           \
  {                                                                                                     \
    if (few)                                                                                            \
      MSA_WINDOW_PAGED((window_paged_rows_kernel<DT, F8, NK, MT>), (window_paged_join<DT, F8, 64 * MT>), total_tokens * q_heads) \
    MSA_WINDOW_PAGED((window_paged_rows_kernel<DT, F8, NK, MT>), (window_paged_join_rows<DT, F8, 64 * MT>), \
                     tile_numbers(total_tokens, num_seqs, ratio, log2_of(64 * MT)) * kv_groups * (4 * MT)) \
  }
#define MSA_WINDOW_PAGED_DIM(DT, F8, NK, MT)                                                            \
  {                                                                                                     \
    if (S.rows == 16)                                                                                   \
      MSA_WINDOW_PAGED((window_paged_kernel<DT, F8, NK>), (window_paged_join<DT, F8, 16>), total_tokens * q_heads) \
    if (S.rows == 64) MSA_WINDOW_PAGED_ROWS(DT, F8, NK, 1)                                              \
    MSA_WINDOW_PAGED_ROWS(DT, F8, NK, MT)                                                               \
  }
#define MSA_WINDOW_PAGED_TYPE(DT, F8)                       \
  {                                                         \
    if (head_dim <= 64) MSA_WINDOW_PAGED_DIM(DT, F8, 2, 2)  \
    if (head_dim <= 128) MSA_WINDOW_PAGED_DIM(DT, F8, 4, 2) \
    MSA_WINDOW_PAGED_DIM(DT, F8, 8, 1)                      \
  }
  if (dtype == kBF16) {
    if (cache_is_fp8) MSA_WINDOW_PAGED_TYPE(kBF16, true)
    MSA_WINDOW_PAGED_TYPE(kBF16, false)
  }
  if (cache_is_fp8) MSA_WINDOW_PAGED_TYPE(kF16, true)
  MSA_WINDOW_PAGED_TYPE(kF16, false)
#undef MSA_WINDOW_PAGED_TYPE
#undef MSA_WINDOW_PAGED_DIM
#undef MSA_WINDOW_PAGED_ROWS
#undef MSA_WINDOW_PAGED
}
