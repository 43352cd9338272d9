// What the kernels of bi_paged_sdpa share: which block computes what, the fold of a row's
// partial results over the keys, and the place of partial results that leave a block.
//
// Arithmetic of a row (query token at position p, one head), the same in every kernel
// launch and for every split of the work, which is what makes its bits independent of the
// batch, of how many tokens arrive together and of where its pages lie:
//   * the keys are taken in blocks of B at fixed positions [B b, B b + B), B = 512 on the
//     tensor cores and 128 on the CUDA cores;
//   * a block's partial result (m, l, o) -- running maximum of the scores in units of log 2,
//     sum of 2^(x - m), and sum of 2^(x - m) v -- starts from nothing in every block;
//   * partial results are joined in order of the blocks (fold below), in fp32.
// A block, or a tile inside one, in which the row sees nothing leaves (m, l, o) as they were
// bit for bit, so it does not matter whether a kernel visits it.
#pragma once

#include "common.cuh"
#include "internal.h"

namespace bi {
namespace psdpa {

constexpr int kTcShift = 9, kSimtShift = 7;  // log 2 of the keys of a block on either route
constexpr int kFineRows = 16;  // tiles of at most so many rows are cheap to split (is_few)
constexpr float kLog2e = 1.4426950408889634f;
constexpr unsigned kErrReasonRange = 2;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The two factors that bring the running (big_m) and the next (m) partial result to their
// common maximum, which becomes big_m.  2^0 = 1 exactly, so a partial result that saw
// nothing (m = -inf, l = 0, o = 0) changes no bit.
__device__ __forceinline__ void fold_factors(float& big_m, float m, float& fa, float& fb) {
  const float top = fmaxf(big_m, m);
  fa = big_m == top ? 1.f : exp2_approx(big_m - top);
  fb = m == top ? (m == -INFINITY ? 0.f : 1.f) : exp2_approx(m - top);
  big_m = top;
}
__device__ __forceinline__ float fold_value(float big, float x, float fa, float fb) {
  return __fmaf_rn(x, fb, __fmul_rn(big, fa));
}

// The row's result from its joined (m, l): 1 / (l + sink's share), 0 for a row that sees
// nothing, whatever its sink (of -inf, -inf - -inf would be NaN).  `sink` is the head's extra
// logit in units of log 2.
__device__ __forceinline__ float row_scale(float m, float l, bool has_sink, float sink) {
  if (l == 0.f) return 0.f;
  float f = 1.f;
  if (has_sink) {
    const float top = fmaxf(m, sink);
    f = m == top ? 1.f : exp2_approx(m - top);
    l = __fadd_rn(__fmul_rn(l, f), exp2_approx(sink - top));
  }
  return __fdiv_rn(f, l);
}
// (+ 0.f: a result of -0 becomes +0, whether or not blocks that add nothing were visited)
__device__ __forceinline__ float row_value(float o, float scale) {
  return scale == 0.f ? 0.f : __fmaf_rn(o, scale, 0.f);
}

// Division of numbers below 2^31 by a fixed d in [1, 2^31): n mul >> shift with
// mul = ceil(2^(31 + l) / d), l = ceil(log2 d) (exact: mul d - 2^(31 + l) < d <= 2^l).
struct Divider {
  unsigned d, mul, shift;
  __device__ __forceinline__ int operator()(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<unsigned>(n)) * mul) >> shift);
  }
};
inline Divider divider(int64_t d) {
  unsigned l = 0;
  while ((1ll << l) < d) ++l;
  const uint64_t top = 1ull << (31 + l);
  return {static_cast<unsigned>(d), static_cast<unsigned>((top + d - 1) / d), 31 + l};
}

// What every kernel of the call knows.
struct Params {
  const void* q;
  int64_t qs[2];
  const void* k;
  const void* v;
  int64_t ks[3], vs[3];
  const int* table;
  int64_t table_stride;
  const int* query_start;
  const int* seq_lens;
  const void* sinks;
  void* out;
  int64_t os[2];
  float scale_log2;        // scale / log 2
  int window;              // INT32_MAX: none
  int first;
  int T, R, H, Hkv, G;     // G = H / Hkv
  int n_pages, page;
  int max_seq;             // tokens a row of the block table holds
  int shift;               // log 2 of the keys of a block
  int tile_tok;            // tokens of a tile
  int groups, group_heads; // a KV head's query heads as groups (tiles cover one group)
  Divider by_tile, by_page, by_head, by_group;  // tile_tok, page, group_heads, groups / Hkv
  int target;              // work items to aim for when a request's keys are split
  int fine_rows;           // tiles of at most so many rows are cheap to split ...
  int finer;               // ... so many times finer
  // partial results of split requests
  int4* head;              // {items of many rows, of few rows, whether a request is split, -}
  int4* info;              // per request {pieces, partial results a row has, first slot, -}
  int2* ends;              // per request {items of many rows up to its own, of few rows}
  float2* part_ml;         // (slot,) (m, l)
  float* part_o;           // D columns a slot (see Part)
  unsigned slots;
};

__device__ __forceinline__ int clampi(int64_t v, int64_t lo, int64_t hi) {
  return static_cast<int>(v < lo ? lo : (v > hi ? hi : v));
}

// n / d: by way of fp32 where that is exact after a correction of one, which is several times
// shorter than the integer division.
__device__ __forceinline__ unsigned divide(unsigned n, unsigned d) {
  if ((n | d) >= (1u << 22)) return n / d;
  unsigned q = __float2uint_rz(__fdividef(static_cast<float>(n), static_cast<float>(d)));
  const int rest = static_cast<int>(n - q * d);
  if (rest < 0) --q;
  if (rest >= static_cast<int>(d)) ++q;
  return q;
}

// Piece `piece` of `pieces` of a list of n blocks: [first, first of the next piece).
__device__ __forceinline__ int piece_start(int n, int piece, int pieces) {
  if (pieces == 1) return piece == 0 ? 0 : n;
  const unsigned each = divide(n, pieces);
  return piece * static_cast<int>(each) + min(piece, n - static_cast<int>(each) * pieces);
}

// The key blocks that the queries at positions [pmin, pmax] need: block i of the list is
// i for i < n_first, then first_win + i - n_first.
struct BlockList {
  int n, n_first, first_win;
  int lo_key;  // first key of the window of pmin
  __device__ __forceinline__ int at(int i) const {
    return i < n_first ? i : first_win + i - n_first;
  }
};
__device__ __forceinline__ BlockList block_list(const Params& p, int pmin, int pmax) {
  BlockList b;
  b.n = b.n_first = b.first_win = b.lo_key = 0;
  if (pmax < 0) return b;
  if (p.window != INT32_MAX) b.lo_key = max(0, max(pmin, 0) - p.window + 1);
  const int all = (pmax >> p.shift) + 1;
  b.first_win = b.lo_key >> p.shift;
  const int firsts = (p.first >> p.shift) + ((p.first & ((1 << p.shift) - 1)) != 0);
  b.n_first = min(firsts, b.first_win);
  b.n = b.n_first + all - b.first_win;
  return b;
}

struct Request {
  int tok, n_tok;  // first row and number of its new tokens
  int seq;         // tokens of its sequence, the new ones among them
};
__device__ __forceinline__ Request request(const Params& p, int r) {
  const int start = p.query_start[r], end = p.query_start[r + 1], seq = p.seq_lens[r];
  Request x;
  x.tok = min(max(start, 0), p.T);
  x.n_tok = min(max(end, x.tok), p.T) - x.tok;
  x.seq = min(max(seq, 0), p.max_seq);
  return x;
}
__device__ __forceinline__ int tiles_of(const Params& p, const Request& x) {
  return p.by_tile(x.n_tok + p.tile_tok - 1);
}
// Most key blocks that any of its tiles lists.
__device__ __forceinline__ int blocks_of(const Params& p, const Request& x) {
  const int all = (x.seq + (1 << p.shift) - 1) >> p.shift;
  if (p.window == INT32_MAX) return all;
  const int64_t keys = static_cast<int64_t>(p.window) + min(p.tile_tok, x.n_tok);
  const int64_t most = (p.first >> p.shift) + (keys >> p.shift) + 3;
  return static_cast<int>(most < all ? most : all);
}

// A tile of few rows: cheap to split, as its partial results are small beside the keys that
// they stand for.  Both sides, 64 requests of 3000 to 8191 keys, in a graph: with 32 heads of 128
// over 8, 1 token each (4 rows) 291 us split finely and 295 not, 4 tokens (16 rows) 325 and 302,
// 5 tokens (20 rows) 339 and 302, 16 tokens (64 rows) 429 and 307; with 32 heads over 1, one token
// (32 rows) 57 and 75.  So it is the number of tiles as much as their rows that decides; what 16
// costs is 8 % for four tokens a request and a third for one token of a large group.
__device__ __forceinline__ bool is_few(const Params& p, const Request& x) {
  return min(x.n_tok, p.tile_tok) * p.group_heads <= p.fine_rows;
}
// Partial results that a tile of n blocks in `pieces` pieces leaves: one a block, but a tile of
// many rows joins its first piece's blocks, the first in order, as it goes (their 64 KiB each
// cost as much as the products: 128 tokens behind 30000, 329 -> 294 us).
__device__ __forceinline__ int entries_of(int n, int pieces, bool few) {
  return few || n == 0 ? n : n - piece_start(n, 1, pieces) + 1;
}
// The first one of piece `piece`, whose first block is i0.
__device__ __forceinline__ int first_entry(int n, int piece, int pieces, bool few, int i0) {
  return few || piece == 0 ? i0 : i0 - piece_start(n, 1, pieces) + 1;
}

struct Work {
  int r, tile, group, kvh, piece, pieces;
  int entries;       // most partial results a row of the request has ...
  int base;          // ... and their first slot (pieces > 1)
  Request x;
};

constexpr unsigned kMuch = 1u << 30;  // sums of slots stop here (the workspace holds fewer)
__device__ __forceinline__ unsigned add_sat(unsigned a, unsigned b) { return min(a + b, kMuch); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  return v;
}
// Inclusive scan over a warp's first n lanes (sums above kMuch stay there).
__device__ __forceinline__ unsigned warp_scan(unsigned a, int n = 32) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int d = 1; d < n; d *= 2) {
    const unsigned x = __shfl_up_sync(0xffffffffu, a, d);
    if (lane >= d) a = add_sat(a, x);
  }
  return a;
}

// The items of a call: request by request -- first the requests whose tiles have many rows,
// whose items are the long ones -- in a request group of heads by group, tile by tile from the
// last (in causal attention the longest) to the first, piece by piece of a tile's keys.
//
// A request's keys are split into pieces only where that shortens the call: a tile whose blocks
// are at most the average load (`span`) is computed in one go, which then keeps the fold in
// registers.  Requests whose tiles have few rows (decode), whose partial results are small
// beside the keys they stand for, are split finer where there are many of them, so that ragged
// lengths spread evenly.  The choice changes no bit of the results.
struct Share {      // one request's share of the items
  Request x;
  int tiles, blocks;
  unsigned pieces, slots, items;
  bool few;
};
struct Spans {
  unsigned span, fine;
};
__device__ __forceinline__ float load_of(const Share& s) {
  return static_cast<float>(s.tiles) * static_cast<float>(s.blocks);
}
__device__ __forceinline__ Spans spans_of(const Params& p, float load) {
  load *= static_cast<float>(p.groups);
  const float t = static_cast<float>(p.target);
  return {load <= t ? 1u : static_cast<unsigned>(ceilf(2.f * load / t)),
          static_cast<unsigned>(fmaxf(1.f, ceilf(load / (static_cast<float>(p.finer) * t))))};
}
__device__ __forceinline__ Share share_of(const Params& p, int r) {
  Share s;
  s.x = r < p.R ? request(p, r) : Request{0, 0, 0};
  s.tiles = tiles_of(p, s.x);
  s.blocks = blocks_of(p, s.x);
  s.few = is_few(p, s.x);
  return s;
}
// Pieces and the slots that the partial results of all its rows take.
__device__ __forceinline__ void split_share(const Params& p, const Spans& sp, Share& s) {
  const unsigned most = s.few ? sp.fine : sp.span;
  s.pieces = s.tiles == 0 ? 0 : max(1u, divide(s.blocks + most - 1, most));
  const unsigned rows = min(s.x.n_tok, p.tile_tok) * p.group_heads;  // as in part_of
  const unsigned entries = s.pieces <= 1 ? 0 : entries_of(s.blocks, s.pieces, s.few);
  const float want = static_cast<float>(s.tiles) * static_cast<float>(p.groups) *
                     static_cast<float>(entries) * static_cast<float>(rows);
  s.slots = s.pieces <= 1 ? 0u : want >= static_cast<float>(kMuch) ? kMuch
                                     : static_cast<unsigned>(s.tiles) * p.groups * entries * rows;
}
// With `end` the slots up to its own: a request whose results do not fit is not split.
__device__ __forceinline__ void count_items(const Params& p, unsigned end, Share& s) {
  if (s.pieces > 1 && end > p.slots) s.pieces = 1;
  s.items = s.tiles * s.pieces * p.groups;
}
// Its item number `in`.
__device__ __forceinline__ Work work_of(const Params& p, int r, const Request& x, int tiles,
                                        int blocks, unsigned pieces, unsigned base, unsigned in) {
  const unsigned per_group = tiles * pieces;
  Work w;
  w.r = r;
  w.pieces = pieces;
  w.entries = entries_of(blocks, pieces, is_few(p, x));
  w.base = base;
  w.x = x;
  w.group = divide(in, per_group);
  const unsigned rest = in - w.group * per_group, q = divide(rest, pieces);
  w.tile = tiles - 1 - static_cast<int>(q);
  w.piece = rest - q * pieces;
  w.kvh = p.by_group(w.group);
  return w;
}

// (64, two a lane, took longer: a block's search grew by more than the small kernel takes.)
constexpr int kFewRequests = 32;

// One warp's view of the items.  Up to 32 requests it works them out by itself, a request a
// lane; beyond, schedule_kernel has left them in the workspace.
struct Finder {
  Share s;
  unsigned base = 0, at = 0;  // its first slot of partial results and first item
  unsigned total;

  __device__ __forceinline__ void begin(const Params& p, bool publish) {
    if (p.R > kFewRequests) {
      const int4 h = *p.head;
      total = h.x + h.y;
      return;
    }
    const int lane = threadIdx.x & 31, n = p.R;
    s = share_of(p, lane);
    split_share(p, spans_of(p, warp_sum(load_of(s))), s);
    unsigned end = 0, many = 0, few = 0;
    if (__any_sync(0xffffffffu, s.slots != 0)) end = warp_scan(s.slots, n);
    base = end - s.slots;
    count_items(p, end, s);
    if (__any_sync(0xffffffffu, !s.few && s.items != 0)) {
      many = warp_scan(s.few ? 0 : s.items, n);
      at = many - s.items;
      many = __shfl_sync(0xffffffffu, many, n - 1);
    }
    if (__any_sync(0xffffffffu, s.few && s.items != 0)) {
      few = warp_scan(s.few ? s.items : 0, n);
      if (s.few) at = many + few - s.items;
      few = __shfl_sync(0xffffffffu, few, n - 1);
    }
    total = many + few;
    if (publish) {
      if (lane < n) {
        const int entries = s.pieces > 1 ? entries_of(s.blocks, s.pieces, s.few) : 0;
        p.info[lane] = make_int4(s.pieces, entries, base, 0);
      }
      const unsigned split = __any_sync(0xffffffffu, s.pieces > 1);
      if (lane == 0) *p.head = make_int4(many, few, split, 0);
    }
  }

  // Items i0 < total and i1 < total, by the whole warp: lanes 0..15 get item i0, the others i1.
  __device__ __forceinline__ Work find(const Params& p, unsigned i0, unsigned i1) const {
    const int lane = threadIdx.x & 31;
    const unsigned i = lane < 16 ? i0 : i1;
    if (p.R <= kFewRequests) {
      const unsigned has0 = __ballot_sync(0xffffffffu, i0 - at < s.items);
      const unsigned has1 = __ballot_sync(0xffffffffu, i1 - at < s.items);
      const int r = __ffs(lane < 16 ? has0 : has1) - 1;
      auto pick = [&](unsigned a) { return __shfl_sync(0xffffffffu, a, r); };
      Request x;
      x.tok = pick(s.x.tok);
      x.n_tok = pick(s.x.n_tok);
      x.seq = pick(s.x.seq);
      const int tiles = pick(s.tiles), blocks = pick(s.blocks);
      const unsigned pieces = pick(s.pieces), b = pick(base), first = pick(at);
      return work_of(p, r, x, tiles, blocks, pieces, b, i - first);
    }
    // the first request whose end lies behind the item, 16-way
    const unsigned many = p.head->x;
    const bool few = i >= many;
    const unsigned v = few ? i - many : i;
    const int half = lane & 16, in = lane & 15;
    int lo = 0, n = p.R;  // it is among [lo, lo + n)
    while (__any_sync(0xffffffffu, n > 1)) {
      const int step = (n + 15) / 16;
      const int last = min(lo + (in + 1) * step, lo + n) - 1;  // of this lane's part
      const int2 e = p.ends[last];
      const unsigned behind =
          __ballot_sync(0xffffffffu, static_cast<unsigned>(few ? e.y : e.x) > v) >> half & 0xffffu;
      const int k = __ffs(behind) - 1;  // (there is one: i < total)
      const int start = lo + k * step;
      n = min(step, lo + n - start);
      lo = start;
    }
    const Share x = share_of(p, lo);
    const int4 info = p.info[lo];
    const unsigned items = x.tiles * info.x * p.groups;
    const int2 e = p.ends[lo];
    return work_of(p, lo, x.x, x.tiles, x.blocks, info.x, info.z,
                   v - (static_cast<unsigned>(few ? e.y : e.x) - items));
  }
};

// Where partial result i of a tile is, of which a request keeps `entries` per tile and `rows`
// per entry: first the place of row 0's (m, l) and of its columns.  Columns lie four by
// four, a row's four next to the other rows', so that a warp with a row per lane stores (and the
// join, with a few rows per warp, reads) whole sectors: row by row, 64 KiB took a block 9000
// clocks to leave.
struct Part {
  int64_t first;
  int rows;
};
__device__ __forceinline__ int part_rows(const Params& p, const Request& x) {
  return min(x.n_tok, p.tile_tok) * p.group_heads;
}
__device__ __forceinline__ Part part_of(const Params& p, const Request& x, unsigned base,
                                        int entries, int tile, int group, int i) {
  const int rows = part_rows(p, x);
  return {static_cast<int64_t>(base) +
              (static_cast<int64_t>(tile * p.groups + group) * entries + i) * rows,
          rows};
}
// Column col (a multiple of 4) of `row`.
template <int D>
__device__ __forceinline__ float4* part_at(const Params& p, const Part& a, int row, int col) {
  return reinterpret_cast<float4*>(p.part_o) + a.first * (D / 4) +
         static_cast<int64_t>(col / 4) * a.rows + row;
}

__device__ __forceinline__ void grid_launch_dependents() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
__device__ __forceinline__ void grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace psdpa

// 16-bit tensor-core route (paged_sdpa_tc.cu); tiles of 128 rows.
bool paged_tc_takes(const PagedSdpaArgs& a);
int launch_paged_tc(const PagedSdpaArgs& a, const psdpa::Params& p, int64_t items,
                    cudaStream_t stream);
}  // namespace bi
