// What the kernels of bi_paged_sdpa share: which block computes what, the fold of a row's
// partial results over the keys, and the place of partial results that leave a block.
//
// Arithmetic of a row (query token at position p, one head), the same in every kernel
// launch and for every split of the work, which is what makes its bits independent of the
// batch, of how many tokens arrive together and of where its pages lie:
//   * the keys are taken in blocks of kBlockKeys at fixed positions [512 b, 512 b + 512);
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

constexpr int kBlockKeys = 512;
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
// nothing.  `sink` is the head's extra logit in units of log 2.
__device__ __forceinline__ float row_scale(float m, float l, bool has_sink, float sink) {
  float f = 1.f;
  if (has_sink) {
    const float top = fmaxf(m, sink);
    f = m == top ? 1.f : exp2_approx(m - top);
    l = __fadd_rn(__fmul_rn(l, f), exp2_approx(sink - top));
  }
  return l == 0.f ? 0.f : __fdiv_rn(f, l);
}
// (+ 0.f: a result of -0 becomes +0, whether or not blocks that add nothing were visited)
__device__ __forceinline__ float row_value(float o, float scale) {
  return scale == 0.f ? 0.f : __fmaf_rn(o, scale, 0.f);
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
  int64_t max_seq;         // tokens a row of the block table holds
  int tile_tok;            // tokens of a tile
  int groups, group_heads; // a KV head's query heads as groups (tiles cover one group)
  int target;              // work items to aim for when a request's keys are split
  int fine_rows;           // tiles of at most so many rows are cheap to split
  // partial results of split requests
  int4* info;              // per request {pieces, blocks a row has, base low, base high}
  int* any_split;
  float2* part_ml;         // (slot,) (m, l)
  float* part_o;           // (slot, D)
  int64_t slots;
};

__device__ __forceinline__ int clampi(int64_t v, int64_t lo, int64_t hi) {
  return static_cast<int>(v < lo ? lo : (v > hi ? hi : v));
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
  const int all = pmax / kBlockKeys + 1;
  b.first_win = b.lo_key / kBlockKeys;
  const int firsts = p.first / kBlockKeys + (p.first % kBlockKeys != 0);
  b.n_first = min(firsts, b.first_win);
  b.n = b.n_first + all - b.first_win;
  return b;
}

struct Request {
  int tok, n_tok;  // first row and number of its new tokens
  int seq;         // tokens of its sequence, the new ones among them
};
__device__ __forceinline__ Request request(const Params& p, int r) {
  Request x;
  x.tok = clampi(p.query_start[r], 0, p.T);
  x.n_tok = clampi(p.query_start[r + 1], x.tok, p.T) - x.tok;
  x.seq = clampi(p.seq_lens[r], 0, p.max_seq);
  return x;
}
__device__ __forceinline__ int tiles_of(const Params& p, const Request& x) {
  return (x.n_tok + p.tile_tok - 1) / p.tile_tok;
}
// Most key blocks that any of its tiles lists.
__device__ __forceinline__ int blocks_of(const Params& p, const Request& x) {
  const int all = x.seq / kBlockKeys + (x.seq % kBlockKeys != 0);
  if (p.window == INT32_MAX) return all;
  const int64_t keys = static_cast<int64_t>(p.window) + min(p.tile_tok, x.n_tok);
  const int64_t most = p.first / kBlockKeys + keys / kBlockKeys + 3;
  return static_cast<int>(most < all ? most : all);
}

struct Work {
  int r, tile, group, kvh, piece, pieces;
  int blocks;        // most blocks a row of the request has
  int64_t base;      // first slot of the request's partial results (pieces > 1)
  Request x;
};

template <int NT>
struct SchedSmem {
  int64_t a[NT / 32], b[NT / 32];
  Work found;
  int hit;
};

template <int NT>
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* s) {
#pragma unroll
  for (int d = 16; d > 0; d /= 2) v += __shfl_xor_sync(0xffffffffu, v, d);
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  int64_t t = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) t += s[w];
  __syncthreads();
  return t;
}

// Exclusive scan over the block; `total` receives the sum.
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* s, int64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = v;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  if (lane == 31) s[warp] = inc;
  __syncthreads();
  int64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) before += s[w];
    total += s[w];
  }
  __syncthreads();
  return before + inc - v;
}

// Work item `item` of the call, found by the whole block (NT threads); false: there is none.
// Items go request by request, in a request group of heads by group, tile by tile from the
// last (in causal attention the longest) to the first, piece by piece of the tile's keys.
//
// A request's keys are split into pieces only where that shortens the call: a tile whose
// blocks are at most the average load of a block slot is computed by one block, which then
// keeps the fold in registers.  Requests whose tiles have few rows (decode), whose partial
// results are small beside the keys they stand for, are split four times finer, so that
// ragged lengths spread evenly.  The choice changes no bit of the results.
template <int NT>
__device__ __forceinline__ bool find_work(const Params& p, int64_t item, SchedSmem<NT>& s,
                                          Work& out, bool publish) {
  const int tid = threadIdx.x;
  if (tid == 0) s.hit = 0;
  int64_t load = 0;
  for (int r = tid; r < p.R; r += NT) {
    const Request x = request(p, r);
    load += static_cast<int64_t>(tiles_of(p, x)) * blocks_of(p, x);
  }
  load = block_sum<NT>(load, s.a) * p.groups;
  const int64_t span = max(static_cast<int64_t>(1), (load + p.target - 1) / p.target);
  const int64_t fine = max(static_cast<int64_t>(1), (load + 4 * p.target - 1) / (4 * p.target));
  int64_t items0 = 0, slots0 = 0;
  int split = 0;
  for (int r0 = 0; r0 < p.R; r0 += NT) {
    const int r = r0 + tid;
    Request x{0, 0, 0};
    int64_t items = 0, slots = 0;
    int pieces = 0, blocks = 0, tiles = 0;
    if (r < p.R) {
      x = request(p, r);
      tiles = tiles_of(p, x);
      blocks = blocks_of(p, x);
      const int64_t rows = static_cast<int64_t>(min(x.n_tok, p.tile_tok)) * p.group_heads;
      const int64_t most = rows <= p.fine_rows ? fine : span;
      pieces = tiles > 0 ? static_cast<int>(max(static_cast<int64_t>(1),
                                                (blocks + most - 1) / most)) : 0;
      if (pieces > 1) slots = static_cast<int64_t>(x.n_tok) * p.H * blocks;
    }
    int64_t total;
    const int64_t base = slots0 + block_scan<NT>(slots, s.b, total);
    slots0 += total;
    if (pieces > 1 && base + slots > p.slots) pieces = 1;  // no room for its partial results
    items = static_cast<int64_t>(tiles) * pieces * p.groups;
    const int64_t at = items0 + block_scan<NT>(items, s.a, total);
    items0 += total;
    if (r < p.R && publish) {
      p.info[r] = make_int4(pieces, blocks, static_cast<int>(base & 0xffffffff),
                            static_cast<int>(base >> 32));
      split |= pieces > 1;
    }
    if (item >= at && item < at + items) {
      const int64_t in = item - at;
      Work w;
      w.r = r;
      w.pieces = pieces;
      w.blocks = blocks;
      w.base = base;
      w.x = x;
      const int per_group = tiles * pieces;
      w.group = static_cast<int>(in / per_group);
      const int rest = static_cast<int>(in - static_cast<int64_t>(w.group) * per_group);
      w.tile = tiles - 1 - rest / pieces;
      w.piece = rest % pieces;
      w.kvh = w.group / (p.groups / p.Hkv);
      s.found = w;
      s.hit = 1;
    }
    if (!publish && items0 > item) break;  // (uniform)
  }
  if (publish) {
    split = __syncthreads_or(split);
    if (tid == 0) *p.any_split = split;
  }
  __syncthreads();
  out = s.found;
  return s.hit != 0;
}

// Slot of the partial result of (row, block i of its tile's list).
__device__ __forceinline__ int64_t part_slot(const Params& p, int64_t base, int blocks,
                                             int tok_in_request, int head, int i) {
  return base + (static_cast<int64_t>(tok_in_request) * p.H + head) * blocks + i;
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
