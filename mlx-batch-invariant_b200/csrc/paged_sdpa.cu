// Attention of new tokens over a KV cache in pages (bi_paged_sdpa): the CUDA-core route, the
// join of partial results and the host side.  The tensor-core route is paged_sdpa_tc.cu.
#include <algorithm>
#include <limits>

#include "paged_sdpa.cuh"

namespace bi {
namespace psdpa {

// ---------------------------------------------------------------------------
// CUDA-core route: any head dim that is a multiple of 32 up to 256, any page size, fp32 too.
// A block takes a tile of up to 16 rows (tokens x heads of a group), four to each warp.  Its
// 128 threads bring 32 keys' K and V rows into shared memory as fp32 (while the 32 before them
// are worked on, where two fit); then per warp a lane takes a key and computes the scores of
// the warp's four rows (K rows 16 bytes apart modulo the banks: no conflicts), (m, l) move by
// warp reductions, and for P V a lane takes every 32nd column.  Keys that a row does not see
// are skipped, so what they hold never reaches it.  Bound by the fp32 FMA pipe for chunks (5
// shared-memory reads per 16 multiply-adds), by the loads' latency for single tokens: 101 fp32
// tokens of 5 requests over up to 950 keys, 8 heads of 64 over 2, take 20 us.
// ---------------------------------------------------------------------------
constexpr int kSimtWarps = 4;
constexpr int kSimtThreads = 32 * kSimtWarps;
constexpr int kSimtRows = 4;  // per warp
constexpr int kSimtTile = kSimtWarps * kSimtRows;
constexpr int kSimtKeys = 32;  // of a step
// Its partial results are one a key block, as those of tiles of few rows are (entries_of).
static_assert(kSimtTile <= kFineRows, "a CUDA-core tile counts as one of few rows");

template <int DC>
struct SimtCfg {
  static constexpr int D = 32 * DC;
  static constexpr int kKRow = D + 4;  // floats
  static constexpr int kBuf = kSimtKeys * (kKRow + D);
  static constexpr int kBufs = DC <= 4 ? 2 : 1;
  static constexpr int kSmem = 4 * (kBufs * kBuf + kSimtTile * D + kSimtTile * kSimtKeys);
};

template <typename T>
struct alignas(16) Vec16 {
  T v[16 / sizeof(T)];
};

template <typename T, int DC>  // head dim 32 * DC
__global__ void __launch_bounds__(kSimtThreads) paged_simt_kernel(const Params p) {
  using C = SimtCfg<DC>;
  constexpr int D = C::D;
  constexpr int VEC = 16 / sizeof(T);
  constexpr int kVecs = D / VEC;                               // of a row
  constexpr int kLoads = kSimtKeys * kVecs / kSimtThreads;     // of a thread, K and V each
  static_assert(kLoads * kSimtThreads == kSimtKeys * kVecs, "whole rows per thread");
  extern __shared__ float s_mem[];
  __shared__ Work s_work;
  __shared__ int s_there;
  float* s_kv = s_mem;
  float* s_q = s_mem + C::kBufs * C::kBuf;  // [row][D]
  float* s_p = s_q + kSimtTile * D;         // [row][key]
  grid_wait();
  grid_launch_dependents();
  if (threadIdx.x < 32) {
    Finder finder;
    finder.begin(p, blockIdx.x == 0);
    const bool there = blockIdx.x < finder.total;
    if (there) {
      const Work w = finder.find(p, blockIdx.x, blockIdx.x);
      if (threadIdx.x == 0) s_work = w;
    }
    if (threadIdx.x == 0) s_there = there;
  }
  __syncthreads();
  if (!s_there) return;
  const Work w = s_work;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int subs = p.groups / p.Hkv;  // groups of a KV head
  const int head0 = w.kvh * p.G + (w.group - w.kvh * subs) * p.group_heads;
  const int heads = min(p.group_heads, (w.kvh + 1) * p.G - head0);
  const int tok0 = w.tile * p.tile_tok;  // in the request
  const int n_tok = min(p.tile_tok, w.x.n_tok - tok0);
  const int rows = n_tok * heads;
  const int pos0 = w.x.seq - w.x.n_tok + tok0, pmax = pos0 + n_tok - 1;
  const BlockList list = block_list(p, pos0, pmax);
  const int i0 = piece_start(list.n, w.piece, w.pieces);
  const int i1 = piece_start(list.n, w.piece + 1, w.pieces);
  if (w.pieces > 1 && i0 == i1) return;

  const T* kbase = static_cast<const T*>(p.k) + w.kvh * p.ks[1];
  const T* vbase = static_cast<const T*>(p.v) + w.kvh * p.vs[1];
  const int* entries = p.table + static_cast<int64_t>(w.r) * p.table_stride;
  const int block_keys = 1 << p.shift;
  // steps of 32 keys: the next one that some row of the tile needs, or -1
  int it_i = i0, it_t = 0;
  auto next_step = [&]() {
    for (; it_i < i1; ++it_i, it_t = 0) {
      const int key0 = list.at(it_i) << p.shift;
      for (; it_t < block_keys; it_t += kSimtKeys) {
        const int t = key0 + it_t;
        if (t > pmax) break;
        if (t + kSimtKeys <= list.lo_key && t >= p.first) continue;
        it_t += kSimtKeys;
        return t;
      }
    }
    return -1;
  };
  // This thread's vectors of a step's K and V rows: zeros for keys past the tile's last and for
  // pages outside the cache.
  Vec16<T> kreg[kLoads], vreg[kLoads];
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int x = tid + i * kSimtThreads, r = x / kVecs, c = x - r * kVecs;
      const int key = t + r;
      int pg = -1, col = 0;
      if (key <= pmax) {
        col = p.by_page(key);
        pg = entries[col];
      }
      if (pg >= 0 && pg < p.n_pages) {
        const int64_t off = key - col * p.page;
        kreg[i] = *reinterpret_cast<const Vec16<T>*>(kbase + pg * p.ks[0] + off * p.ks[2] +
                                                     c * VEC);
        vreg[i] = *reinterpret_cast<const Vec16<T>*>(vbase + pg * p.vs[0] + off * p.vs[2] +
                                                     c * VEC);
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) kreg[i].v[e] = vreg[i].v[e] = from_f32<T>(0.f);
      }
    }
  };
  auto put = [&](float* buf) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int x = tid + i * kSimtThreads, r = x / kVecs, c = x - r * kVecs;
      float* kd = buf + r * C::kKRow + c * VEC;
      float* vd = buf + kSimtKeys * C::kKRow + r * D + c * VEC;
#pragma unroll
      for (int e = 0; e < VEC; e += 4) {
        *reinterpret_cast<float4*>(kd + e) =
            make_float4(to_f32(kreg[i].v[e]), to_f32(kreg[i].v[e + 1]),
                        to_f32(kreg[i].v[e + 2]), to_f32(kreg[i].v[e + 3]));
        *reinterpret_cast<float4*>(vd + e) =
            make_float4(to_f32(vreg[i].v[e]), to_f32(vreg[i].v[e + 1]),
                        to_f32(vreg[i].v[e + 2]), to_f32(vreg[i].v[e + 3]));
      }
    }
  };

  int t = next_step();
  if (t >= 0) fetch(t);
  for (int i = tid; i < kSimtTile * D; i += kSimtThreads) {
    const int r = i / D, e = i - r * D;
    float x = 0.f;
    if (r < rows) {
      const int tk = p.by_head(r);  // (of a partial group the rows are fewer: see below)
      const int tok_r = heads == p.group_heads ? tk : r / heads;
      x = to_f32(static_cast<const T*>(p.q)[static_cast<int64_t>(w.x.tok + tok0 + tok_r) * p.qs[0] +
                                            (head0 + r - tok_r * heads) * p.qs[1] + e]);
    }
    s_q[i] = x;
  }

  int pos[kSimtRows];
  float tot_m[kSimtRows], tot_l[kSimtRows], tot_o[kSimtRows][DC];
  float m[kSimtRows], l[kSimtRows], o[kSimtRows][DC];
  auto clear = [&]() {
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) o[r][c] = 0.f;
    }
  };
  clear();
#pragma unroll
  for (int r = 0; r < kSimtRows; ++r) {
    const int row = warp * kSimtRows + r;
    // a row that is not there (or whose position is negative) sees nothing
    pos[r] = row < rows ? max(-1, pos0 + row / heads) : -1;
    tot_m[r] = m[r];
    tot_l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) tot_o[r][c] = 0.f;
  }
  const bool busy = warp * kSimtRows < rows;
  // The block of the list that `done` is (m, l, o) are complete.
  auto close_block = [&](int done) {
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      const int row = warp * kSimtRows + r;
      if (w.pieces > 1) {
        if (row < rows) {
          const Part at = part_of(p, w.x, w.base, w.entries, w.tile, w.group, done);
          if (lane == 0) p.part_ml[at.first + row] = make_float2(m[r], l[r]);
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const int col = c * 32 + lane;
            reinterpret_cast<float*>(part_at<D>(p, at, row, col & ~3))[col & 3] = o[r][c];
          }
        }
      } else {
        float fa, fb;
        fold_factors(tot_m[r], m[r], fa, fb);
        tot_l[r] = fold_value(tot_l[r], l[r], fa, fb);
#pragma unroll
        for (int c = 0; c < DC; ++c) tot_o[r][c] = fold_value(tot_o[r][c], o[r][c], fa, fb);
      }
    }
    clear();
  };

  int block = i0;  // being worked on
  for (int n = 0; t >= 0; ++n) {
    float* buf = s_kv + (n % C::kBufs) * C::kBuf;
    if (C::kBufs == 1) __syncthreads();
    put(buf);
    __syncthreads();
    const int now = t;
    t = next_step();
    if (t >= 0) fetch(t);
    if (!busy) continue;
    while ((list.at(block) << p.shift) + block_keys <= now) close_block(block++);
    const int key = now + lane;
    unsigned seen[kSimtRows], any = 0;
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      const bool see = key <= pos[r] && (key > pos[r] - p.window || key < p.first);
      seen[r] = __ballot_sync(0xffffffffu, see);
      any |= seen[r];
    }
    if (any == 0) continue;
    const float* krow = buf + lane * C::kKRow;
    const float* qrow = s_q + warp * kSimtRows * D;
    float s[kSimtRows] = {};
#pragma unroll 8
    for (int e = 0; e < D; e += 4) {
      const float4 kv = *reinterpret_cast<const float4*>(krow + e);
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) {
        const float4 qv = *reinterpret_cast<const float4*>(qrow + r * D + e);
        s[r] = __fmaf_rn(qv.x, kv.x, s[r]);
        s[r] = __fmaf_rn(qv.y, kv.y, s[r]);
        s[r] = __fmaf_rn(qv.z, kv.z, s[r]);
        s[r] = __fmaf_rn(qv.w, kv.w, s[r]);
      }
    }
    float* prow = s_p + warp * kSimtRows * kSimtKeys;
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      const bool see = (seen[r] >> lane) & 1u;
      const float x = see ? __fmul_rn(s[r], p.scale_log2) : -INFINITY;
      float top = x;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
      const float nm = fmaxf(m[r], top);
      const float base = nm == -INFINITY ? 0.f : nm;
      const float f = m[r] == nm ? 1.f : exp2_approx(m[r] - nm);
      const float pr = see ? exp2_approx(x - base) : 0.f;
      float sum = pr;
#pragma unroll
      for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
      m[r] = nm;
      l[r] = __fmaf_rn(l[r], f, sum);
#pragma unroll
      for (int c = 0; c < DC; ++c) o[r][c] = __fmul_rn(o[r][c], f);
      prow[r * kSimtKeys + lane] = pr;
    }
    __syncwarp();
    const float* vbuf = buf + kSimtKeys * C::kKRow + lane;
    bool every = true;  // rows that are not there have weights of 0 and are not stored
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      every = every && (seen[r] == 0xffffffffu || warp * kSimtRows + r >= rows);
    }
    if (every) {
#pragma unroll 2
      for (int j = 0; j < kSimtKeys; j += 4) {
        float4 pv[kSimtRows];
#pragma unroll
        for (int r = 0; r < kSimtRows; ++r) {
          pv[r] = *reinterpret_cast<const float4*>(prow + r * kSimtKeys + j);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int c = 0; c < DC; ++c) {
            const float v = vbuf[(j + i) * D + c * 32];
#pragma unroll
            for (int r = 0; r < kSimtRows; ++r) {
              const float pj = i == 0 ? pv[r].x : i == 1 ? pv[r].y : i == 2 ? pv[r].z : pv[r].w;
              o[r][c] = __fmaf_rn(pj, v, o[r][c]);
            }
          }
        }
      }
    } else {
#pragma unroll 1
      for (unsigned left = any; left != 0; left &= left - 1) {
        const int j = __ffs(left) - 1;
#pragma unroll
        for (int r = 0; r < kSimtRows; ++r) {
          if ((seen[r] >> j) & 1u) {
            const float pj = prow[r * kSimtKeys + j];
#pragma unroll
            for (int c = 0; c < DC; ++c) {
              o[r][c] = __fmaf_rn(pj, vbuf[j * D + c * 32], o[r][c]);
            }
          }
        }
      }
    }
    __syncwarp();
  }
  if (!busy) return;
  while (block < i1) close_block(block++);
  if (w.pieces > 1) return;
#pragma unroll
  for (int r = 0; r < kSimtRows; ++r) {
    const int row = warp * kSimtRows + r;
    if (row >= rows) continue;
    const int head = head0 + row % heads;
    const int64_t tok = w.x.tok + tok0 + row / heads;
    const float sink = p.sinks ? to_f32(static_cast<const T*>(p.sinks)[head]) * kLog2e : 0.f;
    const float sc = row_scale(tot_m[r], tot_l[r], p.sinks != nullptr, sink);
    T* dst = static_cast<T*>(p.out) + tok * p.os[0] + head * p.os[1];
#pragma unroll
    for (int c = 0; c < DC; ++c) dst[c * 32 + lane] = from_f32<T>(row_value(tot_o[r][c], sc));
  }
}

// ---------------------------------------------------------------------------
// The items of calls with more requests than a warp keeps in registers: one block, ahead of the
// main kernel, leaves every request's split and the running numbers of items.  (A list of the
// items themselves would save a block another 2 us of search, and take about as long to write.)
// ---------------------------------------------------------------------------
constexpr int kScheduleThreads = 1024;

__global__ void __launch_bounds__(kScheduleThreads) schedule_kernel(const Params p) {
  constexpr int kWarps = kScheduleThreads / 32;
  __shared__ float s_load[kWarps];
  __shared__ unsigned s_slots[kWarps], s_many[kWarps], s_few[kWarps];
  grid_wait();
  grid_launch_dependents();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float load = 0.f;
  for (int r = tid; r < p.R; r += kScheduleThreads) load += load_of(share_of(p, r));
  load = warp_sum(load);
  if (lane == 0) s_load[warp] = load;
  __syncthreads();
  const Spans sp = spans_of(p, warp_sum(s_load[lane]));
  unsigned slots0 = 0, many0 = 0, few0 = 0;
  int split = 0;
  for (int r0 = 0; r0 < p.R; r0 += kScheduleThreads) {
    const int r = r0 + tid;
    Share s = share_of(p, r);
    split_share(p, sp, s);
    const unsigned in_warp = warp_scan(s.slots);
    if (lane == 31) s_slots[warp] = in_warp;
    __syncthreads();
    const unsigned slots = warp_scan(s_slots[lane]);  // up to warp `lane`'s end
    unsigned before = __shfl_sync(0xffffffffu, slots, max(warp - 1, 0));
    const unsigned end = add_sat(add_sat(slots0, warp > 0 ? before : 0u), in_warp);
    slots0 = add_sat(slots0, __shfl_sync(0xffffffffu, slots, 31));
    count_items(p, end, s);
    const unsigned m_in = warp_scan(s.few ? 0 : s.items), f_in = warp_scan(s.few ? s.items : 0);
    if (lane == 31) {
      s_many[warp] = m_in;
      s_few[warp] = f_in;
    }
    __syncthreads();
    const unsigned m = warp_scan(s_many[lane]), f = warp_scan(s_few[lane]);
    before = __shfl_sync(0xffffffffu, m, max(warp - 1, 0));
    const unsigned m_end = many0 + (warp > 0 ? before : 0u) + m_in;
    before = __shfl_sync(0xffffffffu, f, max(warp - 1, 0));
    const unsigned f_end = few0 + (warp > 0 ? before : 0u) + f_in;
    many0 += __shfl_sync(0xffffffffu, m, 31);
    few0 += __shfl_sync(0xffffffffu, f, 31);
    if (r < p.R) {
      const int entries = s.pieces > 1 ? entries_of(s.blocks, s.pieces, s.few) : 0;
      p.info[r] = make_int4(s.pieces, entries, end - s.slots, 0);
      p.ends[r] = make_int2(m_end, f_end);
    }
    split |= s.pieces > 1;
    __syncthreads();
  }
  split = __syncthreads_or(split);
  if (tid == 0) *p.head = make_int4(many0, few0, split, 0);
}

// ---------------------------------------------------------------------------
// Join of the partial results of split requests: a warp takes 64 columns of two neighbouring
// heads of a token (half of its lanes each, four columns a lane) and folds their blocks' partial
// results in order, with the operations of the unsplit kernels; 16 blocks' are in flight at a
// time.  (A warp with all 128 columns had room for 8, and took 3 us longer where a token has 16
// blocks.)  Launched behind every call (the split is decided on the device); where nothing was
// split it reads one word.  Its launch overlaps the main kernel's tail.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 128;

template <typename T, int DC>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
  constexpr int D = 32 * DC;
  constexpr int kParts = (D + 63) / 64;  // of a row's columns
  constexpr int kAhead = 16;             // partial results in flight
  grid_wait();
  const int lane = threadIdx.x & 31;
  // Up to 32 requests: each lane has one, so that what follows waits for memory once.
  const bool small = p.R <= 32;
  const int4 notes = *p.head;
  const Request mine = small && lane < p.R ? request(p, lane) : Request{0, 0, 0};
  const int4 my_info = small && lane < p.R ? p.info[lane] : make_int4(0, 0, 0, 0);
  if (notes.z == 0) return;
  const int h_pairs = (p.H + 1) / 2;
  const int64_t n_pairs = static_cast<int64_t>(p.T) * h_pairs * kParts;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32);
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / 32) + (threadIdx.x >> 5);
       at < n_pairs; at += warps) {
    const int64_t pair = at / kParts;
    const int col = 64 * static_cast<int>(at - pair * kParts) + 4 * (lane >> 1);
    const int tok = static_cast<int>(pair / h_pairs);
    const int head = static_cast<int>(pair - static_cast<int64_t>(tok) * h_pairs) * 2 + (lane & 1);
    Request x;
    int4 info;
    if (small) {
      const unsigned has = __ballot_sync(0xffffffffu, tok >= mine.tok && tok < mine.tok + mine.n_tok);
      const int r = has != 0 ? __ffs(has) - 1 : 0;
      x.tok = __shfl_sync(0xffffffffu, mine.tok, r);
      x.n_tok = __shfl_sync(0xffffffffu, mine.n_tok, r);
      x.seq = __shfl_sync(0xffffffffu, mine.seq, r);
      info.x = __shfl_sync(0xffffffffu, my_info.x, r);
      info.y = __shfl_sync(0xffffffffu, my_info.y, r);
      info.z = __shfl_sync(0xffffffffu, my_info.z, r);
    } else {
      // its request: the last one that starts at or before it (32-way search)
      int lo = 0, hi = p.R;  // answer + 1 is in (lo, hi]
      while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32;
        const int i = lo + lane * step;
        const bool le = i < hi && clampi(p.query_start[i], 0, p.T) <= tok;
        const unsigned bal = __ballot_sync(0xffffffffu, le);
        if (bal == 0) break;
        const int k = 31 - __clz(bal);
        lo = lo + k * step;
        hi = min(hi, lo + step);
      }
      x = request(p, lo);
      info = p.info[lo];
    }
    if (tok < x.tok || tok >= x.tok + x.n_tok || info.x <= 1) continue;
    if (head >= p.H || col >= D) continue;
    const int in = tok - x.tok, tile = p.by_tile(in), first = tile * p.tile_tok;
    const int pos0 = x.seq - x.n_tok + first;
    const int n_tok = min(p.tile_tok, x.n_tok - first);
    const BlockList list = block_list(p, pos0, pos0 + n_tok - 1);
    // its group of heads and its row in the tile, whose rows are tokens x the group's heads
    const int kvh = head / p.G, in_kv = head - kvh * p.G, sub = in_kv / p.group_heads;
    const int group = kvh * (p.groups / p.Hkv) + sub;
    const int heads = min(p.group_heads, p.G - sub * p.group_heads);
    const int row = (in - first) * heads + in_kv - sub * p.group_heads;
    const Part part = part_of(p, x, info.z, info.y, tile, group, 0);
    const int entries = entries_of(list.n, info.x, is_few(p, x));
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i = 0; i < entries; i += kAhead) {
      float2 ml[kAhead];
      float4 po[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool there = i + j < entries;
        const Part b = {part.first + static_cast<int64_t>(i + j) * part.rows, part.rows};
        ml[j] = there ? p.part_ml[b.first + row] : make_float2(-INFINITY, 0.f);
        po[j] = there ? *part_at<D>(p, b, row, col) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float fa, fb;
        fold_factors(m, ml[j].x, fa, fb);
        l = fold_value(l, ml[j].y, fa, fb);
        o.x = fold_value(o.x, po[j].x, fa, fb);
        o.y = fold_value(o.y, po[j].y, fa, fb);
        o.z = fold_value(o.z, po[j].z, fa, fb);
        o.w = fold_value(o.w, po[j].w, fa, fb);
      }
    }
    const float sink = p.sinks ? to_f32(static_cast<const T*>(p.sinks)[head]) * kLog2e : 0.f;
    const float sc = row_scale(m, l, p.sinks != nullptr, sink);
    struct alignas(4 * sizeof(T)) Quad {
      T v[4];
    } q;
    q.v[0] = from_f32<T>(row_value(o.x, sc));
    q.v[1] = from_f32<T>(row_value(o.y, sc));
    q.v[2] = from_f32<T>(row_value(o.z, sc));
    q.v[3] = from_f32<T>(row_value(o.w, sc));
    *reinterpret_cast<Quad*>(static_cast<T*>(p.out) + tok * p.os[0] + head * p.os[1] + col) = q;
  }
}

// A launch that may start before the kernel ahead of it in the stream has ended; every
// kernel here waits for that (grid_wait) before it touches memory.
template <typename... Args>
static cudaError_t launch_early(void (*kernel)(Args...), unsigned grid, unsigned block,
                                size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <typename T, int DC>
static int launch_simt(const Params& p, int64_t items, cudaStream_t stream) {
  constexpr int smem = SimtCfg<DC>::kSmem;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        paged_simt_kernel<T, DC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(paged_sdpa)");
  }
  return cuda_status(launch_early(paged_simt_kernel<T, DC>, static_cast<unsigned>(items),
                                  kSimtThreads, smem, stream, p), "paged_sdpa launch");
}
template <typename T, int DC>
static int launch_join(const Params& p, cudaStream_t stream) {
  const int64_t pairs = static_cast<int64_t>(p.T) * ((p.H + 1) / 2) * ((DC + 1) / 2);
  const int64_t want = (pairs + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(want, 8LL * device_sm_count()));
  return cuda_status(launch_early(join_kernel<T, DC>, grid, kJoinThreads, 0, stream, p),
                     "paged_sdpa join launch");
}

template <typename T>
static int dispatch(const Params& p, int64_t D, int64_t items, bool join, cudaStream_t stream) {
  switch (D / 32) {
#define BI_CASE(n) \
  case n: return join ? launch_join<T, n>(p, stream) : launch_simt<T, n>(p, items, stream);
    BI_CASE(1) BI_CASE(2) BI_CASE(3) BI_CASE(4) BI_CASE(5) BI_CASE(6) BI_CASE(7) BI_CASE(8)
#undef BI_CASE
  }
  return set_error(BI_ERR_UNSUPPORTED, "head dim %lld is not built", static_cast<long long>(D));
}

static int dispatch(const Params& p, int dtype, int64_t D, int64_t items, bool join,
                    cudaStream_t stream) {
  if (dtype == BI_BF16) return dispatch<__nv_bfloat16>(p, D, items, join, stream);
  if (dtype == BI_F16) return dispatch<__half>(p, D, items, join, stream);
  return dispatch<float>(p, D, items, join, stream);
}

constexpr int64_t kMaxPartBytes = 256LL << 20;

static int64_t info_bytes(int64_t R) { return (16 + 24 * R + 255) / 256 * 256; }

}  // namespace psdpa

// Room for the partial results of every row, at most 256 MiB (requests that do not fit are
// not split), and the per-request notes.
int64_t paged_sdpa_workspace(int64_t T, int64_t R, int64_t H, int64_t D, int64_t width,
                             int64_t page) {
  const double blocks = static_cast<double>(width) * static_cast<double>(page) /
                            (1 << psdpa::kSimtShift) + 1.0;
  const double want = static_cast<double>(T) * static_cast<double>(H) * blocks *
                      static_cast<double>(4 * D + 8);
  const int64_t part = want < static_cast<double>(psdpa::kMaxPartBytes)
                           ? static_cast<int64_t>(want) + 256 : psdpa::kMaxPartBytes;
  return psdpa::info_bytes(R) + part;
}

namespace psdpa {
// How the heads and tokens of a call make tiles of `rows` rows.
struct Tiling {
  int64_t group_heads, subs, tile_tok;  // heads of a group, groups of a KV head, tokens of a tile
  int64_t tiles;                        // of all requests: at most one ragged tile each
  explicit Tiling(const PagedSdpaArgs& a) {
    const int64_t rows = paged_tc_takes(a) ? 128 : kSimtTile, G = a.H / a.Hkv;
    group_heads = std::min(G, rows);
    subs = (G + rows - 1) / rows;
    tile_tok = rows / group_heads;
    tiles = a.T / tile_tok + std::min(a.R, a.T);
  }
};
}  // namespace psdpa

bool paged_sdpa_fits(const PagedSdpaArgs& a) {
  const psdpa::Tiling t(a);
  // items are counted in 32 bits that stop at kMuch; the splits of the keys add less than 2^16
  const int64_t most = static_cast<int64_t>(psdpa::kMuch) - (1 << 16);
  return a.R <= most && t.tiles <= most / (a.Hkv * t.subs);
}

int launch_paged_sdpa(const PagedSdpaArgs& a, cudaStream_t stream) {
  using namespace psdpa;
  const bool tc = paged_tc_takes(a);
  const Tiling tiling(a);
  Params p;
  p.q = a.q;
  p.k = a.k;
  p.v = a.v;
  for (int i = 0; i < 2; ++i) {
    p.qs[i] = a.qs[i];
    p.os[i] = a.os[i];
  }
  for (int i = 0; i < 3; ++i) {
    p.ks[i] = a.ks[i];
    p.vs[i] = a.vs[i];
  }
  p.table = a.table;
  p.table_stride = a.table_stride;
  p.query_start = a.query_start;
  p.seq_lens = a.seq_lens;
  p.sinks = a.sinks;
  p.out = a.out;
  // (never 0: the score of a masked key is -inf, and -inf x 0 would be NaN)
  p.scale_log2 = std::max(a.scale * kLog2e, std::numeric_limits<float>::min());
  p.window = a.window <= 0 || a.window >= INT32_MAX ? INT32_MAX : static_cast<int>(a.window);
  p.first = static_cast<int>(std::min<int64_t>(a.first, INT32_MAX));
  if (p.window == INT32_MAX) p.first = 0;
  p.T = static_cast<int>(a.T);
  p.R = static_cast<int>(a.R);
  p.H = static_cast<int>(a.H);
  p.Hkv = static_cast<int>(a.Hkv);
  p.G = p.H / p.Hkv;
  p.n_pages = static_cast<int>(a.n_pages);
  p.page = static_cast<int>(a.page);
  p.shift = tc ? kTcShift : kSimtShift;
  p.max_seq = static_cast<int>(
      std::min<int64_t>(a.width * a.page, INT32_MAX - (1 << kTcShift)));
  p.group_heads = static_cast<int>(tiling.group_heads);
  p.tile_tok = static_cast<int>(tiling.tile_tok);
  p.groups = static_cast<int>(a.Hkv * tiling.subs);
  p.by_tile = divider(p.tile_tok);
  p.by_page = divider(a.page);
  p.by_head = divider(p.group_heads);
  p.by_group = divider(tiling.subs);
  p.target = 2 * device_sm_count();
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.head = reinterpret_cast<int4*>(ws);
  p.info = reinterpret_cast<int4*>(ws + 16);
  p.ends = reinterpret_cast<int2*>(ws + 16 + 16 * a.R);
  const int64_t left = a.workspace_bytes - info_bytes(a.R);
  p.slots = left <= 256 ? 0u : static_cast<unsigned>(
      std::min<int64_t>((left - 256) / (4 * a.D + 8), kMuch - 1));
  p.part_o = reinterpret_cast<float*>(ws + info_bytes(a.R));
  p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<int64_t>(p.slots) * a.D);

  const int64_t tiles = tiling.tiles;
  p.fine_rows = kFineRows;
  // few tiles: one piece for every place is enough; many: finer, to even out ragged lengths
  p.finer = tiles * p.groups >= p.target ? 4 : 1;
  // (the spans are rounded in fp32: a little above finer x target pieces)
  const int64_t items = tiles * p.groups + static_cast<int64_t>(p.finer) * p.target + 64;
  if (a.R > kFewRequests) {
    const int st = cuda_status(launch_early(schedule_kernel, 1u, kScheduleThreads, 0, stream, p),
                               "paged_sdpa schedule launch");
    if (st) return st;
  }
  const int st = tc ? launch_paged_tc(a, p, items, stream)
                    : dispatch(p, a.dtype, a.D, items, false, stream);
  if (st) return st;
  return dispatch(p, a.dtype, a.D, 0, true, stream);
}

}  // namespace bi
