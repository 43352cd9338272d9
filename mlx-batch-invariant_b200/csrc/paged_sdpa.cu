// Attention of new tokens over a KV cache in pages (bi_paged_sdpa): the CUDA-core route, the
// join of partial results and the host side.  The tensor-core route is paged_sdpa_tc.cu.
#include <algorithm>
#include <limits>

#include "paged_sdpa.cuh"

namespace bi {
namespace psdpa {

// ---------------------------------------------------------------------------
// CUDA-core route: any head dim that is a multiple of 32 up to 256, any page size, fp32 too.
// A block takes a tile of up to 16 rows (tokens x heads of a group), four to each warp.
// Per 32 keys a warp computes four scores per lane (lane = key, q out of shared memory),
// updates (m, l) by warp reductions, and adds p v with a lane on every 32nd column.  Keys
// that a row does not see are skipped, so what they hold never reaches it.
// ---------------------------------------------------------------------------
constexpr int kSimtWarps = 4;
constexpr int kSimtThreads = 32 * kSimtWarps;
constexpr int kSimtRows = 4;  // per warp
constexpr int kSimtTile = kSimtWarps * kSimtRows;

template <typename T>
struct alignas(16) Vec16 {
  T v[16 / sizeof(T)];
};

template <typename T, int DC>  // head dim 32 * DC
__global__ void __launch_bounds__(kSimtThreads) paged_simt_kernel(const Params p) {
  constexpr int D = 32 * DC;
  constexpr int VEC = 16 / sizeof(T);
  __shared__ SchedSmem<kSimtThreads, 1> s_sched;
  __shared__ float s_q[kSimtTile][D];
  grid_wait();
  grid_launch_dependents();
  find_work<kSimtThreads, 1>(p, blockIdx.x, s_sched, blockIdx.x == 0);
  __syncthreads();
  if (!s_sched.hit[0]) return;
  const Work w = s_sched.found[0];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int subs = p.groups / p.Hkv;  // groups of a KV head
  const int head0 = w.kvh * p.G + (w.group % subs) * p.group_heads;
  const int heads = min(p.group_heads, (w.kvh + 1) * p.G - head0);
  const int tok0 = w.tile * p.tile_tok;  // in the request
  const int n_tok = min(p.tile_tok, w.x.n_tok - tok0);
  const int rows = n_tok * heads;
  const int pos0 = w.x.seq - w.x.n_tok + tok0;
  const BlockList list = block_list(p, pos0, pos0 + n_tok - 1);
  const int i0 = piece_start(list.n, w.piece, w.pieces);
  const int i1 = piece_start(list.n, w.piece + 1, w.pieces);
  if (w.pieces > 1 && i0 == i1) return;

  for (int i = tid; i < rows * D; i += kSimtThreads) {
    const int r = i / D, d = i - r * D;
    const int64_t tok = w.x.tok + tok0 + r / heads;
    s_q[r][d] = to_f32(static_cast<const T*>(p.q)[tok * p.qs[0] + (head0 + r % heads) * p.qs[1] + d]);
  }
  __syncthreads();
  if (warp * kSimtRows >= rows) return;

  int pos[kSimtRows];
  float tot_m[kSimtRows], tot_l[kSimtRows], tot_o[kSimtRows][DC];
#pragma unroll
  for (int r = 0; r < kSimtRows; ++r) {
    const int row = warp * kSimtRows + r;
    // a row that is not there (or whose position is negative) sees nothing
    pos[r] = row < rows ? max(-1, pos0 + row / heads) : -1;
    tot_m[r] = -INFINITY;
    tot_l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < DC; ++c) tot_o[r][c] = 0.f;
  }
  const int pmax = pos0 + n_tok - 1;
  const T* kbase = static_cast<const T*>(p.k) + w.kvh * p.ks[1];
  const T* vbase = static_cast<const T*>(p.v) + w.kvh * p.vs[1];

  for (int i = i0; i < i1; ++i) {
    const int key0 = list.at(i) * kBlockKeys;
    float m[kSimtRows], l[kSimtRows], o[kSimtRows][DC];
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      m[r] = -INFINITY;
      l[r] = 0.f;
#pragma unroll
      for (int c = 0; c < DC; ++c) o[r][c] = 0.f;
    }
    for (int t = key0; t < key0 + kBlockKeys && t <= pmax; t += 32) {
      if (t + 31 < list.lo_key && t >= p.first) continue;  // no row sees these
      const int key = t + lane;
      unsigned seen[kSimtRows], any = 0;
#pragma unroll
      for (int r = 0; r < kSimtRows; ++r) {
        const bool see = key <= pos[r] && (key > pos[r] - p.window || key < p.first);
        seen[r] = __ballot_sync(0xffffffffu, see);
        any |= seen[r];
      }
      if (any == 0) continue;
      // this lane's key; a page outside the cache reads as zeros
      int64_t pg = -1;
      const int col = p.by_page(key);
      if ((any >> lane) & 1u) pg = p.table[w.r * p.table_stride + col];
      const bool there = pg >= 0 && pg < p.n_pages;
      const int64_t off = there ? key - col * p.page : 0;
      const T* krow = kbase + (there ? pg : 0) * p.ks[0] + off * p.ks[2];
      int64_t voff = (there ? pg : 0) * p.vs[0] + off * p.vs[2];
      float s[kSimtRows] = {};
      if (there) {
#pragma unroll 4
        for (int d = 0; d < D; d += VEC) {
          const Vec16<T> kv = *reinterpret_cast<const Vec16<T>*>(krow + d);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float x = to_f32(kv.v[e]);
#pragma unroll
            for (int r = 0; r < kSimtRows; ++r) {
              s[r] = __fmaf_rn(s_q[warp * kSimtRows + r][d + e], x, s[r]);
            }
          }
        }
      }
      float pr[kSimtRows];
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
        pr[r] = see ? exp2_approx(x - base) : 0.f;
        float sum = pr[r];
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        m[r] = nm;
        l[r] = __fmaf_rn(l[r], f, sum);
#pragma unroll
        for (int c = 0; c < DC; ++c) o[r][c] = __fmul_rn(o[r][c], f);
      }
      const unsigned have = __ballot_sync(0xffffffffu, there);
      for (unsigned left = any; left != 0; left &= left - 1) {
        const int j = __ffs(left) - 1;
        const T* vrow = vbase + __shfl_sync(0xffffffffu, voff, j);
        float v[DC];
#pragma unroll
        for (int c = 0; c < DC; ++c) v[c] = (have >> j) & 1u ? to_f32(vrow[c * 32 + lane]) : 0.f;
#pragma unroll
        for (int r = 0; r < kSimtRows; ++r) {
          const float pj = __shfl_sync(0xffffffffu, pr[r], j);
          if ((seen[r] >> j) & 1u) {
#pragma unroll
            for (int c = 0; c < DC; ++c) o[r][c] = __fmaf_rn(pj, v[c], o[r][c]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < kSimtRows; ++r) {
      const int row = warp * kSimtRows + r;
      if (w.pieces > 1) {
        if (row < rows) {
          const int64_t at = part_slot(p, w.base, w.blocks, tok0 + row / heads,
                                       head0 + row % heads, i);
          if (lane == 0) p.part_ml[at] = make_float2(m[r], l[r]);
#pragma unroll
          for (int c = 0; c < DC; ++c) p.part_o[at * D + c * 32 + lane] = o[r][c];
        }
      } else {
        float fa, fb;
        fold_factors(tot_m[r], m[r], fa, fb);
        tot_l[r] = fold_value(tot_l[r], l[r], fa, fb);
#pragma unroll
        for (int c = 0; c < DC; ++c) tot_o[r][c] = fold_value(tot_o[r][c], o[r][c], fa, fb);
      }
    }
  }
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
// Join of the partial results of split requests: a warp takes one row (token, head) and
// folds its blocks' partial results in order, with the operations of the unsplit kernels.
// Launched behind every call (the split is decided on the device); where nothing was split
// it reads one word.  Its launch overlaps the main kernel's tail.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 128;

template <typename T, int DC>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const Params p) {
  constexpr int D = 32 * DC;
  constexpr int kAhead = 8;  // partial results in flight
  grid_wait();
  if (*p.any_split == 0) return;
  const int lane = threadIdx.x & 31;
  const int64_t n_rows = static_cast<int64_t>(p.T) * p.H;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / 32) + (threadIdx.x >> 5);
       row < n_rows; row += warps) {
    const int tok = static_cast<int>(row / p.H), head = static_cast<int>(row % p.H);
    // its request: the last one that starts at or before it (32-way search)
    int lo = 0, hi = p.R;  // answer + 1 is in (lo, hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const bool le = at < hi && clampi(p.query_start[at], 0, p.T) <= tok;
      const unsigned bal = __ballot_sync(0xffffffffu, le);
      if (bal == 0) break;
      const int k = 31 - __clz(bal);
      lo = lo + k * step;
      hi = min(hi, lo + step);
    }
    const int r = lo;
    const Request x = request(p, r);
    if (tok < x.tok || tok >= x.tok + x.n_tok) continue;
    const int4 info = p.info[r];
    if (info.x <= 1) continue;
    const int in = tok - x.tok, tile = p.by_tile(in);
    const int pos0 = x.seq - x.n_tok + tile * p.tile_tok;
    const int n_tok = min(p.tile_tok, x.n_tok - tile * p.tile_tok);
    const BlockList list = block_list(p, pos0, pos0 + n_tok - 1);
    const int64_t at = part_slot(p, info.z, info.y, in, head, 0);
    float m = -INFINITY, l = 0.f, o[DC];
#pragma unroll
    for (int c = 0; c < DC; ++c) o[c] = 0.f;
    for (int i = 0; i < list.n; i += kAhead) {
      float2 ml[kAhead];
      float po[kAhead][DC];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool in_list = i + j < list.n;
        ml[j] = in_list ? p.part_ml[at + i + j] : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int c = 0; c < DC; ++c) {
          po[j][c] = in_list ? p.part_o[(at + i + j) * D + c * 32 + lane] : 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        float fa, fb;
        fold_factors(m, ml[j].x, fa, fb);
        l = fold_value(l, ml[j].y, fa, fb);
#pragma unroll
        for (int c = 0; c < DC; ++c) o[c] = fold_value(o[c], po[j][c], fa, fb);
      }
    }
    const float sink = p.sinks ? to_f32(static_cast<const T*>(p.sinks)[head]) * kLog2e : 0.f;
    const float sc = row_scale(m, l, p.sinks != nullptr, sink);
    T* dst = static_cast<T*>(p.out) + tok * p.os[0] + head * p.os[1];
#pragma unroll
    for (int c = 0; c < DC; ++c) dst[c * 32 + lane] = from_f32<T>(row_value(o[c], sc));
  }
}

// A launch that may start before the kernel ahead of it in the stream has ended; every
// kernel here waits for that (grid_wait) before it touches memory.
template <typename... Args>
static cudaError_t launch_early(void (*kernel)(Args...), unsigned grid, unsigned block,
                                cudaStream_t stream, Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
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
  return cuda_status(launch_early(paged_simt_kernel<T, DC>, static_cast<unsigned>(items),
                                  kSimtThreads, stream, p), "paged_sdpa launch");
}
template <typename T, int DC>
static int launch_join(const Params& p, cudaStream_t stream) {
  const int64_t rows = static_cast<int64_t>(p.T) * p.H;
  const int64_t want = (rows + kJoinThreads / 32 - 1) / (kJoinThreads / 32);
  const unsigned grid =
      static_cast<unsigned>(std::min<int64_t>(want, 8LL * device_sm_count()));
  return cuda_status(launch_early(join_kernel<T, DC>, grid, kJoinThreads, stream, p),
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

static int64_t info_bytes(int64_t R) { return (16 + 16 * R + 255) / 256 * 256; }

}  // namespace psdpa

// Room for the partial results of every row, at most 256 MiB (requests that do not fit are
// not split), and the per-request notes.
int64_t paged_sdpa_workspace(int64_t T, int64_t R, int64_t H, int64_t D, int64_t width,
                             int64_t page) {
  const double blocks = static_cast<double>(width) * static_cast<double>(page) /
                            psdpa::kBlockKeys + 1.0;
  const double want = static_cast<double>(T) * static_cast<double>(H) * blocks *
                      static_cast<double>(4 * D + 8);
  const int64_t part = want < static_cast<double>(psdpa::kMaxPartBytes)
                           ? static_cast<int64_t>(want) + 256 : psdpa::kMaxPartBytes;
  return psdpa::info_bytes(R) + part;
}

int launch_paged_sdpa(const PagedSdpaArgs& a, cudaStream_t stream) {
  using namespace psdpa;
  const bool tc = paged_tc_takes(a);
  const int rows = tc ? 128 : kSimtTile;
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
  p.max_seq = std::min<int64_t>(a.width * a.page, INT32_MAX - kBlockKeys);
  p.group_heads = std::min(p.G, rows);
  p.tile_tok = rows / p.group_heads;
  const int subs = (p.G + rows - 1) / rows;
  p.groups = p.Hkv * subs;
  p.by_tile = divider(p.tile_tok);
  p.by_page = divider(a.page);
  p.by_head = divider(p.group_heads);
  p.by_group = divider(subs);
  p.target = (tc ? 2 : 8) * device_sm_count();
  p.fine_rows = 16;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.any_split = reinterpret_cast<int*>(ws);
  p.info = reinterpret_cast<int4*>(ws + 16);
  const int64_t left = a.workspace_bytes - info_bytes(a.R);
  p.slots = left <= 256 ? 0u : static_cast<unsigned>(
      std::min<int64_t>((left - 256) / (4 * a.D + 8), kMuch - 1));
  p.part_o = reinterpret_cast<float*>(ws + info_bytes(a.R));
  p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<int64_t>(p.slots) * a.D);

  // tiles of all requests: at most one ragged tile each
  const int64_t tiles = a.T / p.tile_tok + std::min(a.R, a.T);
  // (the spans are rounded in fp32: a little above 4 target pieces)
  const int64_t items = tiles * p.groups + 4LL * p.target + 64;
  if (items > INT32_MAX) return set_error(BI_ERR_UNSUPPORTED, "too many query tiles");
  const int st = tc ? launch_paged_tc(a, p, items, stream)
                    : dispatch(p, a.dtype, a.D, items, false, stream);
  if (st) return st;
  return dispatch(p, a.dtype, a.D, 0, true, stream);
}

}  // namespace bi
