// The token layout of a serving step over a KV cache in pages, and the write of its
// rotated keys and its values into the pages (bi_paged_plan, bi_rope_kv_paged).
#include "common.cuh"
#include "internal.h"

namespace bi {
namespace paged {

// Sites of the device error word (reason 2: a value out of range).
constexpr unsigned kSitePlan = 1;
constexpr unsigned kSiteRope = 2;
constexpr unsigned kErrReasonRange = 2;

__device__ unsigned g_error_word = 0;

// ---------------------------------------------------------------------------
// bi_paged_plan.  With q_r new and c_r cached tokens of request r and pages of P tokens:
//   query_start[r] = sum_{i<r} q_i,   seq_lens[r] = c_r + q_r,
//   need_r = ceil(seq_r / P) - ceil(c_r / P)   pages taken from the free list, in request
//            order, entered into the block table behind the request's own,
//   token t of request r: position p = c_r + t - query_start[r], page = column p div P of
//            the request's row, slot = page * P + p mod P.
//
// One launch.  Each block owns 512 consecutive tokens and scans the request lengths up to
// them by itself (8 bytes a request out of L2): a second launch for the scan, or a look-back
// between blocks, costs more than the scan up to some ten thousand requests.  A request that
// starts among a block's tokens marks its first token there in shared memory, a running
// maximum over the marks then gives every token its request.  The token with p mod P = 0
// enters its page into the block table, so the new pages need no pass of their own.  Bound by
// a launch and two dependent reads: 64 requests take 4.2 us, 4096 with 50000 tokens 7.2.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 512;
constexpr int kPlanItems = 4;  // requests a thread scans at a time

struct Pair {
  int64_t tok, page;
};

__device__ __forceinline__ Pair warp_scan(Pair v, int lane) {
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int64_t a = __shfl_up_sync(0xffffffffu, v.tok, d);
    const int64_t b = __shfl_up_sync(0xffffffffu, v.page, d);
    if (lane >= d) {
      v.tok += a;
      v.page += b;
    }
  }
  return v;
}

__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const PlanArgs a) {
  constexpr int kWarps = kPlanThreads / 32;
  __shared__ Pair s_warp[kWarps];
  __shared__ int s_mark[kPlanThreads];      // the token begins a request: its place here, else -1
  __shared__ int s_req[kPlanThreads], s_ctx[kPlanThreads];
  __shared__ int64_t s_start[kPlanThreads], s_page[kPlanThreads];
  __shared__ int s_top[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t t0 = static_cast<int64_t>(blockIdx.x) * kPlanThreads;
  const bool last_block = blockIdx.x == gridDim.x - 1;
  const int64_t t1 = t0 + kPlanThreads;  // of the last block: everything from t0 on is its own
  // tokens a row of the block table holds (lengths are 32-bit)
  const int64_t cap = a.width * a.page < INT32_MAX ? a.width * a.page : INT32_MAX;
  const int64_t head = a.free_pages != nullptr ? *a.free_head : 0;
  // (positions and page sizes are below 2^31: the 64-bit division is several times longer)
  const unsigned P = static_cast<unsigned>(a.page);
  auto pages_of = [P](int tokens) { return (static_cast<unsigned>(tokens) + P - 1u) / P; };
  bool bad = a.free_pages != nullptr && (head < 0 || head > a.n_free);
  s_mark[tid] = -1;
  __syncthreads();

  Pair run{0, 0};
  for (int64_t base = 0; base < a.R; base += kPlanThreads * kPlanItems) {
    int q[kPlanItems], c[kPlanItems];
    unsigned need[kPlanItems];  // new pages
    const int64_t r0 = base + static_cast<int64_t>(tid) * kPlanItems;
    Pair mine{0, 0};
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      q[i] = c[i] = 0;
      if (r0 + i < a.R) {
        q[i] = a.query_lens[r0 + i];
        c[i] = a.context_lens[r0 + i];
      }
    }
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      if (q[i] < 0 || c[i] < 0 || static_cast<int64_t>(c[i]) + q[i] > cap) {
        bad = true;  // brings no tokens
        q[i] = 0;
        c[i] = c[i] < 0 ? 0 : static_cast<int>(c[i] < cap ? c[i] : cap);
      }
      need[i] = a.free_pages != nullptr ? pages_of(c[i] + q[i]) - pages_of(c[i]) : 0u;
      mine.tok += q[i];
      mine.page += need[i];
    }
    const Pair inc = warp_scan(mine, lane);
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    Pair at{run.tok + inc.tok - mine.tok, run.page + inc.page - mine.page};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const Pair v = s_warp[w];
      if (w < warp) {
        at.tok += v.tok;
        at.page += v.page;
      }
      run.tok += v.tok;
      run.page += v.page;
    }
#pragma unroll
    for (int i = 0; i < kPlanItems; ++i) {
      const int64_t r = r0 + i;
      if (r >= a.R) break;
      if (at.tok >= t0 && (at.tok < t1 || last_block)) {  // the request is this block's
        a.query_start[r] = static_cast<int>(at.tok);
        a.seq_lens[r] = c[i] + q[i];
      }
      if (q[i] > 0 && at.tok < t1 && at.tok + q[i] > t0) {
        const int m = static_cast<int>(at.tok > t0 ? at.tok - t0 : 0);
        s_mark[m] = m;
        s_req[m] = static_cast<int>(r);
        s_ctx[m] = c[i];
        s_start[m] = at.tok;
        s_page[m] = at.page;
      }
      at.tok += q[i];
      at.page += need[i];
    }
    __syncthreads();
    if (run.tok >= t1 && !last_block) break;  // what follows belongs to later blocks
  }

  if (last_block && tid == 0) {
    a.query_start[a.R] = static_cast<int>(run.tok);
    if (run.tok > a.T) bad = true;
    if (a.free_pages != nullptr) {
      const int64_t left = a.n_free - head;
      *a.next_head = static_cast<int>(head + (run.page < left ? run.page : left));
    }
  }

  // every token's request: the latest mark at or before it
  int m = s_mark[tid];
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int o = __shfl_up_sync(0xffffffffu, m, d);
    if (lane >= d) m = max(m, o);
  }
  if (lane == 31) s_top[warp] = m;
  __syncthreads();
  for (int w = 0; w < warp; ++w) m = max(m, s_top[w]);
  const int64_t t = t0 + tid;
  if (t < a.T) {
    int64_t pos = -1, slot = -1;
    if (t < run.tok && m >= 0) {
      const int r = s_req[m], ctx = s_ctx[m];
      pos = ctx + t - s_start[m];
      const int64_t col = static_cast<unsigned>(pos) / P;
      const int64_t old = pages_of(ctx);
      int* entry = a.table + r * a.table_stride + col;
      int page = -1;
      if (a.free_pages != nullptr && col >= old) {
        const int64_t i = head + s_page[m] + col - old;
        if (head >= 0 && i < a.n_free) page = a.free_pages[i];
        if (pos == col * a.page) *entry = page;
      } else {
        page = *entry;
      }
      if (page >= 0) {
        slot = static_cast<int64_t>(page) * a.page + (pos - col * a.page);
      } else {
        bad = true;  // no page: the list of free pages ran out, or the table has none here
      }
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  if (bad) record_error(&g_error_word, (kSitePlan << 8) | kErrReasonRange);
}

// ---------------------------------------------------------------------------
// bi_rope_kv_paged.  Rotate-half RoPE of the first `rot` elements of each q and k head,
// o[i] = x[i] c[i] - x[i+rot/2] s[i],  o[i+rot/2] = x[i+rot/2] c[i] + x[i] s[i]  (fp32, each
// operation rounded, one rounding to the storage type: the operations of bi_rope_kv), the rest
// of the head and the v heads copied; q to q_out, k and v to their token's slot.
//
// A unit is two vectors of one head: the two halves' vectors of a rotated part, two
// neighbouring ones of a copied part.  A block takes one token, so its threads share the
// token's cos / sin rows, and its position and slot are read once; a thread's first unit is
// loaded before they are there.  Bound by HBM: every element is read and written once, in
// 16-byte vectors: 9434 tokens of 32 + 16 bf16 heads of 128 take 38.5 us, 6.2 TB/s of the 6.5 of
// a plain copy (45.4 with the token's place first and 64-bit divisions; 62.7 with three units a
// thread in flight, whose registers cost more threads than the loads gain; 40 with 64 or 192
// threads).  A decode step of 64 tokens is a launch, 3.2 us.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 128;

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

template <typename T, int VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_paged_kernel(const RopePagedArgs a) {
  using V = Vec<T, VEC>;
  const int64_t t = blockIdx.x;
  const int64_t pos = a.positions[t];
  const int64_t slot = a.slots[t];
  const int hd = static_cast<int>(a.hd), half = static_cast<int>(a.rot) / 2;
  const int per_head = hd / (2 * VEC), rot_units = half / VEC;
  const int hq = static_cast<int>(a.hq), hk = static_cast<int>(a.hk);
  const int units = (hq + 2 * hk) * per_head;
  const T* src = static_cast<const T*>(a.qkv) + t * a.qkv_stride;
  V x0, x1;
  int h, e0, e1;  // the unit's head and its vectors' places there
  auto load = [&](int i) {
    const int u = i - (h = i / per_head) * per_head;
    const bool turn = h < hq + hk && u < rot_units;
    e0 = turn ? u * VEC : 2 * u * VEC;
    e1 = turn ? half + u * VEC : e0 + VEC;
    x0 = *reinterpret_cast<const V*>(src + h * hd + e0);
    x1 = *reinterpret_cast<const V*>(src + h * hd + e1);
  };
  if (threadIdx.x < units) load(threadIdx.x);  // before the token's place is known
  if (pos < 0) return;  // a padding row
  const bool store_kv = slot >= 0 && slot < a.n_pages * a.page;
  const bool bad = pos >= a.n_pos || (slot >= 0 && !store_kv);
  if (bad && threadIdx.x == 0) record_error(&g_error_word, (kSiteRope << 8) | kErrReasonRange);
  if (pos >= a.n_pos) return;
  int64_t pg = 0;
  if (store_kv) {  // (the 64-bit division is several times longer)
    pg = (slot | a.page) >> 32 ? slot / a.page
                               : static_cast<uint32_t>(slot) / static_cast<uint32_t>(a.page);
  }
  const int64_t row = slot - pg * a.page;
  T* const kdst = static_cast<T*>(a.k_cache) + pg * a.ks[0] + row * a.ks[2];
  T* const vdst = static_cast<T*>(a.v_cache) + pg * a.vs[0] + row * a.vs[2];
  T* const q_out = static_cast<T*>(a.q_out) + t * hq * hd;
  const float* cs = a.cos_tab + pos * half;
  const float* sn = a.sin_tab + pos * half;
  for (int i = threadIdx.x; i < units;) {
    if (h < hq + hk && e0 < half) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float c = __ldg(cs + e0 + j), s = __ldg(sn + e0 + j);
        const float p = to_f32(x0.v[j]), q = to_f32(x1.v[j]);
        x0.v[j] = from_f32<T>(__fsub_rn(__fmul_rn(p, c), __fmul_rn(q, s)));
        x1.v[j] = from_f32<T>(__fadd_rn(__fmul_rn(q, c), __fmul_rn(p, s)));
      }
    }
    if (h < hq || store_kv) {
      T* dst = h < hq ? q_out + h * hd
                      : h < hq + hk ? kdst + (h - hq) * a.ks[1] : vdst + (h - hq - hk) * a.vs[1];
      *reinterpret_cast<V*>(dst + e0) = x0;
      *reinterpret_cast<V*>(dst + e1) = x1;
    }
    i += kRopeThreads;
    if (i < units) load(i);
  }
}

}  // namespace paged

int launch_paged_plan(const PlanArgs& a, cudaStream_t stream) {
  const int64_t blocks = a.T > 0 ? (a.T + paged::kPlanThreads - 1) / paged::kPlanThreads : 1;
  paged::plan_kernel<<<static_cast<unsigned>(blocks), paged::kPlanThreads, 0, stream>>>(a);
  return cuda_status(cudaGetLastError(), "paged_plan launch");
}

template <typename T>
static int launch_rope_paged_t(const RopePagedArgs& a, cudaStream_t stream) {
  constexpr int kVec = 16 / sizeof(T);
  const unsigned grid = static_cast<unsigned>(a.T);
  auto ok16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; };
  bool vec = a.hd % (2 * kVec) == 0 && a.rot % (2 * kVec) == 0 && a.qkv_stride % kVec == 0 &&
             ok16(a.qkv) && ok16(a.q_out) && ok16(a.k_cache) && ok16(a.v_cache);
  for (int i = 0; i < 3; ++i) vec = vec && a.ks[i] % kVec == 0 && a.vs[i] % kVec == 0;
  if (vec) {
    paged::rope_paged_kernel<T, kVec><<<grid, paged::kRopeThreads, 0, stream>>>(a);
  } else {
    paged::rope_paged_kernel<T, 1><<<grid, paged::kRopeThreads, 0, stream>>>(a);
  }
  return cuda_status(cudaGetLastError(), "rope_kv_paged launch");
}

int launch_rope_paged(const RopePagedArgs& a, int dtype, cudaStream_t stream) {
  if (a.T == 0 || a.hq + 2 * a.hk == 0) return BI_OK;
  if (dtype == BI_BF16) return launch_rope_paged_t<__nv_bfloat16>(a, stream);
  if (dtype == BI_F16) return launch_rope_paged_t<__half>(a, stream);
  return launch_rope_paged_t<float>(a, stream);
}

unsigned read_error_paged(bool clear) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, paged::g_error_word, sizeof(v));
  if (clear && v) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(paged::g_error_word, &z, sizeof(z));
  }
  return v;
}

}  // namespace bi
