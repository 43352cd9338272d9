// Attention of new tokens over a KV cache in pages on the 5th-generation tensor cores:
// fp16 / bf16, head dim 64 or 128, page sizes that divide or are multiples of 128.
//
// A block (two per SM) takes one tile of 128 rows -- 128 / G tokens x the G query heads of a
// KV head -- and walks the tile's keys 128 at a time:
//   warp 4      TMA producer: the tile's q rows once, then K and V of each 128 keys, one box
//               per page (the lanes fetch the pages' numbers one tile ahead);
//   warp 5      tcgen05.mma: S = Q K^T (128 x 128, fp32 in TMEM) and O += P V with P read
//               from TMEM;
//   warps 0..3  one row per thread: maximum, exponentials, sum; P, rounded to the 16-bit
//               type, goes back to TMEM over the scores it came from.
// While one block's softmax runs the other block's products keep the tensor pipe busy.
//
// The running maximum of a 512-key block only moves when a tile's exceeds it by more than
// 2^8: until then the weights are up to 256 times too large, which the 16-bit type and the
// fp32 sums hold, and O needs no rescaling.  Whether it moves is decided row by row (never by
// what other rows of the tile need), so a row's bits do not depend on its neighbours.
//
// Values behind masked keys: their weight is zero, but 0 x NaN is not.  In tiles that some
// row sees only in part the V rows are looked over in shared memory: what no row of the block
// sees is zeroed, and a non-finite value that some rows see is taken out of the product and
// added to those rows' results by hand.
#include "paged_sdpa.cuh"

namespace bi {
namespace psdpa {
namespace tcp {

constexpr int kThreads = 256;
constexpr int kTile = 128;            // rows of a tile and keys of a step
constexpr int kRegsSoftmax = 208;     // 128 x (208 + 48) = 256 x 128, the launch's registers
constexpr int kRegsOther = 48;
constexpr int kTmemCols = 256;        // S at 0 (P over its second half), O at 128
constexpr float kSlack = 8.f;         // log 2 of how far weights may exceed 1

enum : unsigned { kSiteProducer = 1, kSiteMma = 2, kSiteSoftmax = 3, kSiteDrain = 4 };

__device__ unsigned g_error_word_tc = 0;

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;  // K and V tiles alternate
  static constexpr int kSmem = 1024 + (1 + kStages) * kTileBytes;
};

struct Shared {
  SchedSmem<kThreads> sched;
  uint64_t q_full, full[4], empty[4], s_full, p_ready, o_full, mma_done;
  uint32_t tmem;
  int abort_flag;
  int keep_o;         // the softmax warps put values into O: accumulate on them
  unsigned bad[4];    // keys of the tile with a non-finite value that some row sees
};

__device__ __forceinline__ void tmem_ld_x1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_x64(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
      "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, "
      "%35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, "
      "%52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]),
        "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
        "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]),
        "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),
        "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]),
        "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]),
        "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(
          r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
// D(tmem) (+)= A(tmem) x B(smem desc)
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar,
                                            int32_t c0, int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void softmax_sync() {  // the four softmax warps
  asm volatile("bar.sync 1, 128;" ::: "memory");
}

// Two fp32 operations in one instruction, each rounded to nearest.
__device__ __forceinline__ void fma2(float& x0, float& x1, float a, float b) {  // x a + b
  asm("{\n\t.reg .b64 x, y, z;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %2};\n\tmov.b64 z, {%3, %3};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1) : "f"(a), "f"(b));
}
__device__ __forceinline__ void add2(float& x0, float& x1, float y0, float y1) {
  asm("{\n\t.reg .b64 x, y;\n\t"
      "mov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "+f"(x0), "+f"(x1) : "f"(y0), "f"(y1));
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (dtype_of<T>::value == 2) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float unpack(uint32_t w, int hi) {
  const uint16_t h = static_cast<uint16_t>(hi ? w >> 16 : w & 0xffffu);
  return to_f32(*reinterpret_cast<const T*>(&h));
}
// Exponent bits of the two 16-bit values of a word.
template <typename T>
__device__ __forceinline__ constexpr uint32_t exp_mask() {
  return dtype_of<T>::value == 2 ? 0x7f80u : 0x7c00u;
}

// Scores of 64 keys, those that are not visible made -inf.
__device__ __forceinline__ void mask_scores(uint32_t (&s)[64], uint32_t lo, uint32_t hi) {
#pragma unroll
  for (int j = 0; j < 64; ++j) {
    s[j] = ((j < 32 ? lo : hi) >> (j & 31)) & 1u ? s[j] : 0xff800000u;
  }
}

// Steps of 128 keys that block `blk` of the list needs, as a 4-bit set.
__device__ __forceinline__ unsigned steps_of(const Params& p, const BlockList& list, int pmax,
                                             int blk) {
  unsigned set = 0;
#pragma unroll
  for (int s = 0; s < kBlockKeys / kTile; ++s) {
    const int t0 = blk * kBlockKeys + s * kTile;
    if (t0 <= pmax && (t0 + kTile > list.lo_key || t0 < p.first)) set |= 1u << s;
  }
  return set;
}

// The next step behind (i, s) of the blocks [.., i1): its first key, or -1.
struct StepIter {
  int i, i1;
  unsigned left;  // steps of block i still to come
  int blk;
};
__device__ __forceinline__ int next_step(const Params& p, const BlockList& list, int pmax,
                                         StepIter& it) {
  while (it.left == 0) {
    if (it.i >= it.i1) return -1;
    it.blk = list.at(it.i++);
    it.left = steps_of(p, list, pmax, it.blk);
  }
  const int s = __ffs(it.left) - 1;
  it.left &= it.left - 1;
  return it.blk * kBlockKeys + s * kTile;
}

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 2)
    paged_tc_kernel(const __grid_constant__ CUtensorMap map_q,
                    const __grid_constant__ CUtensorMap map_q1,
                    const __grid_constant__ CUtensorMap map_k,
                    const __grid_constant__ CUtensorMap map_v, const Params p) {
  using C = Cfg<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ Shared sh;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_q = smem;
  uint8_t* s_ring = smem + C::kTileBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sh.abort_flag;

  grid_wait();
  grid_launch_dependents();
  Work w;
  if (!find_work<kThreads>(p, blockIdx.x, sh.sched, w, blockIdx.x == 0)) return;
  const int tok0 = w.tile * p.tile_tok;  // in the request
  const int n_tok = min(p.tile_tok, w.x.n_tok - tok0);
  const int rows = n_tok * p.G;
  const int pos0 = w.x.seq - w.x.n_tok + tok0;
  const int pmax = pos0 + n_tok - 1;
  const BlockList list = block_list(p, pos0, pmax);
  const int i0 = static_cast<int>(static_cast<int64_t>(list.n) * w.piece / w.pieces);
  const int i1 = static_cast<int>(static_cast<int64_t>(list.n) * (w.piece + 1) / w.pieces);
  if (w.pieces > 1 && i0 == i1) return;

  if (tid == 0) {
    mbar_init(&sh.q_full, 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.s_full, 1);
    mbar_init(&sh.p_ready, 4);
    mbar_init(&sh.o_full, 1);
    mbar_init(&sh.mma_done, 1);
    sh.abort_flag = 0;
    sh.keep_o = 0;
    fence_barrier_init();
  }
  if (warp == 5) {
    tmem_alloc(&sh.tmem, kTmemCols);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;

  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 4) {
      // ---------------- TMA producer ----------------
      if (lane == 0 && i0 < i1) {
        // a decoding request's one token, or the tile's (and, behind the request's last,
        // other requests': rows that are computed and not stored)
        const bool single = n_tok == 1;
        mbar_arrive_expect_tx(&sh.q_full, static_cast<uint32_t>(
            (single ? 1 : p.tile_tok) * p.G * D * 2));
        for (int h = 0; h < C::kHalves; ++h) {
          tma_load_3d(s_q + h * (kTile * 128), single ? &map_q1 : &map_q, &sh.q_full, h * 64,
                      w.kvh * p.G, w.x.tok + tok0);
        }
      }
      const int box_rows = min(p.page, kTile);
      const int n_box = kTile / box_rows;
      const int* entries = p.table + static_cast<int64_t>(w.r) * p.table_stride;
      auto page_of = [&](int t0) {  // of this lane's box; n_pages (zero fill) where none is
        if (t0 < 0 || lane >= n_box) return p.n_pages;
        const int key = t0 + lane * box_rows;
        if (key > pmax) return p.n_pages;
        const int pg = entries[key / p.page];
        return pg >= 0 && pg < p.n_pages ? pg : p.n_pages;
      };
      StepIter it{i0, i1, 0, 0};
      int t0 = next_step(p, list, pmax, it);
      int pg = page_of(t0);
      int n = 0;
      bool ok = true, any = false;
      while (t0 >= 0 && ok) {
        const int nt = next_step(p, list, pmax, it);
        const int npg = page_of(nt);
        const int row = (t0 + lane * box_rows) % p.page;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++n) {
          const int stage = n % C::kStages;
          const uint32_t phase = (n / C::kStages) & 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&sh.empty[stage], phase ^ 1u, abort_flag));
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&sh.full[stage], C::kTileBytes);
          __syncwarp();
          if (lane < n_box) {
            uint8_t* dst = s_ring + stage * C::kTileBytes + lane * box_rows * 128;
#pragma unroll
            for (int h = 0; h < C::kHalves; ++h) {
              tma_load_4d(dst + h * (kTile * 128), kv == 0 ? &map_k : &map_v, &sh.full[stage],
                          h * 64, row, w.kvh, pg);
            }
          }
          any = true;
        }
        t0 = nt;
        pg = npg;
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        record_error(&g_error_word_tc, (kSiteProducer << 8) | kErrReasonTimeout);
      }
      if (!ok && any) sleep_ns(200000);  // the copies in flight land
    } else if (warp == 5) {
      // ---------------- tcgen05.mma ----------------
      if (lane == 0) {
        constexpr uint32_t fmt = dtype_of<T>::value == 2 ? 1u : 0u;
        constexpr uint32_t idesc_s = umma_idesc_f16(fmt, 0u, kTile, kTile);
        constexpr uint32_t idesc_o = umma_idesc_f16(fmt, 1u, kTile, D);
        StepIter it{i0, i1, 0, 0};
        bool ok = true;
        int n = 0, step = 0;
        if (i0 < i1) ok = mbar_wait(&sh.q_full, 0, abort_flag);
        bool fresh = true;  // the next product starts a key block
        for (int t0 = next_step(p, list, pmax, it); ok && t0 >= 0; ++step) {
          int stage = n % C::kStages;
          ok = mbar_wait(&sh.full[stage], (n / C::kStages) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          const uint32_t qb = smem_u32(s_q), kb = smem_u32(s_ring + stage * C::kTileBytes);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = (k / 4) * (kTile * 128) + (k % 4) * 32;
            umma_f16(tmem, umma_smem_desc(qb + off, 16, 1024, 2),
                     umma_smem_desc(kb + off, 16, 1024, 2), idesc_s, k != 0 ? 1u : 0u);
          }
          umma_commit(&sh.empty[stage]);
          umma_commit(&sh.s_full);
          ++n;
          stage = n % C::kStages;
          ok = mbar_wait(&sh.p_ready, step & 1, abort_flag) &&
               mbar_wait(&sh.full[stage], (n / C::kStages) & 1, abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (*reinterpret_cast<volatile int*>(&sh.keep_o)) {
            fresh = false;
            *reinterpret_cast<volatile int*>(&sh.keep_o) = 0;
          }
          const uint32_t vb = smem_u32(s_ring + stage * C::kTileBytes);
#pragma unroll
          for (int k = 0; k < kTile / 16; ++k) {
            // V (keys x D) is MN-major: 64-column slabs 16 KiB apart, 8-key groups 1 KiB
            umma_f16_ts(tmem + 128, tmem + 64 + k * 8,
                        umma_smem_desc(vb + k * 2048, kTile * 128, 1024, 2), idesc_o,
                        (k != 0 || !fresh) ? 1u : 0u);
          }
          umma_commit(&sh.empty[stage]);
          ++n;
          const bool block_end = it.left == 0;
          if (block_end) umma_commit(&sh.o_full);
          fresh = block_end;
          t0 = next_step(p, list, pmax, it);
        }
        if (!ok) {
          *abort_flag = 1;
          record_error(&g_error_word_tc, (kSiteMma << 8) | kErrReasonTimeout);
        }
        umma_commit(&sh.mma_done);  // every product is done before TMEM is given back
        if (!mbar_wait(&sh.mma_done, 0, nullptr)) {
          record_error(&g_error_word_tc, (kSiteDrain << 8) | kErrReasonTimeout);
        }
      }
    }
  } else {
    // ---------------- softmax: thread = row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const uint32_t lanes = static_cast<uint32_t>(warp * 32) << 16;
    const uint32_t tS = tmem + lanes, tO = tmem + 128 + lanes;
    const int row = warp * 32 + lane;
    const bool live = row < rows;
    const bool warp_live = warp * 32 < rows;
    const int tok = row / p.G, head = w.kvh * p.G + (row - tok * p.G);
    const int pos = live ? max(-1, pos0 + tok) : -1;
    const int lo_key = p.window == INT32_MAX ? 0 : pos - p.window + 1;  // of this row
    float tot_m = -INFINITY, tot_l = 0.f, tot_o[D];
#pragma unroll
    for (int d = 0; d < D; ++d) tot_o[d] = 0.f;
    float m = -INFINITY, l = 0.f;
    bool fresh = true, ok = true;
    int step = 0, block = 0;
    StepIter it{i0, i1, 0, 0};
    for (int t0 = next_step(p, list, pmax, it); t0 >= 0; ++step) {
      const bool block_end = it.left == 0;
      ok = __all_sync(0xffffffffu, mbar_wait(&sh.s_full, step & 1, abort_flag));
      if (!ok) break;
      tc_fence_after();
      // does every row of the tile see every key of the step?
      const bool whole = t0 + kTile - 1 <= pos0 &&
                         (p.window == INT32_MAX || t0 > pmax - p.window ||
                          t0 + kTile <= p.first);
      uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
      if (!whole) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const int k0 = t0 + 32 * b;
          // bits below x of a word, for any x
          auto below = [](int x) { return x <= 0 ? 0u : (x >= 32 ? ~0u : (1u << x) - 1u); };
          vis[b] = below(pos + 1 - k0) & (~below(lo_key - k0) | below(p.first - k0));
        }
      }
      if (warp_live) {
        // The scores of keys 64..127 stay in registers from the maximum to the exponentials;
        // those of keys 0..63 are read twice.  P goes over the second half's scores: keys
        // 0..63 to columns 64..95, keys 64..127 to columns 96..127.
        uint32_t s[64];
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_ld_x64(tS + 64 * h, s);
          tmem_ld_wait();
          if (!whole) mask_scores(s, vis[2 * h], vis[2 * h + 1]);
#pragma unroll
          for (int j = 0; j < 64; j += 8) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              tops[c] = fmaxf(tops[c], fmaxf(__uint_as_float(s[j + 2 * c]),
                                             __uint_as_float(s[j + 2 * c + 1])));
            }
          }
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float t = top == -INFINITY ? top : top * p.scale_log2;
        const bool move = t > m + kSlack;  // (also from m = -inf)
        const float f = move ? exp2_approx(m - t) : 1.f;
        if (move) m = t;
        const float base = m == -INFINITY ? 0.f : -m;
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int h = 1; h >= 0; --h) {
          if (h == 0) {
            tmem_ld_x64(tS, s);
            tmem_ld_wait();
            if (!whole) mask_scores(s, vis[0], vis[1]);
          }
          uint32_t packed[32];
#pragma unroll
          for (int j = 0; j < 64; j += 2) {
            float x0 = __uint_as_float(s[j]), x1 = __uint_as_float(s[j + 1]);
            fma2(x0, x1, p.scale_log2, base);
            x0 = exp2_approx(x0);
            x1 = exp2_approx(x1);
            add2(sum[j % 4], sum[j % 4 + 1], x0, x1);
            packed[j / 2] = pack2<T>(x0, x1);
          }
          tmem_st_x32(tS + 64 + 32 * h, packed);
        }
        l = __fmaf_rn(l, f, __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3])));
        if (!fresh && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(tO + c, o);
            tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__fmul_rn(__uint_as_float(o[j]), f));
            tmem_st_x32(tO + c, o);
          }
        }
        tmem_st_wait();
      }
      if (!whole) {
        // V of this step: thread = key
        const int n = 2 * step + 1, stage = n % C::kStages;
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.full[stage], (n / C::kStages) & 1, abort_flag));
        if (!ok) break;
        uint8_t* vrow = s_ring + stage * C::kTileBytes + row * 128;
        const int key = t0 + row;
        const bool seen = key <= pmax && (key >= list.lo_key || key < p.first);
        constexpr uint32_t em = exp_mask<T>();
        bool bad = false;
#pragma unroll 1
        for (int c = 0; c < C::kHalves * 8; ++c) {
          uint4* at = reinterpret_cast<uint4*>(vrow + (c >> 3) * (kTile * 128) +
                                               (((c + row) & 7) << 4));
          uint4 x = *at;
          uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
          bool hit = false;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if ((xw[e] & em) == em) {
              xw[e] &= 0xffff0000u;
              hit = true;
            }
            if (((xw[e] >> 16) & em) == em) {
              xw[e] &= 0xffffu;
              hit = true;
            }
          }
          if (hit) *at = x;
          bad |= hit;
        }
        const unsigned flags = __ballot_sync(0xffffffffu, bad && seen);
        if (lane == 0) sh.bad[warp] = flags;
        fence_proxy_async_smem();  // the zeros, to the product's reads
        softmax_sync();
        if ((sh.bad[0] | sh.bad[1] | sh.bad[2] | sh.bad[3]) != 0) {
          // add the non-finite values to the rows that see them
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (fresh) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0u;
            } else {
              tmem_ld_32x32b_x32(tO + c, o);
              tmem_ld_wait();
            }
#pragma unroll 1
            for (int k = 0; k < kTile; ++k) {
              if (((sh.bad[k >> 5] >> (k & 31)) & 1u) == 0) continue;
              __syncwarp();
              uint32_t pw;
              tmem_ld_x1(tS + 64 + (k >> 1), pw);
              tmem_ld_wait();
              const float pk = unpack<T>(pw, k & 1);
              const uint32_t word = k < 32 ? vis[0] : k < 64 ? vis[1] : k < 96 ? vis[2] : vis[3];
              if (!live || ((word >> (k & 31)) & 1u) == 0) continue;
              const int kk = t0 + k;
              const int64_t pg = p.table[static_cast<int64_t>(w.r) * p.table_stride + kk / p.page];
              const T* v = static_cast<const T*>(p.v) + pg * p.vs[0] + w.kvh * p.vs[1] +
                           (kk % p.page) * p.vs[2] + c;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float x = to_f32(v[j]);
                if (!isfinite(x)) o[j] = __float_as_uint(__uint_as_float(o[j]) + pk * x);
              }
            }
            __syncwarp();
            tmem_st_x32(tO + c, o);
          }
          tmem_st_wait();
          if (tid == 0) *reinterpret_cast<volatile int*>(&sh.keep_o) = 1;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_ready);
      fresh = false;
      if (block_end) {
        ok = __all_sync(0xffffffffu, mbar_wait(&sh.o_full, block & 1, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {
          if (w.pieces > 1) {
            const int64_t at = part_slot(p, w.base, w.blocks, tok0 + tok, head, i0 + block);
            if (live) p.part_ml[at] = make_float2(m, l);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tO + c, o);
              tmem_ld_wait();
              if (live) {
                float4* dst = reinterpret_cast<float4*>(p.part_o + at * D + c);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  dst[j] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                       __uint_as_float(o[4 * j + 2]),
                                       __uint_as_float(o[4 * j + 3]));
                }
              }
            }
          } else {
            float fa, fb;
            fold_factors(tot_m, m, fa, fb);
            tot_l = fold_value(tot_l, l, fa, fb);
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tO + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                tot_o[c + j] = fold_value(tot_o[c + j], __uint_as_float(o[j]), fa, fb);
              }
            }
          }
        }
        m = -INFINITY;
        l = 0.f;
        fresh = true;
        ++block;
      }
      t0 = next_step(p, list, pmax, it);
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        record_error(&g_error_word_tc, (kSiteSoftmax << 8) | kErrReasonTimeout);
      }
    } else if (w.pieces == 1 && live) {
      const float sink = p.sinks ? to_f32(static_cast<const T*>(p.sinks)[head]) * kLog2e : 0.f;
      const float sc = row_scale(tot_m, tot_l, p.sinks != nullptr, sink);
      T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(w.x.tok + tok0 + tok) * p.os[0] +
               head * p.os[1];
      const bool vec = (p.os[0] % 8 | p.os[1] % 8) == 0 &&
                       (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
#pragma unroll
      for (int d = 0; d < D; d += 8) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          x[j] = pack2<T>(row_value(tot_o[d + 2 * j], sc), row_value(tot_o[d + 2 * j + 1], sc));
        }
        if (vec) {
          *reinterpret_cast<uint4*>(dst + d) = make_uint4(x[0], x[1], x[2], x[3]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t h = static_cast<uint16_t>(j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu);
            dst[d + j] = *reinterpret_cast<const T*>(&h);
          }
        }
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 5) {
    __syncwarp();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int D>
static int launch(const PagedSdpaArgs& a, const Params& p, int64_t items, cudaStream_t stream) {
  using C = Cfg<D>;
  CUtensorMap mq, mq1, mk, mv;
  const uint64_t qdims[3] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.H),
                             static_cast<uint64_t>(a.T)};
  const uint64_t qstr[2] = {static_cast<uint64_t>(a.qs[1]) * 2, static_cast<uint64_t>(a.qs[0]) * 2};
  uint32_t qbox[3] = {64, static_cast<uint32_t>(p.G), static_cast<uint32_t>(p.tile_tok)};
  int st = encode_tiled16(&mq, a.q, 3, qdims, qstr, qbox, a.dtype);
  if (st) return st;
  qbox[2] = 1;
  st = encode_tiled16(&mq1, a.q, 3, qdims, qstr, qbox, a.dtype);
  if (st) return st;
  const uint64_t cdims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(a.page),
                             static_cast<uint64_t>(a.Hkv), static_cast<uint64_t>(a.n_pages)};
  const uint32_t cbox[4] = {64, static_cast<uint32_t>(a.page < kTile ? a.page : kTile), 1, 1};
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t* s = kv == 0 ? a.ks : a.vs;
    const uint64_t cstr[3] = {static_cast<uint64_t>(s[2]) * 2, static_cast<uint64_t>(s[1]) * 2,
                              static_cast<uint64_t>(s[0]) * 2};
    st = encode_tiled16(kv == 0 ? &mk : &mv, kv == 0 ? a.k : a.v, 4, cdims, cstr, cbox, a.dtype);
    if (st) return st;
  }
  cudaError_t e = cudaFuncSetAttribute(paged_tc_kernel<T, D>,
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
  if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(paged_sdpa)");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cuda_status(cudaLaunchKernelEx(&cfg, paged_tc_kernel<T, D>, mq, mq1, mk, mv, p),
                     "paged_sdpa tensor-core launch");
}

}  // namespace tcp
}  // namespace psdpa

// The route is a function of type, head dim, heads and page size; never of the lengths.
bool paged_tc_takes(const PagedSdpaArgs& a) {
  const bool page = a.page >= 128 ? a.page % 128 == 0 : (a.page >= 8 && 128 % a.page == 0);
  return a.dtype != BI_F32 && (a.D == 64 || a.D == 128) && a.H / a.Hkv <= 128 && page;
}

int launch_paged_tc(const PagedSdpaArgs& a, const psdpa::Params& p, int64_t items,
                    cudaStream_t stream) {
  using namespace psdpa::tcp;
  if (a.dtype == BI_BF16) {
    return a.D == 64 ? launch<__nv_bfloat16, 64>(a, p, items, stream)
                     : launch<__nv_bfloat16, 128>(a, p, items, stream);
  }
  return a.D == 64 ? launch<__half, 64>(a, p, items, stream)
                   : launch<__half, 128>(a, p, items, stream);
}

unsigned read_error_paged_sdpa_tc(bool clear) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, psdpa::tcp::g_error_word_tc, sizeof(v));
  if (clear && v) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(psdpa::tcp::g_error_word_tc, &z, sizeof(z));
  }
  return v;
}

}  // namespace bi
