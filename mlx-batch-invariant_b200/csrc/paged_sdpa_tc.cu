// Attention of new tokens over a KV cache in pages on the 5th-generation tensor cores:
// fp16 / bf16, head dim 64 or 128, page sizes that divide or are multiples of 128.
//
// A block (one per SM) works on two items at a time, each a tile of 128 rows -- 128 / G tokens
// x the G query heads of a KV head -- whose keys it walks 128 at a time.  Neighbouring tiles
// of a long chunk share the K and V tiles; otherwise (decode) the two items have their own:
//   warp 8      TMA producer: the tiles' q rows once, then K and V tiles, one box per page
//               (the lanes fetch the pages' numbers ahead), through one ring;
//   warp 9      tcgen05.mma: S = Q K^T (128 x 128, fp32 in TMEM) and O += P V with P read
//               from TMEM, the two items' products in turn;
//   warps 0..3 and 4..7  softmax of the first and of the second item, one row per thread:
//               maximum, exponentials, sum; P, rounded to the 16-bit type, goes back to TMEM
//               over the scores it came from.
// One thread issues both items' products in turn, so while one item's products run the other's
// softmax does: two blocks per SM with an item each fell into step, both in their softmax at
// one time and both waiting for the tensor pipe at another (5000 clocks for two tiles of 128
// keys where the products take 2048; now 3900).
//
// Bound, for chunks, by the chain of a step, which two items overlap only in part and TMEM has
// no room for a third: scores 300 clocks behind the product, maximum 500, exponentials 1900
// (the special-function unit alone takes 1024), the product's turn 1100; and by waves that are
// not full.  2048 tokens behind 6144, 32 heads of 128 over 8: 278 us in a graph (291 called from
// Python), 864 TFLOP/s, 52 % of cuBLAS's burst rate; tensor pipe 38 %, special-function unit
// 47 %, issue slots 36 % of the time.  Its 256 pairs of items make 1.73 waves on 148 SMs, which
// alone is 13 %.  For decode by HBM between the first loads (8 us, the search for the items ahead
// of them) and the last blocks and the join: 64 requests of 3000 to 8191 keys take 274 us in a
// graph (307 called), 5.3 TB/s, 82 % of the copy rate.  (Bringing the next block's first tiles to
// L2 while the last of this one's are worked on changed nothing.)  The softmax keeps a row's
// running result and half its scores in registers; at D = 128 that spills (148 bytes stored, 204
// loaded a thread), at D = 64 hardly (8 and 52).
//
// P is rounded to the caches' 16-bit type because a product's two operands have one type and V
// has that one; the row's sum adds the weights before that rounding.  It adds half a step of the
// type (2^-8 for bf16, 2^-11 for fp16) to each weight, independent from key to key: the result
// is off by 0.0023 of its norm in bf16, where rounding the exact one is off by 0.0017.
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
#include <algorithm>

#include "bounded_wait.h"
#include "paged_sdpa.cuh"

namespace bi {
namespace psdpa {
namespace tcp {

constexpr int kThreads = 384;
constexpr int kTile = 128;            // rows of a tile and keys of a step
constexpr int kRegsSoftmax = 224;     // 2 x 224 + 56 = 3 x 168, the launch's registers
constexpr int kRegsOther = 56;
constexpr int kTmemCols = 512;        // per item: S (P over its second half) and O, 128 each
constexpr float kSlack = 8.f;         // log 2 of how far weights may exceed 1
constexpr int kMaxStages = 12;
constexpr int kBlockKeys = 1 << kTcShift;
constexpr long long kCopyBudgetCycles = 20000000LL;  // about 10 ms

enum : unsigned { kSiteProducer = 1, kSiteMma = 2, kSiteSoftmax = 3, kSiteDrain = 4 };

__device__ unsigned g_error_word_tc = 0;

template <int D>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 5 : 12;  // K and V tiles
  static constexpr int kSmem = 1024 + (2 + kStages) * kTileBytes;
};

__device__ __forceinline__ void tmem_ld_x1(uint32_t taddr, uint32_t& r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr)
               : "memory");
}
// Waits for this warp's TMEM loads; the registers pass through, so that nothing that uses them
// is moved ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
        "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
        "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
        "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
      :
      : "memory");
}
__device__ __forceinline__ void tmem_ld_wait1(uint32_t& r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r) : : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(taddr)
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
                                            uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(static_cast<uint32_t>(accumulate))
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
// A whole warp's wait, bounded like mbar_wait (the flag may be null); a loop of few instructions
// (the kernel's code has to stay within the instruction cache: at 142 KB every step of it was
// fetched anew, and the kernel ran no faster than its code came in).
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity,
                                          const volatile int* abort_flag) {
  const uint32_t addr = smem_u32(bar);
  const bool ok = bounded_wait([&] { return mbar_try_wait(addr, parity); },
                               [] { return clock64(); }, abort_flag, kWaitBudgetCycles);
  return __all_sync(0xffffffffu, ok);
}
// The same for copies of a block that is giving up, with a limit of some milliseconds each.
__device__ __forceinline__ void copy_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t addr = smem_u32(bar);
  bounded_wait([&] { return mbar_try_wait(addr, parity); }, [] { return clock64(); }, nullptr,
               kCopyBudgetCycles);
}
// One lane of the converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }
// Two fp32 numbers in one 64-bit register, two operations in one instruction, each rounded to
// nearest.  (Constants are kept packed: a register short, the compiler would otherwise pack
// them anew at every use.)
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t x, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(x));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
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

// The larger of `top` and 32 scores, in four chains.
__device__ __forceinline__ void max_of(const uint32_t (&s)[32], float (&tops)[4]) {
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      tops[c] = fmaxf(tops[c], fmaxf(__uint_as_float(s[j + 2 * c]),
                                     __uint_as_float(s[j + 2 * c + 1])));
    }
  }
}
// The weights 2^(s scale + base) of 32 scores: added to `sum`, and rounded to T in TMEM.
template <typename T>
__device__ __forceinline__ void weights_of(const uint32_t (&s)[32], uint64_t scale, uint64_t base,
                                           uint64_t (&sum)[2], uint32_t taddr) {
  uint32_t packed[16];
#pragma unroll
  for (int j = 0; j < 32; j += 2) {
    float x0, x1;
    unpair(fma2(pair(__uint_as_float(s[j]), __uint_as_float(s[j + 1])), scale, base), x0, x1);
    x0 = exp2_approx(x0);
    x1 = exp2_approx(x1);
    sum[(j / 2) % 2] = add2(sum[(j / 2) % 2], pair(x0, x1));
    packed[j / 2] = pack2<T>(x0, x1);
  }
  tmem_st_x16(taddr, packed);
}

// What one of a block's two items is.
struct Item {
  int pieces;             // 0: it is not there
  int r, kvh, tok;        // request, KV head, first row
  bool joins;             // keeps a running result of its blocks (else they leave theirs)
  Part part;              // its first partial result (pieces > 1)
  int n_tok, rows, tok0;  // its tile (tok0 in the request)
  int pos0, pmax;         // positions of its first and last token
  // the keys it walks: blocks [i0, i1) of `list`.  Items that share K and V walk the keys that
  // either needs; what a row does not see changes nothing.
  BlockList list;
  int list_pos0, list_pmax;
  int i0, i1;
  int steps;              // of 128 keys
};

// Steps of 128 keys that block `blk` of the list needs, as a 4-bit set.
__device__ __forceinline__ unsigned steps_of(const Params& p, const Item& it, int blk) {
  unsigned set = 0;
#pragma unroll
  for (int s = 0; s < kBlockKeys / kTile; ++s) {
    const int t0 = blk * kBlockKeys + s * kTile;
    if (t0 <= it.list_pmax && (t0 + kTile > it.list.lo_key || t0 < p.first)) set |= 1u << s;
  }
  return set;
}

// Describes the block's items (of which `there` exist): lanes 0..15 of a warp have the first
// one's `w`, the others the second's.  Says whether they share K and V: two tiles of one request
// and group, whose keys are not split.
__device__ __forceinline__ bool make_items(const Params& p, const Work& w, int there,
                                           Item (&out)[2]) {
  const int lane = threadIdx.x & 15, k = (threadIdx.x & 31) >> 4;
  const int other = __shfl_xor_sync(0xffffffffu, w.tile, 16);
  const bool same = __shfl_xor_sync(0xffffffffu, w.r, 16) == w.r &&
                    __shfl_xor_sync(0xffffffffu, w.group, 16) == w.group;
  const bool shared = there == 2 && same && w.pieces == 1;
  Item it;
  it.pieces = 0;
  it.joins = true;
  it.r = it.kvh = it.tok = 0;
  it.part = Part{0, 0};
  it.n_tok = it.rows = it.tok0 = it.pos0 = it.i0 = it.i1 = it.steps = 0;
  it.pmax = it.list_pos0 = it.list_pmax = -1;
  it.list = BlockList{0, 0, 0, 0};
  if (k < there) {
    it.pieces = w.pieces;
    it.r = w.r;
    it.kvh = w.kvh;
    it.tok0 = w.tile * p.tile_tok;
    it.tok = w.x.tok + it.tok0;
    it.n_tok = min(p.tile_tok, w.x.n_tok - it.tok0);
    it.rows = it.n_tok * p.G;
    const int first = w.x.seq - w.x.n_tok;
    it.pos0 = first + it.tok0;
    it.pmax = it.pos0 + it.n_tok - 1;
    it.list_pos0 = it.pos0;
    it.list_pmax = it.pmax;
    if (shared) {  // item 1 is the tile before item 0's
      it.list_pos0 = first + min(w.tile, other) * p.tile_tok;
      it.list_pmax = first + min((max(w.tile, other) + 1) * p.tile_tok, w.x.n_tok) - 1;
    }
    it.list = block_list(p, it.list_pos0, it.list_pmax);
    it.i0 = piece_start(it.list.n, w.piece, w.pieces);
    it.i1 = piece_start(it.list.n, w.piece + 1, w.pieces);
    const bool few = is_few(p, w.x);
    it.joins = w.pieces == 1 || (!few && w.piece == 0);
    it.part = part_of(p, w.x, w.base, w.entries, w.tile, w.group,
                      first_entry(it.list.n, w.piece, w.pieces, few, it.i0));
    for (int i = it.i0 + lane; i < it.i1; i += 16) {
      it.steps += __popc(steps_of(p, it, it.list.at(i)));
    }
  }
  __syncwarp();
#pragma unroll
  for (int d = 8; d > 0; d /= 2) it.steps += __shfl_xor_sync(0xffffffffu, it.steps, d);
  if (lane == 0) out[k] = it;
  return shared;
}

// Walks an item's steps.
struct StepIter {
  int i;
  unsigned left;  // steps of the block still to come
  int blk;
};
// The first key of the next step, or -1.
__device__ __forceinline__ int next_step(const Params& p, const Item& item, StepIter& it) {
  while (it.left == 0) {
    if (it.i >= item.i1) return -1;
    it.blk = item.list.at(it.i++);
    it.left = steps_of(p, item, it.blk);
  }
  const int s = __ffs(it.left) - 1;
  it.left &= it.left - 1;
  return it.blk * kBlockKeys + s * kTile;
}

// The order of the K and V tiles in the ring, which the producer fills and the products empty:
// shared, K(0) V(0) K(1) V(1) ...; else the items' K(0), then round by round V(j) and K(j + 1)
// of item 0, then of item 1.  Place of V(j) of item k:
__device__ __forceinline__ int v_place(bool shared, int l0, int l1, int k, int j) {
  if (shared) return 2 * j + 1;
  int n = (l0 > 0) + (l1 > 0) + min(j, l0) + min(j, max(l0 - 1, 0)) + min(j, l1) +
          min(j, max(l1 - 1, 0));
  if (k == 1) n += (j < l0) + (j + 1 < l0);
  return n;
}

struct Shared {
  uint64_t q_full[2], full[kMaxStages], empty[kMaxStages], s_full[2], p_half[2], p_ready[2],
      o_full[2], looked[2], both, mma_done;
  uint32_t tmem;
  int abort_flag;
  int shared;             // the items share K and V
  int loaded;             // K and V tiles that the producer has asked for
  Item item[2];
  int add[2];             // the item's next product is added to O (it does not start a key block)
  int hit[2];             // 1 + the last step whose V has such a value
  unsigned bad[2][4];     // keys of a step with a non-finite value that some row sees
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
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
  uint8_t* s_ring = smem + 2 * C::kTileBytes;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort_flag = &sh.abort_flag;

  if (warp == 8 && lane == 0) {
    tma_prefetch_desc(&map_q);
    tma_prefetch_desc(&map_q1);
    tma_prefetch_desc(&map_k);
    tma_prefetch_desc(&map_v);
  }
  if (warp == 10 && lane == 0) {
    for (int k = 0; k < 2; ++k) {
      mbar_init(&sh.q_full[k], 1);
      mbar_init(&sh.s_full[k], 1);
      mbar_init(&sh.p_half[k], 4);
      mbar_init(&sh.p_ready[k], 4);
      mbar_init(&sh.o_full[k], 1);
      mbar_init(&sh.looked[k], 4);
      sh.hit[k] = 0;
    }
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.both, 8);
    mbar_init(&sh.mma_done, 1);
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  grid_wait();
  grid_launch_dependents();
  if (warp == 0) {
    Finder finder;
    finder.begin(p, blockIdx.x == 0);
    // alone, as long as there is an SM for every item
    const unsigned per = 2 * finder.total <= static_cast<unsigned>(p.target) ? 1 : 2;
    const unsigned at = blockIdx.x * per;
    const int there = at >= finder.total ? 0 : min(per, finder.total - at);
    Work w = {};
    if (there > 0) w = finder.find(p, at, at + there - 1);
    const bool both = make_items(p, w, there, sh.item);
    if (lane == 0) sh.shared = both;
  } else if (warp == 9) {
    tmem_alloc(&sh.tmem, kTmemCols);
    tmem_relinquish();
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  if (sh.item[0].pieces == 0) {
    if (warp == 9) tmem_dealloc(tmem, kTmemCols);
    return;
  }
  const bool shared = sh.shared;
  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
    if (warp == 8) {
      // ---------------- TMA producer ----------------
      const int side = lane >> 4, sub = lane & 15;  // 16 lanes per item
      const Item item = sh.item[side];
      if (sub == 0 && item.steps > 0) {
        // a decoding request's one token, or the tile's (and, behind the request's last,
        // other requests': rows that are computed and not stored)
        const bool single = item.n_tok == 1;
        mbar_arrive_expect_tx(&sh.q_full[side], static_cast<uint32_t>(
            (single ? 1 : p.tile_tok) * p.G * D * 2));
        for (int h = 0; h < C::kHalves; ++h) {
          tma_load_3d(s_q + side * C::kTileBytes + h * (kTile * 128), single ? &map_q1 : &map_q,
                      &sh.q_full[side], h * 64, item.kvh * p.G, item.tok);
        }
      }
      __syncwarp();
      const int box_rows = min(p.page, kTile);
      const int n_box = kTile / box_rows;
      const int* entries = p.table + static_cast<int64_t>(item.r) * p.table_stride;
      const int kvh = item.kvh;
      auto page_of = [&](int t0) {  // of this lane's box; n_pages (zero fill) where none is
        if (t0 < 0 || sub >= n_box) return p.n_pages;
        const int key = t0 + sub * box_rows;
        if (key > item.list_pmax) return p.n_pages;
        const int pg = entries[p.by_page(key)];
        return pg >= 0 && pg < p.n_pages ? pg : p.n_pages;
      };
      int n = 0;
      bool ok = true;
      auto load = [&](const CUtensorMap* map, int k, int t0, int pg) {
        const int stage = n % C::kStages;
        ok = ok && warp_wait(&sh.empty[stage], ((n / C::kStages) & 1) ^ 1u, abort_flag);
        if (!ok) return;
        ++n;
        if (lane == 0) mbar_arrive_expect_tx(&sh.full[stage], C::kTileBytes);
        __syncwarp();
        if (side == k && sub < n_box) {
          uint8_t* dst = s_ring + stage * C::kTileBytes + sub * box_rows * 128;
          const int key = t0 + sub * box_rows, row = key - p.by_page(key) * p.page;
#pragma unroll
          for (int h = 0; h < C::kHalves; ++h) {
            tma_load_4d(dst + h * (kTile * 128), map, &sh.full[stage], h * 64, row, kvh, pg);
          }
        }
      };
      const int l0 = sh.item[0].steps, l1 = shared ? 0 : sh.item[1].steps, rounds = max(l0, l1);
      StepIter it{item.i0, 0, 0};
      int t0 = next_step(p, item, it), t1 = t0 < 0 ? -1 : next_step(p, item, it);
      int pg0 = page_of(t0), pg1 = page_of(t1);
      if (l0 > 0) load(&map_k, 0, t0, pg0);
      if (l1 > 0) load(&map_k, 1, t0, pg0);
      for (int j = 0; j < rounds && ok; ++j) {
        const int t2 = t1 < 0 ? -1 : next_step(p, item, it);
        const int pg2 = page_of(t2);
        if (j < l0) load(&map_v, 0, t0, pg0);
        if (j + 1 < l0) load(&map_k, 0, t1, pg1);
        if (j < l1) load(&map_v, 1, t0, pg0);
        if (j + 1 < l1) load(&map_k, 1, t1, pg1);
        t0 = t1;
        t1 = t2;
        pg0 = pg1;
        pg1 = pg2;
      }
      if (!ok && lane == 0) {
        *abort_flag = 1;
        record_error(&g_error_word_tc, (kSiteProducer << 8) | kErrReasonTimeout);
      }
      if (lane == 0) sh.loaded = n;
    } else if (warp == 9) {
      // ---------------- tcgen05.mma ----------------
      // The whole warp walks the steps, so that what it computes is uniform, and one lane
      // issues; descriptors advance by constants.
      constexpr uint32_t fmt = dtype_of<T>::value == 2 ? 1u : 0u;
      constexpr uint32_t idesc_s = umma_idesc_f16(fmt, 0u, kTile, kTile);
      constexpr uint32_t idesc_o = umma_idesc_f16(fmt, 1u, kTile, D);
      constexpr uint64_t kTileUnits = C::kTileBytes >> 4;  // of descriptor addresses
      const bool leader = elect_one();
      const int steps0 = uniform(sh.item[0].steps), steps1 = uniform(sh.item[1].steps);
      const bool both = __shfl_sync(0xffffffffu, shared, 0);
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const uint64_t q_desc = umma_smem_desc(smem_u32(s_q), 16, 1024, 2);
      const uint64_t k_desc = umma_smem_desc(smem_u32(s_ring), 16, 1024, 2);
      // V (keys x D) is MN-major: 64-column slabs 16 KiB apart, 8-key groups 1 KiB
      const uint64_t v_desc = umma_smem_desc(smem_u32(s_ring), kTile * 128, 1024, 2);
      bool ok = true;
      int stage = 0;       // of the next tile of the ring ...
      uint32_t phase = 0;  // ... and its barrier's parity
      int next = 0;        // and of the one behind it
      uint32_t next_phase = 0;
      auto behind = [&]() {
        next = stage + 1;
        next_phase = phase;
        if (next == C::kStages) {
          next = 0;
          next_phase ^= 1u;
        }
      };
      auto advance = [&]() {
        behind();
        stage = next;
        phase = next_phase;
      };
      const int rounds = max(steps0, steps1);
      // Round j = -1: the first scores.  Round j: O += P V of each item's step j, then S = Q K^T
      // of its step j + 1.
#pragma unroll 1
      for (int j = -1; j < rounds && ok; ++j) {
#pragma unroll 1
        for (int k = 0; k < 2 && ok; ++k) {
          const int steps = k == 0 ? steps0 : steps1;
          if (j >= steps || steps == 0) continue;
          int ks = stage;
          uint32_t kph = phase;
          const bool waited = both && k == 1;  // for its tiles, in item 0's turn
          if (j < 0) {
            ok = warp_wait(&sh.q_full[k], 0, abort_flag);
          } else {
            behind();
            ks = next;
            kph = next_phase;
            if (!waited) ok = warp_wait(&sh.full[stage], phase, abort_flag);
          }
          if (j + 1 < steps && !waited) ok = ok && warp_wait(&sh.full[ks], kph, abort_flag);
          if (j >= 0) {
            ok = ok && warp_wait(&sh.p_half[k], j & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const bool add = uniform(*const_cast<volatile int*>(&sh.add[k])) != 0;
            // keys 64..127 while the weights of keys 0..63 are still being computed
            const uint64_t vd = v_desc + stage * kTileUnits;
            const uint32_t d = tm + 256 * k;
            if (leader) {
              umma_f16_ts(d + 128, d + 64 + 4 * 8, vd + 4 * (2048 >> 4), idesc_o, add);
#pragma unroll
              for (int i = 5; i < 8; ++i) {
                umma_f16_ts(d + 128, d + 64 + i * 8, vd + i * (2048 >> 4), idesc_o, true);
              }
            }
            __syncwarp();
            ok = warp_wait(&sh.p_ready[k], j & 1, abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (leader) {
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                umma_f16_ts(d + 128, d + 64 + i * 8, vd + i * (2048 >> 4), idesc_o, true);
              }
              if (!both || k == 1) umma_commit(&sh.empty[stage]);
              if (j + 1 == steps) umma_commit(&sh.o_full[k]);
            }
            __syncwarp();
            if (!both) advance();  // (now the K tile, if there is one)
          }
          if (!ok) break;
          if (j + 1 < steps) {
            if (j < 0) tc_fence_after();
            if (leader) {
              const uint64_t qd = q_desc + k * kTileUnits, kd = k_desc + ks * kTileUnits;
#pragma unroll
              for (int i = 0; i < D / 16; ++i) {
                const uint64_t off = ((i / 4) * (kTile * 128) + (i % 4) * 32) >> 4;
                umma_f16(tm + 256 * k, qd + off, kd + off, idesc_s, i != 0 ? 1u : 0u);
              }
              if (!both || k == 1) umma_commit(&sh.empty[ks]);
              umma_commit(&sh.s_full[k]);
            }
            __syncwarp();
            if (!both) advance();
          }
        }
        if (both) {  // V(j) and K(j + 1) served both items
          advance();
          if (j >= 0) advance();
        }
      }
      if (!ok && leader) {
        *abort_flag = 1;
        record_error(&g_error_word_tc, (kSiteMma << 8) | kErrReasonTimeout);
      }
      __syncwarp();
      if (leader) umma_commit(&sh.mma_done);  // every product is done before TMEM is given back
      __syncwarp();
      if (!warp_wait(&sh.mma_done, 0, nullptr) && leader) {
        record_error(&g_error_word_tc, (kSiteDrain << 8) | kErrReasonTimeout);
      }
    }
  } else {
    // ---------------- softmax: thread = row ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
    const int k = warp >> 2;
    const Item& item = sh.item[k];
    const int pieces = item.pieces, steps = item.steps;
    const int row = (warp & 3) * 32 + lane;
    const uint32_t tS = tmem + 256 * k + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t tO = tS + 128;
    const bool live = row < item.rows;
    const bool warp_live = (warp & 3) * 32 < item.rows;
    const int tok = p.by_head(row), head = item.kvh * p.G + (row - tok * p.G);
    const int pos = live ? max(-1, item.pos0 + tok) : -1;
    const int lo_key = p.window == INT32_MAX ? 0 : pos - p.window + 1;  // of this row
    float tot_m = -INFINITY, tot_l = 0.f;
    uint64_t tot_o[D / 2];
#pragma unroll
    for (int d = 0; d < D / 2; ++d) tot_o[d] = 0ull;
    const uint64_t scale2 = pair(p.scale_log2, p.scale_log2);
    float m = -INFINITY, l = 0.f;
    bool fresh = true, ok = true;  // fresh: the step starts a key block
    int block = 0;
    // Barriers of the item's four warps, and of both items' eight, with a bounded wait like all
    // others (a named barrier would wait for good for a warp that gave up).
    int n_looked = 0, n_both = 0;
    auto meet = [&](uint64_t* bar, int& n) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
      return warp_wait(bar, n++ & 1, abort_flag);
    };
    StepIter it{item.i0, 0, 0};
    // do all rows see every key of the step at t0?
    auto whole_for = [&](int t0, int pos0, int pmax) {
      return t0 + kTile - 1 <= pos0 &&
             (p.window == INT32_MAX || t0 > pmax - p.window || t0 + kTile <= p.first);
    };
    // Leaves what O holds for the join, with its (bm, bl), as the item's partial result `entry`.
    auto leave = [&](int entry, float bm, float bl) {
      const Part at = {item.part.first + static_cast<int64_t>(entry) * item.part.rows,
                       item.part.rows};
      if (live) p.part_ml[at.first + row] = make_float2(bm, bl);
#pragma unroll 1
      for (int c = 0; c < D; c += 32) {
        uint32_t o[32];
        tmem_ld_32x32b_x32(tO + c, o);
        tmem_ld_wait(o);
        if (live) {
          float4* dst = part_at<D>(p, at, row, c);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            dst[static_cast<int64_t>(j) * at.rows] =
                make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                            __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
          }
        }
      }
    };
    // The finished key block's O, with its (bm, bl): joined to the running result, or (in a
    // later piece) left for the join.
    auto close_block = [&](float bm, float bl) {
      if (!item.joins) {
        leave(block, bm, bl);
      } else {
        float fa, fb;
        fold_factors(tot_m, bm, fa, fb);
        tot_l = fold_value(tot_l, bl, fa, fb);
        const uint64_t fa2 = pair(fa, fa), fb2 = pair(fb, fb);
#pragma unroll
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld_32x32b_x32(tO + c, o);
          tmem_ld_wait(o);
#pragma unroll
          for (int j = 0; j < 32; j += 2) {  // fold_value, two at a time
            uint64_t& x = tot_o[(c + j) / 2];
            x = fma2(pair(__uint_as_float(o[j]), __uint_as_float(o[j + 1])), fb2, mul2(x, fa2));
          }
        }
      }
      ++block;
    };
    for (int step = 0; step < steps; ++step) {
      const int t0 = next_step(p, item, it);
      const bool whole = whole_for(t0, item.pos0, item.pmax);
      const bool list_whole = whole_for(t0, item.list_pos0, item.list_pmax);
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
      // S of this step; with it the product before it in the queue, the last step's P V, is done
      ok = warp_wait(&sh.s_full[k], step & 1, abort_flag);
      if (!ok) break;
      tc_fence_after();
      uint32_t sa[32], sb[32];
      // keys 64..127 again, behind work that needs the registers
      auto reload = [&]() {
        tmem_ld_32x32b_x32(tS + 64, sa);
        tmem_ld_32x32b_x32(tS + 96, sb);
        tmem_ld_wait(sa);
        tmem_ld_wait(sb);
      };
      float base = 0.f, f = 1.f;
      if (warp_live) {
        if (__builtin_expect(!whole, 0)) {  // keys that the row does not see: a score of -inf
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const uint32_t wa = h == 0 ? vis[0] : vis[2], wb = h == 0 ? vis[1] : vis[3];
            tmem_ld_32x32b_x32(tS + 64 * h, sa);
            tmem_ld_32x32b_x32(tS + 64 * h + 32, sb);
            tmem_ld_wait(sa);
            tmem_ld_wait(sb);
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              sa[j] = (wa >> j) & 1u ? sa[j] : 0xff800000u;
              sb[j] = (wb >> j) & 1u ? sb[j] : 0xff800000u;
            }
            tmem_st_x32(tS + 64 * h, sa);
            tmem_st_x32(tS + 64 * h + 32, sb);
          }
          tmem_st_wait();
        }
        // The scores of keys 64..127 stay in registers from the maximum to the exponentials;
        // those of keys 0..63 are read twice.  P goes over the second half's scores: keys
        // 0..63 to columns 64..95, keys 64..127 to columns 96..127.
        float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          tmem_ld_32x32b_x32(tS + 64 * h, sa);
          tmem_ld_32x32b_x32(tS + 64 * h + 32, sb);
          tmem_ld_wait(sa);
          tmem_ld_wait(sb);
          max_of(sa, tops);
          max_of(sb, tops);
        }
        const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        const float t = top == -INFINITY ? top : top * p.scale_log2;
        if (fresh) {
          const float bm = m, bl = l;
          m = t;
          l = 0.f;
          if (step > 0) {
            close_block(bm, bl);
            reload();
          }
        } else {
          const bool move = t > m + kSlack;  // (also from m = -inf)
          if (move) {
            f = exp2_approx(m - t);
            m = t;
          }
          if (__builtin_expect(__any_sync(0xffffffffu, move), 0)) {
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              uint32_t o[32];
              tmem_ld_32x32b_x32(tO + c, o);
              tmem_ld_wait(o);
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                float x0, x1;
                unpair(mul2(pair(__uint_as_float(o[j]), __uint_as_float(o[j + 1])), pair(f, f)), x0,
                       x1);
                o[j] = __float_as_uint(x0);
                o[j + 1] = __float_as_uint(x1);
              }
              tmem_st_x32(tO + c, o);
            }
            reload();
          }
        }
        base = m == -INFINITY ? 0.f : -m;
      }
      if (__builtin_expect(!list_whole, 0)) {
        // V of this step: thread = key
        const int place = v_place(shared, sh.item[0].steps, sh.item[1].steps, k, step);
        const int stage = place % C::kStages;
        ok = warp_wait(&sh.full[stage], (place / C::kStages) & 1, abort_flag);
        if (!ok) break;
        uint8_t* vrow = s_ring + stage * C::kTileBytes + row * 128;
        const int key = t0 + row;
        const bool seen = key <= item.list_pmax && (key >= item.list.lo_key || key < p.first);
        // seen by every row: the product may have what it holds.  Else look for non-finite values,
        // at first only look: both items' warps read the tile.
        const bool by_all = key <= item.list_pos0 &&
                            (p.window == INT32_MAX || key > item.list_pmax - p.window ||
                             key < p.first);
        constexpr uint32_t em = exp_mask<T>() * 0x10001u;           // both values' exponents
        constexpr uint32_t one = (exp_mask<T>() & -exp_mask<T>()) * 0x10001u;
        constexpr int kChunks = C::kHalves * 8;
        // 16-byte chunk c of a row sits at c ^ (row & 7) of its 128 bytes
        auto chunk = [&](int c) {
          return reinterpret_cast<uint4*>(vrow + (c >> 3) * (kTile * 128) + (((c ^ row) & 7) << 4));
        };
        uint32_t hit = 0;
        if (!by_all) {
#pragma unroll 4
          for (int c = 0; c < kChunks; ++c) {
            const uint4 x = *chunk(c);
            // an exponent of all ones carries into the sign's place
            hit |= ((x.x & em) + one) | ((x.y & em) + one) | ((x.z & em) + one) |
                   ((x.w & em) + one);
          }
        }
        const bool found = (hit & 0x80008000u) != 0;
        if (found) *const_cast<volatile int*>(&sh.hit[k]) = step + 1;
        ok = meet(&sh.looked[k], n_looked);
        if (!ok) break;
        // (both items' warps come to the same answer on shared tiles)
        if (__builtin_expect(*const_cast<volatile int*>(&sh.hit[k]) == step + 1, 0)) {
          // Take them out, and add those that some rows see to these rows' results by hand.
          ok = !shared || meet(&sh.both, n_both);  // both have looked
          if (!ok) break;
          const unsigned flags = __ballot_sync(0xffffffffu, found && seen);
          if (lane == 0) sh.bad[k][warp & 3] = flags;
          if (found) {
#pragma unroll 1
            for (int c = 0; c < kChunks; ++c) {  // (of shared tiles both write the same)
              uint4* at = chunk(c);
              uint4 x = *at;
              uint32_t* xw = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t top = ((xw[e] & em) + one) & 0x80008000u;
                if (top & 0x8000u) xw[e] &= 0xffff0000u;
                if (top & 0x80000000u) xw[e] &= 0xffffu;
              }
              *at = x;
            }
          }
          fence_proxy_async_smem();  // the zeros, to the product's reads
          ok = shared ? meet(&sh.both, n_both) : meet(&sh.looked[k], n_looked);
          if (!ok) break;
          tmem_st_wait();  // O, if this step rescaled it: stores and loads are not ordered
          unsigned bad[4];
#pragma unroll
          for (int b = 0; b < 4; ++b) bad[b] = sh.bad[k][b];
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            if (fresh) {
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = 0u;
            } else {
              tmem_ld_32x32b_x32(tO + c, o);
              tmem_ld_wait(o);
            }
#pragma unroll 1
            for (int i = 0; i < kTile; ++i) {
              const uint32_t bw = i < 32 ? bad[0] : i < 64 ? bad[1] : i < 96 ? bad[2] : bad[3];
              const uint32_t vw = i < 32 ? vis[0] : i < 64 ? vis[1] : i < 96 ? vis[2] : vis[3];
              if (((bw >> (i & 31)) & 1u) == 0) continue;
              __syncwarp();
              uint32_t score;
              tmem_ld_x1(tS + i, score);
              tmem_ld_wait1(score);
              if (!live || ((vw >> (i & 31)) & 1u) == 0) continue;
              const float x = exp2_approx(__fmaf_rn(__uint_as_float(score), p.scale_log2, base));
              const float pi = unpack<T>(pack2<T>(x, x), 0);
              const int key_i = t0 + i;
              const int col = p.by_page(key_i);
              const int64_t pg = p.table[static_cast<int64_t>(item.r) * p.table_stride + col];
              const T* v = static_cast<const T*>(p.v) + pg * p.vs[0] + item.kvh * p.vs[1] +
                           (key_i - col * p.page) * p.vs[2] + c;
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                const float y = to_f32(v[j]);
                if (!isfinite(y)) o[j] = __float_as_uint(__uint_as_float(o[j]) + pi * y);
              }
            }
            __syncwarp();
            tmem_st_x32(tO + c, o);
          }
          fresh = false;  // O holds values now
          reload();
        }
      }
      uint64_t sum[2] = {0ull, 0ull};
      const uint64_t base2 = pair(base, base);
      if (warp_live) {
        weights_of<T>(sa, scale2, base2, sum, tS + 96);
        tmem_ld_32x32b_x32(tS, sa);
        weights_of<T>(sb, scale2, base2, sum, tS + 112);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if ((warp & 3) == 0) *const_cast<volatile int*>(&sh.add[k]) = !fresh;
        mbar_arrive(&sh.p_half[k]);
      }
      if (warp_live) {
        tmem_ld_wait(sa);
        tmem_ld_32x32b_x32(tS + 32, sb);
        weights_of<T>(sa, scale2, base2, sum, tS + 64);
        tmem_ld_wait(sb);
        weights_of<T>(sb, scale2, base2, sum, tS + 80);
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_ready[k]);
      float s0, s1;
      unpair(add2(sum[0], sum[1]), s0, s1);
      l = __fmaf_rn(l, f, __fadd_rn(s0, s1));
      fresh = it.left == 0;
    }
    if (ok && steps > 0) {
      ok = warp_wait(&sh.o_full[k], 0, abort_flag);
      tc_fence_after();
      if (ok && warp_live) {
        close_block(m, l);
        if (item.joins && pieces > 1) {  // the running result, by way of O's columns
#pragma unroll
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
#pragma unroll
            for (int j = 0; j < 32; j += 2) {
              float x0, x1;
              unpair(tot_o[(c + j) / 2], x0, x1);
              o[j] = __float_as_uint(x0);
              o[j + 1] = __float_as_uint(x1);
            }
            tmem_st_x32(tO + c, o);
          }
          tmem_st_wait();
          leave(0, tot_m, tot_l);
        }
      }
    }
    if (!ok) {
      if (lane == 0) {
        *abort_flag = 1;
        record_error(&g_error_word_tc, (kSiteSoftmax << 8) | kErrReasonTimeout);
      }
    } else if (pieces == 1 && live) {
      const float sink = p.sinks ? to_f32(static_cast<const T*>(p.sinks)[head]) * kLog2e : 0.f;
      const float sc = row_scale(tot_m, tot_l, p.sinks != nullptr, sink);
      T* dst = static_cast<T*>(p.out) + static_cast<int64_t>(item.tok + tok) * p.os[0] +
               head * p.os[1];
#pragma unroll
      for (int d = 0; d < D; d += 8) {
        uint32_t x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float o0, o1;
          unpair(tot_o[d / 2 + j], o0, o1);
          x[j] = pack2<T>(row_value(o0, sc), row_value(o1, sc));
        }
        *reinterpret_cast<uint4*>(dst + d) = make_uint4(x[0], x[1], x[2], x[3]);
      }
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 9) {
    __syncwarp();
    tmem_dealloc(tmem, kTmemCols);
  } else if (warp == 8 && __builtin_expect(*abort_flag, 0)) {
    // Somebody gave up, so nobody has waited for the copies in flight: the block's shared memory
    // is not given back while they may still write to it.
    for (int k = 0; k < 2; ++k) {
      if (sh.item[k].steps > 0) copy_wait(&sh.q_full[k], 0);
    }
    const int n = sh.loaded;
    for (int i = max(0, n - C::kStages); i < n; ++i) {
      copy_wait(&sh.full[i % C::kStages], (i / C::kStages) & 1);
    }
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
  // two items a block; no fewer blocks than SMs, for calls whose items each get their own
  cfg.gridDim = dim3(static_cast<unsigned>(
      std::max<int64_t>((items + 1) / 2, std::min<int64_t>(items, device_sm_count()))));
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
