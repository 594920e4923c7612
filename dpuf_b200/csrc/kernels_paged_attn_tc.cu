// kernels_paged_attn_tc.cu - attention of chunks of new tokens over the paged cache on the
// 5th-generation tensor cores (tcgen05, TMEM), 16-bit queries and cache, head_dim <= 128.
//
// An item is 256 rows of one sequence and KV head (two tiles of 128), walked in blocks of 64 keys;
// per tile and block S = Q K^T (M = 128, N = 64) into TMEM, the softmax's weights P from S with the
// running maximum and sum (kernels_paged_attn.cu has the formulas), O += P V with P read from TMEM.
//
//   warps 0..3, 4..7  softmax of tile 0, 1: a thread has one row.  It reads its 64 scores, writes P
//                     (rounded to the cache's type; the sum keeps the unrounded weights) over them,
//                     and scales O in TMEM only when its row's maximum has grown by more than 2^8
//                     since the last time (weights are then at most 2^8, which both types hold with
//                     their full precision; the division by the sum at the end makes up for it),
//                     which after the first blocks is rare.  P has 16 bits because the MMA takes A
//                     and B of one type; a second term would be half as much again of tensor work.
//                     Relative errors against 64 bits, and of the output's rounding alone: four
//                     prompts of 2,048 in fp16 2.7e-4 and 2.1e-4, 512 tokens over 33,280 in bf16
//                     2.1e-3 and 1.7e-3.
//   warp 8            TMA: 64-column boxes of a page's rows (128-byte swizzle) into a ring of key
//                     and value blocks; a page that is not held, or that no row sees, is a box
//                     outside the tensor and arrives as zeros.
//   warps 9, 10       issue tile 0's and tile 1's MMAs (one warp for both was the limit: its waits
//                     left the tensor cores idle); they zero the rows of a value block that no row
//                     of the item sees (stale cache contents may be infinite or NaN, and 0 times
//                     those is NaN; scores of such keys are replaced, not multiplied).
//
// TMEM: each tile has two score buffers of 64 columns (P in the first 32 of each) and O; all 512
// columns.  The second buffer is what the 64-key block buys: the next block's scores are computed
// while the softmax works on this one's.  With one buffer of 128 (P over S, so that QK waits for
// PV and the softmax for both) neither unit was busy half of the time.  The price: at N = 64 the
// QK reads 6 KB of shared memory per 32 tensor cycles, 1.5 times what it delivers.
//
//   warp 11           copies the next item's queries while this one's are in use (two buffers).
//
// Results leave by way of the queries' shared memory: a row is a thread's, and 32 rows' pieces in
// one store cost a cycle a row.
//
// Every wait on an mbarrier is bounded: one that gives up sets the workspace's error word and the
// CTA's abort flag, all roles stop, copies in flight are waited for (bounded) and TMEM is freed.  A
// tile's softmax warps wait each for itself, so they agree on whether one gave up (once an item)
// before they go on to the barriers that need all four.
#include <cuda.h>
#include <math_constants.h>

#include "attn_plan.cuh"
#include "attn_parts.cuh"

namespace dpuf {

namespace {

constexpr int kTile = 128;            // rows of a tile
constexpr int kKeys = 64;             // of a block
constexpr int kItemRows = 2 * kTile;
constexpr int kLoadWarp = 8, kMmaWarp = 9, kQueryWarp = 11;  // kMmaWarp + i: tile i
constexpr int kThreads = 384;
// (The figures of these three are of one input in short bursts; with inputs in rotation, where power
// limits the clock, four prompts of 2,048 take 183 to 189 us.)
// What an item costs beside its blocks, in blocks (four prompts of 2,048: 178 us at 0, 167 at 2, 168 at 3, 174 at 5).
constexpr int kLead = 2;
// Cuts that move to an item's end (a part of 256 rows is 128 KB out and in again).  49 x 216 tokens
// of 3 heads: 31 us at 0, 20 at 3, 19 at 6 and 12; four prompts of 2,048: 170, 167, 167, 170.
constexpr int kSnap = 6;
// Few items are cut into fewer parts (attn_locate).  One prompt of 1,000 tokens, 32/8 heads: 45 us,
// 52 at 0.1, 46 without a limit; 64 tokens over 20,000, 8/2 heads: 67 us, 89 at 0.1, 150 without.
constexpr float kJoin = 0.33f;
// The weights carry a factor 2^7, and so does their sum: at most 2^15, which fp16 holds, while the
// small ones of a long context keep their bits.
constexpr float kLift = 7.0f;
constexpr unsigned long long kWaitNs = 2000000000ull;

typedef unsigned long long u64;

DPUF_DEV uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Shared-memory descriptor of a 128-byte swizzled operand: K-major (lbo unused, sbo between
// groups of 8 rows), or MN-major (lbo between runs of 64 columns, sbo between groups of 8 rows).
DPUF_DEV uint64_t sw128_desc(const void* p, uint32_t lbo, uint32_t sbo) {
  return (uint64_t)((su32(p) >> 4) & 0x3FFF) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16: D fp32, A and B of one type (0 f16, 1 bf16), A K-major, B K- or MN-major, M = 128.
template <typename T>
__host__ __device__ constexpr uint32_t idesc_f16(int n, int b_mn) {
  const uint32_t t = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(kTile >> 4) << 24);
}

// One lane of the warp, the same each time.  The compiler then knows that a single thread issues
// what follows (with a test of the lane it does not, and wraps each MMA in a loop over lanes:
// 700 cycles instead of 400 to 500 for the eight of a product).
DPUF_DEV bool elect_one() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}
DPUF_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((int)acc)
      : "memory");
}
DPUF_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((int)acc)
      : "memory");
}
DPUF_DEV void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(su32(bar))
               : "memory");
}
#define DPUF_R32(v)                                                                                             \
  "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),   \
      "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]),    \
      "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]),   \
      "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
#define DPUF_I32(v)                                                                                             \
  "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), \
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),           \
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]),           \
      "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
// 32 columns of the warp's 32 lanes; the values are there after tmem_wait_ld.
DPUF_DEV void tmem_ld32(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : DPUF_R32(v)
      : "r"(addr));
}
DPUF_DEV void tmem_st32(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::DPUF_I32(v),
      "r"(addr)
      : "memory");
}
// 16 columns, there on return.
DPUF_DEV void tmem_ld16(uint32_t addr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(addr)
      : "memory");
}
DPUF_DEV void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
      "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(addr)
      : "memory");
}
DPUF_DEV void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
DPUF_DEV void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
DPUF_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
DPUF_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

DPUF_DEV unsigned long long gtimer() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
DPUF_DEV void bar_init(uint64_t* bar, int n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(su32(bar)), "r"(n) : "memory");
}
DPUF_DEV void bar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(su32(bar)) : "memory");
}
DPUF_DEV bool bar_try(uint64_t* bar, unsigned par) {
  unsigned ok;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(ok)
               : "r"(su32(bar)), "r"(par)
               : "memory");
  return ok != 0;
}

struct Give {  // where a wait that gives up says so
  volatile int* abort;
  int* err;
};
// Waits of a whole warp: true once the phase is complete, false (for all lanes) after giving up.
DPUF_DEV bool warp_wait(uint64_t* bar, unsigned par, const Give& g) {
  bool ok = bar_try(bar, par);
  if (!ok) {
    const unsigned long long t0 = gtimer();
    for (int it = 1; !ok; it++) {
      ok = bar_try(bar, par);
      if (!ok && (it & 15) == 0 && (*g.abort || gtimer() - t0 > kWaitNs)) {
        *g.abort = 1;
        atomicCAS(g.err, 0, 1);
        break;
      }
    }
  }
  return __all_sync(kFull, ok);
}

DPUF_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DPUF_DEV float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two fp32 values at a time, each rounded as alone.
DPUF_DEV u64 pair(uint32_t a, uint32_t b) {
  u64 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(a), "r"(b));
  return d;
}
DPUF_DEV void split(u64 x, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(x)); }
DPUF_DEV u64 fma2(u64 a, u64 b, u64 c) {
  u64 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
DPUF_DEV u64 add2(u64 a, u64 b) {
  u64 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
DPUF_DEV uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
DPUF_DEV uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}

template <int DP>
struct TileLay {  // shared memory, from a 1,024-byte boundary; operands are 64-column runs of [rows][128 bytes]
  static constexpr int stages = DP == 128 ? 3 : 6;
  static constexpr int tile = kTile * DP * 2;
  static constexpr int block = kKeys * DP * 2;
  static constexpr int q = 0;                   // [2 items][2][tile]
  static constexpr int k = q + 4 * tile;        // [stages][block]
  static constexpr int v = k + stages * block;  // [stages][block]
  static constexpr int bytes = v + stages * block + 1024;
};
constexpr int kQRun = kTile * 128, kKvRun = kKeys * 128;  // bytes of a 64-column run

struct TileArgs {
  AttnArgs p;
  CUtensorMap k_map, v_map;  // (dim, row, head, page), boxes of 64 x min(page_size, 64)
  CUtensorMap q_map, o_map;  // (dim, head, token), boxes of 64 x group x 128 / group: a tile's rows
  int q_boxes, o_boxes;      // whether they are usable: the group divides 128, out has q's type
};

// Positions that an item's rows [r0, r0 + rows) see between them.
DPUF_DEV void item_span(const AttnArgs& p, const AttnSeq& q, int tile, int* lo, int* hi) {
  attn_span(p, q, tile * kItemRows / p.group, min(q.qn - 1, (tile * kItemRows + kItemRows - 1) / p.group), lo, hi);
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads, 1) paged_attention_tc_kernel(const __grid_constant__ TileArgs args) {
  using Lay = TileLay<DP>;
  constexpr int S = Lay::stages;
  extern __shared__ unsigned char raw[];
  __shared__ __align__(8) uint64_t k_full[S], k_empty[S], v_full[S], v_empty[S];
  __shared__ __align__(8) uint64_t q_full[2], q_empty[2], drained[2], s_full[2][2], p_full[2][2], pv_done[2][2];
  __shared__ AttnShare share;
  __shared__ uint32_t tmem_sh;
  __shared__ int abort_sh, flag_sh[2];
  unsigned char* const sm = raw + ((1024 - (su32(raw) & 1023)) & 1023);
  const AttnArgs& p = args.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const AttnParts<kItemRows, DP> parts(p.a.workspace, gridDim.x);
  const Give give{&abort_sh, attn_error(p.a.workspace)};

  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&tmem_sh)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (tid == 0) {
    for (int i = 0; i < S; i++) {
      bar_init(&k_full[i], 1);
      bar_init(&k_empty[i], 2);
      bar_init(&v_full[i], 1);
      bar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 2; i++) {
      bar_init(&q_full[i], 32);
      bar_init(&q_empty[i], 8);
      bar_init(&drained[i], 1);
      for (int h = 0; h < 2; h++) {
        bar_init(&s_full[i][h], 1);
        bar_init(&p_full[i][h], kTile);
        bar_init(&pv_done[i][h], 1);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    abort_sh = 0;
  }
  fence_before();
  AttnRun run = attn_locate<kItemRows, kKeys, kLead, kSnap>(p, share, blockIdx.x, gridDim.x, kJoin);
  attn_zero_unowned(p);
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_sh;
  AttnCursor& c = run.cur;
  const int length = max((int)(run.total / max(run.ctas, 1)), 1);  // of a run, as all CTAs see it
  unsigned it = 0, asked = 0;  // key and value blocks, items' queries requested so far (by their warps)

  if (warp == kLoadWarp) {
    // ================================================================ TMA
    const int box = min(p.a.kv.page_size, kKeys), boxes = kKeys / box;
    bool ok = true;
    for (int left = run.n; ok && left > 0;) {
      int from, to, lo, hi;
      const int done = run.n - left;
      attn_take<kLead, kSnap>(c, left, &from, &to);
      const int n = to - from;
      const AttnOrder order(c, from, n, done, length);
      item_span(p, c.seq, c.tile, &lo, &hi);
      auto page_of = [&](int b) {  // of this lane's box
        const int j = (c.blk0 + b) * kKeys + lane * box;
        int page = p.a.kv.n_pages;  // outside the tensor
        if (lane < boxes && j < hi && j + box > lo) {
          page = p.a.page_table[(size_t)c.s * p.a.table_stride + (j >> p.page_shift)];
          if (page < 0 || page > p.a.kv.n_pages) page = p.a.kv.n_pages;
        }
        return page;
      };
      int page = n ? page_of(order.block(0)) : 0;
      for (int i = 0; ok && i < n; i++, it++) {
        const int b = order.block(i), next = i + 1 < n ? page_of(order.block(i + 1)) : 0;
        const int slot = it % S;
        const unsigned par = (it / S & 1) ^ 1;
        const int row = ((c.blk0 + b) * kKeys + lane * box) & (p.a.kv.page_size - 1);
        auto copy = [&](const CUtensorMap* map, uint64_t* full, unsigned char* dst) {
          if (lane == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(full)), "r"(Lay::block)
                         : "memory");
          __syncwarp();
          if (lane < boxes)
#pragma unroll
            for (int h = 0; h < DP / 64; h++)
              asm volatile(
                  "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
                  "%3, %4, %5}], [%6];" ::"r"(su32(dst + h * kKvRun + lane * box * 128)),
                  "l"(map), "r"(h * 64), "r"(row), "r"(c.head), "r"(page), "r"(su32(full))
                  : "memory");
        };
        if (!(ok = warp_wait(&k_empty[slot], par, give))) break;
        copy(&args.k_map, &k_full[slot], sm + Lay::k + slot * Lay::block);
        if (!(ok = warp_wait(&v_empty[slot], par, give))) {
          it++;  // (its keys are on the way)
          break;
        }
        copy(&args.v_map, &v_full[slot], sm + Lay::v + slot * Lay::block);
        page = next;
      }
      if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
    }
  } else if (warp == kQueryWarp) {
    // ================================================================ queries, an item ahead
    constexpr int kCh = DP / 8, kStep = 32 / kCh;  // 16-byte chunks of a row, rows of a pass
    const int ch = lane % kCh;
    const bool in = ch * 8 < p.a.kv.head_dim;
    bool ok = true;
    for (int left = run.n; ok && left > 0;) {
      const unsigned seg = asked;
      int from, to;
      attn_take<kLead, kSnap>(c, left, &from, &to);
      if (from == to) {
        if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
        continue;
      }
      if (!(ok = warp_wait(&q_empty[seg & 1], (seg >> 1 & 1) ^ 1, give))) break;
      const int total = c.seq.qn * p.group, r0 = c.tile * kItemRows;
      const uint32_t dst = su32(sm + Lay::q + (seg & 1) * 2 * Lay::tile);
      const int rows = total - r0 > kTile ? kItemRows : kTile;
      if (args.q_boxes) {  // rows beyond the sequence are the next one's or zeros: nobody reads their results
        if (lane == 0) {
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(su32(&q_full[seg & 1])),
                       "r"(rows / kTile * Lay::tile)
                       : "memory");
          for (int i = 0; i < rows / kTile; i++)
#pragma unroll
            for (int h = 0; h < DP / 64; h++)
              asm volatile(
                  "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
                  "%3, %4}], [%5];" ::"r"(dst + i * Lay::tile + h * kQRun),
                  "l"(&args.q_map), "r"(h * 64), "r"(c.head * p.group), "r"(c.seq.q0 + (r0 + i * kTile) / p.group),
                  "r"(su32(&q_full[seg & 1]))
                  : "memory");
        } else {
          bar_arrive(&q_full[seg & 1]);
        }
        asked++;
        if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
        continue;
      }
      const char* const base = (const char*)p.a.q + ch * 16;
      int rr = r0 + lane / kCh, tok = rr / p.group, g = rr - tok * p.group;
      const int step_t = kStep / p.group, step_g = kStep - step_t * p.group;
#pragma unroll 4
      for (int r = lane / kCh; r < rows; r += kStep) {
        const bool have = in && rr < total;
        const int64_t at = have ? ((int64_t)(c.seq.q0 + tok) * p.a.q_stride[0] +
                                   (int64_t)(c.head * p.group + g) * p.a.q_stride[1]) * 2 : -(int64_t)ch * 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         dst + (r >> 7) * Lay::tile + (ch >> 3) * kQRun + (r & 127) * 128 + (((ch & 7) ^ (r & 7)) << 4)),
                     "l"(base + at), "r"(have ? 16 : 0)
                     : "memory");
        rr += kStep;
        tok += step_t;
        g += step_g;
        if (g >= p.group) {
          g -= p.group;
          tok++;
        }
      }
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(su32(&q_full[seg & 1])) : "memory");
      asked++;
      if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // nothing in flight at exit
  } else if (warp >= kMmaWarp) {
    // ================================================================ MMA of tile w
    constexpr uint32_t kIdPv = idesc_f16<T>(DP, 1);
    const uint32_t id_qk = idesc_f16<T>(kKeys, 0) | (p.a.scale < 0.0f ? 1u << 13 : 0u);  // Q negated
    const int w = warp - kMmaWarp;
    const uint64_t dq0 = sw128_desc(sm + Lay::q + w * Lay::tile, 16, 1024);
    const uint64_t dk = sw128_desc(sm + Lay::k, 16, 1024), dv = sw128_desc(sm + Lay::v, kKvRun, 1024);
    const uint32_t ts = tmem + w * kTile, to_ = tmem + 2 * kTile + w * kTile;
    unsigned base = 0;                // blocks of earlier items
    unsigned seg = 0, blocks = 0;     // items, and blocks of this tile so far
    bool ok = true;
    for (int left = run.n; ok && left > 0;) {
      int from, to, lo, hi;
      const int done = run.n - left;
      attn_take<kLead, kSnap>(c, left, &from, &to);
      const int n = to - from;
      const AttnOrder order(c, from, n, done, length);
      if (n == 0) {
        if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
        continue;
      }
      item_span(p, c.seq, c.tile, &lo, &hi);
      const bool mine = w == 0 || c.seq.qn * p.group - c.tile * kItemRows > kTile;
      const uint64_t dq = dq0 + (uint64_t)((seg & 1) * (2 * Lay::tile >> 4));
      // scores of block b into its buffer, whose earlier weights have been read
      auto scores = [&](int b) {
        const unsigned g = base + b, e = blocks + b;
        const int slot = g % S;
        ok = warp_wait(&k_full[slot], g / S & 1, give);
        if (ok && e >= 2) ok = warp_wait(&pv_done[w][e & 1], (e - 2) >> 1 & 1, give);
        if (!ok) return;
        if (elect_one()) {
          fence_after();
          const uint64_t db = dk + (uint64_t)(slot * (Lay::block >> 4));
          const uint32_t d = ts + (e & 1) * kKeys;
#pragma unroll
          for (int s = 0; s < DP / 16; s++)  // 16 columns = 32 bytes a step
            mma_ss(d, dq + (uint64_t)((s / 4) * (kQRun >> 4) + (s % 4) * 2),
                   db + (uint64_t)((s / 4) * (kKvRun >> 4) + (s % 4) * 2), id_qk, s > 0);
          mma_commit(&s_full[w][e & 1]);
          mma_commit(&k_empty[slot]);
        }
      };
      // in both tiles' warps, also for an item of one tile: a wait for a phase is only good if the
      // one before it was seen
      ok = warp_wait(&q_full[seg & 1], seg >> 1 & 1, give);
      if (!mine) {  // the other tile alone: this one's share of the ring's bookkeeping
        for (int b = 0; ok && b < n; b++) {
          const unsigned g = base + b;
          if (!(ok = warp_wait(&k_full[g % S], g / S & 1, give))) break;
          if (lane == 0) bar_arrive(&k_empty[g % S]);
          if (!(ok = warp_wait(&v_full[g % S], g / S & 1, give))) break;
          if (lane == 0) bar_arrive(&v_empty[g % S]);
        }
      } else {
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the copies may be generic writes
        if (ok) scores(0);
        if (ok && n > 1) scores(1);
        for (int b = 0; ok && b < n; b++) {
          const unsigned g = base + b, e = blocks + b;
          const int slot = g % S;
          if (!(ok = warp_wait(&v_full[slot], g / S & 1, give))) break;
          const int j0 = (c.blk0 + order.block(b)) * kKeys;
          const int z0 = max(lo - j0, 0), z1 = min(hi - j0, kKeys);  // rows that the item sees
          if (z0 > 0 || z1 < kKeys) {  // (both tiles' warps write these zeros)
            unsigned char* v = sm + Lay::v + slot * Lay::block;
            for (int r = lane >> 3; r < kKeys; r += 4)
              if (r < z0 || r >= z1)
#pragma unroll
                for (int h = 0; h < DP / 64; h++)
                  *(uint4*)(v + h * kKvRun + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
          }
          if (!(ok = warp_wait(&p_full[w][e & 1], e >> 1 & 1, give))) break;
          if (elect_one()) {
            fence_after();
            const uint64_t db = dv + (uint64_t)(slot * (Lay::block >> 4));
#pragma unroll
            for (int s = 0; s < kKeys / 16; s++)  // 16 keys = 2,048 bytes of V, 8 columns of P a step
              mma_ts(to_, ts + (e & 1) * kKeys + s * 8, db + (uint64_t)(s * 128), kIdPv, b > 0 || s > 0);
            mma_commit(&pv_done[w][e & 1]);
            mma_commit(&v_empty[slot]);
          }
          if (b + 2 < n) scores(b + 2);
        }
        blocks += n;
      }
      seg++;
      base += n;
      if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
    }
  } else {
    // ================================================================ softmax: tile w, this thread's row
    const int w = warp >> 2, t = tid & (kTile - 1);
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + w * kTile + lanes, tO = tmem + 2 * kTile + w * kTile + lanes;
    // not 0, so that a hidden score (-inf) stays one
    const float sl = fmaxf(fabsf(p.a.scale) * 1.44269504088896341f, 1e-37f);
    const int hd = p.a.kv.head_dim;
    unsigned blocks = 0, seg = 0;
    uint64_t* pending = nullptr;  // to arrive on once the TMA store has read the buffer (thread 0)
    auto stored = [&]() {
      if (pending) {
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        bar_arrive(pending);
        pending = nullptr;
      }
    };
    bool ok = true;
    auto wg_sync = [&]() { asm volatile("bar.sync %0, 128;" ::"r"(1 + w) : "memory"); };
    // Whether none of the tile's four warps gave up a wait: they leave together or meet at every wg_sync.
    auto agree = [&](bool mine) {
      int all;
      asm volatile(
          "{ .reg .pred p, q; setp.ne.b32 p, %2, 0; bar.red.and.pred q, %1, 128, p; selp.s32 %0, 1, 0, q; }"
          : "=r"(all)
          : "r"(1 + w), "r"((int)mine)
          : "memory");
      return all != 0;
    };
    for (int left = run.n; ok && left > 0;) {
      int from, to;
      const int done = run.n - left;
      attn_take<kLead, kSnap>(c, left, &from, &to);
      const int n = to - from;
      const AttnOrder order(c, from, n, done, length);
      if (n == 0) {
        if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
        continue;
      }
      const int total = c.seq.qn * p.group, r0 = c.tile * kItemRows + w * kTile;
      unsigned char* const qs = sm + Lay::q + ((seg & 1) * 2 + w) * Lay::tile;  // free once the last scores are in
      uint64_t* const q_done = &q_empty[seg & 1];
      seg++;
      const bool alone = total - c.tile * kItemRows <= kTile;  // one tile only
      if (w == 1 && alone) {  // (tile 0 arrives on q_done for both, when the item is done)
        stored();
        if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
        continue;
      }
      const int r = r0 + t;
      const bool live = r < total;
      const int tok = live ? r / p.group : 0;
      int lo = 0, hi = 0;
      if (live) attn_span(p, c.seq, tok, tok, &lo, &hi);
      float m = -CUDART_INF_F, l = 0.0f;  // m: the maximum that the weights refer to
      for (int b = 0; b < n; b++, blocks++) {
        const int j0 = (c.blk0 + order.block(b)) * kKeys, h = blocks & 1;
        if (!(ok = warp_wait(&s_full[w][h], blocks >> 1 & 1, give))) break;
        fence_after();
        uint32_t s[kKeys];
        tmem_ld32(tS + h * kKeys, s);
        tmem_ld32(tS + h * kKeys + 32, s + 32);
        tmem_wait_ld();
        if (!__all_sync(kFull, lo <= j0 && j0 + kKeys <= hi)) {
          const int a = lo - j0, e = hi - j0;
#pragma unroll
          for (int i = 0; i < kKeys; i++)
            if (i < a || i >= e) s[i] = 0xFF800000u;  // -inf
        }
        float t4[4];
#pragma unroll
        for (int i = 0; i < 4; i++) t4[i] = fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 4]));
#pragma unroll
        for (int i = 8; i < kKeys; i += 8)
#pragma unroll
          for (int e = 0; e < 4; e++) t4[e] = max3(t4[e], __uint_as_float(s[i + e]), __uint_as_float(s[i + e + 4]));
        const float top = max3(fmaxf(t4[0], t4[1]), t4[2], t4[3]);
        const bool grow = b == 0 || m == -CUDART_INF_F ? top > m : (top - m) * sl > 8.0f;
        if (__any_sync(kFull, grow)) {
          const float m2 = grow ? top : m;
          const float f = !grow ? 1.0f : m == -CUDART_INF_F ? 0.0f : ex2((m - m2) * sl);
          l *= f;
          m = m2;
          if (b > 0) {  // O as the product of the block before leaves it
            if (!(ok = warp_wait(&pv_done[w][h ^ 1], (blocks - 1) >> 1 & 1, give))) break;
            fence_after();
#pragma unroll 1
            for (int i = 0; i < DP / 16; i++) {
              uint32_t o[16];
              tmem_ld16(tO + 16 * i, o);
#pragma unroll
              for (int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st16(tO + 16 * i, o);
            }
          }
        }
        const float ref = m == -CUDART_INF_F ? 0.0f : __fmaf_rn(m, sl, -kLift);
        const u64 sl2 = pair(__float_as_uint(sl), __float_as_uint(sl));
        const u64 ref2 = pair(__float_as_uint(-ref), __float_as_uint(-ref));
        u64 l2[2] = {0, 0};
#pragma unroll
        for (int i = 0; i < kKeys; i += 2) {
          float a, e;
          split(fma2(pair(s[i], s[i + 1]), sl2, ref2), a, e);
          a = ex2(a);
          e = ex2(e);
          l2[i / 2 & 1] = add2(l2[i / 2 & 1], pair(__float_as_uint(a), __float_as_uint(e)));
          s[i / 2] = pack2(a, e, T());
        }
        float la, lb;
        split(add2(l2[0], l2[1]), la, lb);
        l += la + lb;
        tmem_st32(tS + h * kKeys, s);
        tmem_wait_st();
        fence_before();
        bar_arrive(&p_full[w][h]);
        stored();  // the item before's, long read by now
      }
      if (ok) ok = warp_wait(&pv_done[w][(blocks - 1) & 1], (blocks - 1) >> 1 & 1, give);
      if (!(ok = agree(ok))) break;
      fence_after();

      // ---- the whole item, or a part of it
      const bool whole = from == 0 && to == c.n_blk;
      bool join = false;
      int c0 = 0, c1 = 0;
      if (!whole) {
        const size_t slot = 2 * (size_t)blockIdx.x + (from == 0 ? 1 : 0);
        const int pr = w * kTile + t;
        parts.ml[slot * kItemRows + pr] = make_float2(m == -CUDART_INF_F ? m : m * sl, l);
#pragma unroll
        for (int i = 0; i < DP / 32; i++) {
          uint32_t o[32];
          tmem_ld32(tO + 32 * i, o);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; e++)  // [dim][row]: a warp's rows are adjacent
            parts.o[(slot * DP + 32 * i + e) * kItemRows + pr] = __uint_as_float(o[e]);
        }
        attn_owners<kLead, kSnap>(run, c, &c0, &c1);
        __threadfence();
        wg_sync();
        if (t == 0) flag_sh[w] = attn_arrive(parts.count + 2 * c0 + w, c1 - c0 + 1);
        wg_sync();
        join = flag_sh[w] != 0;
        if (join) {
          float top = -CUDART_INF_F;
          for (int cc = c0; cc <= c1; cc++)
            top = fmaxf(top, __ldcg(&parts.ml[(2 * (size_t)cc + (cc == c0)) * kItemRows + pr]).x);
          m = top;
          l = 0.0f;
          for (int cc = c0; cc <= c1; cc++) {
            const float2 x = __ldcg(&parts.ml[(2 * (size_t)cc + (cc == c0)) * kItemRows + pr]);
            l = __fmaf_rn(x.y, x.x == -CUDART_INF_F ? 0.0f : ex2(x.x - top), l);
          }
        }
      }
      if (whole || join) {
        const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
        // by way of the queries' shared memory, so that a store covers whole rows and not a piece
        // of 32 of them; a round is DP * 2 bytes of every row.  A full tile in q's type leaves by
        // TMA, which the next item's first block does not wait for.
        const bool boxes = args.o_boxes && r0 + kTile <= total;
        if (boxes && t == 0) pending = q_done;
        auto write = [&](auto wide) {
          constexpr bool kF32 = decltype(wide)::value;
          constexpr int kCh = DP / 8, kDims = kF32 ? 4 : 8;  // chunks of a row and round, dims of a chunk
#pragma unroll
          for (int i = 0; i < DP / 64; i++) {
            uint32_t o[64];
            if (whole) {
              tmem_ld32(tO + 64 * i, o);
              tmem_ld32(tO + 64 * i + 32, o + 32);
              tmem_wait_ld();
            } else {
              const int pr = w * kTile + t;
#pragma unroll
              for (int e = 0; e < 64; e++) o[e] = 0;
#pragma unroll 1
              for (int cc = c0; cc <= c1; cc++) {
                const size_t slot = 2 * (size_t)cc + (cc == c0);
                const float x = __ldcg(&parts.ml[slot * kItemRows + pr]).x;
                const float* src = parts.o + (slot * DP + 64 * i) * kItemRows + pr;
                float y[64];
#pragma unroll
                for (int e = 0; e < 64; e++) y[e] = __ldcg(src + e * kItemRows);
                const float f = x == -CUDART_INF_F ? 0.0f : ex2(x - m);
#pragma unroll
                for (int e = 0; e < 64; e++) o[e] = __float_as_uint(__fmaf_rn(y[e], f, __uint_as_float(o[e])));
              }
            }
#pragma unroll
            for (int z = 0; z < 64 / kDims; z++) {
              const int dim = 64 * i + z * kDims, chunk = dim / kDims % kCh;
              uint4 x;
              if (kF32) {
                x.x = __float_as_uint(__uint_as_float(o[z * 4]) * inv);
                x.y = __float_as_uint(__uint_as_float(o[z * 4 + 1]) * inv);
                x.z = __float_as_uint(__uint_as_float(o[z * 4 + 2]) * inv);
                x.w = __float_as_uint(__uint_as_float(o[z * 4 + 3]) * inv);
              } else {
                uint32_t h[4];
#pragma unroll
                for (int e = 0; e < 4; e++)
                  h[e] = pack2(__uint_as_float(o[(z * 8 + 2 * e) & 63]) * inv,
                               __uint_as_float(o[(z * 8 + 2 * e + 1) & 63]) * inv, T());
                x = make_uint4(h[0], h[1], h[2], h[3]);
              }
              *(uint4*)(qs + (chunk >> 3) * kQRun + t * 128 + (((chunk & 7) ^ (t & 7)) << 4)) = x;
              if (chunk == kCh - 1) {  // the round is full
                if (!kF32 && boxes) {
                  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                  wg_sync();
                  if (t == 0) {
#pragma unroll
                    for (int h = 0; h < DP / 64; h++)
                      asm volatile(
                          "cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                              &args.o_map),
                          "r"(h * 64), "r"(c.head * p.group), "r"(c.seq.q0 + r0 / p.group), "r"(su32(qs + h * kQRun))
                          : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                  }
                  continue;
                }
                wg_sync();
                const int ch = t % kCh, d0 = dim / (kCh * kDims) * (kCh * kDims) + ch * kDims;
                if (d0 < hd) {
                  // token and head of the first row, and their steps
                  int tk = (r0 + t / kCh) / p.group, hh = r0 + t / kCh - tk * p.group;
                  const int step_t = kTile / kCh / p.group, step_h = kTile / kCh - step_t * p.group;
#pragma unroll 4
                  for (int rr = t / kCh; rr < kTile; rr += kTile / kCh) {
                    const size_t to_at = ((size_t)(c.seq.q0 + tk) * p.a.n_q + c.head * p.group + hh) * hd + d0;
                    if (r0 + rr < total)
                      *(uint4*)((char*)p.a.out + to_at * (kF32 ? 4 : 2)) =
                          *(const uint4*)(qs + (ch >> 3) * kQRun + rr * 128 + (((ch & 7) ^ (rr & 7)) << 4));
                    tk += step_t;
                    hh += step_h;
                    if (hh >= p.group) {
                      hh -= p.group;
                      tk++;
                    }
                  }
                }
                wg_sync();
              }
            }
          }
        };
        if (p.a.out_dtype == DPUF_TYPE_F32) write(std::true_type());
        else write(std::false_type());
      }
      // what this thread wrote to and read from the queries' shared memory comes before the TMA load
      // of the item after next into it
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (alone) bar_arrive(q_done);
        if (!pending) bar_arrive(q_done);
      }
      fence_before();  // O is read: the next item's products may overwrite it once its P arrives
      if (left > 0) attn_next_item<kItemRows, kKeys, kLead>(p, c);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // nothing in flight at exit
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (abort_sh) {  // nothing in flight at exit: bounded waits for the copies and the products asked for
    auto settle = [&](uint64_t* bar, unsigned par) {
      const unsigned long long t0 = gtimer();
      while (!bar_try(bar, par) && gtimer() - t0 < kWaitNs / 100) {}
    };
    if (warp == kLoadWarp)
      for (unsigned i = it > S ? it - S : 0; i < it; i++) {
        settle(&k_full[i % S], i / S & 1);
        settle(&v_full[i % S], i / S & 1);
      }
    if (warp == kQueryWarp)
      for (unsigned i = asked > 2 ? asked - 2 : 0; i < asked; i++) settle(&q_full[i & 1], i >> 1 & 1);
    if (warp >= kMmaWarp && warp < kQueryWarp) {
      if (elect_one()) mma_commit(&drained[warp - kMmaWarp]);
      settle(&drained[warp - kMmaWarp], 0);
    }
    __syncthreads();
  }
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                             const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                             CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeFn)f;
  }();
  return fn;
}

// `strides` of dimensions 1.. in elements of 2 bytes.
bool encode(CUtensorMap* map, int dtype, void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
            const cuuint32_t* box) {
  cuuint64_t bytes[3];
  for (int i = 0; i + 1 < rank; i++) bytes[i] = strides[i] * 2;
  const cuuint32_t one[4] = {1, 1, 1, 1};
  return encoder()(map, dtype == DPUF_TYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                   rank, base, dims, bytes, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                   CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP>
cudaError_t launch(const TileArgs& a, cudaStream_t s) {
  const cudaError_t e = smem_limit_once<paged_attention_tc_kernel<T, DP>>(TileLay<DP>::bytes);
  if (e != cudaSuccess) return e;
  paged_attention_tc_kernel<T, DP><<<kAttnSms, kThreads, TileLay<DP>::bytes, s>>>(a);
  return cudaGetLastError();
}

}  // namespace

size_t paged_attention_tc_workspace() { return AttnParts<kItemRows, 128>::bytes(kAttnSms); }

cudaError_t launch_paged_attention_tc(const AttnArgs& p, cudaStream_t s) {
  if (!encoder()) return cudaErrorNotSupported;
  TileArgs a;
  a.p = p;
  const DpufPagedKv& kv = p.a.kv;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.n_kv,
                              (cuuint64_t)kv.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv.row_stride, (cuuint64_t)kv.head_stride, (cuuint64_t)kv.page_stride};
  const cuuint32_t box[4] = {64, (cuuint32_t)std::min(kv.page_size, kKeys), 1, 1};
  if (!encode(&a.k_map, kv.dtype, kv.k, 4, dims, strides, box) || !encode(&a.v_map, kv.dtype, kv.v, 4, dims, strides, box))
    return cudaErrorNotSupported;  // strides that a tensor map cannot hold
  const cuuint64_t q_dims[3] = {(cuuint64_t)kv.head_dim, (cuuint64_t)p.a.n_q, (cuuint64_t)p.a.n_tokens};
  const cuuint64_t q_strides[2] = {(cuuint64_t)p.a.q_stride[1], (cuuint64_t)p.a.q_stride[0]};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)p.group, (cuuint32_t)(kTile / p.group)};
  a.q_boxes = kTile % p.group == 0 && encode(&a.q_map, kv.dtype, (void*)p.a.q, 3, q_dims, q_strides, q_box);
  const cuuint64_t o_strides[2] = {(cuuint64_t)kv.head_dim, (cuuint64_t)p.a.n_q * kv.head_dim};
  a.o_boxes = a.q_boxes && p.a.out_dtype == p.a.dtype && encode(&a.o_map, kv.dtype, p.a.out, 3, q_dims, o_strides, q_box);
  const bool small = kv.head_dim <= 64;
  if (kv.dtype == DPUF_TYPE_F16) return small ? launch<__half, 64>(a, s) : launch<__half, 128>(a, s);
  return small ? launch<__nv_bfloat16, 64>(a, s) : launch<__nv_bfloat16, 128>(a, s);
}

}  // namespace dpuf
