// attn_plan.cuh - how the paged attention kernels share their work out.
//
// An item is a tile of rows of one sequence and KV head: row r of a sequence is query head
// kv_head * group + r % group of its new token r / group, so all query heads that read a KV head
// sit in the same tiles and its keys are read once for them.  An item walks the key blocks that
// its rows see.  All items' key blocks, laid end to end, are cut into equal runs, one per CTA,
// so that a few long sequences fill the GPU as well as many short ones and ragged batches stay
// balanced; the lengths are read on the device, and the host never waits for them.  An item that
// crosses a cut is computed in parts: each CTA leaves its part's running maximum, sum and
// unnormalised output in the workspace, and the CTA that arrives last (a counter per item, no
// waiting) joins the parts in the order of their keys, so results do not depend on timing.
// An item counts kLead blocks more than it has, for what it costs beside them (queries, results,
// the pipeline's filling): they stand before its first, and a run that ends in them leaves the
// whole item to the next.
// A cut within kSnap places of an item's end moves there: joining parts costs more than the two
// CTAs' work then differs by.
//   part of an item that began in an earlier CTA: slot 2c; part that a later CTA goes on with:
//   slot 2c + 1; the counter is that of the CTA in which the item begins.
#pragma once
#include "serving.cuh"

namespace dpuf {

constexpr int kAttnMaxCtas = 148 * 4;
constexpr int kAttnCounterBytes = (kAttnMaxCtas * 8 + 255) & ~255;

struct AttnArgs {
  DpufPagedAttentionArgs a;
  int group;    // query heads per KV head
  int max_kv;   // positions that a page table row can hold
  int most_q;   // new tokens of a sequence that are looked at (so that 32 bits count its rows)
  int page_shift;
};

struct AttnSeq {
  int q0, qn, kv;  // first new token, new tokens, stored positions
};

DPUF_DEV AttnSeq attn_seq(const AttnArgs& p, int s) {
  AttnSeq i;
  i.q0 = min(max(p.a.q_start[s], 0), p.a.n_tokens);
  i.qn = min(min(max(p.a.q_start[s + 1] - i.q0, 0), p.a.n_tokens - i.q0), p.most_q);
  i.kv = min(max(p.a.kv_len[s], 0), p.max_kv);
  return i;
}

// Positions that the tokens [t0, t1] of a sequence see between them.
DPUF_DEV void attn_span(const AttnArgs& p, const AttnSeq& q, int t0, int t1, int* lo, int* hi) {
  const int first = q.kv - q.qn + t0, last = q.kv - q.qn + t1;
  *hi = p.a.causal ? min(max(last + 1, 0), q.kv) : q.kv;
  *lo = p.a.window > 0 ? max(first - p.a.window + 1, 0) : 0;
}

// Key blocks [*blk0, *blk0 + n) of tile `tile` (at least one, so that rows that see nothing are
// written too).
template <int BM, int BN>
DPUF_DEV int attn_tile_blocks(const AttnArgs& p, const AttnSeq& q, int tile, int* blk0) {
  int lo, hi;
  attn_span(p, q, tile * BM / p.group, min(q.qn - 1, (tile * BM + BM - 1) / p.group), &lo, &hi);
  *blk0 = lo / BN;
  return max((hi + BN - 1) / BN - *blk0, 1);
}

template <int BM>
DPUF_DEV int attn_tiles(const AttnArgs& p, const AttnSeq& q) {
  return (q.qn * p.group + BM - 1) / BM;
}

// A place in the sequence of all key blocks.
struct AttnCursor {
  AttnSeq seq;
  int s, head, tile, tiles;
  int blk0, n_blk;    // the item's key blocks
  int at;             // place within the item, from its lead on
  long long begin;    // the item's first block in the sequence of all
};

// Of an item of n blocks: cuts up to *lo places in move to its start, those from *hi on to its end.
template <int kLead, int kSnap>
DPUF_DEV void attn_snap(int n, int* lo, int* hi) {
  *lo = max(min(kSnap, (n + kLead) / 2), kLead);
  *hi = max(n + kLead - min(kSnap, (n + kLead - 1) / 2), *lo + 1);
}

// The blocks [*from, *to) of the cursor's item that a run with `left` places takes, maybe none.
template <int kLead, int kSnap = 0>
DPUF_DEV void attn_take(const AttnCursor& c, int& left, int* from, int* to) {
  int end = c.at + left, lo, hi;
  attn_snap<kLead, kSnap>(c.n_blk, &lo, &hi);
  left = max(end - (c.n_blk + kLead), 0);
  end = end <= lo ? c.at : end >= hi ? c.n_blk + kLead : end;
  *from = max(c.at - kLead, 0);
  *to = max(end - kLead, 0);
}

// The order in which a run takes its `n` blocks from `from` on of the cursor's item: from a block
// that stands where the run does (`done` places in, modulo a run's length), then round.  The CTAs
// that work on a head's tiles are then at the same keys at the same time, and read them from
// memory once (512 tokens over 33,280 positions: 167 MB instead of 497, of 145).
struct AttnOrder {
  int from, n, first;
  DPUF_DEV AttnOrder(const AttnCursor& c, int from_, int n_, int done, int length) : from(from_), n(n_) {
    int d = (done - c.blk0 - from_) % length;
    if (d < 0) d += length;
    first = d < n_ ? d : 0;
  }
  DPUF_DEV int block(int i) const {
    const int k = i + first;
    return from + (k < n ? k : k - n);
  }
};

template <int BM, int BN, int kLead = 0>
DPUF_DEV void attn_next_item(const AttnArgs& p, AttnCursor& c) {
  c.begin += c.n_blk + kLead;
  c.at = 0;
  if (++c.tile == c.tiles) {
    c.tile = 0;
    if (++c.head == p.a.kv.n_kv) {
      c.head = 0;
      do {
        if (++c.s >= p.a.n_seqs) return;
        c.seq = attn_seq(p, c.s);
        c.tiles = attn_tiles<BM>(p, c.seq);
      } while (c.tiles == 0);
    }
  }
  c.n_blk = attn_tile_blocks<BM, BN>(p, c.seq, c.tile, &c.blk0);
}

struct AttnShare {  // in shared memory
  AttnCursor start;
  long long total;
  long long warp_sum[12];  // of the CTA's warps
  int warp_items[12];
};

struct AttnRun {  // this CTA's run of key blocks
  AttnCursor cur;
  long long total;  // blocks of all items
  int n;            // blocks of this CTA (0: nothing to do)
  int ctas;         // CTAs that have blocks
};

// Key blocks of one KV head of each lane's sequence.  A sequence of many tiles is shared by the
// lanes (a prompt of 2,048 tokens has up to 128, which one thread would walk for microseconds).
template <int BM, int BN, int kLead>
DPUF_DEV long long attn_costs(const AttnArgs& p, const AttnSeq& q) {
  const int lane = threadIdx.x & 31, tiles = attn_tiles<BM>(p, q);
  long long cost = 0;
  int b0;
  unsigned many = __ballot_sync(kFull, tiles > 2);
  if (tiles <= 2)
    for (int t = 0; t < tiles; t++) cost += attn_tile_blocks<BM, BN>(p, q, t, &b0) + kLead;
  for (; many; many &= many - 1) {
    const int j = __ffs(many) - 1;
    const AttnSeq o{__shfl_sync(kFull, q.q0, j), __shfl_sync(kFull, q.qn, j), __shfl_sync(kFull, q.kv, j)};
    long long c = 0;
    for (int t = lane, n = attn_tiles<BM>(p, o); t < n; t += 32) c += attn_tile_blocks<BM, BN>(p, o, t, &b0) + kLead;
#pragma unroll
    for (int i = 16; i; i >>= 1) c += __shfl_xor_sync(kFull, c, i);
    if (lane == j) cost = c;
  }
  return cost;
}
DPUF_DEV long long attn_scan(long long v) {  // inclusive, over the warp
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += t;
  }
  return v;
}

// Fewer CTAs than there are, where an item of n blocks would be cut into more than sqrt(n kJoin)
// parts: a part costs the CTA that joins them about 1 / kJoin of a block's time, one after the other.
//
// All threads of the CTA call this together.  A warp adds up a run of sequences, 32 at a time; the
// warp in whose run the CTA's first block lies finds it.
template <int BM, int BN, int kLead = 0, int kSnap = 0>
DPUF_DEV AttnRun attn_locate(const AttnArgs& p, AttnShare& sh, int cta, int ctas, float join) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int per = (p.a.n_seqs + nw - 1) / nw;
  const int s0 = min(warp * per, p.a.n_seqs), s1 = min(s0 + per, p.a.n_seqs);
  auto seq_of = [&](int s) { return s + lane < s1 ? attn_seq(p, s + lane) : AttnSeq{0, 0, 0}; };
  long long mine = 0, items = 0;
  for (int s = s0; s < s1; s += 32) {
    const AttnSeq q = seq_of(s);
    mine += attn_costs<BM, BN, kLead>(p, q);
    items += attn_tiles<BM>(p, q);
  }
#pragma unroll
  for (int i = 16; i; i >>= 1) {
    mine += __shfl_xor_sync(kFull, mine, i);
    items += __shfl_xor_sync(kFull, items, i);
  }
  mine *= p.a.kv.n_kv;
  if (lane == 0) {
    sh.warp_sum[warp] = mine;
    sh.warp_items[warp] = (int)min(items * p.a.kv.n_kv, (long long)0x7FFFFFF);
  }
  __syncthreads();
  const long long sums = attn_scan(lane < nw ? sh.warp_sum[lane] : 0);
  AttnRun r;
  r.total = __shfl_sync(kFull, sums, 31);
  items = lane < nw ? sh.warp_items[lane] : 0;
#pragma unroll
  for (int i = 16; i; i >>= 1) items += __shfl_xor_sync(kFull, items, i);
  const float parts = items ? fmaxf(sqrtf((float)r.total / (float)items * join), 1.0f) : 0.0f;
  r.ctas = (int)min(min((long long)ctas, r.total), (long long)(parts * (float)items));
  r.n = 0;
  if (cta >= r.ctas) return r;  // the whole CTA
  const long long b = r.total * cta / r.ctas, e = r.total * (cta + 1) / r.ctas;
  r.n = (int)(e - b);
  long long at = __shfl_sync(kFull, sums, warp) - mine;
  if (b >= at && b < at + mine) {  // one warp
    for (int s = s0;; s += 32) {
      AttnCursor c;
      c.seq = seq_of(s);
      const long long k = attn_costs<BM, BN, kLead>(p, c.seq), end = at + attn_scan(k * p.a.kv.n_kv);
      const unsigned in = __ballot_sync(kFull, b < end);
      if (!in) {
        at = __shfl_sync(kFull, end, 31);
        continue;
      }
      const int j = __ffs(in) - 1;
      const long long cost = __shfl_sync(kFull, k, j);
      at = __shfl_sync(kFull, end, j) - cost * p.a.kv.n_kv;
      c.seq = AttnSeq{__shfl_sync(kFull, c.seq.q0, j), __shfl_sync(kFull, c.seq.qn, j), __shfl_sync(kFull, c.seq.kv, j)};
      c.s = s + j;
      c.head = (int)((b - at) / cost);
      at += c.head * cost;
      c.tiles = attn_tiles<BM>(p, c.seq);
      for (int t0 = 0;; t0 += 32) {  // 32 tiles at a time
        c.n_blk = t0 + lane < c.tiles ? attn_tile_blocks<BM, BN>(p, c.seq, t0 + lane, &c.blk0) : 0;
        const int places = t0 + lane < c.tiles ? c.n_blk + kLead : 0;
        const long long tile_end = at + attn_scan(places);
        const unsigned hit = __ballot_sync(kFull, b < tile_end);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            c.tile = t0 + lane;
            c.begin = tile_end - places;
            c.at = (int)(b - c.begin);
            sh.start = c;
          }
          break;
        }
        at = __shfl_sync(kFull, tile_end, 31);
      }
      break;
    }
  }
  __syncthreads();
  r.cur = sh.start;
  int lo, hi;
  attn_snap<kLead, kSnap>(r.cur.n_blk, &lo, &hi);
  if (r.cur.at <= lo) {
    r.n += r.cur.at;
    r.cur.at = 0;
  } else if (r.cur.at >= hi) {
    r.n = max(r.n - (r.cur.n_blk + kLead - r.cur.at), 0);
    if (r.n) attn_next_item<BM, BN, kLead>(p, r.cur);
  }
  return r;
}

// The first and last CTA that have parts of the cursor's item.
template <int kLead = 0, int kSnap = 0>
DPUF_DEV void attn_owners(const AttnRun& r, const AttnCursor& c, int* c0, int* c1) {
  int lo, hi;
  attn_snap<kLead, kSnap>(c.n_blk, &lo, &hi);
  auto holds = [&](long long x) { return (int)(((x + 1) * r.ctas - 1) / r.total); };  // place x of all
  *c0 = holds(c.begin + lo);
  *c1 = holds(c.begin + hi - 1);
}

// Zeros for the tokens before the first sequence's and after the last one's (padding of a batch): each
// CTA takes some of them.
DPUF_DEV void attn_zero_unowned(const AttnArgs& p) {
  const int n = p.a.n_tokens;
  const int first = min(max(p.a.q_start[0], 0), n), end = max(min(p.a.q_start[p.a.n_seqs], n), first);
  const int rows = first + n - end;
  if (rows == 0) return;
  const int64_t bytes = (int64_t)p.a.n_q * p.a.kv.head_dim * (p.a.out_dtype == DPUF_TYPE_F32 ? 4 : 2);  // 16 k
  for (int r = blockIdx.x; r < rows; r += gridDim.x) {
    uint4* const row = (uint4*)((char*)p.a.out + (r < first ? r : r - first + end) * bytes);
    for (int64_t i = threadIdx.x; i < bytes / 16; i += blockDim.x) row[i] = make_uint4(0, 0, 0, 0);
  }
}

// Cache offset (elements) of head 0, row 0 of the page that holds position j of sequence s, or -1.
DPUF_DEV int64_t attn_page(const AttnArgs& p, int s, int j) {
  const int page = p.a.page_table[(size_t)s * p.a.table_stride + (j >> p.page_shift)];
  return page < 0 || page >= p.a.kv.n_pages ? -1 : (int64_t)page * p.a.kv.page_stride;
}

}  // namespace dpuf
