// kernels_rope.cu - rotary positions fused with the store of new keys and values into the paged
// cache.
//
// Per token at position p and pair i of the first rot dimensions, with c = cos_tab[p][i] and
// s = sin_tab[p][i] (the host's tables carry whatever stretches the angles for long contexts):
//   (a, b) -> (a c - b s, b c + a s)
// in fp32, each product and the sum rounded, then one rounding to the stored type.  The tables
// are read and not computed: at position 10^5 an fp32 angle is off by 2^-8, a table made in 64
// bits is not.
//
// Bound by bytes: every element of q, k and v is read once and written once.  A thread takes one
// unit of 16 dimensions (for half layout 8 and their 8 partners) of up to kRopeHeads heads of
// one token, so the 64 bytes of table that a unit needs are read once for those heads instead of
// once per head (a head's unit itself is 32 bytes in 16 bits), and its loads are in flight
// together.  Neighbouring threads take neighbouring units.
#include "serving.cuh"

namespace dpuf {

namespace {

constexpr int kRopeHeads = 2;
constexpr int kRopeThreads = 128;

// Where sequence s's key and value at `pos` go: the element offset of (its page, head 0, its row), or -1.
DPUF_DEV int64_t cache_row(const DpufRopeAppendArgs& a, int s, int pos) {
  const int j = pos / a.kv.page_size;
  if (s < 0 || s >= a.n_seqs || j >= a.pages_per_seq) return -1;
  const int page = a.page_table[(size_t)s * a.table_stride + j];
  if (page < 0 || page >= a.kv.n_pages) return -1;
  return (int64_t)page * a.kv.page_stride + (int64_t)(pos % a.kv.page_size) * a.kv.row_stride;
}

// Eight elements as they were loaded.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  DPUF_DEV void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = __ldcs((const uint4*)p + i);
  }
  DPUF_DEV void values(float (&v)[8]) const { load8((const T*)w, v); }
};

// Units of 16 dimensions (head_dim and rot multiples of 16, everything 16-byte aligned).
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ DpufRopeAppendArgs a,
                                                                    int per_token, int units) {
  // 32 bits hold a block's first thread for any grid, and divide faster
  const unsigned id = blockIdx.x * (unsigned)kRopeThreads + threadIdx.x;
  const int t = (int)(id / (unsigned)per_token);
  if (t >= a.n_tokens) return;
  const int pos = __ldg(a.pos + t), seq = __ldg(a.seq + t);
  const int in_token = (int)(id - (unsigned)t * (unsigned)per_token);
  int g = in_token / units;
  const int c = in_token - g * units;
  const int gq = (a.n_q + kRopeHeads - 1) / kRopeHeads, gk = (a.kv.n_kv + kRopeHeads - 1) / kRopeHeads;
  const int kind = g < gq ? 0 : g < gq + gk ? 1 : 2;  // q, k, v
  g -= kind == 0 ? 0 : kind == 1 ? gq : gq + gk;
  const int heads = kind == 0 ? a.n_q : a.kv.n_kv;
  const int h0 = g * kRopeHeads, nh = min(kRopeHeads, heads - h0);
  const bool turn = kind != 2 && c * 16 < a.rotary_dim;
  // the unit's two runs of 8 dimensions
  const int d0 = turn && !kInterleaved ? c * 8 : c * 16;
  const int d1 = turn && !kInterleaved ? c * 8 + (a.rotary_dim >> 1) : c * 16 + 8;

  const int64_t* st = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
  const T* x = (const T*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (int64_t)t * st[0] + (int64_t)h0 * st[1];
  Raw8<T> raw0[kRopeHeads], raw1[kRopeHeads];
#pragma unroll
  for (int i = 0; i < kRopeHeads; i++)
    if (i < nh) {
      raw0[i].load(x + i * st[1] + d0);
      raw1[i].load(x + i * st[1] + d1);
    }
  const bool in_table = pos >= 0 && pos < a.n_pos;
  const int64_t row = kind == 0 || !in_table ? -1 : cache_row(a, seq, pos);
  float cs[8], sn[8];
  if (turn && in_table) {
    load8(a.cos_tab + (size_t)pos * (a.rotary_dim >> 1) + c * 8, cs);
    load8(a.sin_tab + (size_t)pos * (a.rotary_dim >> 1) + c * 8, sn);
  }
  if (kind != 0 && row < 0) return;
  void* const dst = kind == 0 ? a.q_out : kind == 1 ? a.kv.k : a.kv.v;
  const int type = kind == 0 ? a.out_dtype : a.kv.dtype;
  const int64_t step = kind == 0 ? a.kv.head_dim : a.kv.head_stride;
  int64_t o = kind == 0 ? ((int64_t)t * a.n_q + h0) * a.kv.head_dim : row + (int64_t)h0 * a.kv.head_stride;
#pragma unroll
  for (int i = 0; i < kRopeHeads; i++, o += step)
    if (i < nh) {
      float lo[8], hi[8];
      raw0[i].values(lo);
      raw1[i].values(hi);
      if (!in_table) {  // a query of padding, or without a table row
#pragma unroll
        for (int e = 0; e < 8; e++) lo[e] = hi[e] = pos < 0 ? 0.0f : __int_as_float(0x7FC00000);
      } else if (turn) {
        if (kInterleaved) {  // the unit's 16 dimensions are 8 pairs: pair e is elements 2e, 2e + 1
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float p0 = lo[2 * e], q0 = lo[2 * e + 1], p1 = hi[2 * e], q1 = hi[2 * e + 1];
            lo[2 * e] = p0 * cs[e] - q0 * sn[e];
            lo[2 * e + 1] = q0 * cs[e] + p0 * sn[e];
            hi[2 * e] = p1 * cs[e + 4] - q1 * sn[e + 4];
            hi[2 * e + 1] = q1 * cs[e + 4] + p1 * sn[e + 4];
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float p = lo[e], q = hi[e];
            lo[e] = p * cs[e] - q * sn[e];
            hi[e] = q * cs[e] + p * sn[e];
          }
        }
      }
      store8_as(dst, (size_t)o + d0, type, lo);
      store8_as(dst, (size_t)o + d1, type, hi);
    }
}

// Any rotary size, any alignment of q, k and v: a thread takes 8 neighbouring dimensions, as one
// access where q, k and v are 16-byte aligned, and fetches the partners of the turned ones one by
// one (they are another thread's run, so from the cache).  A head's threads are in one warp, which
// has read all of the head before it writes any: q may be turned in place.
template <typename T>
__global__ void __launch_bounds__(kRopeThreads) rope_append_runs_kernel(const __grid_constant__ DpufRopeAppendArgs a,
                                                                         int aligned) {
  const int hd = a.kv.head_dim, runs = hd >> 3, rh = a.rotary_dim >> 1;
  const int heads = a.n_q + 2 * a.kv.n_kv;
  const int lane = threadIdx.x & 31, per_warp = 32 / runs, in_warp = lane / runs;
  const int64_t row_id = ((int64_t)blockIdx.x * (kRopeThreads / 32) + (threadIdx.x >> 5)) * per_warp + in_warp;
  const int d0 = (lane - in_warp * runs) * 8;
  const int64_t tok = row_id / heads;
  const bool live = in_warp < per_warp && tok < a.n_tokens;
  const int t = live ? (int)tok : 0;
  const int pos = __ldg(a.pos + t), seq = __ldg(a.seq + t);
  int h = live ? (int)(row_id - tok * heads) : 0;
  const int kind = h < a.n_q ? 0 : h < a.n_q + a.kv.n_kv ? 1 : 2;
  h -= kind == 0 ? 0 : kind == 1 ? a.n_q : a.n_q + a.kv.n_kv;
  const int64_t* st = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
  const T* x = (const T*)(kind == 0 ? a.q : kind == 1 ? a.k : a.v) + (int64_t)t * st[0] + (int64_t)h * st[1];
  float v[8];
  if (aligned) {
    load8(x + d0, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = to_f32(x[d0 + e]);
  }
  const bool in_table = pos >= 0 && pos < a.n_pos;
  const int64_t row = kind == 0 || !in_table ? -1 : cache_row(a, seq, pos);
  if (!in_table) {  // a query of padding, or without a table row
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = pos < 0 ? 0.0f : __int_as_float(0x7FC00000);
  } else if (kind != 2 && d0 < a.rotary_dim) {
    const float* const cs = a.cos_tab + (size_t)pos * rh;
    const float* const sn = a.sin_tab + (size_t)pos * rh;
    if (a.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        if (d0 + e < a.rotary_dim) {
          const int i = (d0 + e) >> 1;
          const float p = v[e], q = v[e + 1];
          v[e] = p * cs[i] - q * sn[i];
          v[e + 1] = q * cs[i] + p * sn[i];
        }
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) {
        const int d = d0 + e;
        if (d < rh) v[e] = v[e] * cs[d] - to_f32(x[d + rh]) * sn[d];
        else if (d < a.rotary_dim) v[e] = v[e] * cs[d - rh] + to_f32(x[d - rh]) * sn[d - rh];
      }
    }
  }
  __syncwarp();
  if (!live || (kind != 0 && row < 0)) return;
  if (kind == 0) {
    const size_t o = ((size_t)t * a.n_q + h) * hd + d0;
    if (aligned) {
      store8_as(a.q_out, o, a.out_dtype, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) store_as(a.q_out, o + e, a.out_dtype, v[e]);
    }
    return;
  }
  store8_as(kind == 1 ? a.kv.k : a.kv.v, (size_t)(row + (int64_t)h * a.kv.head_stride) + d0, a.kv.dtype, v);
}

template <typename T>
void launch_runs(const DpufRopeAppendArgs& a, bool aligned, unsigned grid, cudaStream_t s) {
  rope_append_runs_kernel<T><<<grid, kRopeThreads, 0, s>>>(a, aligned);
}

template <typename T>
void launch_units(const DpufRopeAppendArgs& a, int per_token, unsigned grid, cudaStream_t s) {
  const int units = a.kv.head_dim >> 4;
  if (a.interleaved) rope_append_kernel<T, true><<<grid, kRopeThreads, 0, s>>>(a, per_token, units);
  else rope_append_kernel<T, false><<<grid, kRopeThreads, 0, s>>>(a, per_token, units);
}

}  // namespace

cudaError_t launch_rope_append(const DpufRopeAppendArgs& a, bool aligned, cudaStream_t s) {
  const int gq = (a.n_q + kRopeHeads - 1) / kRopeHeads, gk = (a.kv.n_kv + kRopeHeads - 1) / kRopeHeads;
  const int64_t per_token = (int64_t)(a.kv.head_dim >> 4) * (gq + 2 * gk);
  // Units of 16 dimensions where sizes and alignment allow (and 32 bits count the threads); 8,191
  // tokens of 32 + 2 x 8 heads of 128 in bf16, half turned: 42 us, as runs of 8: 66 us.
  if (aligned && a.kv.head_dim % 16 == 0 && a.rotary_dim % 16 == 0 &&
      (int64_t)a.n_tokens * per_token + kRopeThreads < ((int64_t)1 << 32)) {
    const unsigned grid = (unsigned)(((int64_t)a.n_tokens * per_token + kRopeThreads - 1) / kRopeThreads);
    if (a.dtype == DPUF_TYPE_F32) launch_units<float>(a, (int)per_token, grid, s);
    else if (a.dtype == DPUF_TYPE_F16) launch_units<__half>(a, (int)per_token, grid, s);
    else launch_units<__nv_bfloat16>(a, (int)per_token, grid, s);
    return cudaGetLastError();
  }
  const int64_t per_block = (int64_t)(kRopeThreads / 32) * (32 / (a.kv.head_dim >> 3));  // heads
  const int64_t grid = ((int64_t)a.n_tokens * (a.n_q + 2 * a.kv.n_kv) + per_block - 1) / per_block;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (a.dtype == DPUF_TYPE_F32) launch_runs<float>(a, aligned, (unsigned)grid, s);
  else if (a.dtype == DPUF_TYPE_F16) launch_runs<__half>(a, aligned, (unsigned)grid, s);
  else launch_runs<__nv_bfloat16>(a, aligned, (unsigned)grid, s);
  return cudaGetLastError();
}

}  // namespace dpuf
