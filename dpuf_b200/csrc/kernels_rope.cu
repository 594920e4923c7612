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

// Any head and rotary size, any alignment of q, k and v: a thread takes one pair (or one
// dimension beyond the turned ones, or one pair of neighbouring dimensions of v).
__global__ void __launch_bounds__(kRopeThreads) rope_append_pairs_kernel(const __grid_constant__ DpufRopeAppendArgs a) {
  const int hd = a.kv.head_dim, half = hd >> 1;
  const int heads = a.n_q + 2 * a.kv.n_kv;
  const int64_t id = (int64_t)blockIdx.x * kRopeThreads + threadIdx.x;
  const int64_t row_id = id / half;
  const int c = (int)(id - row_id * half);
  const int t = (int)(row_id / heads);
  if (t >= a.n_tokens) return;
  int h = (int)(row_id - (int64_t)t * heads);
  const int kind = h < a.n_q ? 0 : h < a.n_q + a.kv.n_kv ? 1 : 2;
  h -= kind == 0 ? 0 : kind == 1 ? a.n_q : a.n_q + a.kv.n_kv;
  const int rh = a.rotary_dim >> 1;
  const bool turn = kind != 2 && c < rh;
  const int d0 = turn && !a.interleaved ? c : 2 * c, d1 = turn && !a.interleaved ? c + rh : 2 * c + 1;
  const int64_t* st = kind == 0 ? a.q_stride : kind == 1 ? a.k_stride : a.v_stride;
  const void* x = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
  const size_t at = (size_t)((int64_t)t * st[0] + (int64_t)h * st[1]);
  float lo = load_as(x, at + d0, a.dtype), hi = load_as(x, at + d1, a.dtype);
  const int pos = a.pos[t];
  const bool in_table = pos >= 0 && pos < a.n_pos;
  if (turn && in_table) {
    const float cs = a.cos_tab[(size_t)pos * rh + c], sn = a.sin_tab[(size_t)pos * rh + c];
    const float p = lo, q = hi;
    lo = p * cs - q * sn;
    hi = q * cs + p * sn;
  }
  if (kind == 0) {
    if (!in_table) lo = hi = pos < 0 ? 0.0f : __int_as_float(0x7FC00000);
    const size_t o = ((size_t)t * a.n_q + h) * hd;
    store_as(a.q_out, o + d0, a.out_dtype, lo);
    store_as(a.q_out, o + d1, a.out_dtype, hi);
    return;
  }
  if (!in_table) return;
  const int64_t row = cache_row(a, a.seq[t], pos);
  if (row < 0) return;
  void* dst = kind == 1 ? a.kv.k : a.kv.v;
  const size_t o = (size_t)(row + (int64_t)h * a.kv.head_stride);
  store_as(dst, o + d0, a.kv.dtype, lo);
  store_as(dst, o + d1, a.kv.dtype, hi);
}

template <typename T>
void launch_units(const DpufRopeAppendArgs& a, int per_token, unsigned grid, cudaStream_t s) {
  const int units = a.kv.head_dim >> 4;
  if (a.interleaved) rope_append_kernel<T, true><<<grid, kRopeThreads, 0, s>>>(a, per_token, units);
  else rope_append_kernel<T, false><<<grid, kRopeThreads, 0, s>>>(a, per_token, units);
}

}  // namespace

cudaError_t launch_rope_append(const DpufRopeAppendArgs& a, bool vectors, cudaStream_t s) {
  const int gq = (a.n_q + kRopeHeads - 1) / kRopeHeads, gk = (a.kv.n_kv + kRopeHeads - 1) / kRopeHeads;
  const int64_t per_token = (int64_t)(a.kv.head_dim >> 4) * (gq + 2 * gk);
  // (the units' kernel counts threads in 32 bits)
  if (vectors && (int64_t)a.n_tokens * per_token + kRopeThreads < ((int64_t)1 << 32)) {
    const unsigned grid = (unsigned)(((int64_t)a.n_tokens * per_token + kRopeThreads - 1) / kRopeThreads);
    if (a.dtype == DPUF_TYPE_F32) launch_units<float>(a, (int)per_token, grid, s);
    else if (a.dtype == DPUF_TYPE_F16) launch_units<__half>(a, (int)per_token, grid, s);
    else launch_units<__nv_bfloat16>(a, (int)per_token, grid, s);
    return cudaGetLastError();
  }
  const int64_t threads = (int64_t)a.n_tokens * (a.kv.head_dim >> 1) * (a.n_q + 2 * a.kv.n_kv);
  const int64_t grid = (threads + kRopeThreads - 1) / kRopeThreads;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  rope_append_pairs_kernel<<<(unsigned)grid, kRopeThreads, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace dpuf
