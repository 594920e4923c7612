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

constexpr int kRopeHeads = 4;
constexpr int kRopeThreads = 128;

// Where token t's key and value go: the element offset of (its page, head 0, its row), or -1.
DPUF_DEV int64_t cache_row(const DpufRopeAppendArgs& a, int t, int pos) {
  const int s = a.seq[t];
  const int j = pos / a.kv.page_size;
  if (s < 0 || s >= a.n_seqs || j >= a.pages_per_seq) return -1;
  const int page = a.page_table[(size_t)s * a.table_stride + j];
  if (page < 0 || page >= a.kv.n_pages) return -1;
  return (int64_t)page * a.kv.page_stride + (int64_t)(pos % a.kv.page_size) * a.kv.row_stride;
}

// Units of 16 dimensions (head_dim and rot multiples of 16, everything 16-byte aligned).
template <typename T, bool kInterleaved>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(const __grid_constant__ DpufRopeAppendArgs a) {
  const int units = a.kv.head_dim >> 4;
  const int gq = (a.n_q + kRopeHeads - 1) / kRopeHeads, gk = (a.kv.n_kv + kRopeHeads - 1) / kRopeHeads;
  const int per_token = units * (gq + 2 * gk);
  const int64_t id = (int64_t)blockIdx.x * kRopeThreads + threadIdx.x;
  const int t = (int)(id / per_token);
  if (t >= a.n_tokens) return;
  const int in_token = (int)(id - (int64_t)t * per_token);
  const int c = in_token % units;
  int g = in_token / units;
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
  float lo[kRopeHeads][8], hi[kRopeHeads][8];
#pragma unroll
  for (int i = 0; i < kRopeHeads; i++)
    if (i < nh) {
      load8(x + i * st[1] + d0, lo[i]);
      load8(x + i * st[1] + d1, hi[i]);
    }
  const int pos = a.pos[t];
  const bool in_table = pos >= 0 && pos < a.n_pos;
  if (turn && in_table) {
    float cs[8], sn[8];
    load8(a.cos_tab + (size_t)pos * (a.rotary_dim >> 1) + c * 8, cs);
    load8(a.sin_tab + (size_t)pos * (a.rotary_dim >> 1) + c * 8, sn);
#pragma unroll
    for (int i = 0; i < kRopeHeads; i++)
      if (i < nh) {
        float nl[8], nu[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
          if (kInterleaved) {  // the unit's 16 dimensions are 8 pairs: pair e is element 2e, 2e + 1
            const float p = e < 4 ? lo[i][(2 * e) & 7] : hi[i][(2 * e) & 7];
            const float q = e < 4 ? lo[i][(2 * e + 1) & 7] : hi[i][(2 * e + 1) & 7];
            float* o = e < 4 ? nl : nu;
            o[(2 * e) & 7] = p * cs[e] - q * sn[e];
            o[(2 * e + 1) & 7] = q * cs[e] + p * sn[e];
          } else {
            nl[e] = lo[i][e] * cs[e] - hi[i][e] * sn[e];
            nu[e] = hi[i][e] * cs[e] + lo[i][e] * sn[e];
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          lo[i][e] = nl[e];
          hi[i][e] = nu[e];
        }
      }
  }
  if (kind == 0) {
    if (!in_table) {
      const float fill = pos < 0 ? 0.0f : __int_as_float(0x7FC00000);
#pragma unroll
      for (int i = 0; i < kRopeHeads; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) lo[i][e] = hi[i][e] = fill;
    }
    const size_t o = ((size_t)t * a.n_q + h0) * a.kv.head_dim;
#pragma unroll
    for (int i = 0; i < kRopeHeads; i++)
      if (i < nh) {
        store8_as(a.q_out, o + (size_t)i * a.kv.head_dim + d0, a.out_dtype, lo[i]);
        store8_as(a.q_out, o + (size_t)i * a.kv.head_dim + d1, a.out_dtype, hi[i]);
      }
    return;
  }
  if (!in_table) return;
  const int64_t row = cache_row(a, t, pos);
  if (row < 0) return;
  void* dst = kind == 1 ? a.kv.k : a.kv.v;
#pragma unroll
  for (int i = 0; i < kRopeHeads; i++)
    if (i < nh) {
      const size_t o = (size_t)(row + (int64_t)(h0 + i) * a.kv.head_stride);
      store8_as(dst, o + d0, a.kv.dtype, lo[i]);
      store8_as(dst, o + d1, a.kv.dtype, hi[i]);
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
  const int64_t row = cache_row(a, t, pos);
  if (row < 0) return;
  void* dst = kind == 1 ? a.kv.k : a.kv.v;
  const size_t o = (size_t)(row + (int64_t)h * a.kv.head_stride);
  store_as(dst, o + d0, a.kv.dtype, lo);
  store_as(dst, o + d1, a.kv.dtype, hi);
}

template <typename T>
void launch_units(const DpufRopeAppendArgs& a, unsigned grid, cudaStream_t s) {
  if (a.interleaved) rope_append_kernel<T, true><<<grid, kRopeThreads, 0, s>>>(a);
  else rope_append_kernel<T, false><<<grid, kRopeThreads, 0, s>>>(a);
}

}  // namespace

cudaError_t launch_rope_append(const DpufRopeAppendArgs& a, bool vectors, cudaStream_t s) {
  const int gq = (a.n_q + kRopeHeads - 1) / kRopeHeads, gk = (a.kv.n_kv + kRopeHeads - 1) / kRopeHeads;
  const int64_t threads = vectors ? (int64_t)a.n_tokens * (a.kv.head_dim >> 4) * (gq + 2 * gk)
                                  : (int64_t)a.n_tokens * (a.kv.head_dim >> 1) * (a.n_q + 2 * a.kv.n_kv);
  const int64_t grid = (threads + kRopeThreads - 1) / kRopeThreads;
  if (grid > 0x7FFFFFFF) return cudaErrorInvalidValue;
  if (!vectors) rope_append_pairs_kernel<<<(unsigned)grid, kRopeThreads, 0, s>>>(a);
  else if (a.dtype == DPUF_TYPE_F32) launch_units<float>(a, (unsigned)grid, s);
  else if (a.dtype == DPUF_TYPE_F16) launch_units<__half>(a, (unsigned)grid, s);
  else launch_units<__nv_bfloat16>(a, (unsigned)grid, s);
  return cudaGetLastError();
}

}  // namespace dpuf
