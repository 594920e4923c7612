// kernels_paged_attn.cu - attention of new tokens over the paged cache.
//
// One pass over the keys with the running maximum m and sum l of the softmax: for a block of
// keys with scores s_j = scale * q . k_j,
//   m' = max(m, max s_j),  p_j = exp(s_j - m'),  l' = l e^{m-m'} + sum p_j,
//   o' = o e^{m-m'} + sum p_j v_j,  at the end out = o / l (0 where l = 0).
// Scores are kept in units of log 2 (scale * log2(e) is folded into the product), so every
// exponential is one ex2.  A row that has seen nothing has m = -inf and l = 0.  A score that is NaN
// does not raise m, but makes l and o NaN; they stay that whatever they are multiplied by.
#include <math_constants.h>

#include <algorithm>

#include "attn_parts.cuh"

namespace dpuf {

namespace {

constexpr float kLog2e = 1.44269504088896341f;

DPUF_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ fp32 arithmetic, any types
// Chunks over an fp32 cache, and fp32 queries of heads over 128.  Bound by shared-memory reads (a
// float4 of K or V feeds 4 or 8 multiply-adds).  A CTA takes 16 rows and blocks of 32 keys, both widened to fp32 in shared memory.  Thread
// (row = tid / 16, x = tid % 16) has the scores of keys x and x + 16 and the output's dimensions
// 4 x + 64 i of its row; a row's 16 threads are half a warp.
constexpr int kGenRows = 16, kGenKeys = 32, kGenThreads = 256;
constexpr float kJoin = 8.0f;

template <typename TK, int DP>  // DP: head_dim rounded up to 64, 128 or 256
__global__ void __launch_bounds__(kGenThreads) paged_attention_f32_kernel(const __grid_constant__ AttnArgs p) {
  extern __shared__ __align__(16) float sm[];
  constexpr int kStride = DP + 4;  // rows 16 bytes apart in banks: eight rows' float4 do not collide
  float* qs = sm;                              // [kGenRows][DP]
  float* ks = qs + kGenRows * DP;              // [kGenKeys][kStride]
  float* vs = ks + kGenKeys * kStride;         // [kGenKeys][kStride]
  float* ps = vs + kGenKeys * kStride;         // [kGenRows][kGenKeys + 1]
  __shared__ AttnShare share;
  __shared__ int flag;
  const int tid = threadIdx.x, row = tid >> 4, x = tid & 15;
  const int hd = p.a.kv.head_dim;
  AttnRun run = attn_locate<kGenRows, kGenKeys>(p, share, blockIdx.x, gridDim.x, kJoin);
  attn_zero_unowned(p);
  if (run.n == 0) return;
  const AttnParts<kGenRows, DP> parts(p.a.workspace, gridDim.x);
  AttnCursor& c = run.cur;
  const float scale = p.a.scale * kLog2e;

  for (int left = run.n; left > 0;) {
    const int from = c.at, to = min(c.n_blk, c.at + left);
    left -= to - from;
    // ---- the item's rows
    const int r0 = c.tile * kGenRows, r = r0 + row;
    const bool live = r < c.seq.qn * p.group;
    const int tok = live ? r / p.group : 0, head = c.head * p.group + (live ? r % p.group : 0);
    __syncthreads();
    for (int i = tid; i < kGenRows * DP; i += kGenThreads) {
      const int rr = r0 + i / DP, d = i % DP;
      float v = 0.0f;
      if (rr < c.seq.qn * p.group && d < hd)
        v = load_as(p.a.q, (size_t)((int64_t)(c.seq.q0 + rr / p.group) * p.a.q_stride[0] +
                                    (int64_t)(c.head * p.group + rr % p.group) * p.a.q_stride[1] + d), p.a.dtype);
      qs[i] = v;
    }
    int lo = 0, hi = 0;  // positions that this row sees
    if (live) attn_span(p, c.seq, tok, tok, &lo, &hi);
    int tlo, thi;        // positions that the tile sees
    attn_span(p, c.seq, r0 / p.group, min(c.seq.qn - 1, (r0 + kGenRows - 1) / p.group), &tlo, &thi);
    float m = -CUDART_INF_F, l = 0.0f;
    float o[DP / 64][4] = {};

    for (int b = from; b < to; b++) {
      const int j0 = (c.blk0 + b) * kGenKeys;
      __syncthreads();
      for (int i = tid; i < kGenKeys * (DP / 8); i += kGenThreads) {
        const int key = i / (DP / 8), d = i % (DP / 8) * 8, j = j0 + key;
        float kv[8] = {}, vv[8] = {};
        if (j >= tlo && j < thi && d < hd) {
          const int64_t page = attn_page(p, c.s, j);
          if (page >= 0) {
            const int64_t at = page + (int64_t)c.head * p.a.kv.head_stride +
                               (int64_t)(j & (p.a.kv.page_size - 1)) * p.a.kv.row_stride + d;
            load8((const TK*)p.a.kv.k + at, kv);
            load8((const TK*)p.a.kv.v + at, vv);
          }
        }
        store8_as(ks, key * kStride + d, DPUF_TYPE_F32, kv);
        store8_as(vs, key * kStride + d, DPUF_TYPE_F32, vv);
      }
      __syncthreads();
      float s0 = 0.0f, s1 = 0.0f;
#pragma unroll 8
      for (int d = 0; d < DP; d += 4) {
        const float4 q = *(const float4*)(qs + row * DP + d);
        const float4 a = *(const float4*)(ks + x * kStride + d), e = *(const float4*)(ks + (x + 16) * kStride + d);
        s0 = fmaf(q.x, a.x, fmaf(q.y, a.y, fmaf(q.z, a.z, fmaf(q.w, a.w, s0))));
        s1 = fmaf(q.x, e.x, fmaf(q.y, e.y, fmaf(q.z, e.z, fmaf(q.w, e.w, s1))));
      }
      s0 = j0 + x >= lo && j0 + x < hi ? s0 * scale : -CUDART_INF_F;
      s1 = j0 + x + 16 >= lo && j0 + x + 16 < hi ? s1 * scale : -CUDART_INF_F;
      float top = fmaxf(s0, s1);
#pragma unroll
      for (int i = 8; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, i));
      const bool sees = j0 < hi && j0 + kGenKeys > lo;  // this row, of the block
      if (sees) {
        // (a NaN score does not raise the maximum, but reaches l and o: the factors are never skipped)
        const float m2 = fmaxf(m, top), ref = m2 == -CUDART_INF_F ? 0.0f : m2;
        const float f = m == -CUDART_INF_F ? 0.0f : ex2(m - m2);
        const float p0 = ex2(s0 - ref), p1 = ex2(s1 - ref);
        ps[row * (kGenKeys + 1) + x] = p0;
        ps[row * (kGenKeys + 1) + x + 16] = p1;
        l = fmaf(l, f, p0 + p1);  // this thread's keys only; summed over the row at the end
        m = m2;
#pragma unroll
        for (int i = 0; i < DP / 64; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[i][e] *= f;
      }
      __syncwarp();
      if (sees)
        for (int k = 0; k < kGenKeys; k++) {
          const float w = ps[row * (kGenKeys + 1) + k];
#pragma unroll
          for (int i = 0; i < DP / 64; i++) {
            const float4 v = *(const float4*)(vs + k * kStride + 64 * i + 4 * x);
            o[i][0] = fmaf(w, v.x, o[i][0]);
            o[i][1] = fmaf(w, v.y, o[i][1]);
            o[i][2] = fmaf(w, v.z, o[i][2]);
            o[i][3] = fmaf(w, v.w, o[i][3]);
          }
        }
    }
#pragma unroll
    for (int i = 8; i; i >>= 1) l += __shfl_xor_sync(kFull, l, i);

    // ---- the whole item, or a part of it
    const bool whole = from == 0 && to == c.n_blk;
    bool join = false;
    int c0 = 0, c1 = 0;
    if (!whole) {
      const size_t slot = 2 * (size_t)blockIdx.x + (from == 0 ? 1 : 0);
      if (x == 0) parts.ml[slot * kGenRows + row] = make_float2(m, l);
#pragma unroll
      for (int i = 0; i < DP / 64; i++)
        *(float4*)(parts.o + (slot * kGenRows + row) * DP + 64 * i + 4 * x) =
            make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
      attn_owners(run, c, &c0, &c1);
      join = attn_last_part(parts.count + 2 * c0, c1 - c0 + 1, &flag);
      if (join) {
        m = -CUDART_INF_F;
        for (int cc = c0; cc <= c1; cc++)
          m = fmaxf(m, __ldcg(&parts.ml[(2 * (size_t)cc + (cc == c0 ? 1 : 0)) * kGenRows + row]).x);
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < DP / 64; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[i][e] = 0.0f;
        for (int cc = c0; cc <= c1; cc++) {
          const size_t at = (2 * (size_t)cc + (cc == c0 ? 1 : 0)) * kGenRows + row;
          const float2 part = __ldcg(&parts.ml[at]);
          const float f = part.x == -CUDART_INF_F ? 0.0f : ex2(part.x - m);
          l = fmaf(part.y, f, l);
#pragma unroll
          for (int i = 0; i < DP / 64; i++) {
            const float4 v = __ldcg((const float4*)(parts.o + at * DP + 64 * i + 4 * x));
            o[i][0] = fmaf(v.x, f, o[i][0]);
            o[i][1] = fmaf(v.y, f, o[i][1]);
            o[i][2] = fmaf(v.z, f, o[i][2]);
            o[i][3] = fmaf(v.w, f, o[i][3]);
          }
        }
      }
    }
    if ((whole || join) && live) {
      const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
      const size_t at = ((size_t)(c.seq.q0 + tok) * p.a.n_q + head) * hd;
#pragma unroll
      for (int i = 0; i < DP / 64; i++)
#pragma unroll
        for (int e = 0; e < 4; e++)
          if (64 * i + 4 * x + e < hd) store_as(p.a.out, at + 64 * i + 4 * x + e, p.a.out_dtype, o[i][e] * inv);
    }
    if (left > 0) attn_next_item<kGenRows, kGenKeys>(p, c);
  }
}

// ------------------------------------------------------------------ fp32 cache, up to 4 rows
// Decode steps.  Bound by the bytes of K and V: eight lanes take a key, each some of its dimensions
// straight into registers (a step ahead), so a warp has four keys at a time and nothing goes
// through shared memory but the queries; the eight lanes' sums meet in three shuffles a row.  Every
// group of eight lanes keeps a softmax of its own; they are joined at the item's end.
constexpr int kFewRows = 4, kFewWarps = 4, kFewKeys = 64;
constexpr float kFewJoin = 16.0f;
// CTAs an SM: registers for all that is in flight (64 tokens at 2,304, head_dim 128: 220 us with 2, 305
// with 3, which spills; 2 tokens at 10,029, head_dim 64: 38 and 36).
__host__ __device__ constexpr int few_ctas(int dp) { return dp == 64 ? 3 : 2; }

template <int DP>  // head_dim rounded up to 64 or 128
__global__ void __launch_bounds__(kFewWarps * 32, few_ctas(DP)) paged_attention_f32_few_kernel(const __grid_constant__ AttnArgs p) {
  constexpr int R = kFewRows, NV = DP / 32, kStep = kFewWarps * 4;  // float4 of a lane, keys of a step
  __shared__ AttnShare share;
  __shared__ int flag;
  __shared__ __align__(16) float qs[R][DP];
  __shared__ __align__(16) float merge[kFewWarps][R][DP];
  __shared__ float2 ml_sh[kFewWarps][R];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, grp = lane >> 3, gl = lane & 7;
  const int hd = p.a.kv.head_dim;
  AttnRun run = attn_locate<R, kFewKeys>(p, share, blockIdx.x, gridDim.x, kFewJoin);
  attn_zero_unowned(p);
  if (run.n == 0) return;
  const AttnParts<R, DP> parts(p.a.workspace, gridDim.x);
  AttnCursor& c = run.cur;

  for (int left = run.n; left > 0;) {
    const int from = c.at, to = min(c.n_blk, c.at + left);
    left -= to - from;
    const int total = c.seq.qn * p.group, r0 = c.tile * R, rows = min(R, total - r0);
    __syncthreads();
    for (int i = tid; i < R * DP; i += kFewWarps * 32) {
      const int r = i / DP, d = i % DP, tok = (r0 + r) / p.group;
      qs[r][d] = r < rows && d < hd ? load_as(p.a.q, (size_t)((int64_t)(c.seq.q0 + tok) * p.a.q_stride[0] +
                                              (int64_t)(c.head * p.group + r0 + r - tok * p.group) * p.a.q_stride[1] + d),
                                              p.a.dtype) * (p.a.scale * kLog2e)
                                    : 0.0f;
    }
    int lo[R], hi[R];  // positions that each row sees
#pragma unroll
    for (int r = 0; r < R; r++) {
      lo[r] = hi[r] = 0;
      if (r < rows) attn_span(p, c.seq, (r0 + r) / p.group, (r0 + r) / p.group, &lo[r], &hi[r]);
    }
    int tlo, thi;  // positions that the tile sees
    attn_span(p, c.seq, r0 / p.group, min(c.seq.qn - 1, (r0 + R - 1) / p.group), &tlo, &thi);
    __syncthreads();
    float m[R], l[R], o[R][NV * 4];
#pragma unroll
    for (int r = 0; r < R; r++) {
      m[r] = -CUDART_INF_F;
      l[r] = 0.0f;
#pragma unroll
      for (int e = 0; e < NV * 4; e++) o[r][e] = 0.0f;
    }
    const int first = (c.blk0 + from) * kFewKeys + warp * 4 + grp, steps = (to - from) * (kFewKeys / kStep);
    auto page_of = [&](int step) -> int64_t {
      const int j = first + step * kStep;
      return step < steps && j >= tlo && j < thi ? attn_page(p, c.s, j) : -1;
    };
    float4 k[NV], v[NV];
    auto fetch = [&](int step, int64_t page, float4 (&kk)[NV], float4 (&vv)[NV]) {
      const int j = first + step * kStep;
      const int64_t at = page + (int64_t)c.head * p.a.kv.head_stride +
                         (int64_t)(j & (p.a.kv.page_size - 1)) * p.a.kv.row_stride + gl * 4;
#pragma unroll
      for (int i = 0; i < NV; i++) {
        kk[i] = vv[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (page >= 0 && i * 32 + gl * 4 < hd) {
          kk[i] = __ldcs((const float4*)((const float*)p.a.kv.k + at + i * 32));
          vv[i] = __ldcs((const float4*)((const float*)p.a.kv.v + at + i * 32));
        }
      }
    };
    int64_t page = page_of(0);
    fetch(0, page, k, v);
    page = page_of(1);
    for (int step = 0; step < steps; step++) {
      float4 k2[NV], v2[NV];
      fetch(step + 1, page, k2, v2);
      page = page_of(step + 2);
      const int j = first + step * kStep;
      float s[R], f[R];
#pragma unroll
      for (int r = 0; r < R; r++) {
        s[r] = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; i++) {
          const float4 q = *(const float4*)&qs[r][i * 32 + gl * 4];
          s[r] = fmaf(q.x, k[i].x, fmaf(q.y, k[i].y, fmaf(q.z, k[i].z, fmaf(q.w, k[i].w, s[r]))));
        }
      }
      bool grew = false;
#pragma unroll
      for (int r = 0; r < R; r++) {
#pragma unroll
        for (int i = 1; i < 8; i <<= 1) s[r] += __shfl_xor_sync(kFull, s[r], i);
        if (!(j >= lo[r] && j < hi[r])) s[r] = -CUDART_INF_F;
        const float m2 = fmaxf(m[r], s[r]);
        f[r] = m2 == m[r] ? 1.0f : ex2(m[r] - m2);
        s[r] = s[r] == -CUDART_INF_F ? 0.0f : ex2(s[r] - m2);
        grew = grew || f[r] != 1.0f;
        l[r] = fmaf(l[r], f[r], s[r]);
        m[r] = m2;
      }
      if (__any_sync(kFull, grew))
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int e = 0; e < NV * 4; e++) o[r][e] *= f[r];
#pragma unroll
      for (int r = 0; r < R; r++)
#pragma unroll
        for (int i = 0; i < NV; i++) {
          o[r][4 * i] = fmaf(s[r], v[i].x, o[r][4 * i]);
          o[r][4 * i + 1] = fmaf(s[r], v[i].y, o[r][4 * i + 1]);
          o[r][4 * i + 2] = fmaf(s[r], v[i].z, o[r][4 * i + 2]);
          o[r][4 * i + 3] = fmaf(s[r], v[i].w, o[r][4 * i + 3]);
        }
#pragma unroll
      for (int i = 0; i < NV; i++) {
        k[i] = k2[i];
        v[i] = v2[i];
      }
    }
    // ---- the warp's four groups, then the warps
#pragma unroll
    for (int r = 0; r < R; r++) {
#pragma unroll
      for (int x = 8; x < 32; x <<= 1) {
        const float om = __shfl_xor_sync(kFull, m[r], x), ol = __shfl_xor_sync(kFull, l[r], x);
        const float m2 = fmaxf(m[r], om);
        const float g = m[r] == -CUDART_INF_F ? 0.0f : ex2(m[r] - m2), og = om == -CUDART_INF_F ? 0.0f : ex2(om - m2);
        l[r] = l[r] * g + ol * og;
        m[r] = m2;
#pragma unroll
        for (int e = 0; e < NV * 4; e++) {
          const float y = __shfl_xor_sync(kFull, o[r][e], x);
          o[r][e] = o[r][e] * g + y * og;
        }
      }
      if (grp == 0)
#pragma unroll
        for (int i = 0; i < NV; i++)
          *(float4*)&merge[warp][r][i * 32 + gl * 4] =
              make_float4(o[r][4 * i], o[r][4 * i + 1], o[r][4 * i + 2], o[r][4 * i + 3]);
      if (lane == 0) ml_sh[warp][r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    const bool whole = from == 0 && to == c.n_blk;
    const int r = tid / (DP / 4), d = tid % (DP / 4) * 4;  // one float4 of the tile's output a thread
    const bool mine = r < rows;
    float top = -CUDART_INF_F, sum = 0.0f;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    auto add = [&](float2 ml, float4 y) {
      const float g = ml.x == -CUDART_INF_F ? 0.0f : ex2(ml.x - top);
      sum = fmaf(ml.y, g, sum);
      x.x = fmaf(y.x, g, x.x);
      x.y = fmaf(y.y, g, x.y);
      x.z = fmaf(y.z, g, x.z);
      x.w = fmaf(y.w, g, x.w);
    };
    if (mine) {
#pragma unroll
      for (int w = 0; w < kFewWarps; w++) top = fmaxf(top, ml_sh[w][r].x);
#pragma unroll
      for (int w = 0; w < kFewWarps; w++) add(ml_sh[w][r], *(const float4*)&merge[w][r][d]);
    }
    bool join = false;
    if (!whole) {
      const size_t slot = 2 * (size_t)blockIdx.x + (from == 0 ? 1 : 0);
      if (mine) {
        if (d == 0) parts.ml[slot * R + r] = make_float2(top, sum);
        *(float4*)(parts.o + (slot * R + r) * DP + d) = x;
      }
      int c0, c1;
      attn_owners(run, c, &c0, &c1);
      join = attn_last_part(parts.count + 2 * c0, c1 - c0 + 1, &flag);
      if (join && mine) {
        top = -CUDART_INF_F;
        sum = 0.0f;
        x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        auto at = [&](int cc) { return (2 * (size_t)cc + (cc == c0)) * R + r; };
#pragma unroll 8
        for (int cc = c0; cc <= c1; cc++) top = fmaxf(top, __ldcg(&parts.ml[at(cc)]).x);
#pragma unroll 8
        for (int cc = c0; cc <= c1; cc++) add(__ldcg(&parts.ml[at(cc)]), __ldcg((const float4*)(parts.o + at(cc) * DP + d)));
      }
    }
    if ((whole || join) && mine && d < hd) {
      const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
      const int tok = (r0 + r) / p.group, head = c.head * p.group + r0 + r - tok * p.group;
      store4_as(p.a.out, ((size_t)(c.seq.q0 + tok) * p.a.n_q + head) * hd + d, p.a.out_dtype, x.x * inv, x.y * inv,
                x.z * inv, x.w * inv);
    }
    if (left > 0) attn_next_item<R, kFewKeys>(p, c);
  }
}

template <typename TK, int DP>
cudaError_t launch_f32(const AttnArgs& p, cudaStream_t s) {
  constexpr size_t smem = sizeof(float) * (kGenRows * DP + 2 * kGenKeys * (DP + 4) + kGenRows * (kGenKeys + 1));
  const cudaError_t e = smem_limit_once<paged_attention_f32_kernel<TK, DP>>((int)smem);
  if (e != cudaSuccess) return e;
  paged_attention_f32_kernel<TK, DP><<<kAttnSms * 2, kGenThreads, smem, s>>>(p);
  return cudaGetLastError();
}

}  // namespace

int64_t paged_attention_workspace() {
  static_assert(kAttnSms * 3 <= kAttnMaxCtas, "counters");
  return (int64_t)std::max({AttnParts<kGenRows, 256>::bytes(kAttnSms * 2), AttnParts<kFewRows, 128>::bytes(kAttnSms * 3),
                            paged_attention_tc_workspace()});
}

cudaError_t paged_attention_status(void* workspace, bool* gave_up, cudaStream_t s) {
  int word = 0;
  cudaError_t e = cudaMemcpyAsync(&word, attn_error(workspace), sizeof(word), cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  *gave_up = word != 0;
  if (e == cudaSuccess && word) e = cudaMemsetAsync(workspace, 0, kAttnHeader + kAttnCounterBytes, s);
  return e;
}

cudaError_t launch_paged_attention(const DpufPagedAttentionArgs& a, cudaStream_t s) {
  AttnArgs p;
  p.a = a;
  p.group = a.n_q / a.kv.n_kv;
  p.page_shift = 31 - __builtin_clz((unsigned)a.kv.page_size);
  p.max_kv = (int)std::min<int64_t>((int64_t)a.pages_per_seq << p.page_shift, 1 << 30);
  p.most_q = std::min(1 << 24, (1 << 30) / p.group);
  if (a.kv.dtype == DPUF_TYPE_F32) {
    // Up to 4 rows, one tile of the streaming kernel (64 tokens at 2,304, 32 / 8 heads of 128: 220 us; by
    // the 16-row tiles 680).  More rows would read the keys once per 4 and still take less up to about 14
    // (from a flushed L2: 7 rows, 28 / 4 heads, 231 us against 395; 8, 16 / 2 heads, 128 and 209; 16,
    // 16 / 1 heads, 137 and 129): the limit is not where the two meet.
    if (a.max_q * p.group <= kFewRows && a.kv.head_dim <= 128) {
      if (a.kv.head_dim <= 64)
        paged_attention_f32_few_kernel<64><<<kAttnSms * few_ctas(64), kFewWarps * 32, 0, s>>>(p);
      else
        paged_attention_f32_few_kernel<128><<<kAttnSms * few_ctas(128), kFewWarps * 32, 0, s>>>(p);
      return cudaGetLastError();
    }
    if (a.kv.head_dim <= 64) return launch_f32<float, 64>(p, s);
    if (a.kv.head_dim <= 128) return launch_f32<float, 128>(p, s);
    return launch_f32<float, 256>(p, s);
  }
  if (a.dtype == DPUF_TYPE_F32 && a.kv.head_dim > 128)
    return a.kv.dtype == DPUF_TYPE_F16 ? launch_f32<__half, 256>(p, s) : launch_f32<__nv_bfloat16, 256>(p, s);
  // more rows than one mma.sync tile: 32 sequences of 2,000 positions with 32 / 64 rows each take the
  // tensor-core kernel 87 / 87 us, the streaming one 105 / 186; one of 16 rows at 2,304 17 us there
  if (a.dtype != DPUF_TYPE_F32 && a.kv.head_dim <= 128 && a.max_q * p.group > 16) {
    const cudaError_t e = launch_paged_attention_tc(p, s);
    if (e != cudaErrorNotSupported) return e;  // (a cache whose strides no tensor map holds streams)
  }
  return launch_paged_attention_rows(p, s);
}

}  // namespace dpuf
