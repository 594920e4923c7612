// kernels_paged_attn_rows.cu - attention of few rows over a 16-bit paged cache: decode steps (the
// query heads of one KV head and one to a few tokens), and every chunk whose queries are fp32.
//
// Bound by the bytes of K and V: a key is read once for the 16 rows of an item, 4 head_dim x 16
// flops for 4 head_dim bytes.  The arithmetic runs on mma.sync (m16n8k16: the 16 rows are the M
// side), which leaves the issue slots nearly idle, and the kernel's work is to keep loads in
// flight: each warp streams its own 16 keys of every block of 16 x kWarps through a ring of its
// own with cp.async, runs ahead across items, and never waits for another warp within an item.
// At an item's end the warps' maxima, sums and outputs are joined through shared memory.
//
// fp32 queries stay exact: q is scaled by a power of two per row and split into kTerms terms of
// the cache's type (2 of fp16 carry 22 bits, 3 of bf16 24), and so are the weights; each product
// is kTerms MMAs.  The weights carry a factor 2^12, which the sum carries too, so that in fp16 the
// small ones of a long context keep their bits (a weight of 2^-26 of the largest is still normal).
//
// 16-bit queries take their weights in one term, rounded to the cache's type (the sum keeps them
// unrounded): the output is rounded to that type once more anyway, and the largest weight, a power
// of two, is exact.  Relative errors against 64 bits, and of the output's rounding alone: 64 tokens
// at 2,304 in fp16 2.15e-4 and 2.07e-4; one at 131,071 in bf16 1.68e-3 and 1.66e-3.
#include <cuda_bf16.h>
#include <math_constants.h>

#include "attn_parts.cuh"

namespace dpuf {

namespace {

constexpr int kRows = 16;
constexpr float kLift = 12.0f;
// A block's time over that of one row of a part in the CTA that joins it.
constexpr float kJoin = 64.0f;

DPUF_DEV uint32_t su32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
DPUF_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DPUF_DEV uint32_t pack2(float a, float b, __half) {
  const __half2 h = __floats2half2_rn(a, b);
  return *(const uint32_t*)&h;
}
DPUF_DEV uint32_t pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}
DPUF_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
DPUF_DEV void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
DPUF_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __half) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
DPUF_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, __nv_bfloat16) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, "
      "%2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The first term of x in type T, and what is left of x.
template <typename T>
DPUF_DEV float rest(float x) {
  return x - to_f32(from_f32<T>(x));
}

template <int DP>
struct RowsLay {
  static constexpr int warps = DP == 256 ? 2 : 4;  // two CTAs fit an SM: one joins while the other streams
  static constexpr int keys = 16 * warps;         // of a block
  static constexpr int stages = DP == 64 ? 6 : 3;
  static constexpr int half = 16 * DP * 2;        // bytes of a warp's keys (or values) of a block
  static constexpr int ring = stages * 2 * half;  // of a warp
  static constexpr int merge = warps * ring;      // [warps][8][DP] floats
  static constexpr int bytes = merge + warps * 8 * DP * 4;
};

template <typename T, int DP, int kTerms>  // kTerms 1: queries of type T, else fp32
__global__ void __launch_bounds__(RowsLay<DP>::warps * 32, 2)
paged_attention_rows_kernel(const __grid_constant__ AttnArgs p) {
  using Lay = RowsLay<DP>;
  constexpr int W = Lay::warps, kKeys = Lay::keys, S = Lay::stages;
  extern __shared__ __align__(128) unsigned char sm[];
  __shared__ AttnShare share;
  __shared__ int flag;
  __shared__ float2 ml_sh[W][kRows];
  float* const merge = (float*)(sm + Lay::merge);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hd = p.a.kv.head_dim;
  const AttnParts<kRows, DP> parts(p.a.workspace, gridDim.x);
  AttnRun run = attn_locate<kRows, kKeys>(p, share, blockIdx.x, gridDim.x, kJoin / (float)min(kRows, p.a.max_q * p.group));
  attn_zero_unowned(p);
  if (run.n == 0) return;

  // ---- the warp's stream of keys and values
  const uint32_t ring = su32(sm) + warp * Lay::ring;
  AttnCursor pc = run.cur;  // block that is requested next
  int requested = 0, span_lo, span_hi;
  auto span = [&](const AttnCursor& c, int* lo, int* hi) {
    attn_span(p, c.seq, c.tile * kRows / p.group, min(c.seq.qn - 1, (c.tile * kRows + kRows - 1) / p.group), lo, hi);
  };
  span(pc, &span_lo, &span_hi);
  // pages of the warp's keys [j, j + 8) and [j + 8, j + 16) of the cursor's block, -1 for none
  auto pages = [&](int* pg) {
    const int j = (pc.blk0 + pc.at) * kKeys + warp * 16;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      pg[i] = -1;
      if (j + 8 * i < span_hi && j + 8 * i + 8 > span_lo) {
        const int page = p.a.page_table[(size_t)pc.s * p.a.table_stride + ((j + 8 * i) >> p.page_shift)];
        pg[i] = page < p.a.kv.n_pages ? page : -1;
      }
    }
  };
  int pg[2];
  pages(pg);
  auto request = [&]() {
    if (requested < run.n) {
      constexpr int kChunks = DP / 8, kPer = 32 / kChunks >= 1 ? 32 / kChunks : 1;  // rows per pass
      const int ch = lane % kChunks, r0 = lane / kChunks;
      const int j = (pc.blk0 + pc.at) * kKeys + warp * 16;
      const uint32_t dst = ring + (requested % S) * 2 * Lay::half;
      const char* const kb = (const char*)p.a.kv.k + (int64_t)pc.head * p.a.kv.head_stride * 2 + ch * 16;
      const char* const vb = (const char*)p.a.kv.v + (int64_t)pc.head * p.a.kv.head_stride * 2 + ch * 16;
#pragma unroll
      for (int i = 0; i < 16 / kPer; i++) {
        const int r = i * kPer + r0, jj = j + r;
        const int page = pg[r >> 3];
        const bool ok = page >= 0 && jj >= span_lo && jj < span_hi && ch * 8 < hd;
        const int64_t at = ok ? ((int64_t)page * p.a.kv.page_stride +
                                 (int64_t)(jj & (p.a.kv.page_size - 1)) * p.a.kv.row_stride) * 2 : -(int64_t)ch * 16;
        const uint32_t o = dst + r * (DP * 2) + ((ch ^ (r & 7)) << 4);
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(o), "l"(kb + at), "r"(ok ? 16 : 0) : "memory");
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(o + Lay::half), "l"(vb + at),
                     "r"(ok ? 16 : 0) : "memory");
      }
      if (++requested < run.n) {
        if (++pc.at == pc.n_blk) {
          attn_next_item<kRows, kKeys>(p, pc);
          span(pc, &span_lo, &span_hi);
        }
        pages(pg);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < S - 1; i++) request();

  AttnCursor& c = run.cur;
  int used = 0;
  for (int left = run.n; left > 0;) {
    const int from = c.at, to = min(c.n_blk, c.at + left);
    left -= to - from;
    const int total = c.seq.qn * p.group, r0 = c.tile * kRows;
    const int rows = min(kRows, total - r0);
    // ---- this thread's rows: lane / 4 and lane / 4 + 8
    uint32_t q[kTerms][DP / 16][4];
    int lo[2], hi[2];
    float mul[2];
#pragma unroll
    for (int e = 0; e < 2; e++) {
      const int r = r0 + (lane >> 2) + 8 * e;
      const bool live = r < total;
      lo[e] = hi[e] = 0;
      if (live) attn_span(p, c.seq, r / p.group, r / p.group, &lo[e], &hi[e]);
      mul[e] = p.a.scale * 1.44269504088896341f;
      const int64_t at = live ? (int64_t)(c.seq.q0 + r / p.group) * p.a.q_stride[0] +
                                    (int64_t)(c.head * p.group + r % p.group) * p.a.q_stride[1] : 0;
      if (kTerms == 1) {
        const T* src = (const T*)p.a.q + at;
#pragma unroll
        for (int s = 0; s < DP / 16; s++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int d = s * 16 + h * 8 + (lane & 3) * 2;
            q[0][s][2 * h + e] = live && d < hd ? *(const uint32_t*)(src + d) : 0u;
          }
      } else {
        const float* src = (const float*)p.a.q + at;
        float top = 0.0f;
#pragma unroll
        for (int s = 0; s < DP / 8; s++) {
          const int d = s * 8 + (lane & 3) * 2;
          if (live && d < hd) {
            const float2 x = *(const float2*)(src + d);
            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
          }
        }
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
        top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
        // the power of two that brings the largest element into [1, 2) (rows of 0 or infinity: none)
        const int ex = top >= 1.2e-38f && top < CUDART_INF_F ? (int)(__float_as_uint(top) >> 23) - 127 : 0;
        const float down0 = __uint_as_float((uint32_t)(127 - ex / 2) << 23);
        const float down1 = __uint_as_float((uint32_t)(127 - (ex - ex / 2)) << 23);
        mul[e] = mul[e] * __uint_as_float((uint32_t)(127 + ex / 2) << 23) *
                 __uint_as_float((uint32_t)(127 + ex - ex / 2) << 23);
#pragma unroll
        for (int s = 0; s < DP / 16; s++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int d = s * 16 + h * 8 + (lane & 3) * 2;
            float2 x = make_float2(0.0f, 0.0f);
            if (live && d < hd) x = *(const float2*)(src + d);
            x.x = x.x * down0 * down1;
            x.y = x.y * down0 * down1;
#pragma unroll
            for (int k = 0; k < kTerms; k++) {
              q[k][s][2 * h + e] = pack2(x.x, x.y, T());
              x.x = rest<T>(x.x);
              x.y = rest<T>(x.y);
            }
          }
      }
    }
    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.0f, 0.0f};

    for (int b = from; b < to; b++, used++) {
      request();
      asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
      __syncwarp();
      const uint32_t kt = ring + (used % S) * 2 * Lay::half, vt = kt + Lay::half;
      float s[2][4] = {};
      {
        const int r = (lane & 7) + ((lane >> 4) << 3);
        const uint32_t base = kt + r * (DP * 2);
#pragma unroll
        for (int ks = 0; ks < DP / 16; ks++) {
          uint32_t k4[4];
          ldsm4(k4, base + (((ks * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4));
#pragma unroll
          for (int k = kTerms - 1; k >= 0; k--) {  // small terms first
            mma16816(s[0], q[k][ks], k4[0], k4[1], T());
            mma16816(s[1], q[k][ks], k4[2], k4[3], T());
          }
        }
      }
      const int j = (c.blk0 + b) * kKeys + warp * 16 + (lane & 3) * 2;
      uint32_t pa[kTerms][4];
      bool grew = false;
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float t = -CUDART_INF_F;
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const int jj = j + n * 8 + x;
            float& v = s[n][2 * e + x];
            v = jj >= lo[e] && jj < hi[e] ? v * mul[e] : -CUDART_INF_F;
            t = fmaxf(t, v);
          }
        t = fmaxf(t, __shfl_xor_sync(kFull, t, 1));
        t = fmaxf(t, __shfl_xor_sync(kFull, t, 2));
        const float m2 = fmaxf(m[e], t);
        f[e] = m[e] == -CUDART_INF_F ? 0.0f : ex2(m[e] - m2);
        grew = grew || m2 != m[e];
        m[e] = m2;
        const float ref = m2 == -CUDART_INF_F ? 0.0f : m2 - kLift;
        float w[4];
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
          for (int x = 0; x < 2; x++) w[2 * n + x] = ex2(s[n][2 * e + x] - ref);
        l[e] = __fmaf_rn(l[e], f[e], (w[0] + w[1]) + (w[2] + w[3]));
#pragma unroll
        for (int k = 0; k < kTerms; k++) {
          pa[k][e] = pack2(w[0], w[1], T());
          pa[k][2 + e] = pack2(w[2], w[3], T());
          if (k + 1 < kTerms)
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = rest<T>(w[i]);
        }
      }
      if (__any_sync(kFull, grew))
#pragma unroll
        for (int i = 0; i < DP / 8; i++) {
          o[i][0] *= f[0];
          o[i][1] *= f[0];
          o[i][2] *= f[1];
          o[i][3] *= f[1];
        }
      {
        const int r = (lane & 7) + (((lane >> 3) & 1) << 3);
        const uint32_t base = vt + r * (DP * 2);
#pragma unroll
        for (int d = 0; d < DP / 16; d++) {
          uint32_t v4[4];
          ldsm4_t(v4, base + (((d * 2 + (lane >> 4)) ^ (r & 7)) << 4));
#pragma unroll
          for (int k = kTerms - 1; k >= 0; k--) {
            mma16816(o[2 * d], pa[k], v4[0], v4[1], T());
            mma16816(o[2 * d + 1], pa[k], v4[2], v4[3], T());
          }
        }
      }
      __syncwarp();  // the stage is read: the next request may overwrite it
    }

    // ---- the warps' results joined: rows 0..7, then 8..15
    const bool whole = from == 0 && to == c.n_blk;
    const size_t slot = 2 * (size_t)blockIdx.x + (from == 0 ? 1 : 0);
#pragma unroll
    for (int e = 0; e < 2; e++) {
      l[e] += __shfl_xor_sync(kFull, l[e], 1);
      l[e] += __shfl_xor_sync(kFull, l[e], 2);
      if ((lane & 3) == 0) ml_sh[warp][(lane >> 2) + 8 * e] = make_float2(m[e], l[e]);
    }
    for (int e = 0; 8 * e < rows; e++) {
      float* mine = merge + (warp * 8 + (lane >> 2)) * DP + (lane & 3) * 2;
#pragma unroll
      for (int i = 0; i < DP / 8; i++)
        *(float2*)(mine + i * 8) = e == 0 ? make_float2(o[i][0], o[i][1]) : make_float2(o[i][2], o[i][3]);
      __syncthreads();
      for (int i = tid; i < 8 * DP / 4; i += W * 32) {
        const int rr = i / (DP / 4), d = i % (DP / 4) * 4, r = 8 * e + rr;
        if (r >= rows) break;
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < W; w++) top = fmaxf(top, ml_sh[w][r].x);
        float sum = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < W; w++) {
          const float2 ml = ml_sh[w][r];
          const float g = ml.x == -CUDART_INF_F ? 0.0f : ex2(ml.x - top);
          sum = __fmaf_rn(ml.y, g, sum);
          const float4 y = *(const float4*)(merge + (w * 8 + rr) * DP + d);
          x.x = __fmaf_rn(y.x, g, x.x);
          x.y = __fmaf_rn(y.y, g, x.y);
          x.z = __fmaf_rn(y.z, g, x.z);
          x.w = __fmaf_rn(y.w, g, x.w);
        }
        if (whole) {
          const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
          const int tok = (r0 + r) / p.group, head = c.head * p.group + (r0 + r) % p.group;
          const size_t at = ((size_t)(c.seq.q0 + tok) * p.a.n_q + head) * hd + d;
          if (d < hd) store4_as(p.a.out, at, p.a.out_dtype, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        } else {
          if (d == 0) parts.ml[slot * kRows + r] = make_float2(top, sum);
          *(float4*)(parts.o + (slot * kRows + r) * DP + d) = x;
        }
      }
      __syncthreads();
    }
    if (!whole) {
      int c0, c1;
      attn_owners(run, c, &c0, &c1);
      if (attn_last_part(parts.count + 2 * c0, c1 - c0 + 1, &flag)) {
        // Of many parts the factors go into shared memory first (where it has room: one long item
        // among many short ones may be cut into hundreds), so that many loads of outputs are in
        // flight; of a few, each thread takes them as it goes.
        const int n = c1 - c0 + 1;
        float* const fac = merge;  // [rows][n]
        const bool staged = n > 8 && rows * n <= W * 8 * DP;
        auto part = [&](int i) { return 2 * (size_t)(c0 + i) + (i == 0); };
        if (staged) {
          for (int r = warp; r < rows; r += W) {
            float top = -CUDART_INF_F;
            for (int i = lane; i < n; i += 32) top = fmaxf(top, __ldcg(&parts.ml[part(i) * kRows + r]).x);
            top = warp_max(top);
            float sum = 0.0f;
            for (int i = lane; i < n; i += 32) {
              const float2 ml = __ldcg(&parts.ml[part(i) * kRows + r]);
              const float g = ml.x == -CUDART_INF_F ? 0.0f : ex2(ml.x - top);
              fac[r * n + i] = g;
              sum = __fmaf_rn(ml.y, g, sum);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(kFull, sum, o);
            if (lane == 0) ml_sh[0][r].y = sum;
          }
          __syncthreads();
        }
        for (int i = tid; i < rows * (DP / 4); i += W * 32) {
          const int r = i / (DP / 4), d = i % (DP / 4) * 4;
          float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          float sum = 0.0f;
          auto add = [&](int k, float g) {
            const float4 y = __ldcg((const float4*)(parts.o + (part(k) * kRows + r) * DP + d));
            x.x = __fmaf_rn(y.x, g, x.x);
            x.y = __fmaf_rn(y.y, g, x.y);
            x.z = __fmaf_rn(y.z, g, x.z);
            x.w = __fmaf_rn(y.w, g, x.w);
          };
          if (staged) {
            sum = ml_sh[0][r].y;
#pragma unroll 16
            for (int k = 0; k < n; k++) add(k, fac[r * n + k]);
          } else {
            float top = -CUDART_INF_F;
#pragma unroll 4
            for (int k = 0; k < n; k++) top = fmaxf(top, __ldcg(&parts.ml[part(k) * kRows + r]).x);
#pragma unroll 4
            for (int k = 0; k < n; k++) {
              const float2 ml = __ldcg(&parts.ml[part(k) * kRows + r]);
              const float g = ml.x == -CUDART_INF_F ? 0.0f : ex2(ml.x - top);
              sum = __fmaf_rn(ml.y, g, sum);
              add(k, g);
            }
          }
          const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
          const int tok = (r0 + r) / p.group, head = c.head * p.group + (r0 + r) - tok * p.group;
          const size_t at = ((size_t)(c.seq.q0 + tok) * p.a.n_q + head) * hd + d;
          if (d < hd) store4_as(p.a.out, at, p.a.out_dtype, x.x * inv, x.y * inv, x.z * inv, x.w * inv);
        }
        if (staged) __syncthreads();
      }
    }
    if (left > 0) attn_next_item<kRows, kKeys>(p, c);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

template <typename T, int DP, int kTerms>
cudaError_t launch(const AttnArgs& p, cudaStream_t s) {
  const cudaError_t e = smem_limit_once<paged_attention_rows_kernel<T, DP, kTerms>>(RowsLay<DP>::bytes);
  if (e != cudaSuccess) return e;
  paged_attention_rows_kernel<T, DP, kTerms><<<kAttnSms * 2, RowsLay<DP>::warps * 32, RowsLay<DP>::bytes, s>>>(p);
  return cudaGetLastError();
}

template <typename T, int kTerms>
cudaError_t launch(const AttnArgs& p, cudaStream_t s) {
  if (p.a.kv.head_dim <= 64) return launch<T, 64, kTerms>(p, s);
  if (kTerms > 1 || p.a.kv.head_dim <= 128) return launch<T, 128, kTerms>(p, s);
  return launch<T, 256, 1>(p, s);
}

}  // namespace

cudaError_t launch_paged_attention_rows(const AttnArgs& p, cudaStream_t s) {
  const bool f32 = p.a.dtype == DPUF_TYPE_F32;
  if (p.a.kv.dtype == DPUF_TYPE_F16) return f32 ? launch<__half, 2>(p, s) : launch<__half, 1>(p, s);
  return f32 ? launch<__nv_bfloat16, 3>(p, s) : launch<__nv_bfloat16, 1>(p, s);
}

}  // namespace dpuf
