// kernels_sample.cu - sampling on the device: temperature, top-k, top-p and min-p from given
// uniforms, one row of logits per thread-block cluster.
//
// With m the row's maximum, an entry's weight is w = exp((l - m) / T) in fp32, taken into sums
// as the integer f = round(w 2^43): sums of integers do not depend on their order, so neither do
// the thresholds and the id (an entry below 2^-44 of the maximum's weight has f = 0 and is never
// kept).  The entries kept by top-k and by top-p are the first ones in the order (logit down,
// index up), i.e. all entries above a threshold value and the first few, by index, of those
// equal to it.  The thresholds come from histograms of counts and weights instead of a sort: one
// over 2,048 equal steps of (m - l) / T, then, inside the step that holds the threshold, over
// ranges of the value's bits (made monotone) until the range is one value.
//
// A row is read from memory once: the cluster's CTAs keep a slice each in shared memory, and
// exchange histograms and running sums through distributed shared memory.  Each CTA adds up one
// segment of the bins over all CTAs, then all look the threshold's bin up in the segments.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>

#include "serving.cuh"

namespace cg = cooperative_groups;

namespace dpuf {

namespace {

constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr float kFix = 8796093022208.0f;  // 2^43
constexpr float kReach = 30.6f;           // > 44 ln 2: beyond it f is 0

typedef unsigned long long u64;

// Unsigned integers in the order of the values; NaN below everything.
DPUF_DEV uint32_t value_key(float v) {
  if (v != v) return 0;
  const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals 0
  return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
DPUF_DEV float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7FFFFFFFu : ~k); }

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab, slice, cached;  // cached: entries of a slice kept in shared memory
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* ids;
  float* probs;
};

struct Found {  // the bin in which a running sum passes its target, and the sums above it
  int bin;
  uint32_t count, above;
  u64 mass_above, mass;
};

struct SampleShared {
  uint32_t count[kBins], m0[kBins], m1[kBins], m2[kBins];  // weights in three parts of 15 bits
  uint32_t seg_count[kBins];                               // this CTA's segment, summed over the CTAs
  u64 seg_mass[kBins];
  uint32_t seg_count_sum;
  u64 seg_mass_sum;
  u64 best;           // maximum's key and lowest index
  u64 exchange[2];
  u64 warp_sum[kSampWarps];
  Found found;
  int pick;
  float pick_w;
};

DPUF_DEV u64 block_inclusive(u64 v, u64* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
  for (int w = 0; w < warp; w++) v += warp_sum[w];
  return v;
}
DPUF_DEV u64 block_sum(u64 v, u64* warp_sum) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kSampWarps; w++) v += warp_sum[w];
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kSampThreads) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  SampleShared& sh = *(SampleShared*)dyn;
  T* cache = (T*)(dyn + ((sizeof(SampleShared) + 15) & ~(size_t)15));
  cg::cluster_group cl = cg::this_cluster();
  const int R = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / R;
  const int tid = threadIdx.x;
  const T* src = (const T*)a.logits + (int64_t)row * a.row_stride;
  const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
  src += base;
  auto at = [&](int i) { return to_f32(i < a.cached ? cache[i] : src[i]); };

  // ---- the slice, and the row's maximum (lowest index)
  u64 best = 0;
  for (int i = tid; i < n; i += kSampThreads) {
    const T v = src[i];
    if (i < a.cached) cache[i] = v;
    const u64 k = ((u64)value_key(to_f32(v)) << 32) | (uint32_t)~(uint32_t)(base + i);
    best = max(best, k);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(kFull, best, o));
  if ((tid & 31) == 0) sh.warp_sum[tid >> 5] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 0; w < kSampWarps; w++) best = max(best, sh.warp_sum[w]);
    sh.best = best;
  }
  cl.sync();
  for (int r = 0; r < R; r++) best = max(best, cl.map_shared_rank(&sh, r)->best);
  const uint32_t key_max = (uint32_t)(best >> 32);
  const float m = key_value(key_max);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const bool nothing = key_max <= value_key(-CUDART_INF_F);
  if (nothing || !(temp > 0.0f)) {
    if (rank == 0 && tid == 0) {
      a.ids[row] = nothing ? -1 : (int)~(uint32_t)best;
      if (a.probs) a.probs[row] = nothing ? 0.0f : 1.0f;
    }
    cl.sync();  // the others may still read this CTA's maximum
    return;
  }
  const float inv_t = 1.0f / temp;
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  const float min_p = fminf(a.min_p ? a.min_p[row] : 0.0f, 1.0f);
  auto weight = [&](float v) {
    const float w = v == m ? 1.0f : expf((v - m) * inv_t);
    return w > 0.0f ? w : 0.0f;  // NaN has none
  };
  auto fixed = [&](float w) { return (u64)__float2ull_rn(w * kFix); };
  const float step = (float)kBins / kReach * inv_t;  // bins per unit of m - l
  auto first_bin = [&](float v) { return v == m ? 0 : (int)fminf((m - v) * step, (float)(kBins - 1)); };

  // ---- histogram of the entries that `bin` gives a bin (>= 0), summed over the cluster
  const int seg = kBins / R;
  auto histogram = [&](auto bin) {
    for (int b = tid; b < kBins; b += kSampThreads) sh.count[b] = sh.m0[b] = sh.m1[b] = sh.m2[b] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kSampThreads) {
      const float v = at(i);
      const u64 f = fixed(weight(v));
      const int b = f ? bin(v) : -1;
      if (b < 0) continue;
      atomicAdd(&sh.count[b], 1u);
      atomicAdd(&sh.m0[b], (uint32_t)f & 0x7FFF);
      atomicAdd(&sh.m1[b], (uint32_t)(f >> 15) & 0x7FFF);
      atomicAdd(&sh.m2[b], (uint32_t)(f >> 30));
    }
    cl.sync();
    u64 cs = 0, ms = 0;
    for (int b = tid; b < seg; b += kSampThreads) {
      uint32_t c = 0;
      u64 f = 0;
      for (int r = 0; r < R; r++) {
        const SampleShared* o = cl.map_shared_rank(&sh, r);
        const int g = rank * seg + b;
        c += o->count[g];
        f += (u64)o->m0[g] + ((u64)o->m1[g] << 15) + ((u64)o->m2[g] << 30);
      }
      sh.seg_count[b] = c;
      sh.seg_mass[b] = f;
      cs += c;
      ms += f;
    }
    cs = block_sum(cs, sh.warp_sum);
    ms = block_sum(ms, sh.warp_sum);
    if (tid == 0) {
      sh.seg_count_sum = (uint32_t)cs;
      sh.seg_mass_sum = ms;
    }
    cl.sync();
  };
  // ---- the bin in which the count (by_count) or the weight reaches the target
  auto find = [&](bool by_count, uint32_t count0, u64 mass0, uint32_t k_target, double p_target) {
    __syncthreads();
    if (tid < 32) {
      uint32_t c = count0;
      u64 f = mass0;
      auto reached = [&](uint32_t cc, u64 ff) { return by_count ? cc >= k_target : (double)ff >= p_target; };
      int r = 0;
      for (; r < R - 1; r++) {
        const SampleShared* o = cl.map_shared_rank(&sh, r);
        if (reached(c + o->seg_count_sum, f + o->seg_mass_sum)) break;
        c += o->seg_count_sum;
        f += o->seg_mass_sum;
      }
      // a lane's run of bins, then the bin within the run
      const SampleShared* o = cl.map_shared_rank(&sh, r);
      const int per = seg / 32;
      uint32_t lc = 0;
      u64 lf = 0;
      for (int b = 0; b < per; b++) {
        lc += o->seg_count[tid * per + b];
        lf += o->seg_mass[tid * per + b];
      }
      uint32_t ic = lc;
      u64 jf = lf;
#pragma unroll
      for (int s = 1; s < 32; s <<= 1) {
        const uint32_t tc = __shfl_up_sync(kFull, ic, s);
        const u64 tf = __shfl_up_sync(kFull, jf, s);
        if (tid >= s) {
          ic += tc;
          jf += tf;
        }
      }
      const unsigned hit = __ballot_sync(kFull, reached(c + ic, f + jf) && lc > 0);
      const unsigned any = __ballot_sync(kFull, lc > 0);
      const int lane = hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : 0;
      if (tid == lane) {
        c += ic - lc;
        f += jf - lf;
        int b = 0, last = 0;
        uint32_t c2 = c, lastc = c;
        u64 f2 = f, lastf = f;
        for (; b < per; b++) {
          const uint32_t bc = o->seg_count[tid * per + b];
          const u64 bf = o->seg_mass[tid * per + b];
          if (bc) {
            last = b;
            lastc = c2;
            lastf = f2;
            if (reached(c2 + bc, f2 + bf)) break;
          }
          c2 += bc;
          f2 += bf;
        }
        sh.found = Found{r * seg + tid * per + last, o->seg_count[tid * per + last], lastc, lastf,
                         o->seg_mass[tid * per + last]};
      }
    }
    __syncthreads();
    return sh.found;
  };
  // ---- from the first histogram's bin to one value: its key, and what lies above it
  auto refine = [&](Found f1, bool by_count, uint32_t k_target, double p_target, uint32_t* key, Found* cls) {
    const int b1 = f1.bin;
    const float lo_v = m - (float)(b1 + 1) / step, hi_v = m - (float)b1 / step;
    const float slack = 1e-5f * (fabsf(m) + fabsf(lo_v)) + 1e-30f;
    uint32_t hi = b1 == 0 ? key_max : min(key_max, value_key(hi_v + slack));
    uint32_t lo = b1 == kBins - 1 ? 1u : value_key(lo_v - slack);
    if (!(lo_v - slack <= hi_v + slack)) lo = 1u, hi = key_max;  // m or the step is not finite
    Found f = f1;
    for (;;) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)kBins) shift++;
      histogram([&](float v) {
        const uint32_t kv = value_key(v);
        return first_bin(v) == b1 && kv >= lo && kv <= hi ? (int)((hi - kv) >> shift) : -1;
      });
      f = find(by_count, f.above, f.mass_above, k_target, p_target);
      const uint32_t top = hi - ((uint32_t)f.bin << shift);
      if (shift == 0) {
        *key = top;
        *cls = f;
        return;
      }
      lo = max(lo, top - ((1u << shift) - 1));
      hi = top;
    }
  };

  uint32_t key_t = 0;          // kept: keys above it,
  uint32_t ties = 0xFFFFFFFFu;  // and the first `ties` entries equal to it
  const bool limit_k = k >= 1 && k < a.vocab, limit_p = top_p < 1.0f;
  if (limit_k || limit_p) {
    histogram(first_bin);
    uint32_t count = 0;
    u64 mass = 0;
    for (int r = 0; r < R; r++) {
      const SampleShared* o = cl.map_shared_rank(&sh, r);
      count += o->seg_count_sum;
      mass += o->seg_mass_sum;
    }
    const bool by_k = limit_k && (uint32_t)k < count;
    Found fk{}, fp{};
    if (by_k) fk = find(true, 0, 0, (uint32_t)k, 0.0);
    // the weight that top-p has to hold is known once top-k's threshold is: both start from the
    // first histogram, so the refinements (which overwrite it) come after the look-ups
    if (!by_k) {
      if (limit_p && top_p > 0.0f) fp = find(false, 0, 0, 0, (double)top_p * (double)mass);
    } else {
      Found cls;
      refine(fk, true, (uint32_t)k, 0.0, &key_t, &cls);
      ties = (uint32_t)k - cls.above;
      mass = cls.mass_above + cls.mass / cls.count * ties;
      if (limit_p && top_p > 0.0f) {
        histogram(first_bin);
        fp = find(false, 0, 0, 0, (double)top_p * (double)mass);
      }
    }
    if (limit_p) {
      if (!(top_p > 0.0f)) {
        key_t = key_max;
        ties = 1;
      } else {
        const double target = (double)top_p * (double)mass;
        Found cls;
        refine(fp, false, 0, target, &key_t, &cls);
        const u64 each = cls.mass / cls.count;
        // the fewest of the class that reach the target
        u64 c = (double)cls.mass_above >= target ? 1 : (u64)((target - (double)cls.mass_above) / (double)each);
        while (c > 1 && (double)(cls.mass_above + (c - 1) * each) >= target) c--;
        while (c < cls.count && (double)(cls.mass_above + c * each) < target) c++;
        ties = (uint32_t)max((u64)1, c);
      }
    }
  }

  // ---- index order: a thread's run of the slice is contiguous, of odd length (no bank conflicts)
  const int per = ((n + kSampThreads - 1) / kSampThreads) | 1;
  const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
  uint32_t before = 0;  // entries equal to the threshold at lower indices
  if (ties != 0xFFFFFFFFu) {
    uint32_t mine = 0;
    for (int i = i0; i < i1; i++) mine += value_key(at(i)) == key_t;
    const u64 incl = block_inclusive(mine, sh.warp_sum);
    if (tid == kSampThreads - 1) sh.exchange[0] = incl;
    cl.sync();
    before = (uint32_t)incl - mine;
    for (int r = 0; r < rank; r++) before += (uint32_t)cl.map_shared_rank(&sh, r)->exchange[0];
  }
  auto kept = [&](float v, uint32_t& tie) -> u64 {
    const uint32_t kv = value_key(v);
    if (kv < key_t) return 0;
    if (kv == key_t && tie++ >= ties) return 0;
    const float w = weight(v);
    return w >= min_p ? fixed(w) : 0;
  };
  u64 mine = 0;
  {
    uint32_t tie = before;
    for (int i = i0; i < i1; i++) mine += kept(at(i), tie);
  }
  u64 incl = block_inclusive(mine, sh.warp_sum);
  if (tid == kSampThreads - 1) sh.exchange[1] = incl;
  cl.sync();
  u64 total = 0, lower = 0;
  for (int r = 0; r < R; r++) {
    const u64 e = cl.map_shared_rank(&sh, r)->exchange[1];
    if (r < rank) lower += e;
    total += e;
  }
  incl += lower;
  const double target = (double)a.u[row] * (double)total;
  auto passed = [&](u64 c) { return (double)c > target || c >= total; };
  if (mine && passed(incl) && !(incl - mine > 0 && passed(incl - mine))) {  // one thread of the cluster
    u64 run = incl - mine;
    uint32_t tie = before;
    for (int i = i0; i < i1; i++) {
      const float v = at(i);
      const u64 f = kept(v, tie);
      run += f;
      if (f && passed(run)) {
        a.ids[row] = base + i;
        if (a.probs) a.probs[row] = (float)((double)weight(v) * (double)kFix / (double)total);
        break;
      }
    }
  }
  cl.sync();  // no CTA leaves while others read its shared memory
}

template <typename T>
cudaError_t launch(const SampleArgs& args, cudaStream_t s) {
  SampleArgs a = args;
  int cluster = 1;
  while (cluster < kMaxCluster && a.vocab > cluster * 4096) cluster *= 2;
  a.slice = (a.vocab + cluster - 1) / cluster;
  const size_t head = (sizeof(SampleShared) + 15) & ~(size_t)15;
  const size_t room = 200 * 1024 - head;
  a.cached = (int)std::min((size_t)a.slice, room / sizeof(T));
  const size_t smem = head + (size_t)a.cached * sizeof(T);
  cudaError_t e = cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * cluster);
  cfg.blockDim = dim3(kSampThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sample_rows_kernel<T>, a);
}

}  // namespace

cudaError_t launch_sample_rows(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const float* u,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               int32_t* ids, float* probs, cudaStream_t s) {
  const SampleArgs a{logits, row_stride, rows, vocab, 0, 0, u, temperature, top_k, top_p, min_p, ids, probs};
  if (dtype == DPUF_TYPE_F32) return launch<float>(a, s);
  if (dtype == DPUF_TYPE_F16) return launch<__half>(a, s);
  return launch<__nv_bfloat16>(a, s);
}

}  // namespace dpuf
