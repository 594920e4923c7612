// kernels_sample.cu - sampling on the device: temperature, top-k, top-p and min-p from given
// uniforms, one row of logits per thread-block cluster.
//
// With m the row's maximum, an entry's weight is w = exp((l - m) / T) in fp32, taken into sums
// as the integer f = round(w 2^43): sums of integers do not depend on their order, so neither do
// the thresholds and the id (an entry below 2^-44 of the maximum's weight has f = 0 and is never
// kept; rounding down instead would lose half a unit an entry, and 10^5 entries' worth moves ids).  All three filters keep a prefix of the order (logit down, index up), i.e. all entries
// above a threshold value and the first few, by index, of those equal to it.  No sort of the row:
//
//  1. the row's slices go to the cluster's shared memory, once; the maximum.
//  2. a histogram of counts over 1,024 equal steps of (m - l) / T down to the smallest entry, or
//     to where weights end, summed over the cluster.  The
//     step in which top-k ends follows exactly, for top-p a step by which it has ended for sure
//     (a step's weight is between its count times its ends' weights), for min-p the same.
//  3. the entries down to that step are handed to one CTA of the cluster (the others are then
//     done): mostly a few dozen.
//  4. up to 256 of them, a thread each, it ranks by comparing all with all, which gives each one's
//     running weight too.  Of more, the thresholds are searched by histograms of counts and weights
//     over ranges of the value's bits (made monotone), each range the bin of the one before, until
//     it is one value.  Where they are too many to hand over (a nucleus of much of the vocabulary)
//     the cluster does the same together, each CTA adding up one segment of the bins.
//  5. the running weight in index order passes u times the kept weight at the id.
//
// Bound by latency for few rows (the cluster's barriers and the block's), by the passes over the
// slices for many; the row is read from memory once.
#include <cooperative_groups.h>
#include <math_constants.h>

#include <algorithm>

#include "attn_parts.cuh"

namespace cg = cooperative_groups;

namespace dpuf {

namespace {

constexpr int kSampThreads = 512;
constexpr int kSampWarps = kSampThreads / 32;
constexpr int kBins = 1024;
constexpr int kMaxCluster = 16;
constexpr int kListCap = 3 * kBins;       // entries that one CTA hands over (in the histograms' place)
constexpr int kFewCap = 256;              // entries that are ranked by comparison
constexpr float kFix = 8796093022208.0f;  // 2^43
constexpr float kReach = 30.6f;           // > 44 ln 2: beyond it f is 0

typedef unsigned long long u64;

// Unsigned integers in the order of the values (0 for NaN); of the 16-bit types without the low
// bits that their fp32 form does not use, so that neighbouring values have neighbouring keys.
template <typename T>
struct Key {
  static constexpr int drop = std::is_same<T, float>::value ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  static DPUF_DEV uint32_t of(float v) {
    if (v != v) return 0;
    const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);  // -0 equals 0
    return ((b & 0x80000000u) ? ~b : b | 0x80000000u) >> drop;
  }
  static DPUF_DEV float value(uint32_t k) {
    const uint32_t b = k << drop;
    return __uint_as_float((b & 0x80000000u) ? b & 0x7FFFFFFFu : ~(b | ((1u << drop) - 1)));
  }
};

struct SampleArgs {
  const void* logits;
  int64_t row_stride;
  int rows, vocab, slice, cached;  // cached: entries of a slice kept in shared memory
  int given, given_i;              // entries that rank 0 can be given (in its slice's place), offset of their indices
  const float* u;
  const float* temperature;
  const int* top_k;
  const float* top_p;
  const float* min_p;
  int* ids;
  float* probs;
};

struct Found {  // the bin in which a running sum reaches its target, and the sums above it
  int bin;      // -1: not reached
  uint32_t count, above;
  u64 mass_above, mass;
};

struct SampleShared {
  uint32_t count[kBins];
  union {  // one after the other
    struct {  // what a CTA hands over, in index order
      float list_v[kListCap];
      int list_i[kListCap];
    };
    struct {
      uint32_t m0[kBins], m1[kBins], m2[kBins];  // weights in three parts of 15 bits
      uint32_t bin_count[kBins];                 // this CTA's segment of the bins, summed over the CTAs
      u64 bin_mass[kBins];
    };
  };
  float few_v[kFewCap];  // in rank 0: the entries in no order,
  int few_i[kFewCap];
  u64 few_f[kFewCap], few_x[kFewCap];  // their weights; their places in the order
  unsigned few_n;
  uint32_t first;  // where this CTA's entries go
  uint32_t seg_count;
  u64 seg_mass;
  u64 best;  // maximum's key and lowest index
  float low;  // minimum
  u64 exchange[4];
  u64 warp_sum[kSampWarps];
  float warp_lo[kSampWarps], warp_hi[kSampWarps];
  Found found;
  int step_k, step_p, step_lo;
  float hi_k, hi_m;
};

DPUF_DEV u64 warp_inclusive(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
DPUF_DEV uint32_t warp_inclusive32(uint32_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(kFull, v, o);
    if (lane >= o) v += t;
  }
  return v;
}
DPUF_DEV u64 block_inclusive(u64 v, u64* warp_sum) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_inclusive(v);
  __syncthreads();
  if (lane == 31) warp_sum[warp] = v;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kSampWarps; w++)
    if (w < warp) v += warp_sum[w];
  return v;
}
DPUF_DEV u64 block_sum(u64 v, u64* warp_sum) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) warp_sum[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kSampWarps; w++) v += warp_sum[w];
  return v;
}

// Bit j: entry j of 16 bytes is `cut` or more (NaN is not).
DPUF_DEV uint32_t at_least(uint4 x, float cut, float) {
  return (uint32_t)(__uint_as_float(x.x) >= cut) | (uint32_t)(__uint_as_float(x.y) >= cut) << 1 |
         (uint32_t)(__uint_as_float(x.z) >= cut) << 2 | (uint32_t)(__uint_as_float(x.w) >= cut) << 3;
}
DPUF_DEV uint32_t at_least_bits(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // from two 16-bit masks each
  const uint32_t t = (a & 0x00010001u) | (b & 0x00010001u) << 2 | (c & 0x00010001u) << 4 | (d & 0x00010001u) << 6;
  return (t | t >> 15) & 0xFFu;
}
DPUF_DEV uint32_t at_least(uint4 x, float cut, __half) {
  const __half2 c = __half2half2(__float2half_ru(cut)), *e = (const __half2*)&x;
  return at_least_bits(__hge2_mask(e[0], c), __hge2_mask(e[1], c), __hge2_mask(e[2], c), __hge2_mask(e[3], c));
}
DPUF_DEV uint32_t at_least(uint4 x, float cut, __nv_bfloat16) {
  const __nv_bfloat162 c = __bfloat162bfloat162(__float2bfloat16_ru(cut)), *e = (const __nv_bfloat162*)&x;
  return at_least_bits(__hge2_mask(e[0], c), __hge2_mask(e[1], c), __hge2_mask(e[2], c), __hge2_mask(e[3], c));
}

template <typename T>
__global__ void __launch_bounds__(kSampThreads, 2) sample_rows_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) unsigned char dyn[];
  SampleShared& sh = *(SampleShared*)dyn;
  T* cache = (T*)(dyn + ((sizeof(SampleShared) + 15) & ~(size_t)15));
  cg::cluster_group cl = cg::this_cluster();
  const int R = (int)cl.num_blocks(), rank = (int)cl.block_rank();
  const int row = blockIdx.x / R;
  const int tid = threadIdx.x, lane = tid & 31;
  const T* src = (const T*)a.logits + (int64_t)row * a.row_stride;
  const int base = min(rank * a.slice, a.vocab), n = min(a.slice, a.vocab - base);
  src += base;
  auto at = [&](int i) { return to_f32(i < a.cached ? cache[i] : src[i]); };
  auto of = [&](int r) { return cl.map_shared_rank(&sh, r); };
  // a sum over the cluster of a u64 that each CTA has in exchange[e] (after a cluster barrier)
  auto over_cluster = [&](int e) {
    u64 v = lane < R ? of(lane)->exchange[e] : 0;
#pragma unroll
    for (int o = kMaxCluster / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return __shfl_sync(kFull, v, 0);
  };
  // and the sum of the lower ranks' only
  auto below_rank = [&](int e) {
    u64 v = lane < rank ? of(lane)->exchange[e] : 0;
#pragma unroll
    for (int o = kMaxCluster / 2; o; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return __shfl_sync(kFull, v, 0);
  };

  // ---- 1. the slice, and the row's maximum (lowest index)
  float top_v = -CUDART_INF_F;
  int top_i = -1;
  float low_v = CUDART_INF_F;
  auto see = [&](float v, int i) {
    if (v > top_v) {
      top_v = v;
      top_i = i;
    }
    low_v = fminf(low_v, v);
  };
  const bool vectors = ((uintptr_t)src & 15) == 0;
  constexpr int kVec = 16 / sizeof(T);
  const int in_vectors = vectors ? min(n, a.cached) / kVec * kVec : 0;
#pragma unroll 4
  for (int i = tid * kVec; i < in_vectors; i += kSampThreads * kVec) {
    const uint4 x = __ldcs((const uint4*)(src + i));
    *(uint4*)(cache + i) = x;
    const T* e = (const T*)&x;
#pragma unroll
    for (int j = 0; j < kVec; j++) see(to_f32(e[j]), i + j);
  }
#pragma unroll 8
  for (int i = in_vectors + tid; i < n; i += kSampThreads) {
    const T v = src[i];
    if (i < a.cached) cache[i] = v;
    see(to_f32(v), i);
  }
  // an empty thread's key is 0 (that of NaN); the lowest index wins among equal keys
  u64 best = top_i < 0 ? 0 : ((u64)Key<T>::of(top_v) << 32) | (uint32_t)~(uint32_t)(base + top_i);
#pragma unroll
  for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(kFull, best, o));
  low_v = -warp_max(-low_v);
  if (lane == 0) {
    sh.warp_sum[tid >> 5] = best;
    sh.warp_lo[tid >> 5] = low_v;
  }
  for (int b = tid; b < kBins; b += kSampThreads) sh.count[b] = 0;
  if (tid == 0) sh.few_n = 0;
  __syncthreads();
  if (tid < 32) {
    best = lane < kSampWarps ? sh.warp_sum[lane] : 0;
    low_v = lane < kSampWarps ? sh.warp_lo[lane] : CUDART_INF_F;
#pragma unroll
    for (int o = kSampWarps / 2; o; o >>= 1) best = max(best, __shfl_xor_sync(kFull, best, o));
    low_v = -warp_max(-low_v);
    if (lane == 0) {
      sh.best = best;
      sh.low = low_v;
    }
  }
  cl.sync();
  best = lane < R ? of(lane)->best : 0;
  low_v = -warp_max(lane < R ? -of(lane)->low : -CUDART_INF_F);
#pragma unroll
  for (int o = kMaxCluster / 2; o; o >>= 1) best = max(best, __shfl_xor_sync(kFull, best, o));
  best = __shfl_sync(kFull, best, 0);
  const uint32_t key_max = (uint32_t)(best >> 32);
  const float m = Key<T>::value(key_max);
  const float temp = a.temperature ? a.temperature[row] : 1.0f;
  const bool nothing = key_max <= Key<T>::of(-CUDART_INF_F);
  const int k = a.top_k ? a.top_k[row] : 0;
  const float top_p = a.top_p ? a.top_p[row] : 1.0f;
  if (nothing || !(temp > 0.0f) || k == 1 || top_p <= 0.0f) {  // the first maximum is all that is kept
    if (rank == 0 && tid == 0) {
      a.ids[row] = nothing ? -1 : (int)~(uint32_t)best;
      if (a.probs) a.probs[row] = nothing ? 0.0f : 1.0f;
    }
    cl.sync();  // the others may still read this CTA's maximum
    return;
  }
  const float inv_t = 1.0f / temp;
  const float min_p = fminf(a.min_p ? a.min_p[row] : 0.0f, 1.0f);
  const float u = a.u[row];
  auto weight = [&](float v) {
    const float w = v == m ? 1.0f : expf((v - m) * inv_t);
    return w > 0.0f ? w : 0.0f;  // NaN has none
  };
  // round(w 2^43) of w in [0, 1]: the 24-bit significand, shifted (half up)
  auto fixed = [&](float w) -> u64 {
    const uint32_t b = __float_as_uint(w);
    const int n = 146 - (int)(b >> 23);
    return n > 63 ? 0 : (((u64)((b & 0x7FFFFFu) | 0x800000u) << 39) + (1ull << (n - 1))) >> n;
  };
  // steps per unit of (m - l) / T; a little more than the row's span, so that its smallest entry is inside
  const float span = (m - low_v) * inv_t * 1.0001f + 1e-6f;
  const float reach = span < kReach ? span : kReach;  // (kReach for an infinite or undefined span)
  const float per_step = (float)kBins / reach, per_unit = inv_t * per_step;
  // every entry of the slice, in no order: 16 bytes at a time
  auto each = [&](auto f) {
    const int full = min(n, a.cached) / kVec * kVec;
    for (int i = tid * kVec; i < full; i += kSampThreads * kVec) {
      const uint4 x = *(const uint4*)(cache + i);
      const T* e = (const T*)&x;
#pragma unroll
      for (int j = 0; j < kVec; j++) f(to_f32(e[j]));
    }
    for (int i = full + tid; i < n; i += kSampThreads) f(at(i));
  };
  auto finish = [&](int id, float w, u64 total) {
    a.ids[row] = id;
    if (a.probs) a.probs[row] = (float)((double)w * (double)kFix / (double)total);
  };

  // ---- 2. the step by which the kept prefix has ended
  const bool limit_k = k >= 1 && k < a.vocab, limit_p = top_p < 1.0f;
  bool by_k = false, by_p = false;  // filters that may end the prefix
  u64 mass = 0;                     // weight of what top-k keeps, where by_p
  int last_step = kBins;            // kBins: the whole slice stays the domain
  int first_step = 0;               // top-p ends no earlier
  if (limit_k || limit_p) {
    auto whole_mass = [&]() {
      u64 mine = 0;
      each([&](float v) { mine += fixed(weight(v)); });
      mine = block_sum(mine, sh.warp_sum);
      if (tid == 0) sh.exchange[0] = mine;
    };
    if (m < CUDART_INF_F && per_unit < CUDART_INF_F)
      each([&](float v) {
        const float z = (m - v) * per_unit;
        if (z < (float)kBins) atomicAdd(&sh.count[(int)z], 1u);  // (not for NaN)
      });
    else  // m - m may be no number, and the steps' factor no finite one
      each([&](float v) {
        const float z = v == m ? 0.0f : (m - v) * inv_t;
        if (z < reach) atomicAdd(&sh.count[min((int)(z * per_step), kBins - 1)], 1u);
      });
    const bool mass_now = limit_p && !limit_k && !(min_p > 0.0f);  // else it may not be needed
    if (mass_now) whole_mass();
    cl.sync();
    if (mass_now) mass = over_cluster(0);
    // bins 2 tid and 2 tid + 1: counts, and bounds of their weights (wide enough for the rounding
    // of the sums)
    uint32_t c[2] = {0, 0};
#pragma unroll 8
    for (int r = 0; r < R; r++) {
      const uint2 x = *(const uint2*)&of(r)->count[2 * tid];
      c[0] += x.x;
      c[1] += x.y;
    }
    const float w0 = expf(-(float)(2 * tid) / per_step), w1 = expf(-(float)(2 * tid + 1) / per_step),
                w2 = tid == kSampThreads - 1 ? 0.0f : expf(-(float)(2 * tid + 2) / per_step);
    const float hi[2] = {c[0] * w0 * 1.001f, c[1] * w1 * 1.001f}, lo[2] = {c[0] * w1 * 0.999f, c[1] * w2 * 0.999f};
    uint32_t cc = c[0] + c[1];
    float sl = lo[0] + lo[1], sh_ = hi[0] + hi[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t z = __shfl_up_sync(kFull, cc, o);
      const float x = __shfl_up_sync(kFull, sl, o), y = __shfl_up_sync(kFull, sh_, o);
      if (lane >= o) {
        cc += z;
        sl += x;
        sh_ += y;
      }
    }
    if (lane == 31) {
      sh.warp_sum[tid >> 5] = cc;
      sh.warp_lo[tid >> 5] = sl;
      sh.warp_hi[tid >> 5] = sh_;
    }
    if (tid == 0) {
      sh.step_k = sh.step_p = kBins;
      sh.step_lo = 0;
      sh.hi_k = sh.hi_m = 0.0f;
    }
    __syncthreads();
    float all_lo = 0.0f;
#pragma unroll
    for (int w = 0; w < kSampWarps; w++) {
      if (w < (tid >> 5)) {
        cc += (uint32_t)sh.warp_sum[w];
        sl += sh.warp_lo[w];
        sh_ += sh.warp_hi[w];
      }
      all_lo += sh.warp_lo[w];
    }
    // running sums at the ends of bins 2 tid and 2 tid + 1
    const uint32_t run[2] = {cc - c[1], cc};
    const float run_lo[2] = {sl - lo[1], sl}, run_hi[2] = {sh_ - hi[1], sh_};
    // bounded before it becomes an integer: a flat row's steps are so narrow that it may pass 2^31
    const int step_m =
        min_p > 0.0f ? (int)fminf(-logf(min_p) * per_step * 1.0001f, (float)(kBins - 2)) + 1 : kBins - 1;
#pragma unroll
    for (int e = 0; e < 2; e++) {
      if (limit_k && run[e] > (uint32_t)k && run[e] - c[e] <= (uint32_t)k) {  // strictly more than k up to here
        sh.step_k = 2 * tid + e;
        sh.hi_k = run_hi[e];
      }
      if (2 * tid + e == step_m) sh.hi_m = run_hi[e];
    }
    __syncthreads();
    by_k = limit_k && sh.step_k < kBins;
    // min-p may end the prefix before top-p for sure
    by_p = limit_p && (by_k || min_p <= 0.0f || sh.hi_m >= top_p * all_lo * 0.999f);
    if (by_p && !by_k && !mass_now) {
      whole_mass();
      cl.sync();
      mass = over_cluster(0);
    }
    if (by_p) {
      // at most the upper bound of top-k's weight where it is not known yet
      const float target = top_p * (by_k ? sh.hi_k : (float)((double)mass / (double)kFix)) * 1.001f;
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (run_lo[e] >= target && (2 * tid + e == 0 || run_lo[e] - lo[e] < target)) atomicMin(&sh.step_p, 2 * tid + e);
      // and the last step before which it has not ended for sure
      const float least = top_p * (float)((double)mass / (double)kFix) * 0.999f;
#pragma unroll
      for (int e = 0; e < 2; e++)
        if (!by_k && run_hi[e] < least) atomicMax(&sh.step_lo, 2 * tid + e + 1);
      __syncthreads();
      first_step = min(sh.step_lo, kBins - 1);
    }
    // top-p after a top-k that ends the prefix needs all that top-k keeps for its weight
    last_step = by_k ? sh.step_k : sh.step_p;
    if (min_p > 0.0f && !(by_k && by_p)) last_step = min(last_step, step_m);
  }

  // ---- 3. the entries down to that step to rank 0: at once while they are few, else once its
  // slice is free.  In index order: a thread's run is contiguous.
  float cut = -CUDART_INF_F;
  bool local = false;  // rank 0 goes on alone, over what it has been given
  int have = 0;
  T* const given_v = cache;
  int* const given_i = (int*)(dyn + a.given_i);
  if (last_step < kBins) {
    const float low = m - (float)(last_step + 1) / per_step * temp;
    cut = fminf(low - 1e-5f * (fabsf(m) + fabsf(low)) - 1e-30f, m);  // at or below every entry wanted
    if (!(cut <= m)) cut = -CUDART_INF_F;                             // the step's end is not finite
    // runs of an odd number of 16 bytes (no bank conflicts), eight at a time, as bits
    const int vectors_ = (n + kVec - 1) / kVec, per = ((vectors_ + kSampThreads - 1) / kSampThreads) | 1;
    const int v0 = min(tid * per, vectors_), v1 = min(v0 + per, vectors_);
    typedef typename std::conditional<kVec == 8, u64, uint32_t>::type Bits;
    auto wanted = [&](int first) {
      Bits in = 0;
#pragma unroll
      for (int x = 0; x < 8; x++) {
        const int i = (first + x) * kVec;
        if (first + x >= v1) break;
        if (i + kVec <= min(n, a.cached))
          in |= (Bits)at_least(*(const uint4*)(cache + i), cut, T()) << x * kVec;
        else
          for (int j = 0; j < kVec && i + j < n; j++) in |= (Bits)(at(i + j) >= cut) << (x * kVec + j);
      }
      return in;
    };
    uint32_t mine = 0;
    for (int v = v0; v < v1; v += 8) mine += sizeof(Bits) == 8 ? __popcll(wanted(v)) : __popc((uint32_t)wanted(v));
    uint32_t o = warp_inclusive32(mine);
    if (lane == 31) sh.warp_sum[tid >> 5] = o;
    __syncthreads();
    o -= mine;
    uint32_t all = 0;  // the CTA's entries; o: where this thread's begin
#pragma unroll
    for (int w = 0; w < kSampWarps; w++) {
      if (w < (tid >> 5)) o += (uint32_t)sh.warp_sum[w];
      all += (uint32_t)sh.warp_sum[w];
    }
    if (tid == 0) {
      sh.exchange[1] = all <= kListCap ? all : 1u << 30;
      sh.first = all == 0 || all > kFewCap ? kFewCap : atomicAdd(&of(0)->few_n, all);
    }
    SampleShared* const to = of(0);
    if (all <= kFewCap) __syncthreads();
    if (mine && all <= kListCap) {
      const uint32_t first = all <= kFewCap ? sh.first : kFewCap;
      for (int v = v0; v < v1; v += 8)
        for (Bits in = wanted(v); in; in &= in - 1) {
          const int i = v * kVec + (sizeof(Bits) == 8 ? __ffsll(in) : __ffs((uint32_t)in)) - 1;
          const float x = at(i);
          if (first + o < kFewCap) {
            to->few_v[first + o] = x;
            to->few_i[first + o] = base + i;
          }
          sh.list_v[o] = x;
          sh.list_i[o++] = base + i;
        }
    }
    cl.sync();  // rank 0's slice is not needed any more if the lists fit
    const u64 entries = over_cluster(1);
    if (entries <= kFewCap) {
      have = (int)entries;
      local = true;
      cl.barrier_arrive();  // this CTA has read the others' counts; they wait for that before they leave
      if (rank != 0) {
        cl.barrier_wait();
        return;
      }
    } else if (entries <= (u64)a.given) {
      local = true;
      have = (int)entries;
      T* const tv = (T*)((unsigned char*)to + ((unsigned char*)given_v - dyn));
      int* const ti = (int*)((unsigned char*)to + ((unsigned char*)given_i - dyn));
      const int first = (int)below_rank(1), mine_n = (int)sh.exchange[1];
      for (int i = tid; i < mine_n; i += kSampThreads) {
        tv[first + i] = from_f32<T>(sh.list_v[i]);
        ti[first + i] = sh.list_i[i];
      }
      cl.sync();
      if (rank != 0) return;
    }
  } else if (limit_p) {
    cl.sync();  // the counts are read: the histograms below may overwrite them
  }

  if (local && have <= kFewCap) {
    // ---- 4. few: thread t has an entry; its rank and the weight before it by comparison with all
    const int threads = (have + 31) & ~31;  // whole warps; they meet at barrier 1
    if (tid < threads) {
      auto meet = [&]() { asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory"); };
      const bool real = tid < have;
      const float v = real ? sh.few_v[tid] : 0.0f;
      const int id = real ? sh.few_i[tid] : 0;
      const float w = real ? weight(v) : 0.0f;
      const u64 f = fixed(w);
      const u64 x = ((u64)Key<T>::of(v) << 32) | (uint32_t)~(uint32_t)id;  // larger: ahead
      if (real) {
        sh.few_x[tid] = x;
        sh.few_f[tid] = f;
      }
      meet();
      int place = 0;
      u64 before = 0;
#pragma unroll 8
      for (int j = 0; j < have; j++) {
        const u64 ahead = (u64)0 - (u64)(sh.few_x[j] > x);  // all ones or 0
        place -= (int)ahead;
        before += sh.few_f[j] & ahead;
      }
      const bool in_k = real && (!by_k || place < k);
      if (by_k && by_p) {  // the weight of what top-k keeps
        if (real && place == min(k, have) - 1) sh.exchange[2] = before + f;
        meet();
        mass = sh.exchange[2];
      }
      const bool keep = in_k && (!by_p || place == 0 || (double)before < (double)top_p * (double)mass) && w >= min_p;
      const u64 g = keep ? f : 0;
      meet();
      if (real) sh.few_f[tid] = g;
      meet();
      u64 total = 0, cdf = 0;
#pragma unroll 8
      for (int j = 0; j < have; j++) {
        const u64 gj = sh.few_f[j];
        total += gj;
        cdf += gj & ((u64)0 - (u64)(sh.few_i[j] <= id));
      }
      const double target = (double)u * (double)total;
      auto passed = [&](u64 c) { return (double)c > target || c >= total; };
      if (g && passed(cdf) && !(cdf > g && passed(cdf - g))) finish(id, w, total);
    }
    cl.barrier_wait();  // the others have read this CTA's count
    return;
  }

  // ---- 4. many: thresholds by histograms, of what rank 0 has been given or of all slices
  const int dn = local ? have : n;
  auto value = [&](int i) { return local ? to_f32(given_v[i]) : at(i); };
  auto reached = [&](bool by_count, u64 c, u64 f, uint32_t k_target, double p_target) {
    return by_count ? c >= k_target : (double)f >= p_target;
  };
  // Entries with keys in [lo, hi] into bins of 2^shift keys from the top, and the bin in which the
  // count (by_count) or the weight, from the sums above, reaches the target.
  // `tail`: the range is all that lies below its top, so what lies above is the rest of the whole.
  // (top-p's first range is top-k's: its histogram is kept where top-k needed no other.)
  uint32_t built_lo = 1, built_hi = 0;
  auto level = [&](uint32_t lo, uint32_t hi, int shift, bool by_count, Found above, uint32_t k_target,
                   double p_target, bool tail) {
    const bool again = lo == built_lo && hi == built_hi;
    const bool single = shift == 0;  // a key a bin: its weight is that of one entry, times the count
    built_lo = lo;
    built_hi = hi;
    __syncthreads();
    if (!again)
      for (int b = tid; b < kBins; b += kSampThreads) {
        sh.count[b] = 0;
        if (!single) sh.m0[b] = sh.m1[b] = sh.m2[b] = 0;
      }
    if (tid == 0) sh.found = Found{-1, 0, 0, 0, 0};
    __syncthreads();
#pragma unroll 4
    for (int i = tid; i < (again ? 0 : dn); i += kSampThreads) {
      const float v = value(i);
      const uint32_t kv = Key<T>::of(v);
      if (kv < lo || kv > hi) continue;
      const int b = (int)((hi - kv) >> shift);
      if (single) {
        atomicAdd(&sh.count[b], 1u);
      } else if (const u64 f = fixed(weight(v))) {
        atomicAdd(&sh.count[b], 1u);
        atomicAdd(&sh.m0[b], (uint32_t)f & 0x7FFF);
        atomicAdd(&sh.m1[b], (uint32_t)(f >> 15) & 0x7FFF);
        atomicAdd(&sh.m2[b], (uint32_t)(f >> 30));
      }
    }
    auto key_mass = [&](int b) { return fixed(weight(Key<T>::value(hi - (uint32_t)b))); };  // (hi - b >= lo)
    if (local) {
      __syncthreads();
      u64 c[2], f[2];
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int b = 2 * tid + e;
        c[e] = sh.count[b];
        if (single) {
          const u64 one = c[e] ? key_mass(b) : 0;
          f[e] = one * c[e];
          if (!one) c[e] = 0;
        } else {
          f[e] = (u64)sh.m0[b] + ((u64)sh.m1[b] << 15) + ((u64)sh.m2[b] << 30);
        }
      }
      u64 ci = block_inclusive(c[0] + c[1], sh.warp_sum) + above.above - c[0] - c[1];
      u64 fi = block_inclusive(f[0] + f[1], sh.warp_sum) + above.mass_above - f[0] - f[1];
#pragma unroll
      for (int e = 0; e < 2; e++) {  // one bin of one thread is the first to reach the target
        if (c[e] && reached(by_count, ci + c[e], fi + f[e], k_target, p_target) &&
            ((ci == above.above && fi == above.mass_above) || !reached(by_count, ci, fi, k_target, p_target)))
          sh.found = Found{2 * tid + e, (uint32_t)c[e], (uint32_t)ci, fi, f[e]};
        ci += c[e];
        fi += f[e];
      }
      __syncthreads();
      return sh.found;
    }
    const int seg = kBins / R;
    if (!again) {
      cl.sync();
      for (int i = tid; i < 4 * seg; i += kSampThreads) {  // four threads a bin, each some of the CTAs
        const int g = rank * seg + (i >> 2);
        uint32_t c = 0;
        u64 f = 0;
#pragma unroll 4
        for (int r = i & 3; r < R; r += 4) {
          const SampleShared* o = of(r);
          c += o->count[g];
          if (!single) f += (u64)o->m0[g] + ((u64)o->m1[g] << 15) + ((u64)o->m2[g] << 30);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
          c += __shfl_xor_sync(kFull, c, o);
          f += __shfl_xor_sync(kFull, f, o);
        }
        if (single) {
          const u64 one = c ? key_mass(g) : 0;
          f = one * c;
          if (!one) c = 0;
        }
        if ((i & 3) == 0) {
          sh.bin_count[i >> 2] = c;
          sh.bin_mass[i >> 2] = f;
        }
      }
      __syncthreads();
      if (tid < 32) {
        u64 cs = 0, ms = 0;
        for (int b = lane; b < seg; b += 32) {
          cs += sh.bin_count[b];
          ms += sh.bin_mass[b];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) {
          cs += __shfl_xor_sync(kFull, cs, o);
          ms += __shfl_xor_sync(kFull, ms, o);
        }
        if (lane == 0) {
          sh.seg_count = (uint32_t)cs;
          sh.seg_mass = ms;
        }
      }
      cl.sync();
    }
    if (tid < 32) {
      const u64 c0 = lane < R ? of(lane)->seg_count : 0, f0 = lane < R ? of(lane)->seg_mass : 0;
      if (tail) above.mass_above = mass - __shfl_sync(kFull, warp_inclusive(f0), 31);
      const u64 ci = warp_inclusive(c0) + above.above, fi = warp_inclusive(f0) + above.mass_above;
      const unsigned in = __ballot_sync(kFull, lane < R && c0 > 0 && reached(by_count, ci, fi, k_target, p_target));
      if (in) {
        const int r = __ffs(in) - 1;
        u64 c = __shfl_sync(kFull, ci - c0, r), g = __shfl_sync(kFull, fi - f0, r);
        const SampleShared* o = of(r);
        for (int b = 0; b < seg; b += 32) {  // 32 bins at a time
          const u64 bc = o->bin_count[b + lane], bf = o->bin_mass[b + lane];
          const u64 ic = warp_inclusive(bc) + c, jf = warp_inclusive(bf) + g;
          const unsigned hit = __ballot_sync(kFull, bc > 0 && reached(by_count, ic, jf, k_target, p_target));
          if (hit) {
            if (lane == __ffs(hit) - 1)
              sh.found = Found{r * seg + b + lane, (uint32_t)bc, (uint32_t)(ic - bc), jf - bf, bf};
            break;
          }
          c = __shfl_sync(kFull, ic, 31);
          g = __shfl_sync(kFull, jf, 31);
        }
      }
    }
    __syncthreads();
    return sh.found;
  };
  // the value in which the target is reached: its key, the sums above it and its own (bin -1: not
  // reached in the domain)
  auto select = [&](bool by_count, uint32_t k_target, double p_target, uint32_t* key) {
    // down to the domain's end, or to where weights end
    const float end = m - reach * temp, slack = 1e-5f * (fabsf(m) + fabsf(end)) + 1e-30f;
    const float all = end - slack == end - slack ? end - slack : -CUDART_INF_F;
    uint32_t hi = key_max, lo = max(1u, Key<T>::of(fmaxf(cut, all)));
    // over all slices, of a top-p alone: from the step before which it has not ended, down to the
    // smallest weight, so that what is above follows from the whole
    bool tail = false;
    if (!by_count && !by_k && !local && first_step > 0) {
      const float high = m - (float)first_step / per_step * temp + slack;
      if (high >= all && high < m) {
        lo = max(1u, Key<T>::of(all));
        hi = Key<T>::of(high);
        tail = true;
      }
    }
    Found f{0, 0, 0, 0, 0};
    for (;; tail = false) {
      int shift = 0;
      while (((hi - lo) >> shift) >= (uint32_t)kBins) shift++;
      f = level(lo, hi, shift, by_count, f, k_target, p_target, tail);
      if (f.bin < 0) return f;
      const uint32_t top = hi - ((uint32_t)f.bin << shift);
      if (shift == 0) {
        *key = top;
        return f;
      }
      const uint32_t width = (1u << shift) - 1;
      lo = top - lo > width ? top - width : lo;
      hi = top;
    }
  };
  uint32_t key_t = 0;          // kept: keys above it,
  uint32_t ties = 0xFFFFFFFFu;  // and the first `ties` entries equal to it
  if (by_k) {
    const Found f = select(true, (uint32_t)k, 0.0, &key_t);
    if (f.bin >= 0) {
      ties = (uint32_t)k - f.above;
      mass = f.mass_above + f.mass / f.count * ties;
    } else {  // fewer than k have any weight: top-k ends nothing, and they are all in the domain
      key_t = 0;
      u64 mine = 0;
      for (int i = tid; i < dn; i += kSampThreads) mine += fixed(weight(value(i)));
      mine = block_sum(mine, sh.warp_sum);
      if (tid == 0) sh.exchange[0] = mine;
      if (local) {
        mass = mine;
      } else {
        cl.sync();
        mass = over_cluster(0);
      }
    }
  }
  if (by_p) {
    const double target = (double)top_p * (double)mass;
    uint32_t key_p = 0;
    const Found f = select(false, 0, target, &key_p);
    if (f.bin >= 0) {
      const u64 each_f = f.mass / f.count;
      // the fewest of the class that reach the target
      u64 c = (double)f.mass_above >= target ? 1 : (u64)((target - (double)f.mass_above) / (double)each_f);
      while (c > 1 && (double)(f.mass_above + (c - 1) * each_f) >= target) c--;
      while (c < f.count && (double)(f.mass_above + c * each_f) < target) c++;
      const uint32_t ties_p = (uint32_t)max((u64)1, c);
      // the shorter of the two prefixes
      if (key_p > key_t || (key_p == key_t && ties_p < ties)) {
        key_t = key_p;
        ties = ties_p;
      }
    }
  }

  // ---- 5. index order: a thread's run of the domain is contiguous
  const int dper = ((dn + kSampThreads - 1) / kSampThreads) | 1;
  const int d0 = min(tid * dper, dn), d1 = min(d0 + dper, dn);
  uint32_t before = 0;  // entries equal to the threshold at lower indices
  if (ties != 0xFFFFFFFFu) {
    uint32_t mine = 0;
    for (int i = d0; i < d1; i++) mine += Key<T>::of(value(i)) == key_t;
    const u64 incl = block_inclusive(mine, sh.warp_sum);
    before = (uint32_t)(incl - mine);
    if (!local) {
      if (tid == kSampThreads - 1) sh.exchange[2] = incl;
      cl.sync();
      before += (uint32_t)below_rank(2);
    }
  }
  auto kept = [&](float v, uint32_t& tie) -> u64 {
    const uint32_t kv = Key<T>::of(v);
    if (kv < key_t) return 0;
    if (kv == key_t && tie++ >= ties) return 0;
    const float w = weight(v);
    return w >= min_p ? fixed(w) : 0;
  };
  u64 mine = 0;
  {
    uint32_t tie = before;
    for (int i = d0; i < d1; i++) mine += kept(value(i), tie);
  }
  u64 incl = block_inclusive(mine, sh.warp_sum);
  if (tid == kSampThreads - 1) sh.exchange[3] = incl;
  u64 total;
  if (local) {
    __syncthreads();
    total = sh.exchange[3];
  } else {
    cl.sync();
    total = over_cluster(3);
    incl += below_rank(3);
  }
  const double target = (double)u * (double)total;
  auto passed = [&](u64 c) { return (double)c > target || c >= total; };
  if (mine && passed(incl) && !(incl - mine > 0 && passed(incl - mine))) {  // one thread
    u64 run = incl - mine;
    uint32_t tie = before;
    for (int i = d0; i < d1; i++) {
      const float v = value(i);
      const u64 f = kept(v, tie);
      run += f;
      if (f && passed(run)) {
        finish(local ? given_i[i] : base + i, weight(v), total);
        break;
      }
    }
  }
  if (!local) cl.sync();  // no CTA leaves while others read its shared memory
}

template <typename T>
cudaError_t launch(const SampleArgs& args, cudaStream_t s) {
  SampleArgs a = args;
  // CTAs per row: slices of which two fit an SM (76 KB beside the 36 KB of tables), so that one
  // CTA's barriers and passes overlap another's; more, up to 16 and down to 2,048 entries each,
  // while the rows leave SMs idle.  256 rows of 151,936 in bf16: 133 us with 4 CTAs a row, 148 with
  // 2, 181 with 8.
  int cluster = 1;
  while (cluster < 8 && (int64_t)a.vocab * (int)sizeof(T) > (int64_t)cluster * 76 * 1024) cluster *= 2;
  while (cluster < kMaxCluster && a.vocab > cluster * 4096 && (int64_t)a.rows * cluster * 2 <= 2 * kAttnSms) cluster *= 2;
  const int align = 16 / (int)sizeof(T);
  a.slice = ((a.vocab + cluster - 1) / cluster + align - 1) / align * align;
  const size_t head = (sizeof(SampleShared) + 15) & ~(size_t)15;
  const size_t room = 200 * 1024 - head;
  a.cached = (int)std::min((size_t)a.slice, room / sizeof(T) / align * align);
  const size_t smem = head + (size_t)a.cached * sizeof(T);
  a.given = (int)((size_t)a.cached * sizeof(T) / (sizeof(T) + 4)) / 8 * 8;
  a.given_i = (int)(head + (size_t)a.given * sizeof(T));
  static bool wide[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev < 0 || dev >= 64 || !wide[dev])) {
    e = cudaFuncSetAttribute(sample_rows_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && dev >= 0 && dev < 64) wide[dev] = true;
  }
  if (e == cudaSuccess) e = smem_limit_once<sample_rows_kernel<T>>(200 * 1024);
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
  const SampleArgs a{logits, row_stride, rows, vocab, 0, 0, 0, 0, u, temperature, top_k, top_p, min_p, ids, probs};
  if (dtype == DPUF_TYPE_F32) return launch<float>(a, s);
  if (dtype == DPUF_TYPE_F16) return launch<__half>(a, s);
  return launch<__nv_bfloat16>(a, s);
}

}  // namespace dpuf
