// attn_parts.cuh - the workspace of the paged attention kernels: what the parts of an item that
// crosses CTAs leave behind, their counters, and the error word.
#pragma once
#include <algorithm>
#include <type_traits>

#include "attn_plan.cuh"

namespace dpuf {

constexpr int kAttnSms = 148;
constexpr int kAttnHeader = 256;  // the error word
static_assert(kAttnHeader + kAttnCounterBytes <= DPUF_PAGED_ATTENTION_ZEROED, "what is zero before the first use");

// Set to 1 when a bounded wait gave up.
DPUF_HD int* attn_error(void* ws) { return (int*)ws; }

template <int kRows, int kDim>
struct AttnParts {
  unsigned* count;  // [kAttnMaxCtas][2], zero between calls
  float2* ml;       // [2 CTAs][kRows]: maximum (in units of log 2) and sum
  float* o;         // [2 CTAs][kRows x kDim], unnormalised
  static constexpr size_t bytes(int ctas) {
    return kAttnHeader + kAttnCounterBytes + (size_t)2 * ctas * kRows * (sizeof(float2) + kDim * sizeof(float));
  }
  DPUF_DEV AttnParts(void* ws, int ctas) {
    count = (unsigned*)((char*)ws + kAttnHeader);
    ml = (float2*)((char*)ws + kAttnHeader + kAttnCounterBytes);
    o = (float*)(ml + (size_t)2 * ctas * kRows);
  }
};

// One thread, after its CTA's (or warpgroup's) parts are written and fenced: whether this was the
// last of the item's parts.  The counter is then zero again, as the next call finds it.
DPUF_DEV int attn_arrive(unsigned* counter, int parts) {
  const bool last = atomicAdd(counter, 1u) == (unsigned)(parts - 1);
  if (last) *counter = 0;
  __threadfence();
  return last;
}

// True in the CTA that has to join the item's parts; all of its threads see the others' parts.
DPUF_DEV bool attn_last_part(unsigned* counter, int parts, int* flag) {
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *flag = attn_arrive(counter, parts);
  __syncthreads();
  return *flag != 0;
}

// Raises a kernel's dynamic shared-memory limit on its first launch on each device.
template <auto kernel>
cudaError_t smem_limit_once(int bytes) {
  static bool done[64] = {};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || (dev >= 0 && dev < 64 && done[dev])) return e;
  e = cudaFuncSetAttribute((const void*)kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev] = true;
  return e;
}

// 16-bit queries and cache, head_dim <= 128 (kernels_paged_attn_tc.cu); cudaErrorNotSupported where
// no tensor map holds the cache's strides.
cudaError_t launch_paged_attention_tc(const AttnArgs& p, cudaStream_t s);
size_t paged_attention_tc_workspace();
// 16-bit cache, queries of its type or (head_dim <= 128) fp32 (kernels_paged_attn_rows.cu).
cudaError_t launch_paged_attention_rows(const AttnArgs& p, cudaStream_t s);

}  // namespace dpuf
