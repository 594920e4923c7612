// serving.cuh - what the serving kernels (rotary append, paged attention, sampling) share:
// element access in the three types, the paged cache's addresses, and the launchers.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "dpuf_cuda.h"

namespace dpuf {

DPUF_DEV float to_f32(float v) { return v; }
DPUF_DEV float to_f32(__half v) { return __half2float(v); }
DPUF_DEV float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
DPUF_DEV T from_f32(float v);
template <>
DPUF_DEV float from_f32<float>(float v) { return v; }
template <>
DPUF_DEV __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
DPUF_DEV __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One element in a type known at run time.
DPUF_DEV float load_as(const void* p, size_t i, int dtype) {
  if (dtype == DPUF_TYPE_F32) return ((const float*)p)[i];
  if (dtype == DPUF_TYPE_F16) return __half2float(((const __half*)p)[i]);
  return __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
DPUF_DEV void store_as(void* p, size_t i, int dtype, float v) {
  if (dtype == DPUF_TYPE_F32) ((float*)p)[i] = v;
  else if (dtype == DPUF_TYPE_F16) ((__half*)p)[i] = __float2half_rn(v);
  else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(v);
}

// Eight consecutive elements from a 16-byte aligned address.
DPUF_DEV void load8(const float* p, float (&v)[8]) {
  const float4 a = ((const float4*)p)[0], b = ((const float4*)p)[1];
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
DPUF_DEV void load8(const __half* p, float (&v)[8]) {
  const uint4 u = *(const uint4*)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*(const __half2*)&w[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
DPUF_DEV void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 u = *(const uint4*)p;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
// Eight consecutive elements, index i of p with i and p 16-byte aligned, type known at run time.
DPUF_DEV void store8_as(void* p, size_t i, int dtype, const float (&v)[8]) {
  if (dtype == DPUF_TYPE_F32) {
    float4* d = (float4*)((float*)p + i);
    d[0] = make_float4(v[0], v[1], v[2], v[3]);
    d[1] = make_float4(v[4], v[5], v[6], v[7]);
    return;
  }
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; j++) {
    if (dtype == DPUF_TYPE_F16) {
      const __half2 h = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *(const uint32_t*)&h;
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
      w[j] = *(const uint32_t*)&h;
    }
  }
  *(uint4*)((uint16_t*)p + i) = make_uint4(w[0], w[1], w[2], w[3]);
}

// Four consecutive elements, index i of p with i a multiple of 4 and p 16-byte aligned.
DPUF_DEV void store4_as(void* p, size_t i, int dtype, float a, float b, float c, float d) {
  if (dtype == DPUF_TYPE_F32) {
    *(float4*)((float*)p + i) = make_float4(a, b, c, d);
  } else if (dtype == DPUF_TYPE_F16) {
    const __half2 x = __floats2half2_rn(a, b), y = __floats2half2_rn(c, d);
    *(uint2*)((__half*)p + i) = make_uint2(*(const uint32_t*)&x, *(const uint32_t*)&y);
  } else {
    const __nv_bfloat162 x = __floats2bfloat162_rn(a, b), y = __floats2bfloat162_rn(c, d);
    *(uint2*)((__nv_bfloat16*)p + i) = make_uint2(*(const uint32_t*)&x, *(const uint32_t*)&y);
  }
}

// ---- launchers (arguments checked by the callers in ops_serving.cu)
cudaError_t launch_rope_append(const DpufRopeAppendArgs& a, bool aligned, cudaStream_t s);  // aligned: 16-byte accesses to rows
cudaError_t launch_paged_attention(const DpufPagedAttentionArgs& a, cudaStream_t s);
int64_t paged_attention_workspace();
cudaError_t paged_attention_status(void* workspace, bool* gave_up, cudaStream_t s);
cudaError_t launch_sample_rows(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const float* u,
                               const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                               int32_t* ids, float* probs, cudaStream_t s);

}  // namespace dpuf
