// ops_serving.cu - the C entries of the serving operators (include/dpuf_cuda.h): their checks of
// arguments, and the launches.
#include <cmath>
#include <string>

#include "engine_internal.h"
#include "serving.cuh"

// as callers that pack the structures by hand lay them out
static_assert(sizeof(DpufPagedKv) == 64, "DpufPagedKv");
static_assert(sizeof(DpufRopeAppendArgs) == 232, "DpufRopeAppendArgs");
static_assert(sizeof(DpufPagedAttentionArgs) == 184, "DpufPagedAttentionArgs");

namespace dpuf {
namespace {

int32_t refuse(const char* where, const std::string& why) {
  set_error(std::string(where) + ": " + why);
  return -1;
}
int32_t finish(const char* where, cudaError_t e) {
  if (e == cudaSuccess) return 0;
  (void)cudaGetLastError();  // not left for the next call to find
  set_error(std::string(where) + ": launch: " + cudaGetErrorString(e));
  return -4;
}

bool known_type(int t) { return t == DPUF_TYPE_F32 || t == DPUF_TYPE_F16 || t == DPUF_TYPE_BF16; }
int type_bytes(int t) { return t == DPUF_TYPE_F32 ? 4 : 2; }
bool aligned(const void* p, int n) { return ((uintptr_t)p & (uintptr_t)(n - 1)) == 0; }

// "" or what is wrong with the cache and its table (which a call without tokens need not have).
std::string check_cache(const DpufPagedKv& kv, const int32_t* table, int64_t table_stride, int n_seqs,
                        int pages_per_seq, int n_tokens) {
  if (!kv.k || !kv.v || (!table && n_tokens != 0)) return "null cache or page table";
  if (!known_type(kv.dtype)) return "unknown cache type";
  if (kv.n_pages <= 0 || kv.n_kv <= 0) return "a cache needs pages and heads";
  if (kv.page_size < 8 || kv.page_size > 1024 || (kv.page_size & (kv.page_size - 1)))
    return "page_size must be a power of two in [8, 1024]";
  if (kv.head_dim < 8 || kv.head_dim > 256 || kv.head_dim % 8) return "head_dim must be a multiple of 8 up to 256";
  const int b = type_bytes(kv.dtype);
  if (!aligned(kv.k, 16) || !aligned(kv.v, 16) || kv.page_stride * b % 16 || kv.head_stride * b % 16 ||
      kv.row_stride * b % 16)
    return "the cache's bases and strides must be multiples of 16 bytes";
  if (kv.page_stride < 0 || kv.head_stride < 0 || kv.row_stride < kv.head_dim) return "bad cache strides";
  const int least = n_tokens != 0 ? 1 : 0;
  if (n_seqs < least || pages_per_seq < least || table_stride < pages_per_seq) return "bad page table shape";
  return "";
}

}  // namespace
}  // namespace dpuf

using namespace dpuf;

extern "C" {

DPUF_EXPORT int32_t dpuf_cuda_rope_append(const DpufRopeAppendArgs* args, void* stream) {
  const char* me = "dpuf_cuda_rope_append";
  set_error("");
  if (!args) return refuse(me, "null arguments");
  const DpufRopeAppendArgs& a = *args;
  const std::string bad = check_cache(a.kv, a.page_table, a.table_stride, a.n_seqs, a.pages_per_seq, a.n_tokens);
  if (!bad.empty()) return refuse(me, bad);
  if (a.n_tokens < 0) return refuse(me, "negative n_tokens");
  if (a.n_tokens == 0) return 0;
  if (!a.q || !a.k || !a.v || !a.q_out || !a.cos_tab || !a.sin_tab || !a.seq || !a.pos)
    return refuse(me, "null pointer");
  if (!known_type(a.dtype) || !known_type(a.out_dtype)) return refuse(me, "unknown type");
  if (a.n_q <= 0) return refuse(me, "n_q must be positive");
  if (a.rotary_dim < 2 || a.rotary_dim % 2 || a.rotary_dim > a.kv.head_dim)
    return refuse(me, "rotary_dim must be even, at least 2 and at most head_dim");
  if (a.n_pos <= 0) return refuse(me, "empty rotary tables");
  const int b = type_bytes(a.dtype);
  const bool rows_aligned = aligned(a.q, 16) && aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.q_out, 16) &&
                            aligned(a.cos_tab, 16) && aligned(a.sin_tab, 16) && a.q_stride[0] * b % 16 == 0 &&
                            a.q_stride[1] * b % 16 == 0 && a.k_stride[0] * b % 16 == 0 &&
                            a.k_stride[1] * b % 16 == 0 && a.v_stride[0] * b % 16 == 0 && a.v_stride[1] * b % 16 == 0;
  return finish(me, launch_rope_append(a, rows_aligned, (cudaStream_t)stream));
}

DPUF_EXPORT int64_t dpuf_cuda_paged_attention_workspace(void) { return paged_attention_workspace(); }

DPUF_EXPORT int32_t dpuf_cuda_paged_attention(const DpufPagedAttentionArgs* args, void* stream) {
  const char* me = "dpuf_cuda_paged_attention";
  set_error("");
  if (!args) return refuse(me, "null arguments");
  DpufPagedAttentionArgs a = *args;
  const std::string bad = check_cache(a.kv, a.page_table, a.table_stride, a.n_seqs, a.pages_per_seq, a.n_tokens);
  if (!bad.empty()) return refuse(me, bad);
  if (a.n_tokens < 0) return refuse(me, "negative n_tokens");
  if (a.n_tokens == 0) return 0;
  if (!a.q || !a.out || !a.q_start || !a.kv_len) return refuse(me, "null pointer");
  if (a.n_q <= 0 || a.n_q % a.kv.n_kv) return refuse(me, "n_q must be a multiple of the cache's heads");
  if (a.dtype != DPUF_TYPE_F32 && a.dtype != a.kv.dtype) return refuse(me, "q must be float32 or of the cache's type");
  if (a.out_dtype != a.dtype && a.out_dtype != DPUF_TYPE_F32) return refuse(me, "out must be float32 or of q's type");
  if (a.max_q < 1 || a.max_q > (1 << 24)) return refuse(me, "max_q must be in [1, 2^24]");
  if ((int64_t)a.max_q * (a.n_q / a.kv.n_kv) > (1 << 30)) return refuse(me, "max_q times the group is too large");
  if (a.window < 0) return refuse(me, "negative window");
  if (a.window > 0 && !a.causal) return refuse(me, "a window needs causal attention");
  if (!std::isfinite(a.scale)) return refuse(me, "scale must be finite");
  const int b = type_bytes(a.dtype);
  if (!aligned(a.q, 16) || !aligned(a.out, 16) || a.q_stride[0] * b % 16 || a.q_stride[1] * b % 16)
    return refuse(me, "q, its strides and out must be multiples of 16 bytes");
  if (!a.workspace || !aligned(a.workspace, 16) || a.workspace_bytes < paged_attention_workspace())
    return refuse(me, "workspace is null, unaligned or too small");
  if (a.window > (1 << 30)) a.window = 1 << 30;  // no longer than any context: as good as none
  return finish(me, launch_paged_attention(a, (cudaStream_t)stream));
}

DPUF_EXPORT int32_t dpuf_cuda_paged_attention_status(void* workspace, void* stream) {
  const char* me = "dpuf_cuda_paged_attention_status";
  set_error("");
  if (!workspace) return refuse(me, "null workspace");
  bool gave_up = false;
  const int32_t rc = finish(me, paged_attention_status(workspace, &gave_up, (cudaStream_t)stream));
  if (rc != 0 || !gave_up) return rc;
  set_error(std::string(me) + ": a bounded wait in an attention kernel gave up");
  return -6;
}

DPUF_EXPORT uint64_t dpuf_cuda_stream_capture_id(void* stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (cudaStreamGetCaptureInfo((cudaStream_t)stream, &status, &id) != cudaSuccess) {
    (void)cudaGetLastError();  // not left for the next call to find
    return 0;
  }
  return status == cudaStreamCaptureStatusActive ? id : 0;
}

DPUF_EXPORT int32_t dpuf_cuda_sample_rows(const void* logits, int32_t dtype, int64_t row_stride, int32_t rows,
                                          int32_t vocab, const float* u, const float* temperature,
                                          const int32_t* top_k, const float* top_p, const float* min_p,
                                          int32_t* ids, float* probs, void* stream) {
  const char* me = "dpuf_cuda_sample_rows";
  set_error("");
  if (rows < 0) return refuse(me, "negative rows");
  if (rows == 0) return 0;
  if (!logits || !u || !ids) return refuse(me, "null pointer");
  if (!known_type(dtype)) return refuse(me, "unknown type");
  if (vocab < 1 || vocab > (1 << 20)) return refuse(me, "vocab must be in [1, 2^20]");
  if (rows > (1 << 26)) return refuse(me, "too many rows");
  if (!aligned(logits, type_bytes(dtype))) return refuse(me, "logits are not aligned to their type");
  return finish(me, launch_sample_rows(logits, dtype, row_stride, rows, vocab, u, temperature, top_k, top_p, min_p,
                                       ids, probs, (cudaStream_t)stream));
}

}  // extern "C"
