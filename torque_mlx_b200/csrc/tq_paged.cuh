// Shared pieces of the 8-bit paged cache: the batch view of ragged rows, page
// lookup with bounds checks, and the launch helper.
//
// Format: a page holds page_size tokens of one layer as codes
// [kv_heads, page_size, d], one byte each, biased by 128 (code 128 is zero,
// codes 1..255 stand for -127..127), with one fp32 scale for each page and kv
// head, K and V apart.  value = scale * (code - 128).
#pragma once

#include "tq_common.cuh"

namespace tq {

inline bool valid_page_size(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }

// Ragged rows: sequence s holds lengths[s] tokens and brings rows
// [starts[s], starts[s + 1]) (row s alone without starts).
struct RowSpan {
  int64_t first;  // row of the sequence's first new token
  int n;          // new tokens
  int len;        // tokens held before them
};

__device__ __forceinline__ RowSpan row_span(const tq_paged_batch& b, int s) {
  RowSpan r;
  r.len = b.lengths[s];
  int64_t lo = s, hi = (int64_t)s + 1;
  if (b.token_starts) {
    lo = b.token_starts[s];
    hi = b.token_starts[s + 1];
  }
  // rows outside [0, rows) and counts above the announced most are not touched
  if (lo < 0) lo = 0;
  if (hi > b.rows) hi = b.rows;
  int64_t n = hi - lo;
  if (n < 0 || r.len < 0) n = 0;
  if (n > b.max_new_tokens) n = b.max_new_tokens;
  r.first = lo;
  r.n = (int)n;
  if (r.len < 0) r.len = 0;
  return r;
}

// Page id of the idx-th page of sequence s, or -1 where the table has none.
__device__ __forceinline__ int page_id(const tq_paged_kv& kv, const tq_paged_batch& b, int s, int idx) {
  if (idx < 0 || idx >= b.table_width) return -1;
  const int id = b.block_table[(int64_t)s * b.table_stride + idx];
  return (id < 0 || id >= kv.num_pages) ? -1 : id;
}

inline int check_paged_kv(const tq_paged_kv* kv) {
  if (!kv) return TQ_E_ARG;
  if (!valid_head_dim(kv->head_dim)) return TQ_E_HEAD_DIM;
  if (!valid_page_size(kv->page_size) || kv->kv_heads <= 0 || kv->num_pages <= 0 || kv->num_pages > INT32_MAX)
    return TQ_E_SHAPE;
  if (!kv->k_pages || !kv->v_pages || !kv->k_scales || !kv->v_scales) return TQ_E_ARG;
  if ((uintptr_t)kv->k_pages % 16 || (uintptr_t)kv->v_pages % 16) return TQ_E_SHAPE;
  return TQ_OK;
}

inline int check_paged_batch(const tq_paged_batch* b) {
  if (!b) return TQ_E_ARG;
  if (b->seqs < 0 || b->rows < 0 || b->max_new_tokens < 0 || b->table_width < 0 || b->table_stride < b->table_width)
    return TQ_E_SHAPE;
  if (b->seqs > 0 && (!b->lengths || (b->table_width > 0 && !b->block_table))) return TQ_E_ARG;
  if (!b->token_starts && b->rows != b->seqs) return TQ_E_SHAPE;
  return TQ_OK;
}

// The batch with no more rows announced for a sequence than there are: what
// sizes a launch stays within its types, however large the announced number.
inline tq_paged_batch bounded(const tq_paged_batch& batch) {
  tq_paged_batch b = batch;
  if (b.max_new_tokens > b.rows) b.max_new_tokens = (int32_t)b.rows;
  return b;
}

constexpr int kMaxDevices = 64;
inline int device_index() {
  int dev = 0;
  cudaGetDevice(&dev);
  return dev < 0 || dev >= kMaxDevices ? 0 : dev;
}
inline int sm_count() {
  static int sms[kMaxDevices] = {};
  const int dev = device_index();
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    sms[dev] = n;
  }
  return sms[dev];
}

// Launch that may begin while the stream's previous kernel drains: every CTA
// of the kernel runs griddepcontrol.wait before it touches memory that a kernel
// before it may still write.  The attentions' joins read the batch's lengths and
// row starts before that, to plan while the attention runs: its CTAs let them
// start only after their own wait, which covers what wrote those.
template <typename... P, typename... A>
inline int launch_dependent(void (*kernel)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_cuda_error(e);
    return TQ_E_CUDA;
  }
  return TQ_OK;
}

__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_trigger() { asm volatile("griddepcontrol.launch_dependents;"); }

// whether fp16 holds the type's values as they are
template <typename T> struct Exact { static constexpr bool fp16 = false; };
template <> struct Exact<__half> { static constexpr bool fp16 = true; };

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Eight consecutive elements at a 16-byte aligned address.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  const uint4 v = *reinterpret_cast<const uint4*>(p);
  const T* h = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = to_f32<T>(h[i]);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w;
  f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  uint4 v;
  T* h = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < 8; ++i) h[i] = from_f32<T>(f[i]);
  *reinterpret_cast<uint4*>(p) = v;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

}  // namespace tq
