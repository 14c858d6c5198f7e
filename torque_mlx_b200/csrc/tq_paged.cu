// Append to the 8-bit paged cache with the rotary positions applied on the
// way, and the values of whole pages.
//
// Both are bound by memory traffic at prompt sizes and by latency for single
// tokens: a page of one head is quantised by one CTA, which finds the largest
// magnitude of the rows that the page gains (first pass over the rows), fixes
// the page's scale, rescales the tokens held only if the scale grew, and
// writes the new codes (second pass; the rows come from L1/L2 then).  One CTA
// for each page and head means no atomics, so the codes are the same for
// every run, and one launch covers q, k and v.
//
// Measured within a graph: one token of each of 64 sequences, 32 + 2 x 8 heads of
// 128: 4.4 us (1.4 MB: dependent loads bound it), and 6.0 for the values of their
// 64 last pages (25 MB); 7 prompts of 7197 tokens, 16 + 2 x 2 heads of 256: 35 us
// (140 MB, 4.0 TB/s: no load of a next page is in flight while a CTA reduces its
// maximum).
#include "tq_paged.cuh"

namespace tq {

constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kScaleFloor = 7.52316385e-37f;  // 2^-120: a page of zeros keeps a positive scale
constexpr float kScaleMost = 3.402823466e38f * kInv127;

struct RopeArgs {
  const float* cos;
  const float* sin;
  int64_t positions;
  int dim;
  int interleaved;
};

// The rotation of item i of a head's row at one position.  An item is two
// vectors of eight elements, at e0 and e1, such that rotary pairs lie within
// it; the same item of every head of the row shares it.  Values come back with
// the elementwise roundings of separate products and sums (no contraction), so
// that they equal the same formula written with single fp32 operations.
struct ItemRope {
  float c[8], s[8];
  int e0, e1;
  bool live, interleaved;

  __device__ __forceinline__ ItemRope(const RopeArgs& r, int i, bool rotate, int64_t pos) {
    live = rotate && i * 16 < r.dim;
    interleaved = r.interleaved;
    e0 = 16 * i;
    e1 = e0 + 8;
    if (!live) return;
    if (!interleaved) {
      e0 = 8 * i;
      e1 = r.dim / 2 + 8 * i;
    }
    load8(r.cos + pos * (r.dim / 2) + 8 * i, c);
    load8(r.sin + pos * (r.dim / 2) + 8 * i, s);
  }
  __device__ __forceinline__ void apply(float (&a)[8], float (&b)[8]) const {
    if (!live) return;
    if (interleaved) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = a[2 * j], y = a[2 * j + 1], u = b[2 * j], v = b[2 * j + 1];
        a[2 * j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
        a[2 * j + 1] = __fadd_rn(__fmul_rn(x, s[j]), __fmul_rn(y, c[j]));
        b[2 * j] = __fsub_rn(__fmul_rn(u, c[4 + j]), __fmul_rn(v, s[4 + j]));
        b[2 * j + 1] = __fadd_rn(__fmul_rn(u, s[4 + j]), __fmul_rn(v, c[4 + j]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float x = a[j], y = b[j];
        a[j] = __fsub_rn(__fmul_rn(x, c[j]), __fmul_rn(y, s[j]));
        b[j] = __fadd_rn(__fmul_rn(x, s[j]), __fmul_rn(y, c[j]));
      }
    }
  }
};

template <typename T>
__device__ __forceinline__ void load_item(const T* head, int i, const RopeArgs& r, bool rotate, int64_t pos,
                                          float (&a)[8], float (&b)[8], int& e0, int& e1) {
  const ItemRope rope(r, i, rotate, pos);
  e0 = rope.e0;
  e1 = rope.e1;
  load8(head + e0, a);
  load8(head + e1, b);
  rope.apply(a, b);
}

// Biased code of x: a NaN becomes zero (the conversion gives 0 for it).
__device__ __forceinline__ uint32_t code_of(float x) {
  return (uint32_t)(min(127, max(-127, __float2int_rn(x))) + 128);
}

// Biased codes of round(x / scale).  The product with 1 / scale is within 2e-5
// of the quotient (127 of it, three roundings of 2^-24), so its nearest whole
// number is the quotient's unless it lies within 1e-4 of a half; then the
// quotient itself decides.  Adding 1.5 * 2^23 + 128 rounds to even and leaves
// the biased code in the low byte.
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float scale, float inv) {
  constexpr float kMagic = 12582912.f + 128.f;
  uint32_t w[2] = {0, 0};
  bool near = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float y = __fmul_rn(x[i], inv);
    y = y == y ? fminf(fmaxf(y, -127.f), 127.f) : 0.f;
    const float m = __fadd_rn(y, kMagic);
    near |= fabsf(__fsub_rn(y, __fsub_rn(m, kMagic))) > 0.4999f;
    w[i / 4] |= (__float_as_uint(m) & 255u) << (8 * (i & 3));
  }
  if (near) {
    w[0] = w[1] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 4] |= code_of(__fdiv_rn(x[i], scale)) << (8 * (i & 3));
  }
  return make_uint2(w[0], w[1]);
}

// grid (seqs * pages, kv_heads, 2 + q parts): z = 0 the k codes of a page and
// head, 1 its v codes, from 2 on q_each of that kv head's q heads for the
// page's tokens.
//
// A thread keeps the values of its first kHold items from the first pass to
// the second in registers, which covers pages of 64 x 128; longer ones read
// the rest of their rows again.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS)
paged_append_kernel(const tq_paged_kv kv, const tq_paged_batch bt, const T* __restrict__ qkv, int64_t stride, int q_heads,
                    int q_each, const RopeArgs rope, T* __restrict__ q_out, int pages) {
  constexpr int kHold = THREADS == 128 ? 1 : 2;
  __shared__ float red[THREADS / 32];
  grid_wait();
  const int s = blockIdx.x / pages, j = blockIdx.x - s * pages;
  const int h = blockIdx.y, d = kv.head_dim, P = kv.page_size;
  const int shift = d == 64 ? 2 : d == 128 ? 3 : 4, items = 1 << shift;  // items of a head's row
  const RowSpan span = row_span(bt, s);
  const int first_page = span.len / P;
  const int page = first_page + j;
  const int64_t p0 = (int64_t)page * P;                     // first position of the page
  const int lo = j == 0 ? span.len - (int)p0 : 0;           // first slot written
  const int hi = (int)min((int64_t)P, (int64_t)span.len + span.n - p0);  // past the last one
  if (span.n == 0 || hi <= lo) return;
  const int64_t row0 = span.first + (p0 + lo - span.len);   // row of slot lo
  const int tid = threadIdx.x;
  int64_t known = hi - lo;                                  // tokens whose position has a rotary row
  if (rope.dim) known = min(known, max((int64_t)0, rope.positions - (p0 + lo)));

  if (blockIdx.z >= 2) {
    const int group = q_heads / kv.kv_heads, g0 = (blockIdx.z - 2) * q_each, g1 = min(group, g0 + q_each);
    const int total = (hi - lo) * items;
    for (int it = tid; it < total; it += THREADS) {
      const int t = it >> shift, i = it & (items - 1);
      const ItemRope r(rope, i, t < known, p0 + lo + t);
      const T* x = qkv + (row0 + t) * stride + (int64_t)(h * group) * d;
      T* o = q_out + ((row0 + t) * (int64_t)q_heads + h * group) * d;
#pragma unroll 4
      for (int g = g0; g < g1; ++g) {
        float a[8], b[8];
        load8(x + g * d + r.e0, a);
        load8(x + g * d + r.e1, b);
        r.apply(a, b);
        if (t >= known) {
#pragma unroll
          for (int k = 0; k < 8; ++k) a[k] = b[k] = __int_as_float(0x7fffffff);
        }
        store8(o + g * d + r.e0, a);
        store8(o + g * d + r.e1, b);
      }
    }
    return;
  }

  const bool is_v = blockIdx.z == 1;
  const int n = (int)known;
  if (n <= 0) return;
  const T* src = qkv + row0 * stride + (int64_t)(q_heads + (is_v ? kv.kv_heads : 0) + h) * d;
  const int total = n * items;
  float top = 0.f;
  float va[kHold][8], vb[kHold][8];
  int e0[kHold], e1[kHold];
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int it = tid + u * THREADS;
    if (it < total) {
      const int t = it >> shift, i = it & (items - 1);
      load_item(src + t * stride, i, rope, !is_v, p0 + lo + t, va[u], vb[u], e0[u], e1[u]);
    }
  }
  const int id = page_id(kv, bt, s, page);
  if (id < 0) return;
  uint8_t* codes = (is_v ? kv.v_pages : kv.k_pages) + ((int64_t)id * kv.kv_heads + h) * P * d;
  float* scale_at = (is_v ? kv.v_scales : kv.k_scales) + (int64_t)id * kv.kv_heads + h;
  const float was = lo > 0 ? *scale_at : 0.f;
#pragma unroll
  for (int u = 0; u < kHold; ++u)
    if (tid + u * THREADS < total) {
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, fmaxf(fabsf(va[u][k]), fabsf(vb[u][k])));
    }
  for (int it = tid + kHold * THREADS; it < total; it += THREADS) {
    const int t = it >> shift, i = it & (items - 1);
    float a[8], b[8];
    int x0, x1;
    load_item(src + t * stride, i, rope, !is_v, p0 + lo + t, a, b, x0, x1);
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, fmaxf(fabsf(a[k]), fabsf(b[k])));
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();  // also: every thread has read the old scale
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) top = fmaxf(top, red[w]);
  float scale = fminf(fmaxf(__fmul_rn(top, kInv127), kScaleFloor), kScaleMost);
  if (lo > 0) scale = fmaxf(scale, was);
  if (tid == 0) *scale_at = scale;
  const float inv = __fdiv_rn(1.f, scale);

  if (lo > 0 && scale != was) {  // the tokens held move to the larger scale
    const float ratio = __fdiv_rn(was, scale);
    uint4* p = reinterpret_cast<uint4*>(codes);
    for (int i = tid; i < lo * items; i += THREADS) {
      uint4 v = p[i];
      uint32_t* w = &v.x;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t u = 0;
#pragma unroll
        for (int b = 0; b < 4; ++b)
          u |= code_of(__fmul_rn((float)((int)((w[k] >> (8 * b)) & 255) - 128), ratio)) << (8 * b);
        w[k] = u;
      }
      p[i] = v;
    }
  }
#pragma unroll
  for (int u = 0; u < kHold; ++u) {
    const int it = tid + u * THREADS;
    if (it < total) {
      uint8_t* o = codes + (int64_t)(lo + (it >> shift)) * d;
      *reinterpret_cast<uint2*>(o + e0[u]) = codes8(va[u], scale, inv);
      *reinterpret_cast<uint2*>(o + e1[u]) = codes8(vb[u], scale, inv);
    }
  }
  for (int it = tid + kHold * THREADS; it < total; it += THREADS) {
    const int t = it >> shift, i = it & (items - 1);
    float a[8], b[8];
    int x0, x1;
    load_item(src + t * stride, i, rope, !is_v, p0 + lo + t, a, b, x0, x1);
    uint8_t* o = codes + (int64_t)(lo + t) * d;
    *reinterpret_cast<uint2*>(o + x0) = codes8(a, scale, inv);
    *reinterpret_cast<uint2*>(o + x1) = codes8(b, scale, inv);
  }
}

// grid (n * kv_heads, 2): a page and head of k or v, sixteen codes a thread.
template <typename T>
__global__ void __launch_bounds__(256)
paged_dequantize_kernel(const tq_paged_kv kv, const int32_t* __restrict__ ids, T* __restrict__ k_out,
                        T* __restrict__ v_out) {
  grid_wait();
  const int64_t at = blockIdx.x / kv.kv_heads;
  const int h = blockIdx.x % kv.kv_heads;
  const int64_t size = (int64_t)kv.page_size * kv.head_dim;
  const int id = ids[at];
  const bool known = id >= 0 && id < kv.num_pages;
  const int64_t block = (int64_t)(known ? id : 0) * kv.kv_heads + h;
  const uint8_t* codes = (blockIdx.y ? kv.v_pages : kv.k_pages) + block * size;
  T* out = (blockIdx.y ? v_out : k_out) + (at * kv.kv_heads + h) * size;
  const float scale = known ? (blockIdx.y ? kv.v_scales : kv.k_scales)[block] : __int_as_float(0x7fffffff);
  for (int64_t i = threadIdx.x; i < size / 16; i += 256) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (known) v = reinterpret_cast<const uint4*>(codes)[i];
    const uint32_t* w = &v.x;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float f[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        f[k] = __fmul_rn((float)((int)((w[2 * half + k / 4] >> (8 * (k & 3))) & 255) - 128), scale);
      store8(out + i * 16 + half * 8, f);
    }
  }
}

template <typename T>
int launch_append(const tq_paged_kv& kv, const tq_paged_batch& b, const void* qkv, int64_t stride, int q_heads,
                  const RopeArgs& rope, void* q_out, cudaStream_t stream) {
  // pages that max_new_tokens rows can touch, wherever the first one falls
  const int pages = (b.max_new_tokens + kv.page_size - 2) / kv.page_size + 1;
  const int64_t x = (int64_t)b.seqs * pages;
  if (x > INT32_MAX || kv.kv_heads > 65535) return TQ_E_SHAPE;
  // 128 threads while a page gains few tokens (one token of 64 sequences: 4.4 us,
  // 11.0 with 256), 256 for prompts, whose pages of up to 64 x 128 they hold in
  // registers between the passes (prompts of 7197 tokens in pages of 32 x 256
  // take 34.6 us, and 31.2 with 128 threads, so the rule is not the best there).
  // The q heads of a kv head share a CTA (and the angles a thread loads) up to
  // sixteen items a thread: 2, 4, 8 and 16 take 42.4, 37.9, 32.5 and 34.6 us for
  // the same prompts.
  const int rows = b.max_new_tokens < kv.page_size ? b.max_new_tokens : kv.page_size, items = rows * (kv.head_dim / 16);
  const int group = q_heads / kv.kv_heads;
  const bool wide = items > 128;
  const int threads = wide ? 256 : 128;
  int each = 16 * threads / items;
  each = each < 1 ? 1 : (each > group ? group : each);
  const int parts = group ? (group + each - 1) / each : 0;
  if (parts > 65533) return TQ_E_SHAPE;
  const dim3 grid((unsigned)x, kv.kv_heads, 2 + parts);
  if (wide)
    return launch_dependent(paged_append_kernel<T, 256>, grid, dim3(256), 0, stream, kv, b, (const T*)qkv, stride,
                            q_heads, each, rope, (T*)q_out, pages);
  return launch_dependent(paged_append_kernel<T, 128>, grid, dim3(128), 0, stream, kv, b, (const T*)qkv, stride, q_heads,
                          each, rope, (T*)q_out, pages);
}

}  // namespace tq

using namespace tq;

extern "C" {

int tq_paged_append(const tq_paged_kv* kv, const tq_paged_batch* batch, const void* qkv, int x_dtype,
                    int64_t qkv_stride, int q_heads, const float* cos_table, const float* sin_table,
                    int64_t positions, int rotary_dim, int interleaved, void* q_out, tq_stream_t stream) {
  int st = check_paged_kv(kv);
  if (st == TQ_OK) st = check_paged_batch(batch);
  if (st != TQ_OK) return st;
  if (batch->seqs > TQ_PAGED_MAX_SEQS) return TQ_E_SHAPE;
  if (x_dtype != TQ_F32 && x_dtype != TQ_F16 && x_dtype != TQ_BF16) return TQ_E_ARG;
  if (q_heads < 0 || q_heads % kv->kv_heads) return TQ_E_SHAPE;
  const int64_t width = (int64_t)(q_heads + 2 * kv->kv_heads) * kv->head_dim;
  const int per16 = x_dtype == TQ_F32 ? 4 : 8;  // elements of 16 bytes
  if (batch->rows > 1 && (qkv_stride < width || qkv_stride % per16)) return TQ_E_SHAPE;
  if (rotary_dim < 0 || rotary_dim % 16 || rotary_dim > kv->head_dim || positions < 0) return TQ_E_SHAPE;
  if (batch->seqs == 0 || batch->rows == 0 || batch->max_new_tokens == 0) return TQ_OK;
  if (!qkv || (q_heads && !q_out) || (rotary_dim && (!cos_table || !sin_table))) return TQ_E_ARG;
  if ((uintptr_t)qkv % 16 || (uintptr_t)q_out % 16 || (uintptr_t)cos_table % 16 || (uintptr_t)sin_table % 16)
    return TQ_E_SHAPE;
  const RopeArgs rope{cos_table, sin_table, positions, rotary_dim, interleaved};
  const tq_paged_batch b = bounded(*batch);
  cudaStream_t s = (cudaStream_t)stream;
  if (x_dtype == TQ_F16) return launch_append<__half>(*kv, b, qkv, qkv_stride, q_heads, rope, q_out, s);
  if (x_dtype == TQ_BF16) return launch_append<__nv_bfloat16>(*kv, b, qkv, qkv_stride, q_heads, rope, q_out, s);
  return launch_append<float>(*kv, b, qkv, qkv_stride, q_heads, rope, q_out, s);
}

int tq_paged_dequantize(const tq_paged_kv* kv, const int32_t* ids, int64_t n, void* k_out, void* v_out,
                        int out_dtype, tq_stream_t stream) {
  const int st = check_paged_kv(kv);
  if (st != TQ_OK) return st;
  if (out_dtype != TQ_F32 && out_dtype != TQ_F16 && out_dtype != TQ_BF16) return TQ_E_ARG;
  if (n < 0 || n * kv->kv_heads > INT32_MAX) return TQ_E_SHAPE;
  if (n == 0) return TQ_OK;
  if (!ids || !k_out || !v_out) return TQ_E_ARG;
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16) return TQ_E_SHAPE;
  const dim3 grid((unsigned)(n * kv->kv_heads), 2), block(256);
  cudaStream_t s = (cudaStream_t)stream;
  if (out_dtype == TQ_F16)
    return launch_dependent(paged_dequantize_kernel<__half>, grid, block, 0, s, *kv, ids, (__half*)k_out, (__half*)v_out);
  if (out_dtype == TQ_BF16)
    return launch_dependent(paged_dequantize_kernel<__nv_bfloat16>, grid, block, 0, s, *kv, ids, (__nv_bfloat16*)k_out,
                            (__nv_bfloat16*)v_out);
  return launch_dependent(paged_dequantize_kernel<float>, grid, block, 0, s, *kv, ids, (float*)k_out, (float*)v_out);
}

}  // extern "C"
