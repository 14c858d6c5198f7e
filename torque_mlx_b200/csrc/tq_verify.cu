// Verification of drafted tokens against the target's probabilities.
//
// Mathematics: draft i is accepted while u_i q_i(x_i) < p_i(x_i); the next
// token is a draw from max(p - q, 0) (normalised) at the rejected step, taken
// as argmax_v w_v / e_v with given unit-exponential numbers e.  Both are
// comparisons of single fp32 operations, so the result does not depend on the
// order of the work; equal scores go to the lowest index through the key
// (score bits, ~index), compared as one 64-bit number.
//
// Bound: the two or three rows that decide the next token.  A thread block
// cluster takes one sequence: each of its CTAs repeats the acceptance test (a
// few scattered reads), scans its share of the vocabulary, and the CTAs
// exchange their best keys through distributed shared memory, so one launch
// needs no workspace and no counters.  Each CTA arrives at the cluster's barrier
// on entry and waits there before its first store to another one: shared
// memory of a CTA that has not started yet may not be written.
//
// Measured: 4 drafts over 151936 columns: 7.0 us; 64 sequences of up to 8: 22 us
// (3 rows of each, 117 MB, 5.3 TB/s).
#include "tq_paged.cuh"

namespace tq {

constexpr int kVerifyMostThreads = 512;
constexpr int kVerifyMostCluster = 16;

struct VerifyArgs {
  const void* target;
  const void* draft;
  const int32_t* tokens;
  const int32_t* counts;
  const float* uniform;
  const float* noise;
  int32_t* accepted;
  int32_t* out;
  int64_t target_seq, target_row, draft_seq, draft_row, noise_stride, vocab;
  int drafts;
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ uint64_t key_of(float weight, float noise, int64_t v) {
  if (!(weight > 0.f)) return 0;
  const float score = __fdiv_rn(weight, noise);
  if (!(score >= 0.f)) return 0;
  return (uint64_t)__float_as_uint(score) << 32 | (uint32_t)~(uint32_t)v;
}

__device__ __forceinline__ uint64_t best_of(uint64_t a, uint64_t b) { return a > b ? a : b; }

// A thread's best key so far, with a bound that spares most divisions: only a
// weight above least = (best score, less 2^-20 of it) times its noise can have
// a score as large as the best (the product and the quotient are off by 2^-23
// in all; a product below the smallest normal number lets the weight pass).
struct Best {
  uint64_t key = 0;
  float least = 0.f;
  __device__ __forceinline__ bool may(float weight, float noise) const {
    return weight > 0.f && !(weight < least * noise - 2e-38f);
  }
  // eight columns from v: weights a - b, or a without column `taken`
  template <bool DIFF>
  __device__ __forceinline__ void vector(float (&a)[8], const float (&b)[8], const float (&n)[8], int64_t v, int64_t taken) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (DIFF) a[i] = __fsub_rn(a[i], b[i]);
      else if (v + i == taken) a[i] = 0.f;
      any |= may(a[i], n[i]);
    }
    if (any) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (may(a[i], n[i])) take(a[i], n[i], v + i);
    }
  }
  __device__ __forceinline__ void take(float weight, float noise, int64_t v) {
    const uint64_t k = key_of(weight, noise, v);
    if (k > key) {
      key = k;
      least = __uint_as_float((uint32_t)(k >> 32)) * (1.f - 0x1p-20f);
      if (!(least < 3e38f)) least = 3e38f;  // an infinite score: its product with a noise of zero stays a number
    }
  }
};

// The best key of columns [lo, hi): weights p, or max(p - q, 0), or p without
// column `taken`.
template <typename T, bool VEC, bool DIFF>
__device__ __forceinline__ uint64_t scan(const T* __restrict__ p, const T* __restrict__ q, int64_t taken,
                                         const float* __restrict__ e, int64_t lo, int64_t hi) {
  Best best;
  if (VEC) {  // lo, hi multiples of 8, rows at 16-byte boundaries
    constexpr int U = 2;  // vectors of eight in flight
    const int64_t STEP = blockDim.x * 8;
    int64_t v = lo + threadIdx.x * 8;
    for (; v + (U - 1) * STEP < hi; v += U * STEP) {
      float a[U][8], b[U][8], n[U][8];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        load8(p + v + u * STEP, a[u]);
        load8(e + v + u * STEP, n[u]);
        if (DIFF) load8(q + v + u * STEP, b[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) best.vector<DIFF>(a[u], b[u], n[u], v + u * STEP, taken);
    }
    for (; v < hi; v += STEP) {
      float a[8], b[8], n[8];
      load8(p + v, a);
      load8(e + v, n);
      if (DIFF) load8(q + v, b);
      best.vector<DIFF>(a, b, n, v, taken);
    }
  } else {
#pragma unroll 4
    for (int64_t v = lo + threadIdx.x; v < hi; v += blockDim.x) {
      float w = to_f32<T>(p[v]);
      if (DIFF) w = __fsub_rn(w, to_f32<T>(q[v]));
      else if (v == taken) w = 0.f;
      const float n = e[v];
      if (best.may(w, n)) best.take(w, n, v);
    }
  }
  return best.key;
}

// grid (cluster, seqs)
template <typename T, bool VEC>
__global__ void __launch_bounds__(kVerifyMostThreads, 2) verify_kernel(const VerifyArgs a) {
  __shared__ uint64_t warp_best[kVerifyMostThreads / 32];
  __shared__ uint64_t cta_best[2][kVerifyMostCluster];  // written by the cluster's CTAs
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x, size = gridDim.x;
  const int64_t b = blockIdx.y;
  cluster_arrive();  // this CTA has started: the others may write to its shared memory once they have waited for it
  grid_wait();
  const T* target = reinterpret_cast<const T*>(a.target) + b * a.target_seq;
  const T* draft = reinterpret_cast<const T*>(a.draft) + b * a.draft_seq;
  const int32_t* tokens = a.tokens + b * a.drafts;
  int count = a.drafts;
  if (a.counts) count = min(a.drafts, max(0, a.counts[b]));

  // ---- how many drafts stand: every warp for itself ----
  int accepted = count;
  for (int base = 0; base < count; base += 32) {
    const int i = base + lane;
    bool good = false;
    if (i < count) {
      const int32_t x = tokens[i];
      if (x >= 0 && x < a.vocab) {
        const float p = to_f32<T>(target[i * a.target_row + x]);
        const float q = a.draft ? to_f32<T>(draft[i * a.draft_row + x]) : 1.f;
        good = __fmul_rn(a.uniform[b * a.drafts + i], q) < p;
      }
    }
    const unsigned bad = __ballot_sync(FULL, !good && i < count);
    if (bad) {
      accepted = base + __ffs(bad) - 1;
      break;
    }
  }

  // ---- the next token ----
  const int64_t per = ((a.vocab + size - 1) / size + 7) / 8 * 8;
  const int64_t lo = min(a.vocab, rank * per), hi = min(a.vocab, lo + per);
  const T* p = target + accepted * a.target_row;
  const float* e = a.noise + b * a.noise_stride;
  uint64_t best = 0;
  const int first_pass = accepted == count ? 1 : 0;
  for (int pass = first_pass; pass < 2; ++pass) {
    if (pass == 0 && a.draft)
      best = scan<T, VEC, true>(p, draft + accepted * a.draft_row, -1, e, lo, hi);
    else
      best = scan<T, VEC, false>(p, nullptr, pass == 0 ? tokens[accepted] : -1, e, lo, hi);
#pragma unroll
    for (int o = 16; o; o >>= 1) best = best_of(best, __shfl_xor_sync(FULL, best, o));
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    if (pass == first_pass) cluster_wait();  // every CTA of the cluster has started
    if (warp == 0) {
      best = lane < blockDim.x / 32 ? warp_best[lane] : 0;
#pragma unroll
      for (int o = 8; o; o >>= 1) best = best_of(best, __shfl_xor_sync(FULL, best, o));
      if (lane < size) {  // to slot `rank` of the lane-th CTA
        uint32_t at = (uint32_t)__cvta_generic_to_shared(&cta_best[pass][rank]), there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(lane));
        asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there), "l"(best) : "memory");
      }
      __syncwarp();
    }
    cluster_arrive();
    cluster_wait();
    best = 0;
    for (int i = 0; i < size; ++i) best = best_of(best, cta_best[pass][i]);
    if (best) break;  // the same in every CTA of the cluster
  }
  if (rank != 0) return;
  const int32_t next = best ? (int32_t)~(uint32_t)best : 0;
  for (int i = tid; i <= a.drafts; i += blockDim.x)
    a.out[b * (a.drafts + 1) + i] = i < accepted ? tokens[i] : (i == accepted ? next : -1);
  if (tid == 0) a.accepted[b] = accepted;
}

template <typename T, bool VEC>
int launch_verify(const VerifyArgs& a, int64_t seqs, cudaStream_t stream) {
  // Eight CTAs of 256 threads a sequence, or sixteen of 512 while all of those
  // run at once: one sequence of 151936 columns takes 6.8 us instead of 11.4,
  // 14 take 8.8 instead of 11.9, but 16 take 14.2 instead of 13.9 and 64 take
  // 44.7 instead of 22.0.
  const bool few = seqs * 10 <= sm_count();
  const int cluster = few ? 16 : 8;
  static bool allowed[kMaxDevices] = {};
  const int dev = device_index();
  if (!allowed[dev]) {  // clusters of more than eight are opted into, once for each device
    const cudaError_t e = cudaFuncSetAttribute(verify_kernel<T, VEC>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_last_cuda_error(e);
      return TQ_E_CUDA;
    }
    allowed[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cluster, (unsigned)seqs);
  cfg.blockDim = dim3(few ? 512 : 256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, verify_kernel<T, VEC>, a);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_cuda_error(e);
    return TQ_E_CUDA;
  }
  return TQ_OK;
}

template <typename T>
int verify(const VerifyArgs& a, int64_t seqs, cudaStream_t stream) {
  // eight columns at a time where every row starts at 16 bytes
  const int64_t strides = a.target_seq | a.target_row | (a.draft ? a.draft_seq | a.draft_row : 0) | a.noise_stride | a.vocab;
  const uintptr_t at = (uintptr_t)a.target | (uintptr_t)a.draft | (uintptr_t)a.noise;
  return strides % 8 == 0 && at % 16 == 0 ? launch_verify<T, true>(a, seqs, stream) : launch_verify<T, false>(a, seqs, stream);
}

}  // namespace tq

using namespace tq;

extern "C" {

int tq_verify_drafts(const void* target, int64_t target_stride_seq, int64_t target_stride_row, const void* draft,
                     int64_t draft_stride_seq, int64_t draft_stride_row, int dtype, const int32_t* tokens,
                     const int32_t* draft_counts, const float* uniform, const float* noise, int64_t noise_stride,
                     int64_t seqs, int drafts, int64_t vocab, int32_t* accepted, int32_t* out_tokens,
                     tq_stream_t stream) {
  if (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) return TQ_E_ARG;
  if (seqs < 0 || seqs > 65535 || drafts < 0 || vocab <= 0 || vocab > INT32_MAX) return TQ_E_SHAPE;
  if ((seqs > 1 && noise_stride < vocab) || (drafts > 0 && target_stride_row < vocab) ||
      (draft && drafts > 1 && draft_stride_row < vocab) || target_stride_seq < 0 || draft_stride_seq < 0)
    return TQ_E_SHAPE;
  if (seqs == 0) return TQ_OK;
  if (!target || !noise || !accepted || !out_tokens || (drafts && (!tokens || !uniform))) return TQ_E_ARG;
  VerifyArgs a = {};
  a.target = target;
  a.draft = draft;
  a.tokens = tokens;
  a.counts = draft_counts;
  a.uniform = uniform;
  a.noise = noise;
  a.accepted = accepted;
  a.out = out_tokens;
  a.target_seq = target_stride_seq;
  a.target_row = target_stride_row;
  a.draft_seq = draft_stride_seq;
  a.draft_row = draft_stride_row;
  a.noise_stride = noise_stride;
  a.vocab = vocab;
  a.drafts = drafts;
  cudaStream_t s = (cudaStream_t)stream;
  if (dtype == TQ_F16) return verify<__half>(a, seqs, s);
  if (dtype == TQ_BF16) return verify<__nv_bfloat16>(a, seqs, s);
  return verify<float>(a, seqs, s);
}

}  // extern "C"
