// What the two attention kernels over the 8-bit paged cache share: the
// arguments, the division of the work and the conversion of codes.
//
// The chunks of all units (sequence, kv head, tile of query rows) form one
// line that is cut evenly over the CTAs, whatever the sequences' lengths (read
// on the device, so a captured step follows them).  Each unit's stretch starts
// with a lead that stands for its fixed cost.  A unit that falls within one CTA
// is finished there; the parts of a divided one meet in a second launch.
#pragma once

#include "tq_paged.cuh"

namespace tq {

constexpr float kNoScore = -1e30f;  // finite, so that differences of two of them are not NaN
constexpr float kLazy = 8.f;  // a score may pass its reference by 2^8 before the sums are rescaled
// The weights that fp16 holds are taken against a reference 2^7 under the
// largest, which with kLazy is all the room that fp16 has above 1 (2^15): it
// keeps all bits of weights down to 2^-21 of the largest, and 2^-32 of it is
// what the smaller ones are off by at most.
constexpr float kRoom = 7.f;

struct AttendArgs {
  tq_paged_kv kv;
  tq_paged_batch bt;
  const void* q;
  void* out;
  float* lse;
  float* part_o;   // [ctas][2][rows][d] normalised partial outputs
  float* part_l;   // [ctas][2][rows] their base-2 log-sum-exp
  int64_t q_stride;
  int q_heads;
  int group;
  int counted;
  int ctas;
  int whole;       // units are not divided
  uint32_t tries;  // after which a wait of the kernel for many rows gives up
  float scale2;    // softmax scale times log2(e)
};

struct SeqWork {
  int64_t first;  // row of its first token
  int n, base;    // rows; position of the first one
  int tiles;      // query tiles of a kv head
  int chunks;     // chunks of a unit
  int lead;       // what a unit costs besides its chunks, in chunks
  int weight;     // its length on the line: lead and chunks, or 1 where units are not divided
};

template <int ROWS, int CHUNK, int LEAD>
__device__ __forceinline__ SeqWork seq_work(const AttendArgs& a, int s) {
  const RowSpan r = row_span(a.bt, s);
  // a length past the block table is taken as the whole table
  const int64_t most = (int64_t)a.bt.table_width * a.kv.page_size;
  const int held = (int)min((int64_t)r.len, min(most, (int64_t)1 << 30));
  SeqWork w;
  w.first = r.first;
  w.n = r.n;
  w.base = a.counted ? held - r.n : held;
  w.tiles = (int)(((int64_t)r.n * a.group + ROWS - 1) / ROWS);
  w.chunks = max(1, (w.base + r.n + CHUNK - 1) / CHUNK);
  w.lead = a.whole ? 0 : LEAD;
  w.weight = a.whole ? 1 : LEAD + w.chunks;
  return w;
}

// The chunks [c0, c1) of a unit that lie within [rel, rel + room) of its
// stretch of the line (none where only its lead does); returns the positions
// that this takes.
__device__ __forceinline__ int64_t chunk_span(const AttendArgs& a, const SeqWork& w, int rel, int64_t room, int& c0, int& c1) {
  const int to = (int)min((int64_t)w.weight, rel + room);
  c0 = a.whole ? 0 : max(0, rel - w.lead);
  c1 = a.whole ? w.chunks : max(0, to - w.lead);
  return to - rel;
}

// prefix[s] = length of all units before sequence s, for s in [0, seqs].
template <int ROWS, int CHUNK, int LEAD, int THREADS>
__device__ __forceinline__ void plan_prefix(const AttendArgs& a, int64_t* prefix) {
  __shared__ int64_t sums[THREADS / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int64_t carry = 0;
  for (int base = 0; base < a.bt.seqs; base += THREADS) {
    const int s = base + tid;
    int64_t w = 0;
    if (s < a.bt.seqs) {
      const SeqWork q = seq_work<ROWS, CHUNK, LEAD>(a, s);
      w = (int64_t)q.tiles * a.kv.kv_heads * q.weight;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(FULL, w, o);
      if (lane >= o) w += v;
    }
    if (lane == 31) sums[warp] = w;
    __syncthreads();
    int64_t before = carry;
    for (int i = 0; i < THREADS / 32; ++i) {
      if (i < warp) before += sums[i];
      carry += sums[i];
    }
    if (s < a.bt.seqs) prefix[s + 1] = before + w;
    __syncthreads();
  }
  if (tid == 0) prefix[0] = 0;
  __syncthreads();
}

template <int SHARE>
__device__ __forceinline__ int64_t used_ctas(const AttendArgs& a, int64_t total) {
  const int64_t ctas = a.ctas, most = a.whole ? total : (total + SHARE - 1) / SHARE;
  return most < 1 ? 1 : (most < ctas ? most : ctas);
}

// last s with prefix[s] <= x (x < prefix[seqs]): the sequence that holds position x
__device__ __forceinline__ int find_seq(const int64_t* prefix, int seqs, int64_t x) {
  int lo = 0, hi = seqs;  // prefix[lo] <= x < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (prefix[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t r;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(sel));
  return r;
}
// {1024 + u0, 1024 + u1} in fp16 -> {u0 - 128, u1 - 128}, exactly
__device__ __forceinline__ uint32_t unbias(uint32_t x) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(x), "r"(0x64806480u));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Attention of tiles of 128 query rows (tq_paged_prefill.cu): workspace bytes,
// and the launch.
size_t prefill_workspace(int head_dim);
int launch_prefill(const AttendArgs& a, int q_dtype, int64_t max_context, cudaStream_t stream);

}  // namespace tq
