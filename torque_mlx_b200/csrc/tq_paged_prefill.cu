// Attention of many query rows for each kv head over the 8-bit paged cache:
// prompts and their chunks.
//
// Mathematics: as in tq_paged_attend.cu, with one exponential for each score.
// For a page of 2^lv scale, w_j = 2^(s_j + lv - m2) weighs v's codes, and the
// softmax's own sum is l = sum_j w_j 2^-lv.  Where a page's scale is under
// 2^-40 of the largest seen (or 2^-90), its values are left out of the product
// and lv is taken that large, so that l stays exact.
//
// Bound: the two products, 4 d flops for each visible (row, token) pair, on
// the tensor cores, and the exponentials, which take as long at d = 128 (16 a
// clock for each SM).  Both tiles are 128 x 128: S = Q K^T and O += P V by
// tcgen05.mma with fp16 operands and fp32 accumulators in tensor memory; P
// goes back to tensor memory over S, which it replaces.  K and V tiles are
// converted from codes to fp16 once for 128 rows.
//
// A CTA takes 256 rows (128 at d = 256, where tensor memory holds no more):
// for each 128 of them four softmax warps (a thread a row, no shuffles), four
// warps that convert the next tiles meanwhile, once for all rows, and one that
// issues the products.  The two halves take turns: while one's scores are in
// the softmax, the other's products run.
#include "tq_paged_attend.cuh"

namespace tq {

constexpr int kRows = 128;          // query rows of a product
constexpr int kTokens = 128;        // tokens of a tile
constexpr int kPrefillShare = 2;    // smallest share of a CTA, in tiles

// ---- mbarriers, tensor memory and products ----
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// false if the wait gave up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity) {
  for (uint32_t it = 0; it < 20000u; ++it) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity), "r"(100000u)
        : "memory");
    if (done) return true;
  }
  return false;
}
// the same for a whole warp, which goes on together
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity) { return __all_sync(FULL, bar_wait(bar, parity)); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand of 128-byte rows, 16-byte pieces swizzled by the row's
// low three bits, rows in groups of eight (1024 bytes); lead = bytes between
// blocks of 64 elements where those are the operand's outer dimension.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// fp16 operands, fp32 accumulator, M = 128; the second operand's rows are k
// (columns contiguous) where `by_rows`
__host__ __device__ constexpr uint32_t shape(int n, bool by_rows) {
  return 1u << 4 | (by_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kRows >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// 32 columns of the thread's lane
__device__ __forceinline__ void tmem_load32(uint32_t at, float (&v)[32]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
      "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t at, const float (&v)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// pairs of fp32 in one instruction
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

template <int D> struct PrefillShape {
  static constexpr int kHalves = D == 256 ? 1 : 2;
  static constexpr int kUnit = kHalves * kRows;            // query rows of a unit
  static constexpr int kStages = D == 256 ? 1 : 2;         // K and V tiles that are held
  static constexpr int kSoftmax = kHalves * 128;           // threads: softmax, then those that convert, then a warp
  static constexpr int kConvert = D == 256 ? 256 : 128;
  static constexpr int kThreads = kSoftmax + kConvert + 32;
  static constexpr int kOperand = D / 64 * 128 * 128;      // bytes of 128 rows of Q, K or V in fp16
  static constexpr int kSmem = (kHalves + 2 * kStages) * kOperand + 1024;  // from a 1024-byte boundary on
  static constexpr int kColumns = 512;                     // tensor memory of a half: S (P over it), then O
  static constexpr int kRow = D / 16;                      // pieces of 16 codes of a token
  static constexpr int kPieces = 128 * kRow / kConvert;    // a thread's share of a tile
  static constexpr int kTurn = kConvert / kRow;            // tokens from one piece of a thread to its next
  static constexpr int kAges = 4;                          // tiles whose page scales are kept
};

// byte offset of elements [8 q, 8 q + 8) of row t within an operand
__device__ __forceinline__ uint32_t place(int t, int q) { return (uint32_t)((q >> 3) * 16384 + t * 128 + (((q & 7) ^ (t & 7)) << 4)); }

// One half's softmax of a tile: weights of the thread's row to tensor memory.
// lv and inv are of the tile's chunks of sixteen tokens; columns past `seen`
// are hidden where MASKED.
template <bool MASKED>
__device__ __forceinline__ void weigh(uint32_t at, const float* ks, const float* lv, const float* inv, float kf, float m2,
                                      int seen, float& l) {
#pragma unroll 1
  for (int b = 0; b < 4; ++b) {
    float v[32];
    tmem_load32(at + b * 32, v);
    uint32_t p[16];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int chunk = 2 * b + u;
      const bool here = ks[chunk] >= 0.f || ks[chunk] != ks[chunk];
      const float f = here ? ks[chunk] * kf : 0.f, g = here ? lv[chunk] - m2 : -INFINITY;  // no page: weights of zero
      const uint64_t ff = pair(f, f), gg = pair(g, g);
      uint64_t sum = 0;
#pragma unroll
      for (int k = 0; k < 16; k += 2) {
        const float2 s = halves(fma2(pair(v[u * 16 + k], v[u * 16 + k + 1]), ff, gg));
        float x = ex2(s.x), y = ex2(s.y);
        if (MASKED) {
          x = chunk * 16 + k <= seen ? x : 0.f;
          y = chunk * 16 + k + 1 <= seen ? y : 0.f;
        }
        sum = add2(sum, pair(x, y));
        p[u * 8 + k / 2] = half2_bits(x, y);
      }
      const float2 s = halves(sum);
      l = fmaf(s.x + s.y, inv[chunk], l);
    }
    tmem_store16(at + b * 16, p);
  }
}

// The largest exponent of the thread's row in a tile.
template <bool MASKED>
__device__ __forceinline__ float highest(uint32_t at, const float* ks, const float* lv, float kf, int seen) {
  float top = -INFINITY;
#pragma unroll 1
  for (int b = 0; b < 4; ++b) {
    float v[32];
    tmem_load32(at + b * 32, v);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int chunk = 2 * b + u;
      float x = -INFINITY;
#pragma unroll
      for (int k = 0; k < 16; ++k)
        if (!MASKED || chunk * 16 + k <= seen) x = fmaxf(x, v[u * 16 + k]);
      if (ks[chunk] >= 0.f) top = fmaxf(top, fmaf(x, ks[chunk] * kf, lv[chunk]));
    }
  }
  return top;
}

template <int D, typename T>
__global__ void __launch_bounds__(PrefillShape<D>::kThreads, 1) paged_prefill_kernel(const AttendArgs a) {
  using Shape = PrefillShape<D>;
  constexpr int H = Shape::kHalves, ST = Shape::kStages, UNIT = Shape::kUnit;
  extern __shared__ __align__(1024) uint8_t prefill_smem[];
  __shared__ uint64_t bars[4 * ST + 3 * H];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int failed;
  __shared__ float page_k[Shape::kAges][8], page_lv[Shape::kAges][8], page_inv[Shape::kAges][8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(prefill_smem), base = (raw + 1023u) & ~1023u;
  uint8_t* const smem = prefill_smem + (base - raw);
  uint8_t *const sk = smem + H * Shape::kOperand, *const sv = sk + ST * Shape::kOperand;
  const uint32_t k_at = base + H * Shape::kOperand, v_at = k_at + ST * Shape::kOperand;
  int64_t* prefix = reinterpret_cast<int64_t*>(sv + ST * Shape::kOperand);
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  const uint32_t k_full = bar0, k_empty = k_full + 8 * ST, v_full = k_empty + 8 * ST, v_empty = v_full + 8 * ST;  // [stage]
  const uint32_t s_done = v_empty + 8 * ST, p_full = s_done + 8 * H, pv_done = p_full + 8 * H;                     // [half]

  grid_wait();
  plan_prefix<UNIT, kTokens, Shape::kThreads>(a, prefix);
  grid_trigger();
  const int64_t total = prefix[a.bt.seqs];
  const int64_t ctas = used_ctas<kPrefillShare>(a, total);
  if ((int64_t)blockIdx.x >= ctas) return;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      bar_init(k_full + 8 * i, Shape::kConvert);
      bar_init(v_full + 8 * i, Shape::kConvert);
      bar_init(k_empty + 8 * i, 1);
      bar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < H; ++i) {
      bar_init(s_done + 8 * i, 1);
      bar_init(p_full + 8 * i, 128);
      bar_init(pv_done + 8 * i, 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  constexpr int kIssuer = Shape::kThreads / 32 - 1;  // the warp of the products
  if (warp == kIssuer) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(&tmem_at)),
                 "r"((uint32_t)Shape::kColumns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_at;  // half i: S at 256 i, O at 256 i + 128

  const int Hkv = a.kv.kv_heads, P = a.kv.page_size;
  int64_t pos = (int64_t)blockIdx.x * total / ctas;
  const int64_t end = ((int64_t)blockIdx.x + 1) * total / ctas;
  uint32_t tiles_done = 0, half_done[2] = {0, 0};  // of the units before: the barriers' phases
  for (int slot = 0; pos < end; slot = 1) {
    const int s = find_seq(prefix, a.bt.seqs, pos);
    const SeqWork w = seq_work<UNIT, kTokens>(a, s);
    const int64_t rel = pos - prefix[s];
    const int unit = (int)(rel / w.weight), c0 = (int)(rel - (int64_t)unit * w.weight);
    const int c1 = a.whole ? w.chunks : (int)min((int64_t)w.chunks, c0 + (end - pos));
    const int h = unit / w.tiles, r0 = (unit - h * w.tiles) * UNIT;
    const int nr = min(UNIT, w.n * a.group - r0);
    const int last = w.base + (r0 + nr - 1) / a.group;  // last position that a row attends
    const int n = last < 0 ? 0 : max(0, min(c1, last / kTokens + 1) - c0);
    const int live_halves = H == 2 && nr > kRows ? 2 : 1;
    pos += a.whole ? 1 : c1 - c0;

    const int half = H == 2 ? (tid >> 7) & 1 : 0;  // softmax threads
    float kf = 0.f;                                // the row's score factor
    int limit = -1, free_to = 0;
    if (tid < Shape::kSoftmax) {
      // ---- the row's query, times a power of two that makes fp16 hold it, to shared memory ----
      const int r = r0 + tid;
      const bool live = tid < nr;
      const T* row = reinterpret_cast<const T*>(a.q) + (w.first + r / a.group) * a.q_stride +
                     (int64_t)(h * a.group + r % a.group) * D;
      uint8_t* sq = smem + half * Shape::kOperand;
      float up = a.scale2 < 0.f ? -1.f : 1.f, down = 1.f;
      if (!Exact<T>::fp16) {
        float top = 0.f;
        if (live) {
#pragma unroll 4
          for (int q = 0; q < D / 8; ++q) {
            float f[8];
            load8(row + 8 * q, f);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (fabsf(f[k]) <= 3.402823466e38f) top = fmaxf(top, fabsf(f[k]));
          }
        }
        int e = top > 0.f ? 13 - (ilogbf(top) + 1) : 0;
        e = min(120, max(-120, e));
        up *= __int_as_float((e + 127) << 23);
        down = __int_as_float((127 - e) << 23);
      }
#pragma unroll 4
      for (int q = 0; q < D / 8; ++q) {
        float f[8] = {};
        if (live) load8(row + 8 * q, f);
        uint4 v;
        v.x = half2_bits(f[0] * up, f[1] * up);
        v.y = half2_bits(f[2] * up, f[3] * up);
        v.z = half2_bits(f[4] * up, f[5] * up);
        v.w = half2_bits(f[6] * up, f[7] * up);
        *reinterpret_cast<uint4*>(sq + place(tid & 127, q)) = v;
      }
      kf = fabsf(a.scale2) * down;
      limit = w.base + r / a.group;
      free_to = w.base + (r0 + half * kRows) / a.group;  // positions up to here need no mask
      proxy_fence();
    }
    __syncthreads();  // Q is complete; the last unit's accumulators have been read
    bool ok = true;
    float m2 = kNoScore, l = 0.f;

    if (tid < Shape::kSoftmax) {
      // ---- softmax: a row a thread ----
      const uint32_t t_s = tmem + half * 256 + ((uint32_t)((warp & 3) * 32) << 16), t_o = t_s + 128;
      for (int i = 0; i < n && half < live_halves; ++i) {
        const uint32_t ph = (half_done[half] + i) & 1, age = (tiles_done + i) % Shape::kAges;
        if (!(ok = warp_wait(s_done + 8 * half, ph))) break;
        tc_fence_after();
        const int tok = (c0 + i) * kTokens;
        const bool masked = tok + kTokens - 1 > free_to;
        const int seen = limit - tok;  // columns 0..seen are visible
        const float *ks = page_k[age], *lv = page_lv[age], *inv = page_inv[age];
        const float top = masked ? highest<true>(t_s, ks, lv, kf, seen) : highest<false>(t_s, ks, lv, kf, seen);
        if (__any_sync(FULL, top > m2 + kLazy)) {
          const float nm = fmaxf(m2, top), f = ex2(m2 - nm);
          m2 = nm;
          l *= f;
          if (i > 0) {  // the sums of the tiles before: their products are complete
#pragma unroll 1
            for (int b = 0; b < D / 32; ++b) {
              float v[32];
              tmem_load32(t_o + b * 32, v);
#pragma unroll
              for (int k = 0; k < 32; ++k) v[k] *= f;
              tmem_store32(t_o + b * 32, v);
            }
          }
        }
        if (masked) weigh<true>(t_s, ks, lv, inv, kf, m2, seen, l);
        else weigh<false>(t_s, ks, lv, inv, kf, m2, seen, l);
        tmem_store_wait();
        tc_fence_before();
        bar_arrive(p_full + 8 * half);
      }
    } else if (warp != kIssuer) {
      // ---- conversion of the tiles' codes ----
      constexpr int PIECES = Shape::kPieces, TURN = Shape::kTurn;
      const int pt = tid - Shape::kSoftmax, t0 = pt / Shape::kRow, q = pt % Shape::kRow;
      // Lanes of the odd blocks of 64 elements start with the second half of
      // their sixteen, so that eight lanes fill eight columns.
      const int turn = (q >> 2) & 1;
      const uint32_t to_a = place(t0, 2 * q + turn), to_b = place(t0, 2 * q + 1 - turn);
      uint4 kr[PIECES], vr[PIECES];  // codes of the next tile
      float most = -INFINITY;        // log2 of the largest v scale so far
      // lanes 0..7: pages of the chunks of the tile that is loaded next, and the
      // scales of that and of the one that is stored next
      int ids = -1, ids_now = -1;
      float scale_k = 0.f, scale_v = 0.f, scale_k_now = 0.f, scale_v_now = 0.f;
      auto fetch_ids = [&](int i) {
        const int tok = (c0 + i) * kTokens + lane * 16;
        ids = lane < 8 && i < n && tok <= last ? page_id(a.kv, a.bt, s, tok / P) : -1;
      };
      auto fetch_scales = [&]() {
        if (ids >= 0) {
          scale_k = a.kv.k_scales[(int64_t)ids * Hkv + h];
          scale_v = a.kv.v_scales[(int64_t)ids * Hkv + h];
        }
      };
      auto load = [&](const uint8_t* pages, int i, uint4 (&reg)[PIECES]) {
        const int in_page = (c0 + i) * kTokens + t0;
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int id = __shfl_sync(FULL, ids, (t0 + TURN * j) >> 4);
          reg[j] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
          if (id >= 0) {
            const int64_t row = ((int64_t)id * Hkv + h) * P + ((in_page + TURN * j) & (P - 1));
            reg[j] = *reinterpret_cast<const uint4*>(pages + row * D + q * 16);
          }
        }
      };
      auto store = [&](uint8_t* to, const uint4 (&reg)[PIECES]) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const uint32_t x[4] = {reg[j].x, reg[j].y, reg[j].z, reg[j].w};
          uint32_t y[8];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            y[2 * k] = unbias(prmt(x[k], 0x64646464u, 0x4140));
            y[2 * k + 1] = unbias(prmt(x[k], 0x64646464u, 0x4342));
          }
          const uint4 lo = make_uint4(y[0], y[1], y[2], y[3]), hi = make_uint4(y[4], y[5], y[6], y[7]);
          *reinterpret_cast<uint4*>(to + to_a + j * (TURN * 128)) = turn ? hi : lo;
          *reinterpret_cast<uint4*>(to + to_b + j * (TURN * 128)) = turn ? lo : hi;
        }
      };
      fetch_ids(0);
      fetch_scales();
      load(a.kv.k_pages, 0, kr);
      load(a.kv.v_pages, 0, vr);
      for (int i = 0; i < n; ++i) {
        const uint32_t tile = tiles_done + i, st = tile % ST, use = tile / ST;
        ids_now = ids, scale_k_now = scale_k, scale_v_now = scale_v;
        fetch_ids(i + 1);
        if (use > 0 && !(ok = warp_wait(k_empty + 8 * st, (use - 1) & 1))) break;
        // page scales, for the softmax, and chunks whose v is left out
        const float lv = log2f(scale_v_now);
        float top = ids_now >= 0 ? lv : -INFINITY;
#pragma unroll
        for (int o = 4; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
        most = fmaxf(most, __shfl_sync(FULL, top, 0));
        const float least = fmaxf(most - 40.f, -90.f);
        const uint32_t drop = __ballot_sync(FULL, lane < 8 && ids_now >= 0 && lv < least);
        if (pt < 8) {
          const uint32_t age = tile % Shape::kAges;
          const float use_lv = ids_now < 0 ? 0.f : (lv < least ? least : lv);
          page_k[age][lane] = ids_now >= 0 ? scale_k_now : -1.f;
          page_lv[age][lane] = use_lv;
          page_inv[age][lane] = ex2(-use_lv);
        }
        store(sk + st * Shape::kOperand, kr);
        proxy_fence();
        bar_arrive(k_full + 8 * st);
        load(a.kv.k_pages, i + 1, kr);
        fetch_scales();
        if (drop) {
#pragma unroll
          for (int j = 0; j < PIECES; ++j)
            if (drop >> ((t0 + TURN * j) >> 4) & 1) vr[j] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
        }
        if (use > 0 && !(ok = warp_wait(v_empty + 8 * st, (use - 1) & 1))) break;
        store(sv + st * Shape::kOperand, vr);
        proxy_fence();
        bar_arrive(v_full + 8 * st);
        load(a.kv.v_pages, i + 1, vr);
      }
    } else if (lane == 0) {
      // ---- products: S of the first tile, then P V and the next S of each half in turn ----
      auto scores = [&](int i, int x) {
        const uint32_t st = (tiles_done + i) % ST;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
          mma_ss(tmem + x * 256, operand(base + x * Shape::kOperand + off, 16),
                 operand(k_at + st * Shape::kOperand + off, 16), shape(kTokens, false), k > 0);
        }
        tc_commit(s_done + 8 * x);
        if (x == live_halves - 1) tc_commit(k_empty + 8 * st);
      };
      if (n > 0 && (ok = bar_wait(k_full + 8 * (tiles_done % ST), (tiles_done / ST) & 1))) {
        tc_fence_after();
        for (int x = 0; x < live_halves; ++x) scores(0, x);
      }
      for (int i = 0; i < n && ok; ++i) {
        const uint32_t tile = tiles_done + i, st = tile % ST;
        for (int x = 0; x < live_halves; ++x) {
          if (x == 0 && !(ok = bar_wait(v_full + 8 * st, (tile / ST) & 1))) break;
          if (!(ok = bar_wait(p_full + 8 * x, (half_done[x] + i) & 1))) break;
          tc_fence_after();
#pragma unroll
          for (int k = 0; k < kTokens / 16; ++k)
            mma_ts(tmem + x * 256 + 128, tmem + x * 256 + k * 8, operand(v_at + st * Shape::kOperand + k * 2048, 16384),
                   shape(D, true), i > 0 || k > 0);
          tc_commit(pv_done + 8 * x);
          if (x == live_halves - 1) tc_commit(v_empty + 8 * st);
          if (i + 1 < n) {
            if (x == 0) {
              const uint32_t next = tile + 1;
              if (!(ok = bar_wait(k_full + 8 * (next % ST), (next / ST) & 1))) break;
              tc_fence_after();
            }
            scores(i + 1, x);
          }
        }
      }
    }
    if (!ok) failed = 1;
    tiles_done += n;
    half_done[0] += n;
    if (live_halves == 2) half_done[1] += n;

    // ---- the unit's rows ----
    if (tid < Shape::kSoftmax) {
      const bool mine = n > 0 && half < live_halves;
      if (mine && ok && !warp_wait(pv_done + 8 * half, (half_done[half] - 1) & 1)) failed = 1;
      tc_fence_after();
      const bool whole = c0 == 0 && c1 == w.chunks;
      const float inv = failed ? __int_as_float(0x7fffffff) : (l == 0.f ? 0.f : 1.f / l);
      const float lse = l == 0.f ? -INFINITY : m2 + __log2f(l);
      const int r = r0 + tid;
      const int64_t row = w.first + r / a.group, hq = h * a.group + r % a.group;
      const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * UNIT + tid;
      const uint32_t t_o = tmem + half * 256 + 128 + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
      for (int b = 0; b < D / 32 && half < live_halves; ++b) {
        float v[32];
        if (mine) tmem_load32(t_o + b * 32, v);
        if (tid < nr) {
#pragma unroll
          for (int k = 0; k < 32; k += 8) {
            float f[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) f[x] = mine ? v[k + x] * inv : 0.f;
            if (whole) store8(reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D + b * 32 + k, f);
            else store8(a.part_o + part * D + b * 32 + k, f);
          }
        }
      }
      if (tid < nr) {
        if (!whole) a.part_l[part] = lse;
        else if (a.lse) a.lse[row * a.q_heads + hq] = lse * 0.69314718f;
      }
      tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    if (failed) break;  // the phases are not in step any more
  }
  if (failed && tid == 0) {  // products in flight end before the memory goes back
    for (int i = 0; i < H; ++i) bar_wait(pv_done + 8 * i, 0);
  }
  __syncthreads();
  if (warp == kIssuer) {
    __syncwarp();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape::kColumns));
  }
}

// grid (seqs * kv_heads * tiles, rows / 8): a warp joins the parts of a query row.
template <int D, typename T>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const AttendArgs a, int tiles) {
  constexpr int UNIT = PrefillShape<D>::kUnit;
  extern __shared__ __align__(1024) uint8_t prefill_smem[];
  int64_t* prefix = reinterpret_cast<int64_t*>(prefill_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tile = blockIdx.x % tiles, h = (blockIdx.x / tiles) % a.kv.kv_heads, s = blockIdx.x / tiles / a.kv.kv_heads;
  const SeqWork w = seq_work<UNIT, kTokens>(a, s);
  const bool any = tile < w.tiles && tile * UNIT + (int)blockIdx.y * 8 < w.n * a.group;
  int64_t total = 1, ctas = 1, u0 = 0;
  if (any) {
    plan_prefix<UNIT, kTokens, 256>(a, prefix);
    total = prefix[a.bt.seqs];
    ctas = used_ctas<kPrefillShare>(a, total);
    u0 = prefix[s] + ((int64_t)h * w.tiles + tile) * w.weight;
  }
  grid_wait();
  const int in_tile = blockIdx.y * 8 + warp, r = tile * UNIT + in_tile;
  if (!any || r >= w.n * a.group) return;
  const int first = (int)(((u0 + 1) * ctas - 1) / total), last = (int)(((u0 + w.weight) * ctas - 1) / total);
  if (first == last) return;  // finished by its CTA
  const int n = last - first + 1;
  const int slot0 = (int64_t)first * total / ctas < u0 ? 1 : 0;
  auto part_of = [&](int i) { return ((int64_t)(first + i) * 2 + (i == 0 ? slot0 : 0)) * UNIT + in_tile; };
  float top = -INFINITY;
  for (int i = lane; i < n; i += 32) top = fmaxf(top, a.part_l[part_of(i)]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  if (top == -INFINITY) top = 0.f;
  constexpr int E = D / 32;  // elements of a lane: pairs at 2 lane, 64 apart
  float sum = 0.f, v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float f = ex2(a.part_l[part_of(i)] - top);
    const float2* o = reinterpret_cast<const float2*>(a.part_o + part_of(i) * D) + lane;
    sum += f;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const float2 x = o[e * 16];
      v[e] = fmaf(f, x.x, v[e]);
      v[e + 1] = fmaf(f, x.y, v[e + 1]);
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t row = w.first + r / a.group, hq = h * a.group + r % a.group;
  T* out = reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D + 2 * lane;
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    out[e * 32] = from_f32<T>(v[e] * inv);
    out[e * 32 + 1] = from_f32<T>(v[e + 1] * inv);
  }
  if (a.lse && lane == 0) a.lse[row * a.q_heads + hq] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.69314718f;
}

size_t prefill_workspace(int head_dim) {
  const int rows = head_dim == 256 ? PrefillShape<256>::kUnit : PrefillShape<128>::kUnit;
  return (size_t)sm_count() * 2 * rows * (head_dim + 1) * sizeof(float);
}

template <int D, typename T>
int launch_prefill_kernel(AttendArgs a, int64_t max_context, cudaStream_t stream) {
  constexpr int kMostSmem = 227 * 1024 - 1024;
  static bool allowed[kMaxDevices] = {};  // the kernel's attribute is set once for each device
  const int dev = device_index();
  if (!allowed[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(paged_prefill_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_last_cuda_error(e);
      return TQ_E_CUDA;
    }
    allowed[dev] = true;
  }
  constexpr int UNIT = PrefillShape<D>::kUnit;
  a.ctas = sm_count();
  a.part_l = a.part_o + (size_t)a.ctas * 2 * UNIT * D;
  const int prefix_bytes = (a.bt.seqs + 1) * (int)sizeof(int64_t);
  const int tiles = (int)(((int64_t)a.bt.max_new_tokens * a.group + UNIT - 1) / UNIT);
  const int64_t units = (int64_t)a.bt.seqs * a.kv.kv_heads * tiles;
  if (units > INT32_MAX) return TQ_E_SHAPE;
  const int64_t chunks = max_context < 1 ? 1 : (max_context + kTokens - 1) / kTokens;
  a.whole = chunks <= kPrefillShare;
  const int64_t most = a.whole ? units : units * chunks / kPrefillShare + 1;
  if (most < a.ctas) a.ctas = (int)most;
  const int st = launch_dependent(paged_prefill_kernel<D, T>, dim3(a.ctas), dim3(PrefillShape<D>::kThreads),
                                  PrefillShape<D>::kSmem + prefix_bytes, stream, a);
  if (st != TQ_OK || a.ctas == 1 || a.whole) return st;
  const int64_t rows = (int64_t)a.bt.max_new_tokens * a.group;
  const unsigned y = (unsigned)((rows < UNIT ? rows : UNIT) + 7) / 8;
  return launch_dependent(paged_prefill_join_kernel<D, T>, dim3((unsigned)units, y), dim3(256), prefix_bytes,
                          stream, a, tiles);
}

template <typename T>
int launch_prefill_dim(const AttendArgs& a, int64_t max_context, cudaStream_t stream) {
  if (a.kv.head_dim == 64) return launch_prefill_kernel<64, T>(a, max_context, stream);
  if (a.kv.head_dim == 128) return launch_prefill_kernel<128, T>(a, max_context, stream);
  return launch_prefill_kernel<256, T>(a, max_context, stream);
}

int launch_prefill(const AttendArgs& a, int q_dtype, int64_t max_context, cudaStream_t stream) {
  return q_dtype == TQ_F16 ? launch_prefill_dim<__half>(a, max_context, stream)
                           : launch_prefill_dim<__nv_bfloat16>(a, max_context, stream);
}

}  // namespace tq
