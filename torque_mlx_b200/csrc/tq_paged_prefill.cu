// Attention of many query rows for each kv head over the 8-bit paged cache:
// prompts and their chunks.
//
// Mathematics: as in tq_paged_attend.cu, with one exponential for each score.
// For a page of 2^lv scale, w_j = 2^(s_j + lv - m2) weighs v's codes, and the
// softmax's own sum l = sum_j 2^(s_j - m), whose reference m is kept apart as
// there, takes a chunk of one page as (sum_j w_j) 2^-lv 2^(m2 - m).  That holds
// while neither factor leaves fp32's range and no w vanishes before its share of
// l does: up to 2^60 for m2 - m and 2^40 for m2 - m - lv of every page of a step
// (s - m then stays under 55).  Where a row is past that, among pages 2^40 apart
// in scale or beside one whose values have none, the step's scores are summed
// by themselves.
//
// Bound: the two products, 4 d flops for each visible (row, token) pair, on
// the tensor cores, and the exponentials, which take as long at d = 128 (16 a
// clock for each SM).  S = Q K^T and O += P V run on tcgen05.mma with fp16
// operands and fp32 accumulators in tensor memory, 128 rows by 64 tokens a
// step; P goes back to tensor memory over S, which it replaces.  K and V are
// converted from codes to fp16 in shared memory, 128 tokens at a time, once for
// all rows of the CTA.
//
// A CTA takes 256 rows (128 at d = 256, where tensor memory holds no more):
// for each 128 of them four softmax warps (a thread a row, no shuffles), four
// warps that convert the next tiles meanwhile, one that looks up the pages and
// scales of the tiles to come, and one for each half that issues its products.
// Each half has two score buffers, so the next step's scores are ready when a
// softmax ends, whatever the other half does.
//
// Measured: 972 tokens behind 4099, 16 heads over 8 of 128: 72 us, 0.51 PFLOP/s
// (over 8 of 64: 59 us, over 2 of 256: 122 us).  Within a unit a tile of 256
// rows by 128 tokens takes 2.4 us (1.04 PFLOP/s over the card, 2.35 us without a
// reference of l's own); the query rows take 5 us a unit, the output 4, the
// join 8.
#include <atomic>

#include "tq_paged_attend.cuh"

namespace tq {

constexpr int kRows = 128;          // query rows of a product
constexpr int kTokens = 128;        // tokens of a tile
constexpr int kStep = 64;           // tokens of a step
// What a unit costs besides its tiles (its query rows, the output), in tiles.
// 972 tokens alone take 41 us with 0, 39 with 2, 37 with 3, 36 with 5; behind
// 4099 tokens 77, 75, 72, 73; 20 chunks of up to 64 tokens over up to 3000 43,
// 35, 32, 32.
constexpr int kPrefillLead = 3;
constexpr int kPrefillShare = 2;    // smallest share of a CTA, in tiles

// ---- mbarriers, tensor memory and products ----
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
constexpr uint32_t kTries = 20000;  // of 0.1 ms at most, before a wait gives up
std::atomic<uint32_t> wait_tries{kTries};
__device__ uint32_t gave_up_ctas;   // CTAs that left units undone because a wait gave up

// false if the wait gave up
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, uint32_t tries) {
  for (uint32_t it = 0; it < tries; ++it) {
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
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity, uint32_t tries) {
  return __all_sync(FULL, bar_wait(bar, parity, tries));
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// by the one lane that `lead` picks, of a warp that runs this together
__device__ __forceinline__ void tc_commit(uint32_t bar, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred q;\n setp.ne.u32 q, %1, 0;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}\n" ::"r"(bar),
      "r"(lead)
      : "memory");
}
__device__ __forceinline__ uint32_t elect() {
  uint32_t r;
  asm volatile("{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n selp.u32 %0, 1, 0, q;\n}\n" : "=r"(r));
  return r;
}
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// Shared-memory operand of 128-byte rows, 16-byte pieces swizzled by the row's
// low three bits, rows in groups of eight (1024 bytes); lead = bytes between
// blocks of 64 elements where those are the operand's outer dimension.
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t lead) {
  return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(lead >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// the operand `bytes` further on (shared memory ends below the field's range)
__device__ __forceinline__ uint64_t further(uint64_t o, uint32_t bytes) { return o + (bytes >> 4); }
// fp16 operands, fp32 accumulator, M = 128; the second operand's rows are k
// (columns contiguous) where `by_rows`
__host__ __device__ constexpr uint32_t shape(int n, bool by_rows) {
  return 1u << 4 | (by_rows ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kRows >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add, uint32_t lead) {
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %4, 0;\n setp.ne.u32 q, %5, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)add), "r"(lead)
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
// 64 columns of the thread's lane
__device__ __forceinline__ void tmem_load64(uint32_t at, float (&v)[64]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
#pragma unroll
  for (int b = 0; b < 4; ++b)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[16 * b]), "=r"(r[16 * b + 1]), "=r"(r[16 * b + 2]), "=r"(r[16 * b + 3]), "=r"(r[16 * b + 4]),
          "=r"(r[16 * b + 5]), "=r"(r[16 * b + 6]), "=r"(r[16 * b + 7]), "=r"(r[16 * b + 8]), "=r"(r[16 * b + 9]),
          "=r"(r[16 * b + 10]), "=r"(r[16 * b + 11]), "=r"(r[16 * b + 12]), "=r"(r[16 * b + 13]), "=r"(r[16 * b + 14]),
          "=r"(r[16 * b + 15])
        : "r"(at + 16 * b)
        : "memory");
  // the wait names the registers, so that no use of them moves before it
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int k = 0; k < 64; ++k) asm volatile("" : "+r"(r[k]));
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

// 32 elements to consecutive addresses (32-byte boundaries), whole sectors a
// store: a thread writes a row of its own, so narrower stores would send every
// sector twice.
__device__ __forceinline__ void store32(void* p, const uint32_t (&r)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void store_sectors(float* p, const float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 32; k += 8) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = __float_as_uint(v[k + i]);
    store32(p + k, r);
  }
}
template <typename T> __device__ __forceinline__ void store_sectors(T* p, const float (&v)[32]) {
#pragma unroll
  for (int k = 0; k < 32; k += 16) {
    uint32_t r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T lo = from_f32<T>(v[k + 2 * i]), hi = from_f32<T>(v[k + 2 * i + 1]);
      r[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
    }
    store32(p + k, r);
  }
}

template <int D> struct PrefillShape {
  static constexpr int kHalves = D == 256 ? 1 : 2;
  static constexpr int kUnit = kHalves * kRows;            // query rows of a unit
  static constexpr int kStages = D == 256 ? 1 : 2;         // K and V tiles that are held
  static constexpr int kSoftmax = kHalves * 128;           // threads: softmax, then those that convert, then two warps
  static constexpr int kConvert = D == 256 ? 256 : 128;
  static constexpr int kThreads = 512;                     // four warpgroups, not all warps of the last one working
  static constexpr int kWorking = kSoftmax + kConvert + 32 + kHalves * 32;
  static constexpr int kMeeting = kSoftmax + kHalves * 32;    // softmax and products: they meet around a unit
  // Registers of a thread, of 128 at launch: softmax, conversion, the rest.
  static constexpr int kRegsSoftmax = 168, kRegsConvert = 96, kRegsRest = 72;
  static_assert(kHalves * kRegsSoftmax + kConvert / 128 * kRegsConvert + kRegsRest <= 4 * 128, "more than the launch's");
  static constexpr int kOperand = D / 64 * 128 * 128;      // bytes of 128 rows of Q, K or V in fp16
  static constexpr int kSmem = (kHalves + 2 * kStages) * kOperand + 1024;  // from a 1024-byte boundary on
  static constexpr int kColumns = 512;                     // tensor memory of a half: S (P over it), then O
  static constexpr int kRow = D / 16;                      // pieces of 16 codes of a token
  static constexpr int kPieces = 128 * kRow / kConvert;    // a thread's share of a tile
  static constexpr int kTurn = kConvert / kRow;            // tokens from one piece of a thread to its next
  static constexpr int kAges = 4;                          // tiles whose pages and scales are kept
};

// byte offset of elements [8 q, 8 q + 8) of row t within an operand
__device__ __forceinline__ uint32_t place(int t, int q) { return (uint32_t)((q >> 3) * 16384 + t * 128 + (((q & 7) ^ (t & 7)) << 4)); }

// A step's chunks of sixteen tokens as the softmax uses them: products times f
// are the scores, and with the logarithm of v's scale the weights' exponents.
// inv is v's scale inverted.  Without a page f is negative, the logarithm -inf
// and inv 0.
struct StepScales {
  float f[4], lv[4], inv[4];

  __device__ __forceinline__ StepScales(const float* ks, const float* lvs, const float* invs, float kf) {
    const float4 k = *reinterpret_cast<const float4*>(ks), v = *reinterpret_cast<const float4*>(lvs),
                 i = *reinterpret_cast<const float4*>(invs);
    f[0] = k.x, f[1] = k.y, f[2] = k.z, f[3] = k.w;
    lv[0] = v.x, lv[1] = v.y, lv[2] = v.z, lv[3] = v.w;
    inv[0] = i.x, inv[1] = i.y, inv[2] = i.z, inv[3] = i.w;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (f[c] >= 0.f) f[c] *= kf;
  }
};

// The largest exponent of a row's step, or its largest score where SCORE;
// columns past `seen` are hidden where MASKED.
template <bool MASKED, bool SCORE>
__device__ __forceinline__ float highest(const float (&v)[kStep], const StepScales& w, int seen) {
  float x[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int k = 0; k < 16; ++k)
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (!MASKED || c * 16 + k <= seen) x[c] = fmaxf(x[c], v[c * 16 + k]);
  // a NaN (nothing visible, or no page) is passed over
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (SCORE) x[c] = w.f[c] < 0.f ? -INFINITY : x[c] * w.f[c];
    else x[c] = fmaf(x[c], w.f[c], w.lv[c]);
  }
  return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
}

// l and its reference m after a step whose scores are summed by themselves.
template <bool MASKED>
__device__ __forceinline__ void sum_scores(const float (&v)[kStep], const StepScales& w, int seen, float& m, float& l) {
  const float nm = fmaxf(m, highest<MASKED, true>(v, w, seen));
  l *= ex2(m - nm);
  m = nm;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int k = 0; k < 16; ++k)
      if (w.f[c] >= 0.f && (!MASKED || c * 16 + k <= seen)) l += ex2(fmaf(v[c * 16 + k], w.f[c], -m));
}

// The row's weights to tensor memory; returns the sum of 2^(s - m2).
template <bool MASKED>
__device__ __forceinline__ float weigh(uint32_t at, const float (&v)[kStep], const StepScales& w, float m2, int seen) {
  float sums[4];
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    uint64_t s[2][8];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int c = 2 * b + u;
      const float g = w.lv[c] - m2;
      const uint64_t ff = pair(w.f[c], w.f[c]), gg = pair(g, g);
#pragma unroll
      for (int k = 0; k < 8; ++k) s[u][k] = fma2(pair(v[c * 16 + 2 * k], v[c * 16 + 2 * k + 1]), ff, gg);
    }
    uint32_t p[16];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float2 e = halves(s[u][k]);
        float x = ex2(e.x), y = ex2(e.y);
        if (MASKED) {
          const int col = (2 * b + u) * 16 + 2 * k;
          x = col <= seen ? x : 0.f;
          y = col + 1 <= seen ? y : 0.f;
        }
        p[u * 8 + k] = half2_bits(x, y);
        s[u][k] = pair(x, y);
      }
    tmem_store16(at + b * 16, p);
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int o = 4; o; o >>= 1)
#pragma unroll
        for (int k = 0; k < o; ++k) s[u][k] = add2(s[u][k], s[u][k + o]);
      const float2 e = halves(s[u][0]);
      sums[2 * b + u] = e.x + e.y;
    }
  }
  return fmaf(sums[0], w.inv[0], sums[1] * w.inv[1]) + fmaf(sums[2], w.inv[2], sums[3] * w.inv[3]);
}

// A part of a unit that falls to a CTA.
struct Unit {
  int64_t first;       // row of the sequence's first token
  int s, h, base, r0;  // sequence, kv head, position of its first row, first row of the unit
  int nr, last;        // rows; last position that any of them attends
  int c0, n;           // first tile, tiles
  int live_halves, slot;
  bool whole;          // all of the unit's tiles
};

// The CTA's share of the line of tiles, unit by unit.
template <int UNIT> struct UnitLine {
  const AttendArgs& a;
  const int64_t* prefix;
  int64_t pos, end;
  int slot = 0;

  __device__ __forceinline__ UnitLine(const AttendArgs& args, const int64_t* p, int64_t total, int64_t ctas)
      : a(args), prefix(p), pos((int64_t)blockIdx.x * total / ctas), end(((int64_t)blockIdx.x + 1) * total / ctas) {}

  __device__ __forceinline__ bool next(Unit& u) {
    if (pos >= end) return false;
    u.s = find_seq(prefix, a.bt.seqs, pos);
    const SeqWork w = seq_work<UNIT, kTokens, kPrefillLead>(a, u.s);
    const int64_t rel = pos - prefix[u.s];
    const int unit = (int)(rel / w.weight);
    int c1;
    pos += chunk_span(a, w, (int)(rel - (int64_t)unit * w.weight), end - pos, u.c0, c1);
    u.h = unit / w.tiles;
    u.r0 = (unit - u.h * w.tiles) * UNIT;
    u.nr = min(UNIT, w.n * a.group - u.r0);
    u.first = w.first;
    u.base = w.base;
    u.last = w.base + (u.r0 + u.nr - 1) / a.group;
    u.n = u.last < 0 ? 0 : max(0, min(c1, u.last / kTokens + 1) - u.c0);
    u.live_halves = u.nr > kRows ? 2 : 1;
    u.whole = u.c0 == 0 && c1 == w.chunks;
    u.slot = slot;
    slot = 1;
    return c1 > u.c0;  // else the share ends in the unit's lead
  }
};

// a barrier of the working warps, wherever they call it
template <int THREADS> __device__ __forceinline__ void meet() { asm volatile("barrier.sync 1, %0;" ::"n"(THREADS) : "memory"); }
// the same; true for all of them if it is for any
template <int THREADS> __device__ __forceinline__ bool meet_any(bool mine) {
  uint32_t any;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.red.or.pred q, 1, %1, p;\n selp.u32 %0, 1, 0, q;\n}\n"
      : "=r"(any)
      : "n"(THREADS), "r"((uint32_t)mine)
      : "memory");
  return any;
}
template <int THREADS> __device__ __forceinline__ void meet_issuers() { asm volatile("barrier.sync 2, %0;" ::"n"(THREADS) : "memory"); }
template <int REGS, bool MORE> __device__ __forceinline__ void set_registers() {
  if (MORE) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS));
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS));
}

template <int D, typename T>
__global__ void __launch_bounds__(PrefillShape<D>::kThreads, 1) paged_prefill_kernel(const AttendArgs a) {
  using Shape = PrefillShape<D>;
  constexpr int H = Shape::kHalves, ST = Shape::kStages, UNIT = Shape::kUnit;
  extern __shared__ __align__(1024) uint8_t prefill_smem[];
  __shared__ uint64_t bars[4 * ST + 7 * H + 2 * Shape::kAges];
  __shared__ uint32_t tmem_at;
  __shared__ volatile int failed;
  // of a tile's chunks of sixteen tokens: page and head (page 0 and a k scale of
  // -1 where there is none), k's scale, the logarithm and the inverse of v's, and
  // of a step's chunks the smallest logarithm
  __shared__ uint32_t page_at[Shape::kAges][8];
  __shared__ __align__(16) float page_k[Shape::kAges][8], page_lv[Shape::kAges][8], page_inv[Shape::kAges][8];
  __shared__ float page_low[Shape::kAges][2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t raw = (uint32_t)__cvta_generic_to_shared(prefill_smem), base = (raw + 1023u) & ~1023u;
  uint8_t* const smem = prefill_smem + (base - raw);
  uint8_t *const sk = smem + H * Shape::kOperand, *const sv = sk + ST * Shape::kOperand;
  const uint32_t k_at = base + H * Shape::kOperand, v_at = k_at + ST * Shape::kOperand;
  int64_t* prefix = reinterpret_cast<int64_t*>(sv + ST * Shape::kOperand);
  const uint32_t bar0 = (uint32_t)__cvta_generic_to_shared(bars);
  const uint32_t k_full = bar0, k_empty = k_full + 8 * ST, v_full = k_empty + 8 * ST, v_empty = v_full + 8 * ST;  // [stage]
  const uint32_t s_done = v_empty + 8 * ST, p_full = s_done + 16 * H, pv_done = p_full + 16 * H;  // [half][buffer]
  const uint32_t page_full = pv_done + 16 * H, page_empty = page_full + 8 * Shape::kAges;  // [age]
  const uint32_t drained = page_empty + 8 * Shape::kAges;                                   // [half]
  auto warp_wait = [&](uint32_t bar, uint32_t parity) { return all_wait(bar, parity, a.tries); };

  grid_wait();
  plan_prefix<UNIT, kTokens, kPrefillLead, Shape::kThreads>(a, prefix);
  grid_trigger();
  const int64_t total = prefix[a.bt.seqs];
  const int64_t ctas = used_ctas<kPrefillShare>(a, total);
  if ((int64_t)blockIdx.x >= ctas) return;
  if (tid == 0) {
    for (int i = 0; i < ST; ++i) {
      bar_init(k_full + 8 * i, Shape::kConvert);
      bar_init(v_full + 8 * i, Shape::kConvert);
      bar_init(k_empty + 8 * i, H);
      bar_init(v_empty + 8 * i, H);
    }
    for (int i = 0; i < 2 * H; ++i) {
      bar_init(s_done + 8 * i, 1);
      bar_init(p_full + 8 * i, 128);
      bar_init(pv_done + 8 * i, 1);
    }
    for (int i = 0; i < Shape::kAges; ++i) {
      bar_init(page_full + 8 * i, 32);
      bar_init(page_empty + 8 * i, H);
    }
    for (int i = 0; i < H; ++i) bar_init(drained + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    failed = 0;
  }
  constexpr int kIssuer = Shape::kWorking / 32 - H;  // the warps of the products: one for each half
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
  const uint32_t tmem = tmem_at;  // half i: S buffers at 256 i and 256 i + 64, O at 256 i + 128

  const int Hkv = a.kv.kv_heads, P = a.kv.page_size;
  // Each role walks the CTA's units by itself.  Softmax and products meet at the
  // start and at the end of a unit (Q and the accumulators change hands); the
  // others run ahead into the next one as far as the tiles' buffers allow.
  //
  // Every wait has a limit.  A role whose wait gives up sets `failed`; softmax
  // and products decide together, at the end of a unit, whether any of them saw
  // that.  If so the rows not reached become NaN (their parts' sums, where the
  // unit is divided), the products in flight are waited for and the CTA counts
  // itself; the other roles end at their own waits' limit.
  uint32_t tiles_done = 0;  // of the units before: the barriers' phases
  if (tid < Shape::kSoftmax) {
    set_registers<Shape::kRegsSoftmax, true>();
    // ---- softmax: a row a thread ----
    const int half = H == 2 ? tid >> 7 : 0;
    uint32_t pairs_done = 0;  // of this half's steps
    bool gave_up = false;
    UnitLine<UNIT> line(a, prefix, total, ctas);
    for (Unit u; !gave_up && line.next(u);) {
      const int n = u.n, steps = 2 * n, live_halves = u.live_halves;  // even: each buffer's phases stay in step
      float kf = 0.f;  // the row's score factor
      int limit = -1, free_to = 0;
      {
        // ---- the row's query, times a power of two that makes fp16 hold it, to shared memory ----
        const int r = u.r0 + tid;
        const bool live = tid < u.nr;
        const T* row = reinterpret_cast<const T*>(a.q) + (u.first + r / a.group) * a.q_stride +
                       (int64_t)(u.h * a.group + r % a.group) * D;
        uint8_t* sq = smem + half * Shape::kOperand;
        // 64 elements' loads at once, so that their latency is paid once for them
        constexpr int PARTS = D / 64, VECS = 8;
        float up = a.scale2 < 0.f ? -1.f : 1.f, down = 1.f, top = 0.f;
        uint4 x[VECS];
        auto load_part = [&](int part) {
#pragma unroll
          for (int q = 0; q < VECS; ++q) {
            x[q] = make_uint4(0, 0, 0, 0);
            if (live) x[q] = reinterpret_cast<const uint4*>(row)[part * VECS + q];
          }
        };
        if (!Exact<T>::fp16) {
#pragma unroll
          for (int part = PARTS - 1; part >= 0; --part) {
            load_part(part);
#pragma unroll
            for (int q = 0; q < VECS; ++q)
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float f = fabsf(to_f32<T>(reinterpret_cast<const T*>(&x[q])[k]));
                if (f <= 3.402823466e38f) top = fmaxf(top, f);
              }
          }
          int e = top > 0.f ? 13 - (ilogbf(top) + 1) : 0;
          e = min(120, max(-120, e));
          up *= __int_as_float((e + 127) << 23);
          down = __int_as_float((127 - e) << 23);
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          if (Exact<T>::fp16 || part > 0) load_part(part);
#pragma unroll
          for (int q = 0; q < VECS; ++q) {
            float f[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) f[k] = to_f32<T>(reinterpret_cast<const T*>(&x[q])[k]) * up;
            uint4 v;
            v.x = half2_bits(f[0], f[1]);
            v.y = half2_bits(f[2], f[3]);
            v.z = half2_bits(f[4], f[5]);
            v.w = half2_bits(f[6], f[7]);
            *reinterpret_cast<uint4*>(sq + place(tid & 127, part * VECS + q)) = v;
          }
        }
        kf = fabsf(a.scale2) * down;
        limit = u.base + r / a.group;
        free_to = u.base + (u.r0 + half * kRows) / a.group;  // positions up to here need no mask
        proxy_fence();
      }
      meet<Shape::kMeeting>();  // Q is complete
      bool ok = true;
      float m = kNoScore, m2 = kNoScore, l = 0.f;
      {
        const uint32_t t_half = tmem + half * 256 + ((uint32_t)((warp & 3) * 32) << 16), t_o = t_half + 128;
        for (int j = 0; j < steps && half < live_halves; ++j) {
          const uint32_t buf = j & 1, ph = (pairs_done + (j >> 1)) & 1, age = (tiles_done + (j >> 1)) % Shape::kAges;
          if (!(ok = warp_wait(s_done + 8 * (2 * half + buf), ph))) break;
          tc_fence_after();
          const StepScales scales(page_k[age] + 4 * buf, page_lv[age] + 4 * buf, page_inv[age] + 4 * buf, kf);
          const float low = page_low[age][buf];
          float v[kStep];
          tmem_load64(t_half + buf * kStep, v);
          const int tok = u.c0 * kTokens + j * kStep;
          const bool masked = tok + kStep - 1 > free_to;
          const int seen = limit - tok;  // columns 0..seen are visible
          const float top = masked ? highest<true, false>(v, scales, seen) : highest<false, false>(v, scales, seen);
          bool apart = false;
          // one vote while the references hold and l can be taken from the weights
          if (__any_sync(FULL, top > m2 + (kLazy + kRoom) || fabsf(m2 - m) > 60.f || m2 - m - low > 40.f)) {
            if (__any_sync(FULL, top > m2 + (kLazy + kRoom))) {
              const float score = masked ? highest<true, true>(v, scales, seen) : highest<false, true>(v, scales, seen);
              const float nm = fmaxf(m, score), nm2 = fmaxf(m2, top - kRoom), f = ex2(m2 - nm2);
              l *= ex2(m - nm);
              m = nm;
              m2 = nm2;
              if (j > 0) {  // the sums of the steps before, once their products are complete
                if (!(ok = warp_wait(pv_done + 8 * (2 * half + 1 - buf), (pairs_done + ((j - 1) >> 1)) & 1))) break;
                tc_fence_after();
#pragma unroll 1
                for (int b = 0; b < D / 16; ++b) {
                  uint32_t x[16];
                  asm volatile(
                      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                      "\n\ttcgen05.wait::ld.sync.aligned;"
                      : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]),
                        "=r"(x[8]), "=r"(x[9]), "=r"(x[10]), "=r"(x[11]), "=r"(x[12]), "=r"(x[13]), "=r"(x[14]), "=r"(x[15])
                      : "r"(t_o + b * 16)
                      : "memory");
#pragma unroll
                  for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(__uint_as_float(x[k]) * f);
                  tmem_store16(t_o + b * 16, x);
                }
              }
            }
            apart = __any_sync(FULL, fabsf(m2 - m) > 60.f || m2 - m - low > 40.f);
            if (apart) {
              if (masked) sum_scores<true>(v, scales, seen, m, l);
              else sum_scores<false>(v, scales, seen, m, l);
            }
          }
          const float sum = masked ? weigh<true>(t_half + buf * kStep, v, scales, m2, seen)
                                   : weigh<false>(t_half + buf * kStep, v, scales, m2, seen);
          if (!apart) l = fmaf(sum, ex2(m2 - m), l);
          tmem_store_wait();
          tc_fence_before();
          bar_arrive(p_full + 8 * (2 * half + buf));
        }
      }
      tiles_done += n;
      if (half < live_halves) pairs_done += n;
      {
        const bool mine = n > 0 && half < live_halves;
        if (mine && ok) ok = warp_wait(pv_done + 8 * (2 * half + 1), (pairs_done - 1) & 1);
        if (!ok) failed = 1;
        tc_fence_after();
        const bool whole = u.whole;
        // 2^(m2 - m) / l; its power in two halves, since the whole may be under 2^-126
        const float up = ex2(0.5f * (m2 - m)), inv = !ok ? __int_as_float(0x7fffffff) : (l == 0.f ? 0.f : up / l);
        const float lse = !ok ? __int_as_float(0x7fffffff) : (l == 0.f ? -INFINITY : m + __log2f(l));
        const int r = u.r0 + tid;
        const int64_t row = u.first + r / a.group, hq = u.h * a.group + r % a.group;
        const int64_t part = ((int64_t)blockIdx.x * 2 + u.slot) * UNIT + tid;
        const uint32_t t_o = tmem + half * 256 + 128 + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
        for (int b = 0; b < D / 32 && half < live_halves; ++b) {
          float v[32];
          if (mine) tmem_load32(t_o + b * 32, v);
          if (tid < u.nr) {
#pragma unroll
            for (int k = 0; k < 32; ++k) v[k] = mine ? v[k] * inv * up : 0.f;
            if (whole) store_sectors(reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D + b * 32, v);
            else store_sectors(a.part_o + part * D + b * 32, v);
          }
        }
        if (tid < u.nr) {
          if (!whole) a.part_l[part] = lse;
          else if (a.lse) a.lse[row * a.q_heads + hq] = lse * 0.69314718f;
        }
      }
      tc_fence_before();
      gave_up = meet_any<Shape::kMeeting>(!ok || failed);  // the accumulators have been read
      tc_fence_after();
    }
    if (gave_up) {  // the phases are not in step any more: what is left of the share is not computed
      if (tid == 0) atomicAdd(&gave_up_ctas, 1u);
      const float nan = __int_as_float(0x7fffffff);
      for (Unit u; line.next(u);) {
        if (tid >= u.nr) continue;
        if (!u.whole) {
          a.part_l[((int64_t)blockIdx.x * 2 + u.slot) * UNIT + tid] = nan;
          continue;
        }
        const int r = u.r0 + tid;
        const int64_t at = (u.first + r / a.group) * a.q_heads + u.h * a.group + r % a.group;
        for (int k = 0; k < D; ++k) reinterpret_cast<T*>(a.out)[at * D + k] = from_f32<T>(nan);
        if (a.lse) a.lse[at] = nan;
      }
    }
  } else if (tid < Shape::kSoftmax + Shape::kConvert) {
    set_registers<Shape::kRegsConvert, false>();
    // ---- conversion of the tiles' codes ----
    UnitLine<UNIT> line(a, prefix, total, ctas);
    for (Unit u; line.next(u);) {
      const int n = u.n;
      bool ok = true;
      constexpr int PIECES = Shape::kPieces, TURN = Shape::kTurn;
      const int pt = tid - Shape::kSoftmax, t0 = pt / Shape::kRow, q = pt % Shape::kRow;
      // Lanes of the odd blocks of 64 elements start with the second half of
      // their sixteen, so that eight lanes fill eight columns.
      const int turn = (q >> 2) & 1;
      const uint32_t to_a = place(t0, 2 * q + turn), to_b = place(t0, 2 * q + 1 - turn);
      const uint32_t page_bytes = (uint32_t)P * D;  // of a head
      uint4 reg[PIECES];                            // k's codes of a tile, then v's
      // A tile starts at a page boundary, so a piece's place in its page is the
      // same in every tile.
      auto load = [&](const uint8_t* pages, uint32_t age) {
#pragma unroll
        for (int j = 0; j < PIECES; ++j) {
          const int tok = t0 + TURN * j;
          const uint8_t* block = pages + (uint64_t)page_at[age][tok >> 4] * page_bytes;
          reg[j] = *reinterpret_cast<const uint4*>(block + ((tok & (P - 1)) * D + q * 16));
        }
      };
      auto store = [&](uint8_t* to) {
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
      auto pages_of = [&](uint32_t tile) { return warp_wait(page_full + 8 * (tile % Shape::kAges), (tile / Shape::kAges) & 1); };
      if (n > 0 && (ok = pages_of(tiles_done))) load(a.kv.k_pages, tiles_done % Shape::kAges);
      for (int i = 0; i < n && ok; ++i) {
        const uint32_t tile = tiles_done + i, st = tile % ST, use = tile / ST, age = tile % Shape::kAges;
        if (use > 0 && !(ok = warp_wait(k_empty + 8 * st, (use - 1) & 1))) break;
        store(sk + st * Shape::kOperand);
        proxy_fence();
        bar_arrive(k_full + 8 * st);
        load(a.kv.v_pages, age);
        if (i + 1 < n && !(ok = pages_of(tile + 1))) break;
        if (use > 0 && !(ok = warp_wait(v_empty + 8 * st, (use - 1) & 1))) break;
        store(sv + st * Shape::kOperand);
        proxy_fence();
        bar_arrive(v_full + 8 * st);
        if (i + 1 < n) load(a.kv.k_pages, (tile + 1) % Shape::kAges);
      }
      if (!ok) failed = 1;
      tiles_done += n;
      if (!ok) break;
    }
  } else {
    set_registers<Shape::kRegsRest, false>();
    if (warp == kIssuer - 1) {
      // ---- pages and scales of the tiles, ahead of the conversion ----
      UnitLine<UNIT> line(a, prefix, total, ctas);
      for (Unit u; line.next(u);) {
        const int n = u.n;
        bool ok = true;
        auto find = [&](int i) {
          const int tok = (u.c0 + i) * kTokens + lane * 16;
          return lane < 8 && i < n && tok <= u.last ? page_id(a.kv, a.bt, u.s, tok / P) : -1;
        };
        int next = find(0);
        for (int i = 0; i < n; ++i) {
          const uint32_t tile = tiles_done + i, age = tile % Shape::kAges, use = tile / Shape::kAges;
          const int id = next;
          next = find(i + 1);
          const int64_t block = (int64_t)max(id, 0) * Hkv + u.h;
          float ks = -1.f, lv = -INFINITY;
          if (id >= 0) {
            ks = a.kv.k_scales[block];
            lv = log2f(a.kv.v_scales[block]);
            if (ks < 0.f) lv = -INFINITY;  // a negative one stands for no page
          }
          float low = ks < 0.f ? INFINITY : lv;
          low = fminf(low, __shfl_xor_sync(FULL, low, 1));
          low = fminf(low, __shfl_xor_sync(FULL, low, 2));
          if (use > 0 && !(ok = warp_wait(page_empty + 8 * age, (use - 1) & 1))) break;
          if (lane < 8) {
            page_at[age][lane] = (uint32_t)block;
            page_k[age][lane] = ks;
            page_lv[age][lane] = lv;
            page_inv[age][lane] = ks < 0.f ? 0.f : ex2(-lv);
            if ((lane & 3) == 0) page_low[age][lane >> 2] = low;
          }
          __syncwarp();
          bar_arrive(page_full + 8 * age);
        }

        if (!ok) failed = 1;
        tiles_done += n;
        if (!ok) break;
      }
    } else if (warp >= kIssuer && warp < kIssuer + H) {
      // ---- products of a half: S of two steps, then P V of each step and the S after the next ----
      const int x = warp - kIssuer;
      const uint32_t lead = elect(), t_s = tmem + x * 256, t_o = t_s + 128;
      const uint64_t q_op = operand(base + x * Shape::kOperand, 16), k_op = operand(k_at, 16), v_op = operand(v_at, 16384);
      const uint32_t s_bar = s_done + 16 * x, p_bar = p_full + 16 * x, pv_bar = pv_done + 16 * x;
      uint32_t pairs_done = 0;  // of this half's steps
      bool gave_up = false;
      UnitLine<UNIT> line(a, prefix, total, ctas);
      for (Unit u; !gave_up && line.next(u);) {
        const int n = u.n;
        const bool mine = x < u.live_halves, alone = H == 2 && u.live_halves == 1;
        meet<Shape::kMeeting>();
        tc_fence_after();
        bool ok = true;
        // a tile is given back by both halves; the only one at work arrives for both
        auto give_back = [&](uint32_t bar) {
          tc_commit(bar, lead);
          if (alone) tc_commit(bar, lead);
        };
        auto scores = [&](uint32_t st, uint32_t buf) {
          const uint64_t k = further(k_op, st * Shape::kOperand + buf * (kStep * 128));
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {
            const uint32_t off = (i >> 2) * 16384 + (i & 3) * 32;
            mma_ss(t_s + buf * kStep, further(q_op, off), further(k, off), shape(kStep, false), i > 0, lead);
          }
          tc_commit(s_bar + 8 * buf, lead);
          if (buf == 1) give_back(k_empty + 8 * st);
        };
        auto values = [&](uint32_t st, uint32_t buf, bool add) {
          const uint64_t v = further(v_op, st * Shape::kOperand + buf * (kStep * 128));
#pragma unroll
          for (int k = 0; k < kStep / 16; ++k)
            mma_ts(t_o, t_s + buf * kStep + k * 8, further(v, k * 2048), shape(D, true), add || k > 0, lead);
          tc_commit(pv_bar + 8 * buf, lead);
        };
        if (mine && n > 0) {
          uint32_t st = tiles_done % ST;
          ok = warp_wait(k_full + 8 * st, (tiles_done / ST) & 1);
          if (ok) {
            tc_fence_after();
            scores(st, 0);
            scores(st, 1);
          }
          for (int i = 0; i < n && ok; ++i) {
            const uint32_t tile = tiles_done + i, next = tile + 1, ph = (pairs_done + i) & 1;
            st = tile % ST;
            if (!(ok = warp_wait(v_full + 8 * st, (tile / ST) & 1))) break;
            if (!(ok = warp_wait(p_bar, ph))) break;
            tc_fence_after();
            values(st, 0, i > 0);
            if (i + 1 < n) {
              if (!(ok = warp_wait(k_full + 8 * (next % ST), (next / ST) & 1))) break;
              tc_fence_after();
              scores(next % ST, 0);
            }
            if (!(ok = warp_wait(p_bar + 8, ph))) break;
            tc_fence_after();
            values(st, 1, true);
            give_back(v_empty + 8 * st);
            give_back(page_empty + 8 * (tile % Shape::kAges));
            if (i + 1 < n) scores(next % ST, 1);
          }
        }
        if (!ok) failed = 1;
        tiles_done += n;
        if (mine) pairs_done += n;
        gave_up = meet_any<Shape::kMeeting>(!ok || failed);
        tc_fence_after();
      }
      if (gave_up) {  // products in flight end before the memory goes back
        tc_commit(drained + 8 * x, lead);
        all_wait(drained + 8 * x, 0, kTries);
      }
      meet_issuers<32 * H>();
      if (x == 0) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Shape::kColumns));
      }
    }
  }
}

// grid (seqs * kv_heads * tiles, rows / 32): a warp joins the parts of four
// query rows, whose loads run side by side.
constexpr int kJoinRows = 4;

template <int D, typename T>
__global__ void __launch_bounds__(256) paged_prefill_join_kernel(const AttendArgs a, int tiles) {
  constexpr int UNIT = PrefillShape<D>::kUnit, R = kJoinRows;
  extern __shared__ __align__(1024) uint8_t prefill_smem[];
  int64_t* prefix = reinterpret_cast<int64_t*>(prefill_smem);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int tile = blockIdx.x % tiles, h = (blockIdx.x / tiles) % a.kv.kv_heads, s = blockIdx.x / tiles / a.kv.kv_heads;
  const SeqWork w = seq_work<UNIT, kTokens, kPrefillLead>(a, s);
  const int rows = w.n * a.group - tile * UNIT;  // of this unit, at most UNIT of them
  const bool any = tile < w.tiles && (int)blockIdx.y * 8 * R < rows;
  int64_t total = 1, ctas = 1, u0 = 0;
  if (any) {
    plan_prefix<UNIT, kTokens, kPrefillLead, 256>(a, prefix);
    total = prefix[a.bt.seqs];
    ctas = used_ctas<kPrefillShare>(a, total);
    u0 = prefix[s] + ((int64_t)h * w.tiles + tile) * w.weight;
  }
  grid_wait();
  const int r0 = (blockIdx.y * 8 + warp) * R;  // first row, in the unit
  if (!any || r0 >= rows) return;
  const int first = (int)(((u0 + w.lead + 1) * ctas - 1) / total), last = (int)(((u0 + w.weight) * ctas - 1) / total);
  if (first == last) return;  // finished by its CTA
  const int n = last - first + 1, live = min(R, rows - r0);
  const int slot0 = (int64_t)first * total / ctas < u0 ? 1 : 0;
  auto part_of = [&](int i, int k) {  // a row past the last one reads that one again
    return ((int64_t)(first + i) * 2 + (i == 0 ? slot0 : 0)) * UNIT + r0 + min(k, live - 1);
  };
  constexpr int E = D / 32;  // elements of a lane: pairs at 2 lane, 64 apart
  float top[R], sum[R], v[R][E];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    top[k] = -INFINITY, sum[k] = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) v[k][e] = 0.f;
  }
  for (int i0 = 0; i0 < n; i0 += 32) {  // a lane holds a part's sum of each row; the rows' elements do not wait for it
    float f[R];
#pragma unroll
    for (int k = 0; k < R; ++k) f[k] = i0 + lane < n ? a.part_l[part_of(i0 + lane, k)] : -INFINITY;
#pragma unroll
    for (int k = 0; k < R; ++k) {
      float high = f[k];
#pragma unroll
      for (int o = 16; o; o >>= 1) high = fmaxf(high, __shfl_xor_sync(FULL, high, o));
      high = fmaxf(high, top[k]);
      const float ref = high == -INFINITY ? 0.f : high;  // nothing yet: the next parts may lie far below 0
      const float old = ex2(top[k] - ref);
      f[k] = ex2(f[k] - ref);
      top[k] = high;
      sum[k] *= old;
#pragma unroll
      for (int e = 0; e < E; ++e) v[k][e] *= old;
    }
#pragma unroll 2
    for (int i = i0; i < min(n, i0 + 32); ++i) {
#pragma unroll
      for (int k = 0; k < R; ++k) {
        const float2* o = reinterpret_cast<const float2*>(a.part_o + part_of(i, k) * D) + lane;
        const float fi = __shfl_sync(FULL, f[k], i - i0);
        sum[k] += fi;
#pragma unroll
        for (int e = 0; e < E; e += 2) {
          const float2 x = o[e * 16];
          v[k][e] = fmaf(fi, x.x, v[k][e]);
          v[k][e + 1] = fmaf(fi, x.y, v[k][e + 1]);
        }
      }
    }
  }
#pragma unroll
  for (int k = 0; k < R; ++k) {
    if (k >= live) break;
    const int r = tile * UNIT + r0 + k;
    const float inv = sum[k] == 0.f ? 0.f : 1.f / sum[k];
    const int64_t row = w.first + r / a.group, hq = h * a.group + r % a.group;
    uint32_t* out = reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D) + lane;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const T lo = from_f32<T>(v[k][e] * inv), hi = from_f32<T>(v[k][e + 1] * inv);
      out[e * 16] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
    }
    if (a.lse && lane == 0)
      a.lse[row * a.q_heads + hq] = sum[k] == 0.f ? -INFINITY : (top[k] + __log2f(sum[k])) * 0.69314718f;
  }
}

size_t prefill_workspace(int head_dim) {
  const int rows = head_dim == 256 ? PrefillShape<256>::kUnit : PrefillShape<128>::kUnit;
  return (size_t)sm_count() * 2 * rows * (head_dim + 1) * sizeof(float);
}

template <int D, typename T>
int launch_prefill_kernel(AttendArgs a, int64_t max_context, cudaStream_t stream) {
  constexpr int kMostSmem = 227 * 1024 - 2048;  // the static arrays take the rest
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
  a.tries = wait_tries.load(std::memory_order_relaxed);
  a.part_l = a.part_o + (size_t)a.ctas * 2 * UNIT * D;
  const int prefix_bytes = (a.bt.seqs + 1) * (int)sizeof(int64_t);
  const int tiles = (int)(((int64_t)a.bt.max_new_tokens * a.group + UNIT - 1) / UNIT);
  const int64_t units = (int64_t)a.bt.seqs * a.kv.kv_heads * tiles;
  if (units > INT32_MAX) return TQ_E_SHAPE;
  const int64_t chunks = max_context < 1 ? 1 : (max_context + kTokens - 1) / kTokens;
  a.whole = chunks <= kPrefillShare;
  const int64_t most = a.whole ? units : units * (kPrefillLead + chunks) / kPrefillShare + 1;
  if (most < a.ctas) a.ctas = (int)most;
  const int st = launch_dependent(paged_prefill_kernel<D, T>, dim3(a.ctas), dim3(PrefillShape<D>::kThreads),
                                  PrefillShape<D>::kSmem + prefix_bytes, stream, a);
  if (st != TQ_OK || a.ctas == 1 || a.whole) return st;
  const int64_t rows = (int64_t)a.bt.max_new_tokens * a.group;
  const unsigned y = (unsigned)((rows < UNIT ? rows : UNIT) + 8 * kJoinRows - 1) / (8 * kJoinRows);
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

using namespace tq;

extern "C" {

int tq_paged_attend_wait_limit(uint32_t tries) {
  wait_tries.store(tries, std::memory_order_relaxed);
  return TQ_OK;
}

int tq_paged_attend_gave_up(uint32_t* ctas, tq_stream_t stream) {
  if (!ctas) return TQ_E_ARG;
  cudaStream_t s = (cudaStream_t)stream;
  cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
  cudaError_t e = cudaStreamIsCapturing(s, &capturing);
  if (e == cudaSuccess && capturing != cudaStreamCaptureStatusNone) return TQ_E_ARG;
  if (e == cudaSuccess) e = cudaMemcpyFromSymbolAsync(ctas, gave_up_ctas, sizeof(*ctas), 0, cudaMemcpyDeviceToHost, s);
  if (e == cudaSuccess) e = cudaStreamSynchronize(s);
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_last_cuda_error(e);
    return TQ_E_CUDA;
  }
  return TQ_OK;
}

}  // extern "C"
