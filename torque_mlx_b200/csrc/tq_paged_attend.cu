// Attention of a few query rows for each kv head over the 8-bit paged cache.
//
// Mathematics.  For a unit (sequence, kv head, tile of query rows) and its
// tokens j: s_j = q . k_j, o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m) with
// scores in base 2.  Codes are whole numbers up to 127, which fp16 holds
// exactly, so both products run on codes: k's page scale multiplies the
// score, and v's enters the exponent of a second weight
// w_j = 2^(s_j + log2(scale_v) - m2), whose reference m2 is kept apart from
// the softmax's own m, so that pages of very different scale neither overflow
// nor vanish, and 2^7 lower, so that small weights keep their bits in fp16.  A bf16 query is multiplied by a power of two for each row that
// takes its largest element to [2^12, 2^13): fp16 then holds it exactly
// (elements under 2^-30 of the largest are off by 2^-38 of it, less than the
// roundings of an fp32 product with it).  Only the weights w are rounded,
// to fp16; scores, m, m2 and all sums stay in fp32.
//
// Bound: a decode step reads each code once.  At 148 SMs and the measured
// copy rate that is about 11 clocks for a token of one head (d = 128, 256
// bytes), while the tensor cores need 1 clock and the conversions about 12
// issue slots of the 44 there are, so bytes bound it once enough of them are
// in flight: every warp keeps its own ring of 16-token chunks filled by
// asynchronous copies.
//
// Split: the chunks of all units form one line that is cut evenly over the
// CTAs, whatever the sequences' lengths (read on the device, so a captured
// step follows them).  A unit that falls within one CTA is finished there; the
// parts of a divided one meet in a second launch.
//
// Measured: 64 sequences of 16K to 32K tokens, 32 heads over 8 of 128: 482 to
// 507 us by the card (6.3 to 6.6 TB/s of codes); one of 131072, 16 heads over 2 of 256: 34 us (4.0 TB/s);
// one of 512, 8 heads of 128: 7.2 us, of which two launches' latency is most.
#include "tq_paged_attend.cuh"

namespace tq {

constexpr int kAttendWarps = 4;
constexpr int kAttendThreads = kAttendWarps * 32;
constexpr int kChunk = 16;    // tokens of a ring stage
constexpr int kMinChunks = 8; // smallest share of a CTA
// What a unit costs besides its chunks (its query rows, the first copies, the
// warps' parts), in chunks of its CTA.  100 sequences of 1 to 1000 tokens and 8
// heads take 80 us with 0, 51 with 4, 39 with 8, 33 with 16; 64 of 16K to 32K
// take 482 to 485 with each of the last three.
constexpr int kLead = 16;
constexpr int kWholeFew = 16, kWholeMany = 32;  // chunks up to which units stay whole

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at));
  return v;
}

template <int D> struct AttendShape {
  static constexpr int kTile = kChunk * D;                 // bytes of a chunk's k (or v) codes
  static constexpr int kStage = 2 * kTile;
  static constexpr int kStages = D == 64 ? 6 : (D == 128 ? 3 : 2);
  static constexpr int kPieces = D / 16;                   // 16-byte pieces of a token
  // Piece p of token t lies at piece p ^ swizzle(t): the eight lanes that the
  // shared memory serves together then meet eight different 16-byte columns,
  // for the k reads (2 tokens x 4 pieces) and the v reads (4 tokens x 2).
  static __device__ __forceinline__ int swizzle(int t) { return D == 64 ? (t >> 1) & 3 : t & 7; }
};

template <int D, int NT, typename T>
__global__ void __launch_bounds__(kAttendThreads, D * NT <= 128 ? 4 : (D * NT == 256 ? 3 : 2))
paged_attend_kernel(const AttendArgs a) {
  using Shape = AttendShape<D>;
  constexpr int ROWS = 8 * NT, STAGES = Shape::kStages, MT = D / 16, KI = D / 64;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float head[kAttendWarps][STAGES][2];          // page scales of a stage's chunk
  __shared__ float stat[kAttendWarps][ROWS][3];            // m, l, m2 of each warp
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + kAttendWarps * STAGES * Shape::kStage);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  const int Hkv = a.kv.kv_heads, P = a.kv.page_size;

  grid_wait();
  plan_prefix<ROWS, kChunk, kLead, kAttendThreads>(a, prefix);
  grid_trigger();
  const int64_t total = prefix[a.bt.seqs];
  const int64_t ctas = used_ctas<kMinChunks>(a, total);
  if ((int64_t)blockIdx.x >= ctas) return;
  int64_t pos = (int64_t)blockIdx.x * total / ctas;
  const int64_t end = ((int64_t)blockIdx.x + 1) * total / ctas;

  uint8_t* ring = smem + warp * STAGES * Shape::kStage;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t head_at = (uint32_t)__cvta_generic_to_shared(&head[warp][0][0]);

  for (int slot = 0; pos < end; slot = 1) {
    const int s = find_seq(prefix, a.bt.seqs, pos);
    const SeqWork w = seq_work<ROWS, kChunk, kLead>(a, s);
    const int64_t rel = pos - prefix[s];
    const int unit = (int)(rel / w.weight);
    int c0, c1;
    pos += chunk_span(a, w, (int)(rel - (int64_t)unit * w.weight), end - pos, c0, c1);
    if (c0 == c1) break;  // the share ends in the unit's lead
    const int h = unit / w.tiles, r0 = (unit - h * w.tiles) * ROWS;
    const int nr = min(ROWS, w.n * a.group - r0);             // rows of this tile
    const int last = w.base + (r0 + nr - 1) / a.group;        // last position that any of them attends
    const int free_to = w.base + r0 / a.group;                // positions up to here need no mask

    // ---- the warp's chunks: c0 + warp, c0 + warp + 4, ... ----
    const int steps = min(c1, last / kChunk + 1) > c0 + warp && last >= 0
                          ? (min(c1, last / kChunk + 1) - c0 - warp + kAttendWarps - 1) / kAttendWarps
                          : 0;
    uint4 raw[NT][KI][2];  // the query rows' elements, on their way while the copies are issued
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = r0 + nt * 8 + g;
      const T* row = reinterpret_cast<const T*>(a.q) + (w.first + r / a.group) * a.q_stride +
                     (int64_t)(h * a.group + r % a.group) * D;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int piece = D == 64 ? c : 8 * (i >> 1) + 2 * c + (i & 1);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          raw[nt][i][e] = make_uint4(0, 0, 0, 0);
          if (nt * 8 + g < nr) raw[nt][i][e] = reinterpret_cast<const uint4*>(row + piece * 16)[e];
        }
      }
    }
    auto chunk_page = [&](int it) {
      const int ch = c0 + warp + it * kAttendWarps;
      return it < steps ? page_id(a.kv, a.bt, s, ch * kChunk / P) : -1;
    };
    int ids = chunk_page(lane), ids_next = chunk_page(32 + lane);
    int issued = 0;
    auto issue = [&](int st) {  // copies of step `issued` into ring stage st
      if (issued < steps) {
        const int id = __shfl_sync(FULL, ids, issued & 31);
        if (id >= 0) {
          const int ch = c0 + warp + issued * kAttendWarps;
          const int64_t block = (int64_t)id * Hkv + h;
          const int64_t at = (block * P + (ch * kChunk) % P) * D;
          const uint8_t* ks = a.kv.k_pages + at + lane * 16;
          const uint8_t* vs = a.kv.v_pages + at + lane * 16;
          const uint32_t dst = ring_at + st * Shape::kStage;
#pragma unroll
          for (int i = 0; i < kChunk * D / 512; ++i) {
            const int piece = lane + 32 * i, t = piece / Shape::kPieces, p = piece % Shape::kPieces;
            const uint32_t off = t * D + ((p ^ Shape::swizzle(t)) << 4);
            cp_async16(dst + off, ks + 512 * i);
            cp_async16(dst + Shape::kTile + off, vs + 512 * i);
          }
          if (lane < 2) cp_async4(head_at + (st * 2 + lane) * 4, (lane ? a.kv.v_scales : a.kv.k_scales) + block);
        } else if (lane == 0) {
          head[warp][st][0] = -1.f;  // no page: the chunk is not attended
        }
        ++issued;
        if ((issued & 31) == 0) {
          ids = ids_next;
          ids_next = chunk_page(issued + 32 + lane);
        }
      }
      cp_commit();
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);

    // ---- query rows: B fragments of k = (piece, word) steps, exact in fp16 ----
    uint32_t qb[NT][KI * 4][2];
    float kf[NT][2];  // score factor of rows 2c, 2c + 1
    int limit[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float x[KI][16];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x[i][e] = to_f32<T>(reinterpret_cast<const T*>(&raw[nt][i][e / 8])[e % 8]);
          if (fabsf(x[i][e]) <= 3.402823466e38f) top = fmaxf(top, fabsf(x[i][e]));
        }
      top = fmaxf(top, __shfl_xor_sync(FULL, top, 1));
      top = fmaxf(top, __shfl_xor_sync(FULL, top, 2));
      int e = 0;  // power of two that takes the largest element to [2^12, 2^13)
      if (!Exact<T>::fp16 && top > 0.f) {
        e = 13 - (ilogbf(top) + 1);
        e = min(120, max(-120, e));
      }
      const float up = __int_as_float((e + 127) << 23), down = __int_as_float((127 - e) << 23);
#pragma unroll
      for (int i = 0; i < KI; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          qb[nt][i * 4 + k][0] = half2_bits(x[i][4 * k] * up, x[i][4 * k + 1] * up);
          qb[nt][i * 4 + k][1] = half2_bits(x[i][4 * k + 2] * up, x[i][4 * k + 3] * up);
        }
      const float f = a.scale2 * down;
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        kf[nt][k] = __shfl_sync(FULL, f, (2 * c + k) * 4);
        limit[nt][k] = w.base + (r0 + nt * 8 + 2 * c + k) / a.group;
      }
    }

    float o[MT][NT][4];
    float m[NT][2], m2[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int k = 0; k < 2; ++k) m[nt][k] = m2[nt][k] = kNoScore, l[nt][k] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[mt][nt][k] = 0.f;
    }

    int st = 0;
    for (int it = 0; it < steps; ++it, st = st + 1 == STAGES ? 0 : st + 1) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      issue(st == 0 ? STAGES - 1 : st - 1);
      const float ks = head[warp][st][0];
      if (ks < 0.f) continue;
      const float lv = __log2f(head[warp][st][1]);
      const int tok = (c0 + warp + it * kAttendWarps) * kChunk;
      const uint32_t kt = ring_at + st * Shape::kStage, vt = kt + Shape::kTile;

      // scores of tokens g, g + 8 with rows 2c, 2c + 1
      constexpr int CHAINS = D == 256 ? 2 : 1;  // sums that run side by side
      float sums[CHAINS][NT][4];
#pragma unroll
      for (int x = 0; x < CHAINS; ++x)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int k = 0; k < 4; ++k) sums[x][nt][k] = 0.f;
#pragma unroll
      for (int i = 0; i < KI; ++i) {
        const int piece = D == 64 ? c : 8 * (i >> 1) + 2 * c + (i & 1);
        const uint4 lo4 = lds128(kt + g * D + ((piece ^ Shape::swizzle(g)) << 4));
        const uint4 hi4 = lds128(kt + (g + 8) * D + ((piece ^ Shape::swizzle(g + 8)) << 4));
        const uint32_t lo[4] = {lo4.x, lo4.y, lo4.z, lo4.w}, hi[4] = {hi4.x, hi4.y, hi4.z, hi4.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a0 = unbias(prmt(lo[k], 0x64646464u, 0x4140)), a2 = unbias(prmt(lo[k], 0x64646464u, 0x4342));
          const uint32_t a1 = unbias(prmt(hi[k], 0x64646464u, 0x4140)), a3 = unbias(prmt(hi[k], 0x64646464u, 0x4342));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) 
            mma16816(sums[i % CHAINS][nt], a0, a1, a2, a3, qb[nt][i * 4 + k][0], qb[nt][i * 4 + k][1]);
        }
      }
      bool grow = false;
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v = (CHAINS == 1 ? sums[0][nt][k] : sums[0][nt][k] + sums[CHAINS - 1][nt][k]) * (ks * kf[nt][k & 1]);
          if (tok + kChunk - 1 > free_to && tok + g + 8 * (k >> 1) > limit[nt][k & 1]) v = -INFINITY;
          sc[nt][k] = v;
          grow |= v > m[nt][k & 1] + kLazy || v + lv > m2[nt][k & 1] + (kLazy + kRoom);
        }
      if (__any_sync(FULL, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float f2[2];
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float top = fmaxf(sc[nt][k], sc[nt][2 + k]);
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, x));
            const float nm = fmaxf(m[nt][k], top), nm2 = fmaxf(m2[nt][k], top + (lv - kRoom));
            l[nt][k] *= ex2(m[nt][k] - nm);
            f2[k] = ex2(m2[nt][k] - nm2);
            m[nt][k] = nm;
            m2[nt][k] = nm2;
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[mt][nt][k] *= f2[k & 1];
        }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          l[nt][k & 1] += ex2(sc[nt][k] - m[nt][k & 1]);
          p[k] = ex2(sc[nt][k] + (lv - m2[nt][k & 1]));
        }
        pb[nt][0] = transpose8x8(half2_bits(p[0], p[1]));
        pb[nt][1] = transpose8x8(half2_bits(p[2], p[3]));
      }
      // o^T += v^T p^T: tokens 2c, 2c + 1, 2c + 8, 2c + 9; a lane's bytes are
      // the rows "g" (even byte) and "g + 8" (odd byte) of its tiles
      constexpr int VW = D == 64 ? 2 : 4;  // words of a lane's read
#pragma unroll
      for (int u = 0; u < (D == 256 ? 2 : 1); ++u) {
        uint32_t v[4][VW];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int t = 2 * c + (k & 1) + 8 * (k >> 1);
          if (D == 64) {
            const uint2 x = lds64(vt + t * D + (((g >> 1) ^ Shape::swizzle(t)) << 4) + (g & 1) * 8);
            v[k][0] = x.x, v[k][1] = x.y;
          } else {
            const uint4 x = lds128(vt + t * D + (((8 * u + g) ^ Shape::swizzle(t)) << 4));
            v[k][0] = x.x, v[k][1] = x.y, v[k][VW - 2] = x.z, v[k][VW - 1] = x.w;
          }
        }
#pragma unroll
        for (int q = 0; q < VW; ++q)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t sel = half ? 0x7632 : 0x5410;
            const uint32_t x = prmt(v[0][q], v[1][q], sel), y = prmt(v[2][q], v[3][q], sel);
            const uint32_t a0 = unbias(prmt(x, 0x64646464u, 0x4240)), a1 = unbias(prmt(x, 0x64646464u, 0x4341));
            const uint32_t a2 = unbias(prmt(y, 0x64646464u, 0x4240)), a3 = unbias(prmt(y, 0x64646464u, 0x4341));
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[(u * VW + q) * 2 + half][nt], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
          }
      }
    }

    // ---- the warps' parts meet in shared memory ----
    cp_wait<0>();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[nt][k] += __shfl_xor_sync(FULL, l[nt][k], x);
        if (g == 0) {
          stat[warp][nt * 8 + 2 * c + k][0] = m[nt][k];
          stat[warp][nt * 8 + 2 * c + k][1] = l[nt][k];
          stat[warp][nt * 8 + 2 * c + k][2] = m2[nt][k];
        }
      }
    __syncthreads();  // every warp is done with its ring
    float* buf = reinterpret_cast<float*>(smem);  // [warps][rows][d]
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int r = nt * 8 + 2 * c + k;
        float top = stat[0][r][0];
#pragma unroll
        for (int i = 1; i < kAttendWarps; ++i) top = fmaxf(top, stat[i][r][0]);
        const float f = ex2(0.5f * (m2[nt][k] - top));  // twice, since the whole factor may be under 2^-126
        float* dst = buf + (warp * ROWS + r) * D;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          // tile mt of a lane: bytes 2mt, 2mt + 1 of its 16 (8 for d = 64) in each 128 (64) of d
          const int dd = D == 64 ? g * 8 + 2 * mt : (mt / 8) * 128 + g * 16 + 2 * (mt % 8);
          *reinterpret_cast<float2*>(dst + dd) = make_float2(o[mt][nt][k] * f * f, o[mt][nt][2 + k] * f * f);
        }
      }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == w.chunks;
    for (int i = tid; i < nr * (D / 8); i += kAttendThreads) {
      const int r = i / (D / 8), d0 = (i - r * (D / 8)) * 8;
      float top = stat[0][r][0], sum = 0.f;
#pragma unroll
      for (int k = 1; k < kAttendWarps; ++k) top = fmaxf(top, stat[k][r][0]);
#pragma unroll
      for (int k = 0; k < kAttendWarps; ++k) sum += stat[k][r][1] * ex2(stat[k][r][0] - top);
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[k] = 0.f;
#pragma unroll
        for (int i2 = 0; i2 < kAttendWarps; ++i2) v[k] += buf[(i2 * ROWS + r) * D + d0 + k];
        v[k] *= inv;
      }
      const float lse = sum == 0.f ? -INFINITY : top + __log2f(sum);
      if (whole) {
        const int64_t row = w.first + (r0 + r) / a.group, hq = h * a.group + (r0 + r) % a.group;
        store8(reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D + d0, v);
        if (a.lse && d0 == 0) a.lse[row * a.q_heads + hq] = lse * 0.69314718f;
      } else {
        const int64_t part = ((int64_t)blockIdx.x * 2 + slot) * ROWS + r;
        store8(a.part_o + part * D + d0, v);
        if (d0 == 0) a.part_l[part] = lse;
      }
    }
    __syncthreads();  // the buffers are free for the next unit
  }
}

// grid (seqs * kv_heads * tiles, rows, d / DIMS): joins the parts of DIMS
// elements of one query row.  Few units have many parts each: 256 threads read
// sixteen of them side by side, 64 elements a CTA (one sequence of 131072: 33.7
// us with the attention, 48.9 with the small CTAs).  More units have a few: a
// CTA of 64 threads for a row (16 sequences of up to 4001: 13.4 us, 15.5 with
// the large ones).
constexpr int kMaxCtas = 148 * 8;

template <int D, int ROWS, int DIMS, int THREADS, typename T>
__global__ void __launch_bounds__(THREADS) paged_join_kernel(const AttendArgs a, int tiles) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float weight[kMaxCtas];
  __shared__ float red[2][THREADS / 32];
  __shared__ float4 acc[THREADS];
  int64_t* prefix = reinterpret_cast<int64_t*>(smem);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int tile = blockIdx.x % tiles, h = (blockIdx.x / tiles) % a.kv.kv_heads, s = blockIdx.x / tiles / a.kv.kv_heads;
  const int r = blockIdx.y;
  // The attention's CTAs start this kernel after their own wait, so what came
  // before them (the lengths among it) is complete; their parts are read after
  // the wait here, which every CTA makes.
  const SeqWork w = seq_work<ROWS, kChunk, kLead>(a, s);
  const bool live = tile < w.tiles && tile * ROWS + r < w.n * a.group;
  int64_t total = 1, ctas = 1, u0 = 0;
  if (live) {
    plan_prefix<ROWS, kChunk, kLead, THREADS>(a, prefix);
    total = prefix[a.bt.seqs];
    ctas = used_ctas<kMinChunks>(a, total);
    u0 = prefix[s] + ((int64_t)h * w.tiles + tile) * w.weight;
  }
  grid_wait();
  if (!live) return;
  const int first = (int)(((u0 + w.lead + 1) * ctas - 1) / total), last = (int)(((u0 + w.weight) * ctas - 1) / total);
  if (first == last) return;  // finished by its CTA
  const int n = last - first + 1;
  const int slot0 = (int64_t)first * total / ctas < u0 ? 1 : 0;
  auto part_of = [&](int i) { return ((int64_t)(first + i) * 2 + (i == 0 ? slot0 : 0)) * ROWS + r; };

  constexpr int Q = DIMS / 4, STEP = THREADS / Q;  // threads of a part; parts side by side
  const int q = tid % Q, d0 = blockIdx.z * DIMS + 4 * q;
  float top = -INFINITY;
  for (int i = tid; i < n; i += THREADS) {
    const float v = a.part_l[part_of(i)];
    weight[i] = v;
    top = fmaxf(top, v);
  }
  // the first parts are on their way while the weights are formed
  constexpr int AHEAD = 8;
  float4 x[AHEAD];
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) {
    const int i = tid / Q + k * STEP;
    if (i < n) x[k] = *reinterpret_cast<const float4*>(a.part_o + part_of(i) * D + d0);
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  if (lane == 0) red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) top = fmaxf(top, red[0][i]);
  if (top == -INFINITY) top = 0.f;
  float sum = 0.f;
  for (int i = tid; i < n; i += THREADS) {
    const float v = ex2(weight[i] - top);
    weight[i] = v;
    sum += v;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(FULL, sum, o);
  if (lane == 0) red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) sum += red[1][i];

  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](int i, const float4& y) {
    const float f = weight[i];
    v.x = fmaf(f, y.x, v.x), v.y = fmaf(f, y.y, v.y), v.z = fmaf(f, y.z, v.z), v.w = fmaf(f, y.w, v.w);
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k)
    if (tid / Q + k * STEP < n) add(tid / Q + k * STEP, x[k]);
#pragma unroll 8
  for (int i = tid / Q + AHEAD * STEP; i < n; i += STEP)
    add(i, *reinterpret_cast<const float4*>(a.part_o + part_of(i) * D + d0));
  acc[tid] = v;
  __syncthreads();
  if (tid < Q) {
#pragma unroll
    for (int i = 1; i < STEP; ++i) {
      const float4 y = acc[tid + i * Q];
      v.x += y.x, v.y += y.y, v.z += y.z, v.w += y.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int rr = tile * ROWS + r;
    const int64_t row = w.first + rr / a.group, hq = h * a.group + rr % a.group;
    T* o = reinterpret_cast<T*>(a.out) + (row * a.q_heads + hq) * D + d0;
    o[0] = from_f32<T>(v.x * inv), o[1] = from_f32<T>(v.y * inv), o[2] = from_f32<T>(v.z * inv), o[3] = from_f32<T>(v.w * inv);
    if (a.lse && tid == 0 && blockIdx.z == 0)
      a.lse[row * a.q_heads + hq] = sum == 0.f ? -INFINITY : (top + __log2f(sum)) * 0.69314718f;
  }
}

// resident CTAs of an SM, as the launch bounds give them
inline int attend_per_sm(int d, int nt) { return d * nt <= 128 ? 4 : (d * nt == 256 ? 3 : 2); }
inline int attend_ctas(int d, int nt) {
  const int n = sm_count() * attend_per_sm(d, nt);
  return n < kMaxCtas ? n : kMaxCtas;
}

template <int D, int NT, typename T>
int launch_attend(AttendArgs a, int64_t max_context, cudaStream_t stream) {
  const int prefix_bytes = (a.bt.seqs + 1) * (int)sizeof(int64_t);
  const int smem = kAttendWarps * AttendShape<D>::kStages * AttendShape<D>::kStage + prefix_bytes;
  constexpr int kMostSmem = 227 * 1024 - 4096;
  static bool allowed[kMaxDevices] = {};  // the kernel's attribute is set once for each device
  const int dev = device_index();
  if (!allowed[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(paged_attend_kernel<D, NT, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_last_cuda_error(e);
      return TQ_E_CUDA;
    }
    allowed[dev] = true;
  }
  const int tiles = (int)(((int64_t)a.bt.max_new_tokens * a.group + 8 * NT - 1) / (8 * NT));
  const int64_t units = (int64_t)a.bt.seqs * a.kv.kv_heads * tiles;
  if (units > INT32_MAX) return TQ_E_SHAPE;
  const int64_t chunks = (max_context + kChunk - 1) / kChunk;
  // Short units are not divided, since the parts' launch would cost more than
  // it saves: 8 heads of 251 tokens take 6.2 us whole and 7.2 divided, of 501
  // 8.6 and 7.2.  Where many units fill the CTAs anyway, longer ones stay whole
  // too: 512 units of 501 tokens take 17.4 us and 23.4.
  a.whole = chunks <= (units * 4 >= a.ctas ? kWholeMany : kWholeFew);
  const int64_t most = a.whole ? units : units * (kLead + chunks) / kMinChunks + 1;
  if (most < a.ctas) a.ctas = (int)most;
  int st = launch_dependent(paged_attend_kernel<D, NT, T>, dim3(a.ctas), dim3(kAttendThreads), smem, stream, a);
  if (st != TQ_OK || a.ctas == 1 || a.whole) return st;
  const int64_t rows = (int64_t)a.bt.max_new_tokens * a.group;
  const unsigned y = (unsigned)(rows < 8 * NT ? rows : 8 * NT);
  if (units * 16 >= a.ctas)
    return launch_dependent(paged_join_kernel<D, 8 * NT, D, 64, T>, dim3((unsigned)units, y), dim3(64), prefix_bytes,
                            stream, a, tiles);
  return launch_dependent(paged_join_kernel<D, 8 * NT, 64, 256, T>, dim3((unsigned)units, y, D / 64), dim3(256),
                          prefix_bytes, stream, a, tiles);
}

template <int D, typename T>
int launch_rows(const AttendArgs& a, int nt, int64_t max_context, cudaStream_t stream) {
  return nt == 1 ? launch_attend<D, 1, T>(a, max_context, stream) : launch_attend<D, 2, T>(a, max_context, stream);
}

template <typename T>
int launch_dim(const AttendArgs& a, int nt, int64_t max_context, cudaStream_t stream) {
  if (a.kv.head_dim == 64) return launch_rows<64, T>(a, nt, max_context, stream);
  if (a.kv.head_dim == 128) return launch_rows<128, T>(a, nt, max_context, stream);
  return launch_rows<256, T>(a, nt, max_context, stream);
}

// Query rows of a kv head from which on the tiles of 128 rows take over.  8
// sequences and 8 heads of 128, in tiles of 16 and of 128:
//   rows    1000 tokens   4000 tokens   32000 tokens
//   32      20.4  26.5    39.3  47.2
//   40      25.7  27.0    53.2  47.2    304  236
//   41      25.9  27.0    53.5  47.6    305  238
//   64      31.3  27.8    68.6  48.4    408  237
// so from 33 rows on long contexts would gain already, and short ones lose.  The
// count is the largest one of the batch: sequences of one token beside a chunk
// go the chunk's way, which costs them (63 over 4000 tokens with a chunk of 512,
// 32 heads over 8: 405 us in one call, 89 and 69 apart).
constexpr int kPrefillFrom = 41;
inline bool many_rows(int64_t max_new, int group) { return max_new * group >= kPrefillFrom; }

// Tiles of 8 query rows, or 16 where a sequence brings more than 8 for a kv
// head.  8 sequences of 32000 tokens and 8 heads of 128 take 173 us with 12 rows
// in tiles of 8 and 111 in tiles of 16, with 20 rows 229 and 209; of 1000 tokens
// 15.0 and 16.8.  4 rows over 16K to 32K tokens take 79 us and 94.
inline int attend_nt(int64_t max_new, int group) { return max_new * group <= 8 ? 1 : 2; }

}  // namespace tq

using namespace tq;

extern "C" {

int tq_paged_attend_workspace_size(const tq_paged_kv* kv, int q_heads, int max_new_tokens, size_t* bytes) {
  const int st = check_paged_kv(kv);
  if (st != TQ_OK) return st;
  if (!bytes) return TQ_E_ARG;
  if (q_heads <= 0 || q_heads % kv->kv_heads || max_new_tokens < 0) return TQ_E_SHAPE;
  if (many_rows(max_new_tokens, q_heads / kv->kv_heads)) {
    *bytes = prefill_workspace(kv->head_dim);
    return TQ_OK;
  }
  const int nt = attend_nt(max_new_tokens, q_heads / kv->kv_heads);
  *bytes = (size_t)attend_ctas(kv->head_dim, nt) * 2 * 8 * nt * (kv->head_dim + 1) * sizeof(float);
  return TQ_OK;
}

int tq_paged_attend(const tq_paged_kv* kv, const tq_paged_batch* batch, const void* q, int q_dtype, int64_t q_stride,
                    int q_heads, int counted, float scale, int64_t max_context, void* out, float* lse,
                    void* workspace, size_t workspace_bytes, tq_stream_t stream) {
  int st = check_paged_kv(kv);
  if (st == TQ_OK) st = check_paged_batch(batch);
  if (st != TQ_OK) return st;
  if (batch->seqs > TQ_PAGED_MAX_SEQS) return TQ_E_SHAPE;
  if (q_dtype != TQ_F16 && q_dtype != TQ_BF16) return TQ_E_ARG;
  if (q_heads <= 0 || q_heads % kv->kv_heads || max_context < 0) return TQ_E_SHAPE;
  if (batch->rows > 1 && (q_stride < (int64_t)q_heads * kv->head_dim || q_stride % 8)) return TQ_E_SHAPE;
  if (batch->seqs == 0 || batch->rows == 0 || batch->max_new_tokens == 0) return TQ_OK;
  if (!q || !out) return TQ_E_ARG;
  if ((uintptr_t)q % 16 || (uintptr_t)out % 32) return TQ_E_SHAPE;
  size_t need = 0;  // for the announced rows: the kernel for many needs the most
  tq_paged_attend_workspace_size(kv, q_heads, batch->max_new_tokens, &need);
  if (!workspace || workspace_bytes < need || (uintptr_t)workspace % 32) return TQ_E_WORKSPACE;
  AttendArgs a = {};
  a.kv = *kv;
  a.bt = bounded(*batch);
  a.q = q;
  a.out = out;
  a.lse = lse;
  a.q_stride = q_stride;
  a.q_heads = q_heads;
  a.group = q_heads / kv->kv_heads;
  a.counted = counted;
  a.scale2 = scale * 1.44269504f;
  a.part_o = (float*)workspace;
  cudaStream_t s = (cudaStream_t)stream;
  if (many_rows(a.bt.max_new_tokens, a.group)) return launch_prefill(a, q_dtype, max_context, s);
  const int nt = attend_nt(a.bt.max_new_tokens, a.group);
  a.ctas = attend_ctas(kv->head_dim, nt);
  a.part_l = a.part_o + (size_t)a.ctas * 2 * 8 * nt * kv->head_dim;
  return q_dtype == TQ_F16 ? launch_dim<__half>(a, nt, max_context, s) : launch_dim<__nv_bfloat16>(a, nt, max_context, s);
}

}  // extern "C"
