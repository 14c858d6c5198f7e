// Products of a few tokens with a 4-bit weight with group scales.
//
// Mathematics: y[m, i] = sum_g s[i, g] sum_{j in g} (c[i, j] - 8) x[m, j].  A
// code becomes a number of x's type with a logic operation that sets the
// exponent (128 + c in bf16, 1024 + c or 1024 + 16 c in fp16) and one
// arithmetic operation that removes the bias, both exact; the inner sums run
// on mma.sync m16n8k16 with fp32 accumulation, sixteen weight rows by eight
// tokens, and each group's sum is multiplied by its scale in fp32.  x is used
// as it is, so nothing is rounded before y.
//
// Bound: the weight's bytes for any token count the launch takes (each weight
// is converted once for all of them).  At the copy rate an SM must take 512
// bytes of codes every 22 clocks; the conversion, its mma and the scale cost
// about 65 issue slots of the 88 in that time, so loads must never stall the
// warps: each warp keeps a ring of its next fragments filled by asynchronous
// copies, and the ring is filled before x is staged.
//
// Split: a CTA takes a run of row tiles, and its sixteen warps equal runs of
// that run's fragments, so they need not wait for one another: a tile that
// lies within a warp's run is finished in registers, and the pieces of a tile
// that warps share meet in shared memory once, at the end.
//
// Measured: 4 tokens, 151936 x 2048, groups of 64: 36 us (166 MB, 4.6 TB/s;
// 0.69 instructions a clock and scheduler, the logic pipe 52 % busy); 13 tokens,
// 12288 x 2048, groups of 32: 8.5 us; one token, 4096 x 2048: 3.9 us.
#include "tq_paged.cuh"

namespace tq {

constexpr int kW4Threads = 512;
constexpr int kW4Warps = kW4Threads / 32;
constexpr int kW4MaxTokens = TQ_W4_MAX_TOKENS;
constexpr int kW4Block = 128;  // columns of a fragment block
constexpr int kW4Smem = 227 * 1024 - 4096;  // dynamic; the static arrays take the rest

constexpr int kW4Stages = 5;  // fragments of a warp's ring

enum W4Input { kW4Plain = 0, kW4F32 = 1, kW4Rms = 2, kW4Silu = 3 };

struct W4Args {
  const uint4* codes;     // [tiles][blocks][2][32]: word j of half i = columns 64 i + 16 j of the block
  const uint8_t* scales;  // [tiles][blocks][8][groups of a block][2] bf16: rows g and g + 8
  const void* x;
  const void* norm_w;
  const void* residual;
  void* y;
  float* part;            // [k slabs][tokens][n] fp32 when the columns are split over CTAs
  int64_t n, k, x_stride;
  int64_t y_offset;       // first token's row in y and residual
  int tiles, blocks;      // row tiles, column blocks of the weight
  int slab;               // column blocks of a CTA's slab
  int tokens;
  int mode;
  int group;
  float eps;
};

inline bool valid_group(int g) { return g == 32 || g == 64 || g == 128; }
inline int64_t w4_tiles(int64_t n) { return (n + 15) / 16; }
inline int64_t w4_blocks(int64_t k) { return (k + kW4Block - 1) / kW4Block; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
template <int BYTES> __device__ __forceinline__ void cp_scales(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void w4_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void w4_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// A constant that stays in a register: a logic operation holds one immediate
// at most, and two constants folded into it would make two of it.
__device__ __forceinline__ uint32_t kept(uint32_t c) {
  asm volatile("" : "+r"(c));
  return c;
}
// (a & mask) | set
__device__ __forceinline__ uint32_t pick(uint32_t a, uint32_t mask, uint32_t set) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(a), "r"(mask), "r"(set));
  return r;
}

// eight codes of a word -> A fragment of sixteen rows and columns, code - 8
template <typename T> struct W4Math;
template <> struct W4Math<__half> {
  const uint32_t low = kept(0x000f000fu), high = kept(0x00f000f0u), set = kept(0x64006400u), bias = kept(0x64086408u),
                 sixteenth = kept(0x2c002c00u), shifted = kept(0xd480d480u);
  __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) const {
    const uint32_t v = w >> 8;
    a[0] = sub(pick(w, low, set), bias);                 // 1024 + c - 1032
    a[1] = sub(pick(v, low, set), bias);
    a[2] = fma(pick(w, high, set), sixteenth, shifted);  // (1024 + 16 c) / 16 - 72
    a[3] = fma(pick(v, high, set), sixteenth, shifted);
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint32_t fma(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <> struct W4Math<__nv_bfloat16> {
  const uint32_t low = kept(0x000f000fu), set = kept(0x43004300u), bias = kept(0x43084308u);
  __device__ __forceinline__ void expand(uint32_t w, uint32_t (&a)[4]) const {
    a[0] = sub(pick(w, low, set));  // 128 + c - 136
    a[2] = sub(pick(w >> 4, low, set));
    a[1] = sub(pick(w >> 8, low, set));
    a[3] = sub(pick(w >> 12, low, set));
  }
  __device__ __forceinline__ uint32_t sub(uint32_t a) const {
    uint32_t r;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(bias));
    return r;
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

// Eight elements of x' of token m from column k0 (zeros past the last column).
template <typename T>
__device__ __forceinline__ void w4_input(const W4Args& a, int64_t m, int64_t k0, float inv, bool vec, float (&f)[8]) {
  const int64_t row = m * a.x_stride;
  if (a.mode == kW4F32) {
    const float* x = reinterpret_cast<const float*>(a.x) + row;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = k0 + i < a.k ? to_f32<T>(from_f32<T>(x[k0 + i])) : 0.f;
    return;
  }
  const T* x = reinterpret_cast<const T*>(a.x) + row;
  if (vec && k0 + 8 <= a.k) {
    load8(x + k0, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = k0 + i < a.k ? to_f32<T>(x[k0 + i]) : 0.f;
  }
  if (a.mode == kW4Rms) {
    const T* w = reinterpret_cast<const T*>(a.norm_w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < a.k)
        f[i] = to_f32<T>(from_f32<T>(__fmul_rn(to_f32<T>(from_f32<T>(__fmul_rn(f[i], inv))), to_f32<T>(w[k0 + i]))));
  } else if (a.mode == kW4Silu) {
    const T* u = x + a.k;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k0 + i < a.k) {
        const float act = to_f32<T>(from_f32<T>(f[i] / (1.f + expf(-f[i]))));
        f[i] = to_f32<T>(from_f32<T>(__fmul_rn(act, to_f32<T>(u[k0 + i]))));
      }
  }
}

// NT tiles of eight tokens, SG groups of a block.
template <int NT, int SG, typename T>
__global__ void __launch_bounds__(kW4Threads, 1) w4_kernel(const W4Args a) {
  const W4Math<T> math;
  constexpr int UNIT = 1024 + 32 * SG, STAGES = kW4Stages;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  __shared__ float red[kW4Warps][kW4MaxTokens];
  __shared__ float inv_rms[kW4MaxTokens];
  __shared__ int piece_tile[kW4Warps];  // tile whose middle or end a warp left in its piece, or -1
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, c = lane & 3;
  uint8_t* ring = w4_smem + warp * STAGES * UNIT;
  float4* pieces = reinterpret_cast<float4*>(w4_smem + kW4Warps * STAGES * UNIT);  // [warps][NT][32]
  uint8_t* xs = reinterpret_cast<uint8_t*>(pieces + kW4Warps * NT * 32);           // [block][4][token][4] x 16 bytes
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  const int M = a.tokens;
  const int b_lo = blockIdx.y * a.slab, b_hi = min(a.blocks, b_lo + a.slab), nb = b_hi - b_lo;
  const int t_lo = (int)((int64_t)blockIdx.x * a.tiles / gridDim.x);
  const int t_hi = (int)((int64_t)(blockIdx.x + 1) * a.tiles / gridDim.x);
  const int64_t units = (int64_t)(t_hi - t_lo) * nb;
  const int64_t u_lo = warp * units / kW4Warps;
  const int steps = (int)((warp + 1) * units / kW4Warps - u_lo);
  const int first_tile = t_lo + (int)(u_lo / nb), first_block = (int)(u_lo % nb);  // block within the slab

  grid_wait();
  // ---- the ring's first fragments ----
  int left = steps, in_block = first_block;
  const int64_t first_unit = (int64_t)first_tile * a.blocks + b_lo + first_block;
  const uint8_t* src = reinterpret_cast<const uint8_t*>(a.codes) + first_unit * 1024 + lane * 16;
  const uint8_t* ssrc = a.scales + first_unit * (32 * SG) + g * (4 * SG);
  const int64_t skip = a.blocks - nb;  // blocks of other slabs between two tiles
  auto issue = [&](int st) {
    if (left > 0) {
      const uint32_t dst = ring_at + st * UNIT;
      cp16(dst + lane * 16, src);
      cp16(dst + 512 + lane * 16, src + 512);
      if (c == 0) cp_scales<4 * SG>(dst + 1024 + g * (4 * SG), ssrc);
      --left;
      src += 1024;
      ssrc += 32 * SG;
      if (skip && ++in_block == nb) {
        in_block = 0;
        src += skip * 1024;
        ssrc += skip * (32 * SG);
      }
    }
    w4_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(i);

  // ---- x' of this slab in fragment order ----
  const int64_t k_lo = (int64_t)b_lo * kW4Block, k_hi = (int64_t)b_hi * kW4Block;
  const bool vec = a.mode != kW4F32 && a.x_stride % 8 == 0 && ((uintptr_t)a.x & 15) == 0;
  if (tid < kW4Warps) piece_tile[tid] = -1;
  if (a.mode == kW4Rms) {
    for (int m = 0; m < M; ++m) {
      const T* x = reinterpret_cast<const T*>(a.x) + m * a.x_stride;
      float ss = 0.f;
      for (int64_t k = tid; k < a.k; k += kW4Threads) {
        const float v = to_f32<T>(x[k]);
        ss = fmaf(v, v, ss);
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(FULL, ss, o);
      if (lane == 0) red[warp][m] = ss;
    }
    __syncthreads();
    if (tid < M) {
      float ss = 0.f;
      for (int w = 0; w < kW4Warps; ++w) ss += red[w][tid];
      inv_rms[tid] = rsqrtf(ss / (float)a.k + a.eps);
    }
    __syncthreads();
  }
  const int pieces8 = nb * (kW4Block / 8);  // eight columns each
  auto place = [&](int m, int at) {         // four words, sixteen bytes apart
    const int b = at / 16, j = at % 16 / 2, half = at & 1;
    return xs + ((b * 4 + (j >> 1)) * M + m) * 64 + ((j & 1) * 4 + half * 2) * 2;
  };
  auto put = [&](uint8_t* dst, const uint32_t (&w)[4]) {
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<uint32_t*>(dst + q * 16) = w[q];
  };
  if (a.mode == kW4Plain && vec && a.k % 8 == 0) {  // words as they are, four loads of a thread at a time
    constexpr int U = 4;
    const int total = M * pieces8, columns8 = (int)(a.k / 8) - (int)(k_lo / 8);
    for (int i0 = tid; i0 < total; i0 += U * kW4Threads) {
      uint4 v[U];
      int m[U], at[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int i = i0 + u * kW4Threads;
        m[u] = i / pieces8;
        at[u] = i - m[u] * pieces8;
        v[u] = make_uint4(0, 0, 0, 0);
        if (i < total && at[u] < columns8)
          v[u] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.x) + m[u] * a.x_stride + k_lo + at[u] * 8);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kW4Threads < total) {
          const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
          put(place(m[u], at[u]), w);
        }
    }
  } else {
    for (int i = tid; i < M * pieces8; i += kW4Threads) {
      const int m = i / pieces8, at = i - m * pieces8;
      float f[8];
      w4_input<T>(a, m, k_lo + at * 8, a.mode == kW4Rms ? inv_rms[m] : 0.f, vec, f);
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const T lo = from_f32<T>(f[2 * q]), hi = from_f32<T>(f[2 * q + 1]);
        w[q] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
      }
      put(place(m, at), w);
    }
  }
  __syncthreads();
  grid_trigger();

  // ---- the warp's run ----
  float acc[NT][4];
  auto clear = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nt][i] = 0.f;
  };
  auto output = [&](int tile) {  // rows g, g + 8 of a tile, tokens 2c, 2c + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t row = (int64_t)tile * 16 + g + 8 * (i >> 1);
        const int col = nt * 8 + 2 * c + (i & 1);
        if (row < a.n && col < M) {
          float v = acc[nt][i];
          if (a.part) {
            a.part[((int64_t)blockIdx.y * M + col) * a.n + row] = v;
          } else {
            const int64_t o = (a.y_offset + col) * a.n + row;
            if (a.residual) v += to_f32<T>(reinterpret_cast<const T*>(a.residual)[o]);
            reinterpret_cast<T*>(a.y)[o] = from_f32<T>(v);
          }
        }
      }
  };
  clear();
  int tile = first_tile, b = first_block;
  bool begun = first_block == 0;  // the tile's first block was this warp's
  // a lane past the last token reads that one again: its sums are not used
  const uint4 *x0[NT], *xp[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    x0[nt] = reinterpret_cast<const uint4*>(xs) + min(nt * 8 + g, M - 1) * 4 + c;
    xp[nt] = x0[nt] + (int64_t)first_block * M * 16;
  }
  for (int it = 0; it < steps; it += STAGES) {
#pragma unroll
    for (int st = 0; st < STAGES; ++st) {
      if (it + st >= steps) break;
      w4_wait<STAGES - 2>();
      __syncwarp();
      issue(st == 0 ? STAGES - 1 : st - 1);
      const uint8_t* unit = ring + st * UNIT;
      const uint4 wl = *reinterpret_cast<const uint4*>(unit + lane * 16);
      const uint4 wh = *reinterpret_cast<const uint4*>(unit + 512 + lane * 16);
      const uint32_t w[8] = {wl.x, wl.y, wl.z, wl.w, wh.x, wh.y, wh.z, wh.w};
      uint32_t two[SG];  // scales of rows g and g + 8
#pragma unroll
      for (int s = 0; s < SG; ++s) two[s] = reinterpret_cast<const uint32_t*>(unit + 1024)[g * SG + s];
      float sum[NT][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {  // 32 columns
        uint4 x[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          x[nt] = xp[nt][i * (M * 4)];
        }
        if (i % (4 / SG) == 0) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) sum[nt][k] = 0.f;
        }
        uint32_t f[4];
        math.expand(w[2 * i], f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) math.mma(sum[nt], f, x[nt].x, x[nt].y);
        math.expand(w[2 * i + 1], f);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) math.mma(sum[nt], f, x[nt].z, x[nt].w);
        if ((i + 1) % (4 / SG) == 0) {
          const uint32_t s2 = two[i / (4 / SG)];
          const float s0 = __uint_as_float(s2 << 16), s1 = __uint_as_float(s2 & 0xffff0000u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[nt][k] = fmaf(k < 2 ? s0 : s1, sum[nt][k], acc[nt][k]);
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) xp[nt] += M * 16;
      if (++b == nb) {  // the tile ends here
        if (begun) {
          output(tile);
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            pieces[(warp * NT + nt) * 32 + lane] = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
          if (lane == 0) piece_tile[warp] = tile;
        }
        clear();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) xp[nt] = x0[nt];
        b = 0;
        ++tile;
        begun = true;
      }
    }
  }
  if (b != 0 && !begun) {  // the run lies within one tile
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
      pieces[(warp * NT + nt) * 32 + lane] = make_float4(acc[nt][0], acc[nt][1], acc[nt][2], acc[nt][3]);
    if (lane == 0) piece_tile[warp] = tile;
  }
  w4_wait<0>();
  __syncthreads();
  if (b != 0 && begun && steps > 0) {  // the tile begun here goes on in the next warps' pieces
    for (int w = warp + 1; w < kW4Warps; ++w) {
      if (piece_tile[w] != tile) {
        if (piece_tile[w] >= 0) break;
        continue;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float4 v = pieces[(w * NT + nt) * 32 + lane];
        acc[nt][0] += v.x, acc[nt][1] += v.y, acc[nt][2] += v.z, acc[nt][3] += v.w;
      }
    }
    output(tile);
  }
}

// y of the slabs' partial sums, added in their order
template <typename T>
__global__ void __launch_bounds__(256) w4_join_kernel(const float* __restrict__ part, int slabs, int64_t count,
                                                      int64_t offset, const T* __restrict__ residual, T* __restrict__ y) {
  grid_wait();
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= count) return;
  float v = 0.f;
  for (int s = 0; s < slabs; ++s) v += part[s * count + i];
  if (residual) v += to_f32<T>(residual[offset + i]);
  y[offset + i] = from_f32<T>(v);
}

// ---------------------------------------------------------------------------
// weights
// ---------------------------------------------------------------------------
// column of nibble p (p + 4 is the next column) of lane c's word for step j
__device__ __forceinline__ void w4_place(int p, int g, int c, int& row, int& col) {
  row = g + ((p & 2) ? 8 : 0);
  col = 2 * c + ((p & 1) ? 8 : 0);
}

__global__ void __launch_bounds__(256) w4_layout_kernel(const uint8_t* __restrict__ packed,
                                                        const uint16_t* __restrict__ scales, int64_t n, int64_t k,
                                                        int group, int64_t tiles, int64_t blocks,
                                                        uint32_t* __restrict__ out, uint16_t* __restrict__ sout) {
  grid_wait();
  const int64_t stride = (int64_t)gridDim.x * 256, row_bytes = (k + 1) / 2;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < tiles * blocks * 256; i += stride) {
    const int j = (int)(i & 3) + ((int)(i >> 7) & 1) * 4, lane = (int)(i >> 2) & 31, g = lane >> 2, c = lane & 3;
    const int64_t unit = i >> 8, tile = unit / blocks, b = unit - tile * blocks;
    uint32_t w = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      int r, q;
      w4_place(p, g, c, r, q);
      const int64_t row = tile * 16 + r, col = b * kW4Block + j * 16 + q;  // col is even
      uint32_t lo = 8, hi = 8;                                             // code 8: nothing there
      if (row < n && col < k) {
        const uint32_t byte = packed[row * row_bytes + col / 2];
        lo = byte & 15;
        if (col + 1 < k) hi = byte >> 4;
      }
      w |= lo << (4 * p) | hi << (16 + 4 * p);
    }
    out[i] = w;
  }
  const int sg = kW4Block / group;
  const int64_t groups = (k + group - 1) / group;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < tiles * blocks * 16 * sg; i += stride) {
    const int which = (int)(i & 1);
    const int64_t v = i >> 1;
    const int s = (int)(v % sg), g = (int)(v / sg) & 7;
    const int64_t at = v / sg / 8, tile = at / blocks, b = at - tile * blocks;
    const int64_t row = tile * 16 + g + 8 * which, grp = b * sg + s;
    sout[i] = row < n && grp < groups ? scales[row * groups + grp] : 0;
  }
}

// one warp for each row and group
template <typename T>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const T* __restrict__ w, int64_t n, int64_t k, int group,
                                                          uint8_t* __restrict__ packed, uint16_t* __restrict__ scales) {
  grid_wait();
  const int lane = threadIdx.x & 31;
  const int64_t groups = (k + group - 1) / group, row_bytes = (k + 1) / 2;
  const int64_t at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= n * groups) return;
  const int64_t row = at / groups, grp = at - row * groups, k0 = grp * group;
  float top = 0.f;
  for (int i = lane; i < group; i += 32)
    if (k0 + i < k) top = fmaxf(top, fabsf(to_f32<T>(w[row * k + k0 + i])));
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(FULL, top, o));
  const __nv_bfloat16 sb = __float2bfloat16_rn(fminf(fmaxf(__fdiv_rn(top, 7.f), 7.888609052e-31f), 3.3e38f));
  const float s = __bfloat162float(sb);
  if (lane == 0) scales[at] = *reinterpret_cast<const uint16_t*>(&sb);
  for (int i = lane; i < group / 2; i += 32) {
    uint32_t byte = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t col = k0 + 2 * i + h;
      int q = 8;
      // within [-8, 7] before 8 is added: an infinity converts to the largest integer
      if (col < k) q = min(7, max(-8, __float2int_rn(__fdiv_rn(to_f32<T>(w[row * k + col]), s)))) + 8;
      byte |= (uint32_t)q << (4 * h);
    }
    if (k0 + 2 * i < k) packed[row * row_bytes + (k0 / 2) + i] = (uint8_t)byte;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) w4_dequantize_kernel(const uint32_t* __restrict__ codes,
                                                            const uint16_t* __restrict__ scales, int64_t n, int64_t k,
                                                            int group, int64_t tiles, int64_t blocks,
                                                            T* __restrict__ out) {
  grid_wait();
  const int sg = kW4Block / group;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < tiles * blocks * 256; i += (int64_t)gridDim.x * 256) {
    const int j = (int)(i & 3) + ((int)(i >> 7) & 1) * 4, lane = (int)(i >> 2) & 31, g = lane >> 2, c = lane & 3;
    const int64_t unit = i >> 8, tile = unit / blocks, b = unit - tile * blocks;
    const uint32_t w = codes[i];
    const int s = j * 16 / group;
    const int64_t sb = unit * 8 + g;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      int r, q;
      w4_place(p, g, c, r, q);
      const int64_t row = tile * 16 + r, col = b * kW4Block + j * 16 + q;
      const float sc = __uint_as_float((uint32_t)scales[(sb * sg + s) * 2 + (r >= 8)] << 16);
      if (row < n && col < k) out[row * k + col] = from_f32<T>(sc * (float)((int)(w >> (4 * p) & 15) - 8));
      if (row < n && col + 1 < k)
        out[row * k + col + 1] = from_f32<T>(sc * (float)((int)(w >> (16 + 4 * p) & 15) - 8));
    }
  }
}

// ---------------------------------------------------------------------------
// plan
// ---------------------------------------------------------------------------
inline int w4_nt(int tokens) { return tokens <= 8 ? 1 : tokens <= 16 ? 2 : 4; }
inline size_t w4_fixed_smem(int nt, int sg) {
  return (size_t)kW4Warps * (kW4Stages * (1024 + 32 * sg) + nt * 32 * sizeof(float4));
}
// Column blocks of a slab: all of them where x' fits beside the ring, else
// equal shares.
inline int64_t w4_slab(int64_t blocks, int tokens) {
  const int64_t room = (int64_t)(kW4Smem - w4_fixed_smem(w4_nt(tokens), 4)) / (2 * kW4Block * tokens);
  if (blocks <= room) return blocks;
  const int64_t slabs = (blocks + room - 1) / room;
  return (blocks + slabs - 1) / slabs;
}

template <int NT, int SG, typename T>
int launch_w4(const W4Args& a, cudaStream_t stream) {
  auto kernel = w4_kernel<NT, SG, T>;
  static bool allowed[kMaxDevices] = {};
  const int dev = device_index();
  if (!allowed[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kW4Smem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_last_cuda_error(e);
      return TQ_E_CUDA;
    }
    allowed[dev] = true;
  }
  const size_t smem = w4_fixed_smem(NT, SG) + (size_t)a.slab * kW4Block * 2 * a.tokens;
  const int slabs = (a.blocks + a.slab - 1) / a.slab;
  int x = sm_count() / slabs;
  if (x < 1) x = 1;
  if (x > a.tiles) x = a.tiles;
  return launch_dependent(kernel, dim3(x, slabs), dim3(kW4Threads), smem, stream, a);
}

template <int NT, typename T>
int launch_w4_group(const W4Args& a, cudaStream_t stream) {
  if (a.group == 128) return launch_w4<NT, 1, T>(a, stream);
  return a.group == 64 ? launch_w4<NT, 2, T>(a, stream) : launch_w4<NT, 4, T>(a, stream);
}

template <typename T>
int launch_w4_all(const W4Args& a, int nt, cudaStream_t stream) {
  if (nt == 1) return launch_w4_group<1, T>(a, stream);
  return nt == 2 ? launch_w4_group<2, T>(a, stream) : launch_w4_group<4, T>(a, stream);
}

template <typename T>
int gemv_w4(W4Args a, int64_t tokens, void* workspace, cudaStream_t stream) {
  const char* x = (const char*)a.x;
  const size_t item = a.mode == kW4F32 ? 4 : 2;
  for (int64_t m = 0; m < tokens; m += kW4MaxTokens) {
    a.tokens = (int)(tokens - m < kW4MaxTokens ? tokens - m : kW4MaxTokens);
    a.x = x + m * a.x_stride * item;
    a.y_offset = m;
    a.slab = (int)w4_slab(a.blocks, a.tokens);
    const int slabs = (a.blocks + a.slab - 1) / a.slab;
    a.part = slabs > 1 ? (float*)workspace : nullptr;
    int st = launch_w4_all<T>(a, w4_nt(a.tokens), stream);
    if (st == TQ_OK && slabs > 1) {
      const int64_t count = a.tokens * a.n;
      st = launch_dependent(w4_join_kernel<T>, dim3((unsigned)((count + 255) / 256)), dim3(256), 0, stream, a.part,
                            slabs, count, m * a.n, (const T*)a.residual, (T*)a.y);
    }
    if (st != TQ_OK) return st;
  }
  return TQ_OK;
}

inline int check_w4(int64_t n, int64_t k, int group) {
  if (!valid_group(group) || n <= 0 || k <= 0) return TQ_E_SHAPE;
  if (w4_tiles(n) > INT32_MAX / 2 || w4_blocks(k) > INT32_MAX / 256) return TQ_E_SHAPE;
  return TQ_OK;
}

}  // namespace tq

using namespace tq;

extern "C" {

int tq_w4_sizes(int64_t n, int64_t k, int group_size, size_t* code_bytes, size_t* scale_bytes) {
  const int st = check_w4(n, k, group_size);
  if (st != TQ_OK) return st;
  if (!code_bytes || !scale_bytes) return TQ_E_ARG;
  *code_bytes = (size_t)w4_tiles(n) * w4_blocks(k) * 1024;
  *scale_bytes = (size_t)w4_tiles(n) * w4_blocks(k) * 32 * (kW4Block / group_size);
  return TQ_OK;
}

int tq_w4_layout(const uint8_t* packed, const void* scales, int64_t n, int64_t k, int group_size, void* codes_out,
                 void* scales_out, tq_stream_t stream) {
  const int st = check_w4(n, k, group_size);
  if (st != TQ_OK) return st;
  if (!packed || !scales || !codes_out || !scales_out) return TQ_E_ARG;
  if ((uintptr_t)scales % 2 || (uintptr_t)codes_out % 16 || (uintptr_t)scales_out % 16) return TQ_E_SHAPE;
  return launch_dependent(w4_layout_kernel, dim3(sm_count() * 8), dim3(256), 0, (cudaStream_t)stream, packed,
                          (const uint16_t*)scales, n, k, group_size, w4_tiles(n), w4_blocks(k), (uint32_t*)codes_out,
                          (uint16_t*)scales_out);
}

int tq_w4_quantize(const void* weight, int dtype, int64_t n, int64_t k, int group_size, uint8_t* packed,
                   void* scales, tq_stream_t stream) {
  const int st = check_w4(n, k, group_size);
  if (st != TQ_OK) return st;
  if (dtype != TQ_F32 && dtype != TQ_F16 && dtype != TQ_BF16) return TQ_E_ARG;
  if (!weight || !packed || !scales) return TQ_E_ARG;
  const int64_t warps = n * ((k + group_size - 1) / group_size);
  if ((warps + 7) / 8 > INT32_MAX) return TQ_E_SHAPE;
  const dim3 grid((unsigned)((warps + 7) / 8)), block(256);
  cudaStream_t s = (cudaStream_t)stream;
  uint16_t* so = (uint16_t*)scales;
  if (dtype == TQ_F16)
    return launch_dependent(w4_quantize_kernel<__half>, grid, block, 0, s, (const __half*)weight, n, k, group_size, packed, so);
  if (dtype == TQ_BF16)
    return launch_dependent(w4_quantize_kernel<__nv_bfloat16>, grid, block, 0, s, (const __nv_bfloat16*)weight, n, k,
                            group_size, packed, so);
  return launch_dependent(w4_quantize_kernel<float>, grid, block, 0, s, (const float*)weight, n, k, group_size, packed, so);
}

int tq_w4_dequantize(const void* codes, const void* scales, int64_t n, int64_t k, int group_size, void* out,
                     int out_dtype, tq_stream_t stream) {
  const int st = check_w4(n, k, group_size);
  if (st != TQ_OK) return st;
  if (out_dtype != TQ_F32 && out_dtype != TQ_F16 && out_dtype != TQ_BF16) return TQ_E_ARG;
  if (!codes || !scales || !out) return TQ_E_ARG;
  const dim3 grid(sm_count() * 8), block(256);
  cudaStream_t s = (cudaStream_t)stream;
  const uint32_t* cp = (const uint32_t*)codes;
  const uint16_t* sp = (const uint16_t*)scales;
  const int64_t tiles = w4_tiles(n), blocks = w4_blocks(k);
  if (out_dtype == TQ_F16)
    return launch_dependent(w4_dequantize_kernel<__half>, grid, block, 0, s, cp, sp, n, k, group_size, tiles, blocks, (__half*)out);
  if (out_dtype == TQ_BF16)
    return launch_dependent(w4_dequantize_kernel<__nv_bfloat16>, grid, block, 0, s, cp, sp, n, k, group_size, tiles, blocks,
                            (__nv_bfloat16*)out);
  return launch_dependent(w4_dequantize_kernel<float>, grid, block, 0, s, cp, sp, n, k, group_size, tiles, blocks, (float*)out);
}

int tq_gemv_w4_workspace_size(int64_t n, int64_t k, int64_t tokens, size_t* bytes) {
  const int st = check_w4(n, k, 32);
  if (st != TQ_OK) return st;
  if (!bytes) return TQ_E_ARG;
  if (tokens < 0) return TQ_E_SHAPE;
  size_t need = 0;
  const int64_t blocks = w4_blocks(k);
  const int64_t launches[2] = {tokens < kW4MaxTokens ? tokens : kW4MaxTokens, tokens % kW4MaxTokens};
  for (int64_t t : launches) {  // full launches and the last one
    if (t == 0) continue;
    const int64_t slab = w4_slab(blocks, (int)t), slabs = (blocks + slab - 1) / slab;
    const size_t b = slabs > 1 ? (size_t)slabs * t * n * sizeof(float) : 0;
    if (b > need) need = b;
  }
  *bytes = need;
  return TQ_OK;
}

int tq_gemv_w4(const void* codes, const void* scales, int64_t n, int64_t k, int group_size, const void* x,
               int x_dtype, int64_t x_stride, int x_mode, const void* norm_weight, float eps, const void* residual,
               void* y, int64_t tokens, void* workspace, size_t workspace_bytes, tq_stream_t stream) {
  int st = check_w4(n, k, group_size);
  if (st != TQ_OK) return st;
  if (x_mode < kW4Plain || x_mode > kW4Silu) return TQ_E_ARG;
  if (x_dtype != TQ_BF16 && !(x_dtype == TQ_F16 && x_mode == kW4Plain)) return TQ_E_ARG;
  if (tokens < 0 || (tokens > 1 && x_stride < (x_mode == kW4Silu ? 2 * k : k))) return TQ_E_SHAPE;
  if (tokens == 0) return TQ_OK;
  if (!codes || !scales || !x || !y || (x_mode == kW4Rms && !norm_weight)) return TQ_E_ARG;
  if ((uintptr_t)codes % 16 || (uintptr_t)scales % 16) return TQ_E_SHAPE;
  size_t need = 0;
  st = tq_gemv_w4_workspace_size(n, k, tokens, &need);
  if (st != TQ_OK) return st;
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return TQ_E_WORKSPACE;
  W4Args a = {};
  a.codes = (const uint4*)codes;
  a.scales = (const uint8_t*)scales;
  a.x = x;
  a.norm_w = norm_weight;
  a.residual = residual;
  a.y = y;
  a.n = n;
  a.k = k;
  a.x_stride = x_stride;
  a.tiles = (int)w4_tiles(n);
  a.blocks = (int)w4_blocks(k);
  a.mode = x_mode;
  a.group = group_size;
  a.eps = eps;
  cudaStream_t s = (cudaStream_t)stream;
  return x_dtype == TQ_F16 ? gemv_w4<__half>(a, tokens, workspace, s) : gemv_w4<__nv_bfloat16>(a, tokens, workspace, s);
}

}  // extern "C"
