// Input gradients of the quantized products: dA[M, K] = sum_p dC_p[M, N_p] . W_p[K, N_p]^T
// over up to three FP4 / INT4 matrices W_p (one: a linear layer; two: the gate and up
// projections; three: Q, K and V), and the elementwise gradient of SiLU(gate) * up.
//
// The weights are the words of the forward products, read in place: a word holds 8 k of
// one column n, and here n is the contracted axis, so a lane takes 8 words of one word
// row (8 adjacent n, 8 k) and pairs the nibbles of neighbouring n before they are
// converted (pair_words).  Each weight is the fp16 value of the reference's dequantizer,
// products accumulate in fp32 on the matrix cores, and the sum is rounded once.
//
// Gradients have a wider range than activations.  bf16 and fp32 ones, and those of the
// gate/up pair, are carried in fp16 with one power of two per row (k_grad_rows,
// k_swiglu_grad): a row's largest value lands in [2^14, 2^15), so what is lost lies 2^-40
// below it, and the power of two is taken out of the fp32 sums exactly.
#include <algorithm>

#include "mm_common.h"
#include "mm_prefill.h"
#include "mmfp4.h"

namespace {
using namespace mmpf;

constexpr int GR_BN = 64;                 // n per LDS chunk
constexpr int GR_KP = 32;                 // word rows (8 k each) per tile
constexpr int GR_COLS = 8 * GR_KP;        // output columns (k) per tile
constexpr int GR_MAX_TILES = 16384;       // arrival counters at the head of the workspace
constexpr size_t GR_COUNTER_BYTES = (size_t)GR_MAX_TILES * sizeof(uint32_t);

// Zeros that stand in for gradient columns past a matrix's last one.
__device__ __attribute__((aligned(16))) const uint32_t gr_zeros[4] = {0, 0, 0, 0};

struct GradSeg {
  const f16* A;       // gradient of this matrix's output, [M, N], row stride lda
  const uint32_t* B;  // words: [K/8, N], or [N, K/8] (ROWS)
  const f16 *S, *Z;   // [K/g, N]
  int lda, N, ch0;    // ch0: the segment's first chunk
};
struct GradSegs {
  GradSeg s[3];
  int nch;            // chunks of all segments
};

// ---------------------------------------------------------------------------
// Words -> MFMA operands.  w: the words of 8 adjacent n (n0 .. n0 + 7) of one word row;
// b[j] (j = 0..3): the weights of k = 8 kp + 4 wn + j at those n, in n order.  `half`
// selects bytes 0, 1 (wn = 0) or 2, 3 (wn = 1) of two words.
// ---------------------------------------------------------------------------
MM_DEV uint32_t sgpr_const(uint32_t v) {
  asm("" : "+s"(v));   // keeps (x & m) | (y & ~m) one v_bfi_b32 (no literal operand in VOP3)
  return v;
}

// Non-finite scales count as zero (sanitize_scale), two at a time: x + 0x0400 carries the
// all-ones exponent into the sign bit.
MM_DEV f16x2 sanitize2(f16x2 s) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const s16x2 u = __builtin_bit_cast(s16x2, s);
  const s16x2 e = (u & (short)0x7c00) + (short)0x0400;
  return __builtin_bit_cast(f16x2, (s16x2)(u & ~(e >> 15)));
}

template <bool INT4>
struct PairWords;

template <>
struct PairWords<false> {
  // Bytes of e (o) hold the nibble of an even (odd) k of one word below the same of the
  // next word, which is the operand order of the packed convert.
  MM_DEV static void run(const u32x4 (&w)[2], const f16x2 (&s)[4], const f16x2 (&)[4],
                         uint32_t half, f16x8 (&b)[4]) {
    const uint32_t m = sgpr_const(0x0f0f0f0fu);
    uint32_t r[4][4];   // [j][pair of n]
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t P = __builtin_amdgcn_perm(w[q][2], w[q][0], half);   // n, n + 2
      const uint32_t Q = __builtin_amdgcn_perm(w[q][3], w[q][1], half);   // n + 1, n + 3
      const uint32_t e = (P & m) | ((Q << 4) & ~m);
      const uint32_t o = ((P >> 4) & m) | (Q & ~m);
      r[0][2 * q] = __builtin_bit_cast(uint32_t, e2m1_pair_c<0>(e) * s[2 * q]);
      r[2][2 * q] = __builtin_bit_cast(uint32_t, e2m1_pair_c<1>(e) * s[2 * q]);
      r[0][2 * q + 1] = __builtin_bit_cast(uint32_t, e2m1_pair_c<2>(e) * s[2 * q + 1]);
      r[2][2 * q + 1] = __builtin_bit_cast(uint32_t, e2m1_pair_c<3>(e) * s[2 * q + 1]);
      r[1][2 * q] = __builtin_bit_cast(uint32_t, e2m1_pair_c<0>(o) * s[2 * q]);
      r[3][2 * q] = __builtin_bit_cast(uint32_t, e2m1_pair_c<1>(o) * s[2 * q]);
      r[1][2 * q + 1] = __builtin_bit_cast(uint32_t, e2m1_pair_c<2>(o) * s[2 * q + 1]);
      r[3][2 * q + 1] = __builtin_bit_cast(uint32_t, e2m1_pair_c<3>(o) * s[2 * q + 1]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      b[j] = __builtin_bit_cast(f16x8, u32x4{r[j][0], r[j][1], r[j][2], r[j][3]});
  }
};

template <>
struct PairWords<true> {
  // The 16-bit halves of two neighbouring words side by side; a nibble at bits 0..3 of a
  // half under exponent 0x6400 is 1024 + q, at bits 4..7 under 0x5400 it is 64 + q.
  // fp16(q - z) is one rounded subtraction, as in dq_u4_word.
  MM_DEV static void run(const u32x4 (&w)[2], const f16x2 (&s)[4], const f16x2 (&nz)[4],
                         uint32_t half, f16x8 (&b)[4]) {
    const uint32_t mlo = sgpr_const(0x000f000fu), mhi = sgpr_const(0x00f000f0u);
    const f16x2 b1024 = {(f16)-1024.0f, (f16)-1024.0f}, b64 = {(f16)-64.0f, (f16)-64.0f};
    uint32_t r[4][4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const uint32_t x = __builtin_amdgcn_perm(w[p >> 1][2 * (p & 1) + 1], w[p >> 1][2 * (p & 1)],
                                               half);
      const uint32_t y = x >> 8;
      const f16x2 q0 = __builtin_bit_cast(f16x2, (x & mlo) | (~mlo & 0x64006400u)) + b1024;
      const f16x2 q1 = __builtin_bit_cast(f16x2, (x & mhi) | (~mhi & 0x54005400u)) + b64;
      const f16x2 q2 = __builtin_bit_cast(f16x2, (y & mlo) | (~mlo & 0x64006400u)) + b1024;
      const f16x2 q3 = __builtin_bit_cast(f16x2, (y & mhi) | (~mhi & 0x54005400u)) + b64;
      r[0][p] = __builtin_bit_cast(uint32_t, (q0 + nz[p]) * s[p]);
      r[1][p] = __builtin_bit_cast(uint32_t, (q1 + nz[p]) * s[p]);
      r[2][p] = __builtin_bit_cast(uint32_t, (q2 + nz[p]) * s[p]);
      r[3][p] = __builtin_bit_cast(uint32_t, (q3 + nz[p]) * s[p]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      b[j] = __builtin_bit_cast(f16x8, u32x4{r[j][0], r[j][1], r[j][2], r[j][3]});
  }
};

// ---------------------------------------------------------------------------
// The product.  Tiles of BM = 32 * RB * WM rows x 256 columns (k); waves (wm, wn): rows of
// wm, and of every word row's 8 columns the four 4 wn + j, so a wave's tile is 32 * RB rows
// x 128 columns: lane l32 holds columns 8 (kp0 + l32) + 4 wn + j.  Operands go
// global -> LDS directly, STAGES - 1 chunks of 64 n ahead:
//   A  piece (r, c8), 8 halves, at r*8 + (c8 ^ ((r >> 1) & 7))   (as mm_prefill.h)
//   B  Marlin: 32 word rows x 64 words, piece (row, p), 4 words, at row*16 + (p ^ (row & 15)):
//      the 16 lanes of a read pass hit all banks; ROWS: 64 n x 32 words as they lie
//   S, Z  SR group rows x 64 halves: the groups that the tile's 256 k touch
// ks > 1: the chunks are split over gridDim.z and the last block of a tile adds the splits
// in order (k_mid's hand-off: sc1 partials, an arrival counter per tile left at zero).
// ot: the output's type, 0 fp32, 1 fp16, 2 bf16.
// ---------------------------------------------------------------------------
template <bool INT4, int WM, int RB, int SR>
struct GradShape {
  static constexpr int STAGES = 3;
  static constexpr int NWAVE = 2 * WM, NTHR = 64 * NWAVE, BM = 32 * RB * WM;
  static constexpr int A_PIECES = BM * 8, B_PIECES = GR_KP * GR_BN / 4, S_PIECES = SR * 8;
  static constexpr int A_IT = A_PIECES / NTHR, B_IT = B_PIECES / NTHR;
  static constexpr int S_IT = (S_PIECES + NTHR - 1) / NTHR;
  static_assert(A_PIECES % NTHR == 0 && B_PIECES % NTHR == 0 && S_PIECES % 64 == 0, "split");
  static constexpr int LOADS = A_IT + B_IT + S_IT * (INT4 ? 2 : 1);
  static constexpr int A_BYTES = A_PIECES * 16, B_BYTES = B_PIECES * 16, S_BYTES = S_PIECES * 16;
  static constexpr int B_OFF = STAGES * A_BYTES, S_OFF = B_OFF + STAGES * B_BYTES;
  static constexpr int Z_OFF = S_OFF + STAGES * S_BYTES;
  static constexpr int D_OFF = Z_OFF + (INT4 ? STAGES * S_BYTES : 0);   // dump of idle waves
  static constexpr int LDS_BYTES = D_OFF + 1024;
};

MM_DEV uint16_t bf16_bits(float v) {
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40);   // NaN
  return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1)) >> 16);
}

template <bool INT4, bool ROWS, int WM, int RB, int SR>
__global__ void __launch_bounds__(WM * 128)
k_grad(GradSegs segs, void* __restrict__ out, int ot, const float* __restrict__ rowmul, int M,
       int K, int g, int cps, int grp, float* __restrict__ part, uint32_t* __restrict__ counters) {
  using Sh = GradShape<INT4, WM, RB, SR>;
  constexpr int NWAVE = Sh::NWAVE, STAGES = Sh::STAGES;
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS_BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int l32 = lane & 31, h = lane >> 5;
  const int KP = K >> 3, ngroups = K / g;
  // Tile walk of k_prefill2: an XCD takes a run of tiles, groups of grp row tiles
  // column by column.
  const int nx = gridDim.x, ny = gridDim.y, ntile = nx * ny * gridDim.z;
  const int L = blockIdx.x + nx * (blockIdx.y + ny * blockIdx.z);
  const int xq = ntile >> 3, xr = ntile & 7, xcd = L & 7;
  const int lin = xcd * xq + min(xcd, xr) + (L >> 3);
  const int bz = lin / (nx * ny), lt = lin - bz * (nx * ny);
  const int gi = lt / (grp * nx), gw = lt - gi * (grp * nx);
  const int gr = min(grp, ny - gi * grp);
  const int by = gi * grp + gw % gr, bx = gw / gr;
  const int m0 = by * Sh::BM, kp0 = bx * GR_KP;
  const int c_beg = bz * cps, c_end = min(segs.nch, c_beg + cps);
  const int g0 = 8 * kp0 / g;              // first group of the tile

  // Source offsets within a segment that do not change from chunk to chunk.
  int a_row[Sh::A_IT], a_c8[Sh::A_IT];
#pragma unroll
  for (int i = 0; i < Sh::A_IT; ++i) {
    const int p = (i * NWAVE + wave) * 64 + lane, r = p >> 3;
    a_row[i] = min(m0 + r, M - 1);
    a_c8[i] = 8 * ((p & 7) ^ ((r >> 1) & 7));
  }
  auto issue = [&](int ch, int st) {
    const int sg = ch >= segs.s[2].ch0 ? 2 : (ch >= segs.s[1].ch0 ? 1 : 0);
    const GradSeg& s = segs.s[sg];
    const int N = s.N, n0 = (ch - s.ch0) * GR_BN;
#pragma unroll
    for (int i = 0; i < Sh::A_IT; ++i) {
      const f16* src = s.A + (size_t)a_row[i] * s.lda + n0 + a_c8[i];
      if (n0 + GR_BN > N) src = n0 + a_c8[i] < N ? src : (const f16*)gr_zeros;
      gl2lds16(src, smem + st * Sh::A_BYTES + (i * NWAVE + wave) * 1024);
    }
#pragma unroll
    for (int i = 0; i < Sh::B_IT; ++i) {
      const int p = (i * NWAVE + wave) * 64 + lane;
      const uint32_t* src;
      if constexpr (ROWS) {
        const int n = min(n0 + (p >> 3), N - 1), kp = min(kp0 + 4 * (p & 7), KP - 4);
        src = s.B + (size_t)n * KP + kp;
      } else {
        const int row = p >> 4;
        const int n = min(n0 + 4 * ((p & 15) ^ (row & 15)), N - 4);
        src = s.B + (size_t)min(kp0 + row, KP - 1) * N + n;
      }
      gl2lds16(src, smem + Sh::B_OFF + st * Sh::B_BYTES + (i * NWAVE + wave) * 1024);
    }
#pragma unroll
    for (int i = 0; i < Sh::S_IT; ++i) {
      const int wp = i * NWAVE + wave;
      const int p = min(wp * 64 + lane, Sh::S_PIECES - 1);
      const size_t off = (size_t)min(g0 + (p >> 3), ngroups - 1) * N + min(n0 + 8 * (p & 7), N - 8);
      const bool live = wp * 64 < Sh::S_PIECES;
      gl2lds16(s.S + off, smem + (live ? Sh::S_OFF + st * Sh::S_BYTES + wp * 1024 : Sh::D_OFF));
      if constexpr (INT4)
        gl2lds16(s.Z + off, smem + (live ? Sh::Z_OFF + st * Sh::S_BYTES + wp * 1024 : Sh::D_OFF));
    }
  };

  f32x16 acc[RB][4];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[rb][j][v] = 0.0f;

#pragma unroll
  for (int c = 0; c < STAGES - 1; ++c) issue(min(c_beg + c, c_end - 1), c);

  const int arow = wm * 32 * RB + l32, ax = (arow >> 1) & 7;   // rows of all row blocks share ax
  const int srow = 8 * min(kp0 + l32, KP - 1) / g - g0;
  const uint32_t half = wn ? 0x07060302u : 0x05040100u;
  const uint32_t s_off = srow * 128 + h * 16;
  const uint32_t b_row = ROWS ? (h * 8 * 32 + l32) * 4 : l32 * 256, bx15 = l32 & 15;

  auto chunk = [&](int ch, auto stc) {
    constexpr int st = decltype(stc)::value;
    // Chunk ch has landed once at most STAGES - 2 later chunks' loads are outstanding; the
    // barrier publishes it and frees the stage that is refilled next.
    wait_vmcnt<(STAGES - 2) * Sh::LOADS>();
    __builtin_amdgcn_s_barrier();
    issue(min(ch + STAGES - 1, c_end - 1), (st + STAGES - 1) % STAGES);
    f16x8 af[2][RB], bq[2][4];
    u32x4 w[2][2];
    f16x8 sv[2], zv[2];
    auto frag = [&](int t, int slot) {
      if constexpr (ROWS) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[slot][i >> 2][i & 3] = *(const uint32_t*)(smem + Sh::B_OFF + st * Sh::B_BYTES + b_row +
                                                      (16 * t + i) * 128);
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          w[slot][i] = *(const u32x4*)(smem + Sh::B_OFF + st * Sh::B_BYTES + b_row +
                                       ((4 * t + 2 * h + i) ^ bx15) * 16);
      }
      sv[slot] = *(const f16x8*)(smem + Sh::S_OFF + st * Sh::S_BYTES + s_off + t * 32);
      if constexpr (INT4)
        zv[slot] = *(const f16x8*)(smem + Sh::Z_OFF + st * Sh::S_BYTES + s_off + t * 32);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
        af[slot][rb] = *(const f16x8*)(smem + st * Sh::A_BYTES + (arow + 32 * rb) * 128 +
                                       ((2 * t + h) ^ ax) * 16);
    };
    auto decode = [&](int slot) {
      f16x2 s2[4], nz2[4] = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s2[i] = sanitize2(f16x2{sv[slot][2 * i], sv[slot][2 * i + 1]});
        if constexpr (INT4) {
          const f16x2 lim = {(f16)127.0f, (f16)127.0f};
          nz2[i] = -__builtin_elementwise_min(
              __builtin_elementwise_max(f16x2{zv[slot][2 * i], zv[slot][2 * i + 1]}, -lim), lim);
        }
      }
      PairWords<INT4>::run(w[slot], s2, nz2, half, bq[slot]);
    };
    // Step t + 1 is read and decoded while step t's products occupy the matrix cores.
    frag(0, 0);
    decode(0);
#pragma unroll
    for (int t = 0; t < GR_BN / 16; ++t) {
      const int cur = t & 1;
      if (t + 1 < GR_BN / 16) frag(t + 1, cur ^ 1);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[rb][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cur][rb], bq[cur][j], acc[rb][j],
                                                              0, 0, 0);
      if (t + 1 < GR_BN / 16) decode(cur ^ 1);
#pragma unroll
      for (int i = 0; i < RB * 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                    // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, MM_PF2_SCHED_DS, 0);      // DS read
        __builtin_amdgcn_sched_group_barrier(0x002, MM_PF2_SCHED_VALU, 0);    // VALU
      }
    }
  };
  for (int ch = c_beg; ch < c_end; ch += STAGES) {
    static_for(
        [&](auto stc) {
          constexpr int st = decltype(stc)::value;
          if (st == 0 || ch + st < c_end) chunk(ch + st, stc);
        },
        std::make_integer_sequence<int, STAGES>{});
  }
  wait_vmcnt<0>();

  const int ks = gridDim.z;
  if (ks > 1) {
    const int tile = by * nx + bx;
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(part + (size_t)tile * ks * (Sh::BM * GR_COLS));
    auto at = [&](int z, int rb, int j, int q) {
      return 16u * (uint32_t)((((z * RB + rb) * 16 + j * 4 + q) * NWAVE + wave) * 64 + lane);
    };
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          store_agent_x4(prs, at(bz, rb, j, q),
                         f32x4{acc[rb][j][4 * q], acc[rb][j][4 * q + 1], acc[rb][j][4 * q + 2],
                               acc[rb][j][4 * q + 3]});
    __builtin_amdgcn_s_waitcnt(0);   // this wave's partials have reached the coherence point
    __syncthreads();
    uint32_t* const s_last = (uint32_t*)smem;
    if (tid == 0) {
      const uint32_t prev = __hip_atomic_fetch_add(&counters[tile], 1u, __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
      *s_last = prev == (uint32_t)ks - 1u;
    }
    __syncthreads();
    if (!*s_last) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int v = 0; v < 16; ++v) acc[rb][j][v] = 0.0f;
        for (int z = 0; z < ks; z += 2) {
          f32x4 ld[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) ld[i][q] = load_agent_x4(prs, at(min(z + i, ks - 1), rb, j, q));
#pragma unroll
          for (int i = 0; i < 2; ++i)
            if (z + i < ks)
#pragma unroll
              for (int v = 0; v < 16; ++v) acc[rb][j][v] += ld[i][v >> 2][v & 3];
        }
      }
    if (tid == 0)
      __hip_atomic_store(&counters[tile], 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  const int kp = kp0 + l32;
  if (kp >= KP) return;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      const int row = m0 + wm * 32 * RB + rb * 32 + 8 * (v >> 2) + 4 * h + (v & 3);
      if (row >= M) continue;
      const float f = rowmul != nullptr ? rowmul[row] : 1.0f;
      const float x0 = acc[rb][0][v] * f, x1 = acc[rb][1][v] * f;
      const float x2 = acc[rb][2][v] * f, x3 = acc[rb][3][v] * f;
      const size_t at = (size_t)row * K + 8 * kp + 4 * wn;
      if (ot == 1) {
        *(f16x4*)((f16*)out + at) = f16x4{(f16)x0, (f16)x1, (f16)x2, (f16)x3};
      } else if (ot == 2) {
        *(u32x2*)((uint16_t*)out + at) = u32x2{bf16_bits(x0) | (uint32_t)bf16_bits(x1) << 16,
                                               bf16_bits(x2) | (uint32_t)bf16_bits(x3) << 16};
      } else {
        *(f32x4*)((float*)out + at) = f32x4{x0, x1, x2, x3};
      }
    }
}

// ---------------------------------------------------------------------------
// Row conversion: fp16 values v * 2^e with the row's largest in [2^14, 2^15), and
// rowmul[row] = 2^-e.  A zero or non-finite row keeps e = 0.
// ---------------------------------------------------------------------------
constexpr int RW_NT = 512;
constexpr int RW_HOLD = 4;      // 8-value pieces of a row that a thread keeps in registers

MM_DEV float row_exponent(float m, float& inv) {
  int e = 0;
  if (m > 0.0f && m < __builtin_inff()) {
    (void)frexpf(m, &e);          // m = f * 2^e, f in [0.5, 1)
    e = max(-110, min(110, 15 - e));
  }
  inv = ldexpf(1.0f, -e);
  return ldexpf(1.0f, e);
}

MM_DEV float block_max(float m, float* red) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = red[0];
#pragma unroll
  for (int i = 1; i < RW_NT / 64; ++i) m = fmaxf(m, red[i]);
  return m;
}

// 8 values at element offset `at` as fp32.  T: 0 fp32, 1 fp16, 2 bf16.
template <int T>
MM_DEV void load8(const void* p, size_t at, float (&v)[8]) {
  if constexpr (T == 1) {
    const f16x8 x = *(const f16x8*)((const f16*)p + at);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)x[i];
  } else if constexpr (T == 2) {
    const u32x4 x = *(const u32x4*)((const uint16_t*)p + at);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __builtin_bit_cast(float, x[i] << 16);
      v[2 * i + 1] = __builtin_bit_cast(float, x[i] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x4 x = *(const f32x4*)((const float*)p + at + 4 * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = x[j];
    }
  }
}
MM_DEV void store8(f16* p, const float (&v)[8], float mul) {
  f16x8 o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = (f16)(v[i] * mul);
  *(f16x8*)p = o;
}

// One block per row; up to RW_NT * 8 * RW_HOLD columns are read once, wider rows twice.
template <int T>
__global__ void __launch_bounds__(RW_NT)
k_grad_rows(const void* __restrict__ X, f16* __restrict__ Y, float* __restrict__ rowmul, int N) {
  __shared__ float red[RW_NT / 64];
  const size_t base = (size_t)blockIdx.x * N;
  const int np = N / 8;
  float hold[RW_HOLD][8], m = 0.0f;
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) {
      load8<T>(X, base + 8 * (size_t)p, hold[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(hold[i][k]));
    }
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float v[8];
    load8<T>(X, base + 8 * (size_t)p, v);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[k]));
  }
  float inv;
  const float mul = row_exponent(block_max(m, red), inv);
  if (threadIdx.x == 0) rowmul[blockIdx.x] = inv;
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) store8(Y + base + 8 * (size_t)p, hold[i], mul);
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float v[8];
    load8<T>(X, base + 8 * (size_t)p, v);
    store8(Y + base + 8 * (size_t)p, v, mul);
  }
}

// Gradients of silu(g) * u: dg = dh u sig(g) (1 + g (1 - sig(g))), du = dh silu(g), from
// the kept fp16 [g | u], in fp32, written side by side as [dg | du] with the row's power of
// two.  sig(-inf) = 0 with g (1 - sig) = -inf would give NaN where the limit is 0: g is
// bounded below at -1e4 in that term, where sig(g) has long been 0.
MM_DEV void swiglu_grad(float dh, float g, float u, float& dg, float& du) {
  const float sig = 1.0f / (1.0f + __expf(-g));
  const float gb = fmaxf(g, -1.0e4f);
  dg = dh * u * (sig * (1.0f + gb * (1.0f - sig)));
  du = dh * (gb * sig);
}

template <int T>
__global__ void __launch_bounds__(RW_NT)
k_swiglu_grad(const void* __restrict__ dH, const f16* __restrict__ GU, f16* __restrict__ Y,
              float* __restrict__ rowmul, int N) {
  __shared__ float red[RW_NT / 64];
  const size_t hb = (size_t)blockIdx.x * N, gb = 2 * hb;
  const int np = N / 8;
  auto grads = [&](int p, float (&dg)[8], float (&du)[8]) {
    float dh[8], g[8], u[8];
    load8<T>(dH, hb + 8 * (size_t)p, dh);
    load8<1>(GU, gb + 8 * (size_t)p, g);
    load8<1>(GU, gb + N + 8 * (size_t)p, u);
#pragma unroll
    for (int k = 0; k < 8; ++k) swiglu_grad(dh[k], g[k], u[k], dg[k], du[k]);
  };
  float hg[RW_HOLD][8], hu[RW_HOLD][8], m = 0.0f;
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) {
      grads(p, hg[i], hu[i]);
#pragma unroll
      for (int k = 0; k < 8; ++k) m = fmaxf(m, fmaxf(fabsf(hg[i][k]), fabsf(hu[i][k])));
    }
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float dg[8], du[8];
    grads(p, dg, du);
#pragma unroll
    for (int k = 0; k < 8; ++k) m = fmaxf(m, fmaxf(fabsf(dg[k]), fabsf(du[k])));
  }
  float inv;
  const float mul = row_exponent(block_max(m, red), inv);
  if (threadIdx.x == 0) rowmul[blockIdx.x] = inv;
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) {
      store8(Y + gb + 8 * (size_t)p, hg[i], mul);
      store8(Y + gb + N + 8 * (size_t)p, hu[i], mul);
    }
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float dg[8], du[8];
    grads(p, dg, du);
    store8(Y + gb + 8 * (size_t)p, dg, mul);
    store8(Y + gb + N + 8 * (size_t)p, du, mul);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct GradPlan {
  int wm, rb;   // waves along the rows, 32-row blocks per wave
  int ks, cps;
};

GradPlan plan_grad(int M, long ntot_chunks, int K) {
  GradPlan p{1, 1, 1, 0};
  if (M > 128) p = {2, 4, 1, 0};
  else if (M > 64) p = {1, 4, 1, 0};
  else if (M > 32) p = {1, 2, 1, 0};
  const int bm = 32 * p.rb * p.wm;
  const long tiles = (long)mm_cdiv(K, GR_COLS) * mm_cdiv(M, bm);
  const int want = p.rb == 4 && p.wm == 2 ? 200 : 512;
  const int nch = (int)ntot_chunks;
  while (tiles * p.ks < want && p.ks < 64 && nch / (p.ks + 1) >= 4) ++p.ks;
  if (tiles > GR_MAX_TILES) p.ks = 1;
  p.cps = mm_cdiv(nch, p.ks);
  p.ks = mm_cdiv(nch, p.cps);
  return p;
}

size_t grad_ws_bytes(const GradPlan& p, int M, int K) {
  if (p.ks == 1) return GR_COUNTER_BYTES;
  const int bm = 32 * p.rb * p.wm;
  return GR_COUNTER_BYTES +
         (size_t)mm_cdiv(K, GR_COLS) * mm_cdiv(M, bm) * p.ks * bm * GR_COLS * sizeof(float);
}

int grad_chunks(int nmat, const int* N) {
  int c = 0;
  for (int i = 0; i < nmat; ++i) c += mm_cdiv(N[i], GR_BN);
  return c;
}

template <bool INT4, bool ROWS, int WM, int RB, int SR>
int launch_grad(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K, int g,
                const GradPlan& p, void* ws, hipStream_t st) {
  using Sh = GradShape<INT4, WM, RB, SR>;
  const dim3 grid(mm_cdiv(K, GR_COLS), mm_cdiv(M, Sh::BM), p.ks);
  // Row tiles walked together: the walk's A rows (128 B per n) against B words (4 B x 32).
  int grp = 1;
  while (grp * 2 <= (int)grid.y && grp < 4) grp *= 2;
  hipLaunchKernelGGL((k_grad<INT4, ROWS, WM, RB, SR>), grid, dim3(Sh::NTHR), 0, st, s, out, ot,
                     rowmul, M, K, g, p.cps, grp, (float*)((char*)ws + GR_COUNTER_BYTES),
                     (uint32_t*)ws);
  MM_CHECK_LAUNCH("gemm backward");
  return 0;
}

template <bool INT4, bool ROWS, int SR>
int launch_grad_tile(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K,
                     int g, const GradPlan& p, void* ws, hipStream_t st) {
  if (p.wm == 2) return launch_grad<INT4, ROWS, 2, 4, SR>(s, out, ot, rowmul, M, K, g, p, ws, st);
  if (p.rb == 4) return launch_grad<INT4, ROWS, 1, 4, SR>(s, out, ot, rowmul, M, K, g, p, ws, st);
  if (p.rb == 2) return launch_grad<INT4, ROWS, 1, 2, SR>(s, out, ot, rowmul, M, K, g, p, ws, st);
  return launch_grad<INT4, ROWS, 1, 1, SR>(s, out, ot, rowmul, M, K, g, p, ws, st);
}

}  // namespace

extern "C" size_t mm_gemm_backward_workspace_bytes(int nmat, const int* N, int M, int K) {
  if (nmat < 1 || nmat > 3 || N == nullptr || M <= 0 || K <= 0) return GR_COUNTER_BYTES;
  return grad_ws_bytes(plan_grad(M, grad_chunks(nmat, N), K), M, K);
}

extern "C" int mm_gemm_backward(const uint16_t* const* dC, const int* ldc,
                                const float* row_mul, int nmat, const uint32_t* const* B,
                                const uint16_t* const* S, const uint16_t* const* Z, const int* N,
                                int layout, void* dA, int out_type, int M, int K, int g, void* ws,
                                size_t ws_bytes, void* stream) {
  const char* who = "mm_gemm_backward";
  MM_CHECK_ARG(nmat >= 1 && nmat <= 3, "%s: nmat=%d must be 1..3", who, nmat);
  MM_CHECK_ARG(dC != nullptr && ldc != nullptr && B != nullptr && S != nullptr && N != nullptr,
               "%s: null matrix table", who);
  MM_CHECK_ARG(out_type >= 0 && out_type <= 2, "%s: out_type=%d must be 0 (fp32), 1 (fp16) or 2 "
               "(bf16)", who, out_type);
  MM_CHECK_ARG(layout == 0 || layout == 1, "%s: layout=%d must be 0 ([K/8, N] words) or 1 "
               "([N, K/8])", who, layout);
  MM_CHECK_ARG(layout == 0 || Z == nullptr, "%s: row-packed words are FP4 (no zero points)", who);
  MM_CHECK_ARG(M >= 0 && K > 0, "%s: bad shape M=%d K=%d", who, M, K);
  MM_CHECK_ARG(K % (layout ? 32 : 8) == 0, "%s: K=%d must be divisible by %d", who, K,
               layout ? 32 : 8);
  MM_CHECK_ARG(g > 0 && g % 8 == 0 && K % g == 0,
               "%s: group_size=%d must be a multiple of 8 dividing K=%d", who, g, K);
  GradSegs s{};
  uintptr_t al = (uintptr_t)dA;
  int ch = 0;
  for (int i = 0; i < 3; ++i) {
    s.s[i].ch0 = 0x7fffffff;
    if (i >= nmat) continue;
    MM_CHECK_ARG(N[i] > 0 && N[i] % 8 == 0, "%s: N[%d]=%d must be a positive multiple of 8", who,
                 i, N[i]);
    MM_CHECK_ARG(ldc[i] >= N[i] && ldc[i] % 8 == 0,
                 "%s: ldc[%d]=%d must be a multiple of 8, at least N=%d", who, i, ldc[i], N[i]);
    s.s[i] = GradSeg{(const f16*)dC[i], B[i], (const f16*)S[i],
                     Z != nullptr ? (const f16*)Z[i] : nullptr, ldc[i], N[i], ch};
    ch += mm_cdiv(N[i], GR_BN);
    al |= (uintptr_t)dC[i] | (uintptr_t)B[i] | (uintptr_t)S[i] |
          (Z != nullptr ? (uintptr_t)Z[i] : 0);
  }
  s.nch = ch;
  MM_CHECK_ARG((al & 15) == 0, "%s: every operand must be 16-byte aligned", who);
  if (M == 0) return 0;
  const GradPlan p = plan_grad(M, ch, K);
  const size_t need = grad_ws_bytes(p, M, K);
  MM_CHECK_ARG(p.ks == 1 || (ws != nullptr && ws_bytes >= need),
               "%s: workspace of %zu bytes is smaller than the %zu required", who, ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  // A tile's 256 k touch at most 8 groups from g = 32 up, 32 below.
#define MM_GRAD(I4, RW)                                                                       \
  return g >= 32 ? launch_grad_tile<I4, RW, 8>(s, dA, out_type, row_mul, M, K, g, p, ws, st)   \
                 : launch_grad_tile<I4, RW, 32>(s, dA, out_type, row_mul, M, K, g, p, ws, st)
  if (layout == 1) MM_GRAD(false, true);
  if (Z != nullptr) MM_GRAD(true, false);
  MM_GRAD(false, false);
#undef MM_GRAD
}

extern "C" int mm_grad_rows(const void* X, int type, uint16_t* Y, float* row_mul, int M, int N,
                            void* stream) {
  const char* who = "mm_grad_rows";
  MM_CHECK_ARG(type >= 0 && type <= 2, "%s: type=%d must be 0 (fp32), 1 (fp16) or 2 (bf16)", who,
               type);
  MM_CHECK_ARG(M >= 0 && N > 0 && N % 8 == 0, "%s: bad shape M=%d N=%d (N %% 8 == 0)", who, M, N);
  MM_CHECK_ARG((((uintptr_t)X | (uintptr_t)Y) & 15) == 0 && ((uintptr_t)row_mul & 3) == 0,
               "%s: X and Y must be 16-byte aligned", who);
  if (M == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
  switch (type) {
    case 0: hipLaunchKernelGGL(k_grad_rows<0>, dim3(M), dim3(RW_NT), 0, st, X, (f16*)Y, row_mul, N); break;
    case 1: hipLaunchKernelGGL(k_grad_rows<1>, dim3(M), dim3(RW_NT), 0, st, X, (f16*)Y, row_mul, N); break;
    default: hipLaunchKernelGGL(k_grad_rows<2>, dim3(M), dim3(RW_NT), 0, st, X, (f16*)Y, row_mul, N);
  }
  MM_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int mm_swiglu_grad(const void* dH, int type, const uint16_t* gate_up, uint16_t* Y,
                              float* row_mul, int M, int N, void* stream) {
  const char* who = "mm_swiglu_grad";
  MM_CHECK_ARG(type >= 0 && type <= 2, "%s: type=%d must be 0 (fp32), 1 (fp16) or 2 (bf16)", who,
               type);
  MM_CHECK_ARG(M >= 0 && N > 0 && N % 8 == 0, "%s: bad shape M=%d N=%d (N %% 8 == 0)", who, M, N);
  MM_CHECK_ARG((((uintptr_t)dH | (uintptr_t)gate_up | (uintptr_t)Y) & 15) == 0 &&
                   ((uintptr_t)row_mul & 3) == 0,
               "%s: dH, gate_up and Y must be 16-byte aligned", who);
  if (M == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
#define MM_SG(T) hipLaunchKernelGGL(k_swiglu_grad<T>, dim3(M), dim3(RW_NT), 0, st, dH, (const f16*)gate_up, (f16*)Y, row_mul, N)
  if (type == 0) MM_SG(0);
  else if (type == 1) MM_SG(1);
  else MM_SG(2);
#undef MM_SG
  MM_CHECK_LAUNCH(who);
  return 0;
}
