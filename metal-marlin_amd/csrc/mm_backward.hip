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
// k_swiglu_grad): a row's largest finite value lands in [2^14, 2^15), so what is lost lies
// 2^-40 below it, and the power of two is taken out of the fp32 sums exactly.  11 bits of each
// value are held: all of a bf16 one's 8, and of fp32 ones and the pair's dg and du the nearest
// (a second fp16 term of each would double the matrix work; the fp16 gradients of the gated
// block are off by 1.4 times the half step that the result's own rounding costs, bf16 ones by
// no more than that).
#include <algorithm>

#include "mm_common.h"
#include "mm_prefill.h"
#include "mmfp4.h"

namespace {
using namespace mmpf;

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
// all-ones exponent into the sign bit, which the shift spreads.  (Written in C, the shift
// becomes compares and selects, three times the instructions.)
MM_DEV f16x2 sanitize2(f16x2 s) {
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const uint32_t u = __builtin_bit_cast(uint32_t, s);
  const s16x2 e = __builtin_bit_cast(s16x2, u & 0x7c007c00u) + s16x2{0x0400, 0x0400};
  uint32_t m;
  asm("v_pk_ashrrev_i16 %0, 15, %1 op_sel_hi:[0,1]" : "=v"(m) : "v"(__builtin_bit_cast(uint32_t, e)));
  return __builtin_bit_cast(f16x2, u & ~m);
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
// The product, many rows.  Tiles of BM = 32 * RB * WM rows x 256 columns (k); waves
// (wk, wm, wn): wn takes of every word row's 8 columns the four 4 wn + j, so a wave's tile is
// 32 * RB rows x 128 columns: lane l32 holds columns 8 (kp0 + l32) + 4 wn + j.  WK = 4 waves
// share out the 16-n steps of every chunk and add up in LDS at the end: four times the waves
// for a tile of 64 rows, with no weight converted more often.  Operands go global -> LDS
// directly, STAGES - 1 chunks of BN n ahead:
//   A  piece (r, c), 8 halves, at r * BN/8 + (c ^ sw(r)), sw = (r >> 1) & 7 (BN = 64) or
//      r & 15: the 16 lanes of a read pass hit all banks
//   B  Marlin: 32 word rows x BN words, piece (row, p), 4 words, at row * BN/4 +
//      (p ^ (row & 15)); ROWS: BN n x 32 words as they lie
//   S, Z  SR group rows x BN halves: the groups that the tile's 256 k touch
// ks > 1: the chunks are split over gridDim.z and the last block of a tile adds the splits
// in order (k_mid's hand-off: sc1 partials, an arrival counter per tile left at zero).
// ot: the output's type, 0 fp32, 1 fp16, 2 bf16.
// ---------------------------------------------------------------------------
// LDS of a block of NW waves that takes BM rows x KPT word rows (8 k each) in chunks of BN n,
// and its loads.  RED: bytes of the sum over its waves at the end, in the same place.
template <bool INT4, int NW, int BM_, int KPT, int SR, int BN, int STG, int RED>
struct GradShape {
  static constexpr int STAGES = STG, BM = BM_;
  static constexpr int NWAVE = NW, NTHR = 64 * NWAVE;
  static constexpr int A_PIECES = BM * BN / 8, B_PIECES = KPT * BN / 4, S_PIECES = SR * BN / 8;
  static constexpr int A_IT = A_PIECES / NTHR, B_IT = B_PIECES / NTHR;
  static constexpr int S_IT = (S_PIECES + NTHR - 1) / NTHR;
  static_assert(A_PIECES % NTHR == 0 && B_PIECES % NTHR == 0 && S_PIECES % 64 == 0, "split");
  static constexpr int LOADS = A_IT + B_IT + S_IT * (INT4 ? 2 : 1);
  static constexpr int A_BYTES = A_PIECES * 16, B_BYTES = B_PIECES * 16, S_BYTES = S_PIECES * 16;
  static constexpr int B_OFF = STAGES * A_BYTES, S_OFF = B_OFF + STAGES * B_BYTES;
  static constexpr int Z_OFF = S_OFF + STAGES * S_BYTES;
  static constexpr int D_OFF = Z_OFF + (INT4 ? STAGES * S_BYTES : 0);   // dump of idle waves
  static constexpr int LDS_BYTES = D_OFF + 1024 > RED ? D_OFF + 1024 : RED;
  static_assert(LDS_BYTES <= 160 * 1024, "LDS");
};

// The tile of a block, walked as in k_prefill2: an XCD takes a run of tiles, groups of grp row
// tiles column by column.
struct GradTile {
  int bx, by, bz;
};
MM_DEV GradTile grad_tile(int grp) {
  const int nx = gridDim.x, ny = gridDim.y, ntile = nx * ny * gridDim.z;
  const int L = blockIdx.x + nx * (blockIdx.y + ny * blockIdx.z);
  const int xq = ntile >> 3, xr = ntile & 7, xcd = L & 7;
  const int lin = xcd * xq + min(xcd, xr) + (L >> 3);
  const int bz = lin / (nx * ny), lt = lin - bz * (nx * ny);
  const int gi = lt / (grp * nx), gw = lt - gi * (grp * nx);
  const int gr = min(grp, ny - gi * grp);
  return GradTile{gw / gr, gi * grp + gw % gr, bz};
}

// The chunks of a tile on their way to LDS.  Byte offsets of a lane's pieces from bases that
// are uniform: within a segment only the bases move from chunk to chunk, in scalar registers.
template <typename Sh, bool INT4, bool ROWS, int KPT, int BN>
struct GradFeed {
  static constexpr int PA = BN / 8, PB = BN / 4;   // pieces per row of A, of B
  static constexpr int PR = KPT / 4;               // pieces per n of row-packed words
  const GradSegs& segs;
  char* smem;
  int wave, lane, M, KP, ngroups, m0, kp0, g0;
  uint32_t a_off[Sh::A_IT], b_off[Sh::B_IT], s_src[Sh::S_IT];
  const f16* a_base;
  const uint32_t* b_base;
  const f16 *s_base, *z_base;
  int seg_n, seg_n0, seg_next;   // columns of the segment, the chunk's first, its last chunk

  MM_DEV static int aswz(int r) { return BN == 64 ? (r >> 1) & 7 : r & 15; }
  MM_DEV int piece(int i) const { return (i * Sh::NWAVE + wave) * 64 + lane; }
  // n of a row-packed piece.  Tiles of 16 word rows: the four n that the quarters of a wave
  // read together (8 apart) lie side by side, 256 bytes.
  MM_DEV static int rows_n(int p) {
    const int n = p / PR;
    return KPT == 16 ? (n & ~31) | (n & 3) << 3 | (n >> 2 & 7) : n;
  }

  MM_DEV void enter(int ch) {   // chunk ch opens a segment, or the block's range
    const int sg = ch >= segs.s[2].ch0 ? 2 : (ch >= segs.s[1].ch0 ? 1 : 0);
    const GradSeg& s = segs.s[sg];
    const int N = s.N, n0 = (ch - s.ch0) * BN;
    seg_n = N;
    seg_n0 = n0;
    seg_next = sg < 2 ? segs.s[sg + 1].ch0 : 0x7fffffff;
    a_base = s.A + (size_t)m0 * s.lda + n0;
    b_base = ROWS ? s.B + (size_t)n0 * KP + kp0 : s.B + (size_t)kp0 * N + n0;
    s_base = s.S + (size_t)g0 * N + n0;
    if constexpr (INT4) z_base = s.Z + (size_t)g0 * N + n0;
#pragma unroll
    for (int i = 0; i < Sh::A_IT; ++i) {
      const int p = piece(i), r = p / PA;
      a_off[i] = (uint32_t)(min(r, M - 1 - m0) * s.lda + 8 * ((p % PA) ^ aswz(r))) * 2u;
    }
#pragma unroll
    for (int i = 0; i < Sh::B_IT; ++i) {
      const int p = piece(i);
      if constexpr (ROWS)
        b_off[i] = ((uint32_t)rows_n(p) * KP + min(4 * (p % PR), KP - 4 - kp0)) * 4u;
      else
        b_off[i] = ((uint32_t)min(p / PB, KP - 1 - kp0) * N + 4 * ((p % PB) ^ (p / PB & 15))) * 4u;
    }
#pragma unroll
    for (int i = 0; i < Sh::S_IT; ++i) {
      const int p = min(piece(i), Sh::S_PIECES - 1);
      s_src[i] = ((uint32_t)min(p / PA, ngroups - 1 - g0) * N + 8 * (p % PA)) * 2u;
    }
  }
  // A segment's last chunk may reach past its columns: zeros for the gradient, any of the
  // matrix's own words and scales.  (In two forms, so that the common one adds 32-bit offsets
  // to scalar bases.)
  MM_DEV void issue(int st) {
    if (seg_n0 + BN > seg_n) load<true>(st);
    else load<false>(st);
  }
  template <bool TAIL>
  MM_DEV void load(int st) {
#pragma unroll
    for (int i = 0; i < Sh::A_IT; ++i) {
      const char* src = (const char*)a_base + a_off[i];
      if constexpr (TAIL) {
        const int p = piece(i);
        if (seg_n0 + 8 * ((p % PA) ^ aswz(p / PA)) >= seg_n) src = (const char*)gr_zeros;
      }
      gl2lds16(src, smem + st * Sh::A_BYTES + (i * Sh::NWAVE + wave) * 1024);
    }
#pragma unroll
    for (int i = 0; i < Sh::B_IT; ++i) {
      const char* src = (const char*)b_base + b_off[i];
      if constexpr (TAIL) {
        const int p = piece(i);
        const int over = ROWS ? seg_n0 + rows_n(p) - (seg_n - 1)
                              : seg_n0 + 4 * ((p % PB) ^ (p / PB & 15)) - (seg_n - 4);
        if (over > 0) src -= (size_t)over * (ROWS ? KP : 1) * 4;
      }
      gl2lds16(src, smem + Sh::B_OFF + st * Sh::B_BYTES + (i * Sh::NWAVE + wave) * 1024);
    }
#pragma unroll
    for (int i = 0; i < Sh::S_IT; ++i) {
      const int wp = i * Sh::NWAVE + wave;
      const uint32_t off = s_src[i];
      size_t back = 0;
      if constexpr (TAIL) {
        const int p = min(wp * 64 + lane, Sh::S_PIECES - 1);
        back = (size_t)max(0, seg_n0 + 8 * (p % PA) - (seg_n - 8)) * 2;
      }
      const bool live = wp * 64 < Sh::S_PIECES;
      gl2lds16((const char*)s_base - back + off,
               smem + (live ? Sh::S_OFF + st * Sh::S_BYTES + wp * 1024 : Sh::D_OFF));
      if constexpr (INT4)
        gl2lds16((const char*)z_base - back + off,
                 smem + (live ? Sh::Z_OFF + st * Sh::S_BYTES + wp * 1024 : Sh::D_OFF));
    }
  }
  MM_DEV void advance(int ch) {   // to chunk ch, the next one
    if (ch >= seg_next) {
      enter(ch);
      return;
    }
    seg_n0 += BN;
    a_base += BN;
    b_base += ROWS ? (size_t)BN * KP : BN;
    s_base += BN;
    if constexpr (INT4) z_base += BN;
  }
  // The first STAGES chunks of [beg, end).
  MM_DEV void start(int beg, int end) {
    enter(beg);
    issue(0);
#pragma unroll
    for (int c = 1; c < Sh::STAGES; ++c) {
      if (beg + c < end) advance(beg + c);
      issue(c);
    }
  }
};

MM_DEV uint32_t bf16_bits(float v) {
  return __builtin_bit_cast(uint16_t, (__bf16)v);
}
// Four adjacent columns of a row.
MM_DEV void store_grad4(void* out, int ot, size_t at, f32x4 v) {
  if (ot == 1) {
    *(f16x4*)((f16*)out + at) = f16x4{(f16)v[0], (f16)v[1], (f16)v[2], (f16)v[3]};
  } else if (ot == 2) {
    *(u32x2*)((uint16_t*)out + at) =
        u32x2{bf16_bits(v[0]) | bf16_bits(v[1]) << 16, bf16_bits(v[2]) | bf16_bits(v[3]) << 16};
  } else {
    *(f32x4*)((float*)out + at) = v;
  }
}

// The hand-off's second half: true in the block that arrives last at the tile's counter.
MM_DEV bool grad_last(uint32_t* counter, int ks, uint32_t* s_last) {
  __builtin_amdgcn_s_waitcnt(0);   // this wave's partials have reached the coherence point
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t prev =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *s_last = prev == (uint32_t)ks - 1u;
    if (*s_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *s_last != 0;
}

// Gradient values as the operands hold them: sanitised scales, negated clamped zero points.
template <bool INT4>
MM_DEV void grad_scales(f16x8 s, f16x8 z, f16x2 (&s2)[4], f16x2 (&nz2)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s2[i] = sanitize2(f16x2{s[2 * i], s[2 * i + 1]});
    nz2[i] = f16x2{0, 0};
    if constexpr (INT4) {
      const f16x2 lim = {(f16)127.0f, (f16)127.0f};
      nz2[i] = -__builtin_elementwise_min(
          __builtin_elementwise_max(f16x2{z[2 * i], z[2 * i + 1]}, -lim), lim);
    }
  }
}

template <bool INT4, int WM, int WK, int RB, int SR, int BN, int STG>
using GradTall = GradShape<INT4, 2 * WM * WK, 32 * RB * WM, GR_KP, SR, BN, STG,
                           (WK > 1 ? 2 * WM * WK * 4096 : 0)>;   // one (rb, j) of the sum

template <bool INT4, bool ROWS, int WM, int WK, int RB, int SR, int BN, int STG>
__global__ void __launch_bounds__(WM * WK * 128)
k_grad(GradSegs segs, void* __restrict__ out, int ot, const float* __restrict__ rowmul, int M,
       int K, int g, int cps, int grp, float* __restrict__ part, uint32_t* __restrict__ counters) {
  using Sh = GradTall<INT4, WM, WK, RB, SR, BN, STG>;
  static_assert(WK == 1 || WK == 4, "a wave owns all or one of the four row quads");
  constexpr int STAGES = Sh::STAGES;
  constexpr int STEPS = BN / 16 / WK;          // steps per wave and chunk
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS_BYTES];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave & 1, wm = (wave >> 1) % WM, wk = (wave >> 1) / WM;
  const int l32 = lane & 31, h = lane >> 5;
  const int KP = K >> 3;
  const auto [bx, by, bz] = grad_tile(grp);
  const int m0 = by * Sh::BM, kp0 = bx * GR_KP;
  const int c_beg = bz * cps, c_end = min(segs.nch, c_beg + cps);
  const int g0 = 8 * kp0 / g;              // first group of the tile
  GradFeed<Sh, INT4, ROWS, GR_KP, BN> feed{segs, smem, wave, lane, M, KP, K / g, m0, kp0, g0};

  f32x16 acc[RB][4];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[rb][j][v] = 0.0f;

  feed.start(c_beg, c_end);

  const int arow = wm * 32 * RB + l32, ax = feed.aswz(arow);   // rows of all row blocks share ax
  const int srow = 8 * min(kp0 + l32, KP - 1) / g - g0;
  const uint32_t half = wn ? 0x07060302u : 0x05040100u;
  const uint32_t s_off = srow * (BN * 2) + h * 16;
  const uint32_t b_row = ROWS ? (h * 8 * 32 + l32) * 4 : l32 * (BN * 4), bx15 = l32 & 15;

  f16x8 af[2][RB], bq[2][4];
  u32x4 w[2];
  f16x8 sv, zv;
  // Step t0 of this wave in the chunk at stage st: operands of the gradient, words and scales.
  auto frag = [&](auto stc, int t0, int slot) {
    constexpr int st = decltype(stc)::value;
    const int t = wk * STEPS + t0;
    if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2][i & 3] = *(const uint32_t*)(smem + Sh::B_OFF + st * Sh::B_BYTES + b_row +
                                              (16 * t + i) * 128);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = *(const u32x4*)(smem + Sh::B_OFF + st * Sh::B_BYTES + b_row +
                               ((4 * t + 2 * h + i) ^ bx15) * 16);
    }
    sv = *(const f16x8*)(smem + Sh::S_OFF + st * Sh::S_BYTES + s_off + t * 32);
    if constexpr (INT4) zv = *(const f16x8*)(smem + Sh::Z_OFF + st * Sh::S_BYTES + s_off + t * 32);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      af[slot][rb] = *(const f16x8*)(smem + st * Sh::A_BYTES + (arow + 32 * rb) * (BN * 2) +
                                     ((2 * t + h) ^ ax) * 16);
  };
  auto decode = [&](int slot) {
    f16x2 s2[4], nz2[4];
    grad_scales<INT4>(sv, zv, s2, nz2);
    PairWords<INT4>::run(w, s2, nz2, half, bq[slot]);
  };
  // A step is read and converted while the one before it occupies the matrix cores, across
  // chunks too: before a chunk's last step every wave has read that chunk, so its stage is
  // refilled there and the next one, which has landed once at most STAGES - 2 later ones are
  // outstanding, is published by the same barrier.
  auto chunk = [&](int ch, auto stc) {
    constexpr int st = decltype(stc)::value;
#pragma unroll
    for (int t = 0; t < STEPS; ++t) {
      const int cur = t & 1;
      if (t + 1 < STEPS) {
        frag(stc, t + 1, cur ^ 1);
      } else {
        __builtin_amdgcn_s_waitcnt(0xc07f);            // lgkmcnt(0): this wave's reads are done
        wait_vmcnt<(STAGES - 2) * Sh::LOADS>();
        __builtin_amdgcn_s_barrier();
        if (ch + STAGES < c_end) feed.advance(ch + STAGES);
        feed.issue(st);                                // behind the last chunk: again, never read
        frag(std::integral_constant<int, (st + 1) % STAGES>{}, 0, cur ^ 1);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          acc[rb][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(af[cur][rb], bq[cur][j], acc[rb][j],
                                                              0, 0, 0);
      decode(cur ^ 1);
#pragma unroll
      for (int i = 0; i < RB * 4; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                    // MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, MM_PF2_SCHED_DS, 0);      // DS read
        __builtin_amdgcn_sched_group_barrier(0x002, MM_PF2_SCHED_VALU, 0);    // VALU
      }
    }
  };
  static_assert(STEPS % 2 == 0, "the operand slots alternate within a chunk");
  wait_vmcnt<(STAGES - 1) * Sh::LOADS>();
  __builtin_amdgcn_s_barrier();
  frag(std::integral_constant<int, 0>{}, 0, 0);
  decode(0);
  for (int ch = c_beg; ch < c_end; ch += STAGES) {
    static_for(
        [&](auto stc) {
          constexpr int st = decltype(stc)::value;
          if (st == 0 || ch + st < c_end) chunk(ch + st, stc);
        },
        std::make_integer_sequence<int, STAGES>{});
  }
  wait_vmcnt<0>();

  // own[rb][j][q]: rows 8 (q0 + q) + 4 h + i of row block rb.  WK = 4: wave wk sums quad wk
  // of the four waves that share its tile, in their order.
  constexpr int NQ = 4 / WK;
  const int q0 = WK == 1 ? 0 : wk;
  f32x4 own[RB][4][NQ];
  if constexpr (WK == 1) {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          own[rb][j][q] = f32x4{acc[rb][j][4 * q], acc[rb][j][4 * q + 1], acc[rb][j][4 * q + 2],
                                acc[rb][j][4 * q + 3]};
  } else {
    f32x4* red = (f32x4*)smem;   // [wk][wm, wn][quad][lane]
    const int wt = wave % (2 * WM);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q)
          red[(wave * 4 + q) * 64 + lane] = f32x4{acc[rb][j][4 * q], acc[rb][j][4 * q + 1],
                                                  acc[rb][j][4 * q + 2], acc[rb][j][4 * q + 3]};
        __syncthreads();
        own[rb][j][0] = red[(wt * 4 + wk) * 64 + lane];
#pragma unroll
        for (int w = 1; w < WK; ++w) own[rb][j][0] += red[((w * 2 * WM + wt) * 4 + wk) * 64 + lane];
      }
  }
  const int ks = gridDim.z;
  if (ks > 1) {
    const int tile = by * gridDim.x + bx;
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(part + (size_t)tile * ks * (Sh::BM * GR_COLS));
    auto at = [&](int z, int rb, int j, int q) {
      return 16u * (uint32_t)((((z * RB + rb) * 4 + j) * NQ + q) * Sh::NTHR + tid);
    };
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int q = 0; q < NQ; ++q) store_agent_x4(prs, at(bz, rb, j, q), own[rb][j][q]);
    // The flag lies in smem: a second LDS variable would have the compiler wait for every
    // load to LDS before the reads of the main loop (M = 512, 4096 -> 4096 2 ways 40 us, 35 so).
    if (!grad_last(counters + tile, ks, (uint32_t*)smem)) return;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) own[rb][j][q] = f32x4{0, 0, 0, 0};
        for (int z = 0; z < ks; z += 4) {
          f32x4 ld[4][NQ];
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < NQ; ++q) ld[i][q] = load_agent_x4(prs, at(min(z + i, ks - 1), rb, j, q));
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (z + i < ks)
#pragma unroll
              for (int q = 0; q < NQ; ++q) own[rb][j][q] += ld[i][q];
        }
      }
  }
  const int kp = kp0 + l32;
  if (kp >= KP) return;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb)
#pragma unroll
    for (int q = 0; q < NQ; ++q)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = m0 + wm * 32 * RB + rb * 32 + 8 * (q0 + q) + 4 * h + i;
        if (row >= M) continue;
        const float f = rowmul != nullptr ? rowmul[row] : 1.0f;
        store_grad4(out, ot, (size_t)row * K + 8 * kp + 4 * wn,
                    f * f32x4{own[rb][0][q][i], own[rb][1][q][i], own[rb][2][q][i],
                              own[rb][3][q][i]});
      }
}

// ---------------------------------------------------------------------------
// The product, 33 rows up: tiles of 64 rows x 128 columns (16 word rows), 16x16x32 MFMA.  Lane
// (c, q): columns 8 (kp0 + c) + j of word row kp0 + c, gradient rows 16 rb + c, n 8 q .. + 7
// of a step of 32.  A chunk has one step for each of the 8 waves, so every word and every
// gradient value is read from LDS once, and the waves add up in LDS at the end.  While the
// matrix cores take one half of a step's columns, the other half of the next operands is
// converted.  ks > 1: as in k_grad.
//
// Against tiles of 64 x 256: half the columns leave no split to be joined up to 512 rows of K =
// 4096, and every weight costs 1.6 VALU operations (2.0 there, where a wave converts half
// words).  M = 512, 4096 -> 4096: 24.4 us, 700 TFLOP/s (34 there).  A chunk takes 1.27 us, of
// which the matrix cores are busy 0.43: the two waves of a SIMD wait a third of the time for
// each other, and what they issue does not overlap fully.  Reading the next operands before
// the first half (double words) spills and gains nothing.
// ---------------------------------------------------------------------------
constexpr int GN_KP = 16, GN_COLS = 8 * GN_KP, GN_BM = 64, GN_NW = 8, GN_BN = 32 * GN_NW;
constexpr int GN_NTHR = 64 * GN_NW, GN_RED = GN_NW * 2 * 16 * GN_COLS * 4;   // two row blocks

template <bool INT4, int SR, int STG>
using GradNarrow = GradShape<INT4, GN_NW, GN_BM, GN_KP, SR, GN_BN, STG, GN_RED>;

template <bool INT4, bool ROWS, int SR, int STG>
__global__ void __launch_bounds__(GN_NTHR)
k_grad_narrow(GradSegs segs, void* __restrict__ out, int ot, const float* __restrict__ rowmul,
              int M, int K, int g, int cps, int grp, float* __restrict__ part,
              uint32_t* __restrict__ counters) {
  using Sh = GradNarrow<INT4, SR, STG>;
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS_BYTES];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KP = K >> 3;
  const auto [bx, by, bz] = grad_tile(grp);
  const int m0 = by * GN_BM, kp0 = bx * GN_KP;
  const int c_beg = bz * cps, c_end = min(segs.nch, c_beg + cps);
  const int g0 = 8 * kp0 / g;
  GradFeed<Sh, INT4, ROWS, GN_KP, GN_BN> feed{segs, smem, wave, lane, M, KP, K / g, m0, kp0, g0};
  f32x4 acc[4][8];
#pragma unroll
  for (int rb = 0; rb < 4; ++rb)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[rb][j] = f32x4{0, 0, 0, 0};
  feed.start(c_beg, c_end);

  const int srow = 8 * min(kp0 + c, KP - 1) / g - g0;
  const uint32_t s_off = srow * (GN_BN * 2) + (4 * wave + q) * 16;
  const uint32_t a_off = c * (GN_BN * 2) + ((4 * wave + q) ^ c) * 16;
  f16x8 af[2][4], bq[2][4];
  u32x4 w[2];
  f16x8 sv, zv;
  f16x2 s2[4], nz2[4];
  auto frag = [&](auto stc, int slot) __attribute__((always_inline)) {
    constexpr int st = decltype(stc)::value;
    if constexpr (ROWS) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        w[i >> 2][i & 3] = *(const uint32_t*)(smem + Sh::B_OFF + st * Sh::B_BYTES +
                                              (32 * wave + 4 * i + q) * 64 + c * 4);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        w[i] = *(const u32x4*)(smem + Sh::B_OFF + st * Sh::B_BYTES + c * (GN_BN * 4) +
                               ((8 * wave + 2 * q + i) ^ c) * 16);
    }
    sv = *(const f16x8*)(smem + Sh::S_OFF + st * Sh::S_BYTES + s_off);
    if constexpr (INT4) zv = *(const f16x8*)(smem + Sh::Z_OFF + st * Sh::S_BYTES + s_off);
#pragma unroll
    for (int rb = 0; rb < 4; ++rb)
      af[slot][rb] = *(const f16x8*)(smem + st * Sh::A_BYTES + a_off + rb * 16 * (GN_BN * 2));
  };
  // FP4: the even and the odd nibbles of neighbouring words in pairs, for both halves at once
  // (PairWords' e and o, without picking bytes first; 512 rows, 14336 -> 4096 77.2 us with it, 75.0
  // so).
  uint32_t eo[2][4];
  auto decode = [&](auto hfc) __attribute__((always_inline)) {
    constexpr int hf = decltype(hfc)::value;
    if (hf == 0) grad_scales<INT4>(sv, zv, s2, nz2);
    if constexpr (INT4) {
      PairWords<true>::run(w, s2, nz2, hf ? 0x07060302u : 0x05040100u, bq[hf]);
    } else {
      if (hf == 0) {
        const uint32_t m = sgpr_const(0x0f0f0f0fu);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          const uint32_t x = w[p >> 1][2 * (p & 1)], y = w[p >> 1][2 * (p & 1) + 1];
          eo[0][p] = (x & m) | ((y << 4) & ~m);
          eo[1][p] = ((x >> 4) & m) | (y & ~m);
        }
      }
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        u32x4 lo, hi;
#pragma unroll
        for (int p = 0; p < 4; ++p) {
          lo[p] = __builtin_bit_cast(uint32_t, e2m1_pair_c<2 * hf>(eo[o][p]) * s2[p]);
          hi[p] = __builtin_bit_cast(uint32_t, e2m1_pair_c<2 * hf + 1>(eo[o][p]) * s2[p]);
        }
        bq[hf][o] = __builtin_bit_cast(f16x8, lo);
        bq[hf][2 + o] = __builtin_bit_cast(f16x8, hi);
      }
    }
  };
  constexpr std::integral_constant<int, 0> first{};
  constexpr std::integral_constant<int, 1> second{};
  auto half = [&](int slot, int hf) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int rb = 0; rb < 4; ++rb)
        acc[rb][4 * hf + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(af[slot][rb], bq[hf][j],
                                                                     acc[rb][4 * hf + j], 0, 0, 0);
  };
  auto order = [] {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);   // MFMA
      __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);   // DS read
      __builtin_amdgcn_sched_group_barrier(0x002, 5, 0);   // VALU
    }
  };
  auto chunk = [&](int ch, auto stc, int cur) __attribute__((always_inline)) {
    constexpr int st = decltype(stc)::value;
    half(cur, 0);
    decode(second);
    order();
    // Every wave has read this chunk: its stage is refilled, and the next one, which has
    // landed once at most STAGES - 2 later ones are outstanding, is published.
    __builtin_amdgcn_s_waitcnt(0xc07f);            // lgkmcnt(0)
    wait_vmcnt<(STG - 2) * Sh::LOADS>();
    __builtin_amdgcn_s_barrier();
    if (ch + STG < c_end) feed.advance(ch + STG);
    feed.issue(st);                                // behind the last chunk: again, never read
    frag(std::integral_constant<int, (st + 1) % STG>{}, cur ^ 1);
    half(cur, 1);
    decode(first);
    order();
  };
  wait_vmcnt<(STG - 1) * Sh::LOADS>();
  __builtin_amdgcn_s_barrier();
  frag(std::integral_constant<int, 0>{}, 0);
  decode(first);
  // an even number of stages in a round, so that the operand slots are constants
  for (int ch = c_beg; ch < c_end; ch += 2 * STG) {
    static_for(
        [&](auto ic) __attribute__((always_inline)) {
          constexpr int i = decltype(ic)::value;
          if (i == 0 || ch + i < c_end)
            chunk(ch + i, std::integral_constant<int, i % STG>{}, i & 1);
        },
        std::make_integer_sequence<int, 2 * STG>{});
  }
  wait_vmcnt<0>();

  // The sum over the waves, two row blocks at a time: thread (wave, lane) owns row
  // 16 (2 t + wave / 4) + 4 q + wave % 4 and its 8 columns.
  f32x4 own[2][2];
  f32x4* red = (f32x4*)smem;   // [wave][row block][row of a lane][column half][lane]
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    __syncthreads();
#pragma unroll
    for (int rb = 0; rb < 2; ++rb)
#pragma unroll
      for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const f32x4(&a)[8] = acc[2 * t + rb];
          red[(((wave * 2 + rb) * 4 + v) * 2 + hf) * 64 + lane] =
              f32x4{a[4 * hf][v], a[4 * hf + 1][v], a[4 * hf + 2][v], a[4 * hf + 3][v]};
        }
    __syncthreads();
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      own[t][hf] = red[(wave * 2 + hf) * 64 + lane];
#pragma unroll
      for (int k = 1; k < GN_NW; ++k) own[t][hf] += red[((k * 8 + wave) * 2 + hf) * 64 + lane];
    }
  }
  const int ks = gridDim.z;
  if (ks > 1) {
    const int tile = by * gridDim.x + bx;
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(part + (size_t)tile * ks * (GN_BM * GN_COLS));
    auto at = [&](int z, int t, int hf) {
      return 16u * (uint32_t)(((z * 2 + t) * 2 + hf) * GN_NTHR + tid);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) store_agent_x4(prs, at(bz, t, hf), own[t][hf]);
    // the flag lies in smem for k_grad's reason
    if (!grad_last(counters + tile, ks, (uint32_t*)smem)) return;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) own[t][hf] = f32x4{0, 0, 0, 0};
    for (int z = 0; z < ks; z += 4) {
      f32x4 ld[4][2][2];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) ld[i][t][hf] = load_agent_x4(prs, at(min(z + i, ks - 1), t, hf));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (z + i < ks)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) own[t][hf] += ld[i][t][hf];
    }
  }
  if (kp0 + c >= KP) return;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int row = m0 + 16 * (2 * t + (wave >> 2)) + 4 * q + (wave & 3);
    if (row >= M) continue;
    const float f = rowmul != nullptr ? rowmul[row] : 1.0f;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
      store_grad4(out, ot, (size_t)row * K + 8 * (kp0 + c) + 4 * hf, f * own[t][hf]);
  }
}

// ---------------------------------------------------------------------------
// Up to 32 rows: the weights stream HBM -> registers -> 16x16x32 MFMA, as in mm_skinny.h.
// Tiles of 128 columns (16 word rows).  Lane (c, q) of a wave, at a step of 32 n: the words
// of n0 + 8 q .. + 7 of word row kp0 + c (two 16-byte loads: 16 rows x 128 bytes a wave), and
// the gradient's rows 16 mt + c at the same n; words give 8 operands, columns 8 (kp0 + c) + j.
// Converting the words costs 96 VALU operations per 2 KiB of them, a third of what the
// memory rate allows.  The NW waves of a block share out its steps, SPW at a time with all
// loads in flight, and add up in LDS; blocks that split the steps hand over as in k_grad, M
// rows each.
// ---------------------------------------------------------------------------
constexpr int GS_KP = 16, GS_COLS = 128, GS_NW = 8, GS_NTHR = 64 * GS_NW;

template <bool INT4, bool ROWS, int MT, int SPW>
__global__ void __launch_bounds__(GS_NTHR, MT == 1 ? 4 : 2)
k_grad_skinny(GradSegs segs, void* __restrict__ out, int ot, const float* __restrict__ rowmul,
              int M, int K, int g, int rounds, float* __restrict__ part,
              uint32_t* __restrict__ counters) {
  __shared__ __attribute__((aligned(16))) float red[GS_NW][16][GS_COLS];   // one row block
  __shared__ uint32_t s_last;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int KP = K >> 3, kp0 = blockIdx.x * GS_KP, kp = min(kp0 + c, KP - 1);
  const int grow = 8 * kp / g;
  f32x4 acc[MT][8];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[mt][j] = f32x4{0, 0, 0, 0};
  for (int r = 0; r < rounds; ++r) {
    const int st0 = ((blockIdx.y * rounds + r) * GS_NW + wave) * SPW;
    if (st0 >= segs.nch) break;
    u32x4 w[SPW][2];
    f16x8 sv[SPW], zv[SPW], a[SPW][MT];
#pragma unroll
    for (int i = 0; i < SPW; ++i) {
      const int st = min(st0 + i, segs.nch - 1);
      const int sg = st >= segs.s[2].ch0 ? 2 : (st >= segs.s[1].ch0 ? 1 : 0);
      const GradSeg& s = segs.s[sg];
      const int N = s.N, n = (st - s.ch0) * 32 + 8 * q, nc = min(n, N - 8);
      const size_t off = (size_t)grow * N + nc;
      sv[i] = *(const f16x8*)(s.S + off);
      if constexpr (INT4) zv[i] = *(const f16x8*)(s.Z + off);
      if constexpr (ROWS) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[i][k >> 2][k & 3] = __builtin_nontemporal_load(s.B + (size_t)(nc + k) * KP + kp);
      } else {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[i][k] = __builtin_nontemporal_load((const u32x4*)(s.B + (size_t)kp * N + nc + 4 * k));
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        // rows past M, columns past N and steps past the last: zeros
        const bool live = 16 * mt + c < M && n < N && st0 + i < segs.nch;
        a[i][mt] = live ? *(const f16x8*)(s.A + (size_t)(16 * mt + c) * s.lda + n)
                        : f16x8{0, 0, 0, 0, 0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int i = 0; i < SPW; ++i) {
      f16x2 s2[4], nz2[4];
      grad_scales<INT4>(sv[i], zv[i], s2, nz2);
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        f16x8 b[4];
        PairWords<INT4>::run(w[i], s2, nz2, hf ? 0x07060302u : 0x05040100u, b);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[mt][4 * hf + j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                a[i][mt], b[j], acc[mt][4 * hf + j], 0, 0, 0);
      }
    }
  }
  const int ks = gridDim.y, tile = blockIdx.x;
  const __amdgpu_buffer_rsrc_t prs = mm_rsrc(part + (size_t)tile * ks * M * GS_COLS);
  // Item (row, 4 columns) of the tile.
  auto finish = [&](int row, int c4, f32x4 v) {
    if (8 * kp0 + 4 * c4 < K)
      store_grad4(out, ot, (size_t)row * K + 8 * kp0 + 4 * c4,
                  (rowmul != nullptr ? rowmul[row] : 1.0f) * v);
  };
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (mt > 0) __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (16 * mt + 4 * q + i < M)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
          *(f32x4*)&red[wave][4 * q + i][8 * c + 4 * hf] =
              f32x4{acc[mt][4 * hf][i], acc[mt][4 * hf + 1][i], acc[mt][4 * hf + 2][i],
                    acc[mt][4 * hf + 3][i]};
    __syncthreads();
    const int items = min(16, M - 16 * mt) * (GS_COLS / 4);
    for (int e = tid; e < items; e += GS_NTHR) {
      const int row = e / (GS_COLS / 4), c4 = e % (GS_COLS / 4);
      f32x4 v = *(const f32x4*)&red[0][row][4 * c4];
#pragma unroll
      for (int k = 1; k < GS_NW; ++k) v += *(const f32x4*)&red[k][row][4 * c4];
      if (ks == 1) finish(16 * mt + row, c4, v);
      else store_agent_x4(prs, 4u * (uint32_t)((blockIdx.y * M + 16 * mt + row) * GS_COLS + 4 * c4), v);
    }
  }
  if (ks == 1 || !grad_last(counters + tile, ks, &s_last)) return;
  for (int e = tid; e < M * (GS_COLS / 4); e += GS_NTHR) {
    const int row = e / (GS_COLS / 4), c4 = e % (GS_COLS / 4);
    f32x4 v = {0, 0, 0, 0};
    for (int z0 = 0; z0 < ks; z0 += 8) {
      f32x4 ld[8];
#pragma unroll
      for (int z = 0; z < 8; ++z)
        ld[z] = load_agent_x4(prs, 4u * (uint32_t)((min(z0 + z, ks - 1) * M + row) * GS_COLS + 4 * c4));
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (z0 + z < ks) v += ld[z];
    }
    finish(row, c4, v);
  }
}

// ---------------------------------------------------------------------------
// Row conversion: fp16 values v * 2^e with the row's largest finite one in [2^14, 2^15), and
// rowmul[row] = 2^-e.
// ---------------------------------------------------------------------------
constexpr int RW_NT = 512;
constexpr int RW_HOLD = 4;      // 8-value pieces of a row that a thread keeps in registers

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
// The row's factor from largest(finite), its largest magnitude, of the finite values alone or of
// all: a non-finite value stays what it is and leaves the others theirs.  A row that has one
// is looked through twice, so that the others are spared the test of every value.  2^e is up
// to 2^149, so it comes as two factors, the second mostly 1.
struct RowScale {
  float mul, more;
};
template <typename F>
MM_DEV RowScale row_scale(F largest, float* rowmul) {
  float m = largest(std::false_type{});
  if (m == __builtin_inff()) {
    __syncthreads();            // every wave has the first maximum
    m = largest(std::true_type{});
  }
  const int e = carry_exponent(m);
  if (threadIdx.x == 0) rowmul[blockIdx.x] = ldexpf(1.0f, -e);
  return RowScale{ldexpf(1.0f, min(e, 126)), ldexpf(1.0f, max(0, e - 126))};
}
template <bool FINITE>
MM_DEV float max8(float m, const float (&v)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float a = fabsf(v[k]);
    m = !FINITE || a < __builtin_inff() ? fmaxf(m, a) : m;
  }
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
MM_DEV void store8(f16* p, const float (&v)[8], RowScale s) {
  f16x8 o;
  if (s.more == 1.0f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (f16)(v[i] * s.mul);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = (f16)(v[i] * s.mul * s.more);
  }
  *(f16x8*)p = o;
}

// A row's parts, from up to three matrices: pieces of 8 up to the end of each.
struct RowParts {
  const void* x[3];
  int end[3];
  template <int T>
  MM_DEV void load(int row, int p, float (&v)[8]) const {
    const int i = p < end[0] ? 0 : (p < end[1] ? 1 : 2), first = i > 0 ? end[i - 1] : 0;
    load8<T>(x[i], 8 * ((size_t)row * (end[i] - first) + (p - first)), v);
  }
};

// One block per row; up to RW_NT * 8 * RW_HOLD columns are read once, wider rows twice.
template <int T>
__global__ void __launch_bounds__(RW_NT)
k_grad_rows(RowParts parts, f16* __restrict__ Y, float* __restrict__ rowmul) {
  __shared__ float red[RW_NT / 64];
  const int row = blockIdx.x, np = parts.end[2];
  const size_t base = 8 * (size_t)row * np;
  float hold[RW_HOLD][8];
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) parts.load<T>(row, p, hold[i]);
  }
  auto largest = [&](auto finite) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < RW_HOLD; ++i)
      if (threadIdx.x + i * RW_NT < np) m = max8<finite.value>(m, hold[i]);
    for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
      float v[8];
      parts.load<T>(row, p, v);
      m = max8<finite.value>(m, v);
    }
    return block_max(m, red);
  };
  const RowScale scale = row_scale(largest, rowmul);
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) store8(Y + base + 8 * (size_t)p, hold[i], scale);
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float v[8];
    parts.load<T>(row, p, v);
    store8(Y + base + 8 * (size_t)p, v, scale);
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
  float hg[RW_HOLD][8], hu[RW_HOLD][8];
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) grads(p, hg[i], hu[i]);
  }
  auto largest = [&](auto finite) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < RW_HOLD; ++i)
      if (threadIdx.x + i * RW_NT < np)
        m = max8<finite.value>(max8<finite.value>(m, hg[i]), hu[i]);
    for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
      float dg[8], du[8];
      grads(p, dg, du);
      m = max8<finite.value>(max8<finite.value>(m, dg), du);
    }
    return block_max(m, red);
  };
  const RowScale scale = row_scale(largest, rowmul);
#pragma unroll
  for (int i = 0; i < RW_HOLD; ++i) {
    const int p = threadIdx.x + i * RW_NT;
    if (p < np) {
      store8(Y + gb + 8 * (size_t)p, hg[i], scale);
      store8(Y + gb + N + 8 * (size_t)p, hu[i], scale);
    }
  }
  for (int p = threadIdx.x + RW_HOLD * RW_NT; p < np; p += RW_NT) {
    float dg[8], du[8];
    grads(p, dg, du);
    store8(Y + gb + 8 * (size_t)p, dg, scale);
    store8(Y + gb + N + 8 * (size_t)p, du, scale);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
enum { G_SKINNY, G_NARROW, G_64, G_256 };
struct GradPlan {
  int kind;
  int bn;       // n per chunk (step of the skinny kernel)
  int bm, ks;   // rows per tile, splits
  int per;      // chunks per split, or rounds per block
  int spw;
  size_t part;  // partial sums, bytes
};

int grad_chunks(int nmat, const int* N, int bn) {
  int c = 0;
  for (int i = 0; i < nmat; ++i) c += mm_cdiv(N[i], bn);
  return c;
}

GradPlan plan_grad(int nmat, const int* N, int M, int K) {
  GradPlan p{};
  if (M <= 32) {
    p = GradPlan{G_SKINNY, 32, M, 1, 1, 4, 0};
    const int steps = grad_chunks(nmat, N, p.bn), tiles = mm_cdiv(K, GS_COLS);
    if ((long)tiles * mm_cdiv(steps, GS_NW * 4) < 256) p.spw = 2;
    const int blocks_n = mm_cdiv(steps, GS_NW * p.spw);
    p.ks = blocks_n;
    while (p.ks > 1 && ((long)tiles * p.ks > 1024 || p.ks > 32)) p.ks = mm_cdiv(p.ks, 2);
    if (tiles > GR_MAX_TILES) p.ks = 1;
    p.per = mm_cdiv(blocks_n, p.ks);
    p.ks = mm_cdiv(blocks_n, p.per);
    if (p.ks > 1) p.part = (size_t)tiles * p.ks * M * GS_COLS * sizeof(float);
    return p;
  }
  // The tile and the split by a time model (us; MI355X, FP4): rounds of 256 blocks, each its
  // start, a time per chunk (more where all CUs share the memory) and its end, and the
  // hand-off of a split.  Measured, K = 4096, 64 x 128 tiles / 64 x 256 / 256 x 256, each at its
  // best split: M = 64, N = 4096 16.3 (4 ways) / 23 / 82; M = 300 24 / 28 / 89; M = 512 25 / 34 /
  // 89, N = 14336 75 / 82 / 228; M = 1024, N = 4096 50 / 47 / 92; M = 2048 99 / 92 / 103, N =
  // 14336 - / 292 / 266; M = 4096, N = 4096 - / 183 / 147.
  // INT4 and row-packed words are planned by the same times, though their steps cost more: for
  // INT4, M = 300, N = 4096 the model has 24 where the kernel takes 31.
  struct { int kind, bm, cols, bn; double start, chunk, full, split, each; } const kinds[] = {
      {G_NARROW, GN_BM, GN_COLS, GN_BN, 3.6, 1.27, 1.27, 2.2, 1.25},
      {G_64, 64, GR_COLS, 128, 7.8, 1.05, 1.21, 7, 0},
      {G_256, 256, GR_COLS, 64, 16, 1.75, 2.05, 20, 0}};
  double best = 0;
  for (const auto& k : kinds) {
    const long tiles = (long)mm_cdiv(K, k.cols) * mm_cdiv(M, k.bm);
    const int nch = grad_chunks(nmat, N, k.bn);
    for (int ks = 1; ks <= 16 && ks <= nch && (ks == 1 || tiles <= GR_MAX_TILES); ++ks) {
      const int per = mm_cdiv(nch, ks);
      if (mm_cdiv(nch, per) != ks) continue;
      const long rounds = (tiles * ks + 255) / 256;
      const double us = rounds * (k.start + per * (tiles * ks > 192 ? k.full : k.chunk) +
                                  (ks > 1 ? k.split + ks * k.each : 0));
      if (best == 0 || us < best) {
        best = us;
        p = GradPlan{k.kind, k.bn, k.bm, ks, per, 0,
                     ks > 1 ? (size_t)tiles * ks * k.bm * k.cols * sizeof(float) : 0};
      }
    }
  }
  return p;
}

template <bool INT4, bool ROWS, int WM, int WK, int RB, int SR, int BN, int STG>
int launch_grad(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K, int g,
                const GradPlan& p, void* ws, hipStream_t st) {
  using Sh = GradTall<INT4, WM, WK, RB, SR, BN, STG>;
  const dim3 grid(mm_cdiv(K, GR_COLS), mm_cdiv(M, Sh::BM), p.ks);
  int grp = 1;
  while (grp * 2 <= (int)grid.y && grp < 4) grp *= 2;
  hipLaunchKernelGGL((k_grad<INT4, ROWS, WM, WK, RB, SR, BN, STG>), grid, dim3(Sh::NTHR), 0, st, s,
                     out, ot, rowmul, M, K, g, p.per, grp, (float*)((char*)ws + GR_COUNTER_BYTES),
                     (uint32_t*)ws);
  MM_CHECK_LAUNCH("gemm backward");
  return 0;
}

template <bool INT4, bool ROWS, int SR, int STG>
int launch_grad_narrow(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K,
                       int g, const GradPlan& p, void* ws, hipStream_t st) {
  const dim3 grid(mm_cdiv(K, GN_COLS), mm_cdiv(M, GN_BM), p.ks);
  int grp = 1;
  while (grp * 2 <= (int)grid.y && grp < 4) grp *= 2;
  hipLaunchKernelGGL((k_grad_narrow<INT4, ROWS, SR, STG>), grid, dim3(GN_NTHR), 0, st, s, out, ot,
                     rowmul, M, K, g, p.per, grp, (float*)((char*)ws + GR_COUNTER_BYTES),
                     (uint32_t*)ws);
  MM_CHECK_LAUNCH("gemm backward");
  return 0;
}

template <bool INT4, bool ROWS, int MT, int SPW>
int launch_grad_skinny(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K,
                       int g, const GradPlan& p, void* ws, hipStream_t st) {
  hipLaunchKernelGGL((k_grad_skinny<INT4, ROWS, MT, SPW>), dim3(mm_cdiv(K, GS_COLS), p.ks),
                     dim3(GS_NTHR), 0, st, s, out, ot, rowmul, M, K, g, p.per,
                     (float*)((char*)ws + GR_COUNTER_BYTES), (uint32_t*)ws);
  MM_CHECK_LAUNCH("gemm backward (few rows)");
  return 0;
}

// A tile's 256 k touch at most 8 groups from g = 32 up, 32 below.
template <bool INT4, bool ROWS>
int dispatch_grad(const GradSegs& s, void* out, int ot, const float* rowmul, int M, int K, int g,
                  const GradPlan& p, void* ws, hipStream_t st) {
#define MM_GRAD(...) return launch_grad<INT4, ROWS, __VA_ARGS__>(s, out, ot, rowmul, M, K, g, p, ws, st)
#define MM_GRAD_S(...) \
  return launch_grad_skinny<INT4, ROWS, __VA_ARGS__>(s, out, ot, rowmul, M, K, g, p, ws, st)
  if (p.kind == G_SKINNY) {
    if (M <= 16 && p.spw == 2) MM_GRAD_S(1, 2);
    if (M <= 16) MM_GRAD_S(1, 4);
    if (p.spw == 2) MM_GRAD_S(2, 2);
    MM_GRAD_S(2, 4);
  }
#define MM_GRAD_N(...) \
  return launch_grad_narrow<INT4, ROWS, __VA_ARGS__>(s, out, ot, rowmul, M, K, g, p, ws, st)
  if (p.kind == G_NARROW) {
    if (g >= 64) MM_GRAD_N(4, 3);
    if (g >= 32) MM_GRAD_N(8, INT4 ? 2 : 3);
    MM_GRAD_N(16, 2);
  }
  if (g >= 32) {
    if (p.kind == G_256) MM_GRAD(2, 1, 4, 8, 64, 3);
    MM_GRAD(1, 4, 2, 8, 128, 3);
  }
  if (p.kind == G_256) MM_GRAD(2, 1, 4, 32, 64, 3);
  MM_GRAD(1, 4, 2, 32, 128, 3);
#undef MM_GRAD_S
#undef MM_GRAD_N
#undef MM_GRAD
}

}  // namespace

extern "C" size_t mm_gemm_backward_workspace_bytes(int nmat, const int* N, int M, int K) {
  if (nmat < 1 || nmat > 3 || N == nullptr || M <= 0 || K <= 0) return GR_COUNTER_BYTES;
  for (int i = 0; i < nmat; ++i)
    if (N[i] <= 0) return GR_COUNTER_BYTES;
  return GR_COUNTER_BYTES + plan_grad(nmat, N, M, K).part;
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
  for (int i = 0; i < 3; ++i) {
    s.s[i].ch0 = 0x7fffffff;
    if (i >= nmat) continue;
    MM_CHECK_ARG(N[i] > 0 && N[i] % 8 == 0, "%s: N[%d]=%d must be a positive multiple of 8", who,
                 i, N[i]);
    MM_CHECK_ARG(ldc[i] >= N[i] && ldc[i] % 8 == 0,
                 "%s: ldc[%d]=%d must be a multiple of 8, at least N=%d", who, i, ldc[i], N[i]);
    s.s[i] = GradSeg{(const f16*)dC[i], B[i], (const f16*)S[i],
                     Z != nullptr ? (const f16*)Z[i] : nullptr, ldc[i], N[i], 0};
    al |= (uintptr_t)dC[i] | (uintptr_t)B[i] | (uintptr_t)S[i] |
          (Z != nullptr ? (uintptr_t)Z[i] : 0);
  }
  MM_CHECK_ARG((al & 15) == 0, "%s: every operand must be 16-byte aligned", who);
  MM_CHECK_ARG(M <= 64 * 65535, "%s: M=%d is too large", who, M);
  // the kernels address a tile (256 gradient rows, 32 word rows or 128 columns) with 32 bits
  for (int i = 0; i < nmat; ++i)
    MM_CHECK_ARG(ldc[i] < (1 << 22) && N[i] < (1 << 24) && (layout == 0 || K < (1 << 24)),
                 "%s: N[%d]=%d, ldc=%d, K=%d: rows are too long", who, i, N[i], ldc[i], K);
  if (M == 0) return 0;
  const GradPlan p = plan_grad(nmat, N, M, K);
  for (int i = 0; i < nmat; ++i) {
    s.s[i].ch0 = s.nch;
    s.nch += mm_cdiv(N[i], p.bn);
  }
  const size_t need = GR_COUNTER_BYTES + p.part;
  MM_CHECK_ARG(p.ks == 1 || (ws != nullptr && ws_bytes >= need),
               "%s: workspace of %zu bytes is smaller than the %zu required", who, ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  if (layout == 1)
    return dispatch_grad<false, true>(s, dA, out_type, row_mul, M, K, g, p, ws, st);
  if (Z != nullptr)
    return dispatch_grad<true, false>(s, dA, out_type, row_mul, M, K, g, p, ws, st);
  return dispatch_grad<false, false>(s, dA, out_type, row_mul, M, K, g, p, ws, st);
}

extern "C" int mm_grad_rows_multi(const void* const* X, int type, int nmat, const int* N,
                                  uint16_t* Y, float* row_mul, int M, void* stream) {
  const char* who = "mm_grad_rows";
  MM_CHECK_ARG(nmat >= 1 && nmat <= 3 && X != nullptr && N != nullptr,
               "%s: nmat=%d must be 1..3", who, nmat);
  MM_CHECK_ARG(type >= 0 && type <= 2, "%s: type=%d must be 0 (fp32), 1 (fp16) or 2 (bf16)", who,
               type);
  RowParts parts{};
  uintptr_t al = (uintptr_t)Y;
  long pieces = 0;
  for (int i = 0; i < 3; ++i) {
    if (i < nmat) {
      MM_CHECK_ARG(M >= 0 && N[i] > 0 && N[i] % 8 == 0,
                   "%s: bad shape M=%d N=%d (N %% 8 == 0)", who, M, N[i]);
      al |= (uintptr_t)X[i];
      parts.x[i] = X[i];
      pieces += N[i] / 8;
    }
    parts.end[i] = (int)pieces;
  }
  MM_CHECK_ARG(pieces < (1 << 28), "%s: rows are too long", who);
  MM_CHECK_ARG((al & 15) == 0 && ((uintptr_t)row_mul & 3) == 0,
               "%s: X and Y must be 16-byte aligned", who);
  if (M == 0) return 0;
  hipStream_t st = (hipStream_t)stream;
#define MM_GR(T) \
  hipLaunchKernelGGL(k_grad_rows<T>, dim3(M), dim3(RW_NT), 0, st, parts, (f16*)Y, row_mul)
  if (type == 0) MM_GR(0);
  else if (type == 1) MM_GR(1);
  else MM_GR(2);
#undef MM_GR
  MM_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int mm_grad_rows(const void* X, int type, uint16_t* Y, float* row_mul, int M, int N,
                            void* stream) {
  return mm_grad_rows_multi(&X, type, 1, &N, Y, row_mul, M, stream);
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
