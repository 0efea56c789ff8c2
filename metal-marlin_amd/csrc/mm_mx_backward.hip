// Input gradient of the MXFP4 product: dX[M, K] = dY[M, N] . W[N, K], W MXFP4 (mm_mx.h), straight
// through the rounding of x.
//
// The contraction runs along N, across the rows of W, whose scales change from row to row: the
// scaled matrix instructions cannot take them.  A quarter of every MXFP4 value is a bf16 number,
// though: 2 bits of E2M1, and magnitudes from 2^-130, a subnormal one, to 1.5 * 2^127.  (Of the
// values themselves those of scale codes 253 and 254 reach 1.5 * 2^129: infinities, which make NaNs
// of zeros of dY.)  So quarters of the weights are converted exactly, 64 rows of a stage at a time,
// into an LDS tile [n][k], from which ds_read_b64_tr_b16 takes columns as 32x32x16 operands, and the
// sums are multiplied by 4.  bf16 dY is multiplied as it is.  fp16 dY is, too, in stages whose
// quarters are normal fp16 numbers, as those of a trained matrix are; in others it is two bf16 terms
// (11 bits in 8 + 8).  fp32 is three (24 bits; what lies below 2^-133, bf16's smallest step, is cut
// off).  Products are exact, sums fp32, rounded once.
//
// Bound by LDS and the matrix cores in turn: a stage of a 128 x 256 tile reads 128 KiB of operands
// and writes 58, about 0.5 us, and multiplies for 0.43; it takes 1.2 where the last-level cache
// holds the operands (2048 x 14336 x 4096: 270 us of bf16, 0.89 PFLOP/s; 323 of fp16, 588 with two
// terms throughout; 1093 of fp32).  Where they come out of HBM (eight sets of operands in turn) bf16
// takes 326 us, 0.74 PFLOP/s.
#include <algorithm>

#include "mm_mx_gemm.h"
#include "mmfp4.h"

using namespace mmmx;

namespace {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// Pieces of dY past its last column.
__device__ __attribute__((aligned(16))) const uint32_t mx_zeros[4] = {0, 0, 0, 0};

// WK x WM waves of 32 KB x 32 MB each.  A stage is 128 bytes of every row of dY: BN = 64 columns
// (32 of fp32), and as many rows of W.  LDS holds three stages of dY, three of W's words and scales
// and two of converted weights: what is copied has two stages' time to arrive.
template <int T, int WK_, int WM_, int KB_, int MB_>
struct GradTile {
  static constexpr int WK = WK_, WM = WM_, KB = KB_, MB = MB_;
  static constexpr int WN = WK, NB = KB;                  // as the results' columns
  static constexpr int NWAVE = WK * WM, NTHR = NWAVE * 64;
  static constexpr int TK = WK * KB * 32, TM = WM * MB * 32;
  static constexpr int BN = 128 / kBytes<T>, STEPS = BN / 16;
  static constexpr int BLOCKS = BN * TK / 32;             // of W per stage
  static constexpr int A = TM * 128, B = BN * TK * 2;     // bytes of a stage of dY and of W in bf16
  static constexpr int WP = BLOCKS / 64, SP = (BLOCKS + 255) / 256;   // copies of words, of scales
  static constexpr int RAW = WP * 1024 + SP * 256;
  static constexpr int STAGES = 3 * (A + RAW) + 2 * B, OUT = NWAVE * 32 * (KB * 128 + 16);
  static constexpr int LDS = (STAGES > OUT ? STAGES : OUT) + 16;      // and which stages are wide
  static constexpr int IT = TM / 8 / NWAVE, WIT = (WP + NWAVE - 1) / NWAVE,
                       SIT = (SP + NWAVE - 1) / NWAVE;    // copies per wave and stage
  static constexpr int COPIES = IT + WIT + SIT;
  static constexpr int TERMS = T == BF16 ? 1 : (T == F16 ? 2 : 3);
  static_assert(TM % (8 * NWAVE) == 0 && NWAVE % 2 == 0 && BLOCKS <= NTHR && BLOCKS % 64 == 0,
                "copies per wave, blocks per thread");
};

struct Grad {
  const uint8_t *dY, *W, *S;
  void* out;           // dX, or (split) fp32 partial sums [splits, M, K]
  // ldy: row stride of dY; ks: of the scales, a multiple of 4; per: stages of a split
  int out_type, M, N, K, ldy, ks, stages, per;
};

// Columns n .. n + 7 of a row of dY as bf16 terms whose sum they are: each term is the leading 8
// bits of what the terms before it leave.  (Cut off, not rounded: the largest finite fp32 values
// stay finite.)  What is not finite lies in the first term alone.
template <int T>
MM_DEV void terms(const char* p0, const char* p1, bf16x8 (&t)[T == BF16 ? 1 : (T == F16 ? 2 : 3)]) {
  if constexpr (T == BF16) {
    t[0] = *(const bf16x8*)p0;
  } else {
    constexpr int TERMS = T == F16 ? 2 : 3;
    float v[8];
    if constexpr (T == F16) {
      const f16x8 h = *(const f16x8*)p0;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)h[i];
    } else {
      const f32x4 a = *(const f32x4*)p0, b = *(const f32x4*)p1;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = a[i] == a[i] ? a[i] : __builtin_nanf("");   // a NaN whose leading bits tell
        v[4 + i] = b[i] == b[i] ? b[i] : __builtin_nanf("");
      }
    }
#pragma unroll
    for (int s = 0; s < TERMS; ++s) {
      u32x4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[i] = __builtin_amdgcn_perm(u32_of(v[2 * i + 1]), u32_of(v[2 * i]), 0x07060302u);
      t[s] = __builtin_bit_cast(bf16x8, w);
      if (s + 1 < TERMS)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float rest = v[i] - f32_of(u32_of(v[i]) & 0xffff0000u);
          v[i] = rest == rest ? rest : 0.0f;
        }
    }
  }
}

// Weights 2 I, 2 I + 1 of a word as fp16 or bf16 under the scale s.
template <bool HALF, int I>
MM_DEV uint32_t two(uint32_t w, float s) {
  if constexpr (HALF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, s, I));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, I));
}
// The same as bf16 under a scale below 2^-127, the least that the conversion knows: the leading
// halves of fp32 products, which are multiples of 2^-130.
template <int I>
MM_DEV uint32_t two_small(uint32_t w, float s) {
  const f32x2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, I);
  return __builtin_amdgcn_perm(u32_of(v.y * s), u32_of(v.x * s), 0x07060302u);
}

template <class Sh, int T>
__global__ void __launch_bounds__(Sh::NTHR) k_mx_grad(Grad a, int gm, int gk) {
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Sh::WK, wk = wave % Sh::WK, l32 = lane & 31, h = lane >> 5;
  // each XCD takes a stretch of tiles, row tiles innermost: they share their weights
  const int total = gm * gk, q = total >> 3, rem = total & 7, xcd = blockIdx.x & 7;
  const int lin = xcd * q + min(xcd, rem) + (int)(blockIdx.x >> 3);
  const int m0 = lin % gm * Sh::TM, k0 = lin / gm * Sh::TK;
  const int u0 = blockIdx.y * a.per, u1 = min(a.stages, u0 + a.per);
  const int row_bytes = (a.N * kBytes<T> + 15) / 16 * 16;

  const uint8_t* src[Sh::IT];
#pragma unroll
  for (int i = 0; i < Sh::IT; ++i) {
    const int r = (i * Sh::NWAVE + wave) * 8 + lane / 8;
    src[i] = a.dY + (size_t)min(m0 + r, a.M - 1) * a.ldy * kBytes<T>;
  }
  const int at = 16 * ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7));
  // Stages past the last one: that one again, which nobody uses.
  auto issue_dy = [&](int v, int slot) {
    const int u = min(v, u1 - 1);
#pragma unroll
    for (int i = 0; i < Sh::IT; ++i) {
      const int b = u * 128 + at;
      copy16(b < row_bytes ? src[i] + b : (const uint8_t*)mx_zeros,
             smem + slot * Sh::A + (i * Sh::NWAVE + wave) * 1024);
    }
  };
  // Block b of a stage is block b % RB of row b / RB; rows past N meet zeros of dY, blocks past K
  // are not stored.
  constexpr int RB = Sh::TK / 32;
  char* const raw = smem + 3 * Sh::A;
  char* const conv = raw + 3 * Sh::RAW;
  auto issue_w = [&](int v, int slot) {
    const int u = min(v, u1 - 1);
#pragma unroll
    for (int i = 0; i < Sh::WIT; ++i) {      // waves to spare copy the last piece again
      const int c = min(i * Sh::NWAVE + wave, Sh::WP - 1), b = c * 64 + lane;
      const int n = min(u * Sh::BN + b / RB, a.N - 1);
      copy16(a.W + (size_t)n * (a.K / 2) + min(k0 / 2 + b % RB * 16, a.K / 2 - 16),
             raw + slot * Sh::RAW + c * 1024);
    }
#pragma unroll
    for (int i = 0; i < Sh::SIT; ++i) {
      const int c = min(i * Sh::NWAVE + wave, Sh::SP - 1), b = min((c * 64 + lane) * 4, Sh::BLOCKS - 4);
      const int n = min(u * Sh::BN + b / RB, a.N - 1);
      copy4(a.S + (size_t)n * a.ks + min(k0 / 32 + b % RB, a.ks - 4),
            raw + slot * Sh::RAW + Sh::WP * 1024 + c * 256);
    }
  };
  // Thread b converts block b.  [n][k] in 64-byte blocks, block c of row n at c ^ (n % 4): the 4
  // rows that a transposed read takes lie in different banks.
  const bool idle = Sh::BLOCKS != Sh::NTHR && tid >= Sh::BLOCKS;
  auto store = [&](u32x4 wv, uint32_t code, int half_of, auto half) __attribute__((always_inline)) {
    constexpr bool HALF = decltype(half)::value;
    if (idle) return;
    const int n = tid / RB, c = tid % RB;
    char* const d = conv + half_of * Sh::B + n * (Sh::TK * 2) + (c ^ (n & 3)) * 64;
    const float s = scale_of(max(code, 2u) - 2u);        // a quarter
    const uint32_t nan = !HALF && code == 255u ? 0x7fc07fc0u : 0u;
    // lanes of one round write all of the 16 pieces that banks tell apart
    const int turn = (tid >> 2) & 3;
    if (turn & 1) wv = u32x4{wv[1], wv[2], wv[3], wv[0]};
    if (turn & 2) wv = u32x4{wv[2], wv[3], wv[0], wv[1]};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t w = wv[j];
      lds_store16(d + 16 * ((j + turn) & 3), u32x4{two<HALF, 0>(w, s) | nan, two<HALF, 1>(w, s) | nan,
                                    two<HALF, 2>(w, s) | nan, two<HALF, 3>(w, s) | nan});
    }
    if (!HALF && code < 2u) {
      const float t = f32_of(0x00100000u << code);       // 2^-129, 2^-128
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = j == 0 ? wv[0] : (j == 1 ? wv[1] : (j == 2 ? wv[2] : wv[3]));
        lds_store16(d + 16 * ((j + turn) & 3), u32x4{two_small<0>(w, t), two_small<1>(w, t),
                                                     two_small<2>(w, t), two_small<3>(w, t)});
      }
    }
  };
  // A stage of fp16 dY is wide, two bf16 terms, if a quarter of one of its weights is no normal
  // fp16 number: 0.5 .. 6 times 2^-13 .. 2^13, or zeros under any scale but NaN.  Whoever finds one
  // leaves the stage's number in its half's word.
  int* const wide = (int*)(smem + Sh::LDS - 16);
  constexpr std::true_type HALF{};
  constexpr std::false_type BF{};
  const auto convert = [&](int u, int slot, int half_of) __attribute__((always_inline)) {
    const char* const r = raw + slot * Sh::RAW;
    const int b = min(tid, Sh::BLOCKS - 1);
    const u32x4 wv = *(const u32x4*)(r + b * 16);
    const uint32_t code = *(const uint8_t*)(r + Sh::WP * 1024 + b);
    if constexpr (T == F16) {
      const u32x4 m = wv & 0x77777777u;
      if (code - 116u > 26u && (code == 255u || (m.x | m.y | m.z | m.w) != 0u))
        lds_store4(wide + half_of, (uint32_t)u);
      stores_done();
      block_barrier();
      if (wide[half_of] != u) return store(wv, code, half_of, HALF);
    }
    store(wv, code, half_of, BF);
  };
  f32x16 acc[Sh::KB][Sh::MB];
#pragma unroll
  for (int k = 0; k < Sh::KB; ++k)
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[k][m][i] = 0.0f;

  // A transposed read: lane s of a group of 16 points at row s / 4, columns 4 (s % 4) on, of a
  // 4 x 16 block, and gets column s of it.  Groups 2 h + g take rows 8 h (+ 4) and columns 16 g.
  const int tr_n = 8 * h + (lane & 15) / 4, tr_c = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
  auto compute = [&](int slot, int half_of, auto half) __attribute__((always_inline)) {
    constexpr bool HALF = decltype(half)::value;
    const char* const dA = smem + slot * Sh::A;
    char* const dB = conv + half_of * Sh::B;
#pragma unroll
    for (int j = 0; j < Sh::STEPS; ++j) {
      bf16x8 wv[Sh::KB];
#pragma unroll
      for (int k = 0; k < Sh::KB; ++k) {
        s16x4 p[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = 16 * j + tr_n + 4 * i, c = wk * Sh::KB + k;
          p[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4)(dB + n * (Sh::TK * 2) + (c ^ (n & 3)) * 64 + tr_c * 2));
        }
        const short __attribute__((ext_vector_type(8))) both =
            __builtin_shufflevector(p[0], p[1], 0, 1, 2, 3, 4, 5, 6, 7);
        wv[k] = __builtin_bit_cast(bf16x8, both);
      }
#pragma unroll
      for (int m = 0; m < Sh::MB; ++m) {
        const int r = (wm * Sh::MB + m) * 32 + l32, sw = (r >> 1) & 7;
        const char* const row = dA + r * 128;
        if constexpr (HALF) {
          const f16x8 v = *(const f16x8*)(row + 16 * ((2 * j + h) ^ sw));
#pragma unroll
          for (int k = 0; k < Sh::KB; ++k)
            acc[k][m] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, wv[k]), v,
                                                               acc[k][m], 0, 0, 0);
          continue;
        }
        bf16x8 t[Sh::TERMS];
        if constexpr (T == F32)
          terms<T>(row + 16 * ((4 * j + 2 * h) ^ sw), row + 16 * ((4 * j + 2 * h + 1) ^ sw), t);
        else
          terms<T>(row + 16 * ((2 * j + h) ^ sw), nullptr, t);
#pragma unroll
        for (int k = 0; k < Sh::KB; ++k)
#pragma unroll
          for (int s = 0; s < Sh::TERMS; ++s)
            acc[k][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[k], t[s], acc[k][m], 0, 0, 0);
      }
    }
  };
  if (u0 < u1) {
    if (T == F16 && tid < 2) wide[tid] = -1;
    issue_w(u0, 0);
    issue_dy(u0, 0);
    issue_w(u0 + 1, 1);
    issue_dy(u0 + 1, 1);
    issue_w(u0 + 2, 2);
    wait_loads<2 * Sh::COPIES>();
    stores_done();
    block_barrier();
    convert(u0, 0, 0);
    int slot = 0, half_of = 0;
#pragma unroll 1
    for (int u = u0; u < u1; ++u) {
      // dY of this stage, words of the next and this stage's converted weights are there, and all
      // have done with the stage before
      wait_loads<Sh::COPIES>();
      stores_done();
      block_barrier();
      const int next = slot == 2 ? 0 : slot + 1;
      issue_dy(u + 2, next == 2 ? 0 : next + 1);
      issue_w(u + 3, slot);
      convert(u + 1, next, half_of ^ 1);
      if (T == F16 && wide[half_of] != u) compute(slot, half_of, HALF);
      else compute(slot, half_of, BF);
      slot = next;
      half_of ^= 1;
    }
    wait_loads<0>();
  }
#pragma unroll
  for (int k = 0; k < Sh::KB; ++k)
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[k][m][i] *= 4.0f;
  __syncthreads();
  const size_t base = blockIdx.y * sum_pitch((size_t)a.M * a.K);      // 0 unless split
  tile_out<Sh>(acc, smem, a.out, a.out_type, a.M - m0, k0, a.K,
               [=, K = a.K](int m) { return base + (size_t)(m0 + m) * K; });
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr size_t COUNTERS = 65536;

// Tiles of dX: a stage of the only block on a CU takes `one` us, of two that share it `two`, a
// block's beginning and end `ends` (bf16; measured at 64 .. 2048 rows of 14336 x 4096, 4096 x 14336
// and 4096 x 4096, operands in the last-level cache; fp16 takes 1.2 times as long, which changes no
// choice).
struct Cost {
  int tm, tk;
  float one, two, ends;
};
constexpr Cost COSTS[] = {{128, 256, 1.2f, 2.4f, 4.0f}, {64, 128, 0.83f, 1.15f, 2.5f},
                          {32, 128, 0.6f, 0.85f, 2.0f}};
constexpr int CUS = 256, MAX_SPLITS = 16;

struct Plan {
  int tile, splits, per, stages;
};
// With few tiles N is split, and the splits' sums are joined by another launch: 2.5 us and their
// bytes at about 3 TB/s.  us, best tile and split: 2048 x 14336 x 4096 270 (of 64 x 128 524, in two
// splits 298), 509 x 4096 x 4096 35 in four (unsplit 79), 128 x 4096 x 4096 22 (30 of 128 x 256).
Plan plan_of(int M, int N, int K, int type) {
  Plan best{0, 1, 0, mm_cdiv(N, type == F32 ? 32 : 64)};
  float least = 0;
  for (int t = 0; t < 3; ++t) {
    const Cost& c = COSTS[t];
    const long tiles = (long)mm_cdiv(M, c.tm) * mm_cdiv(K, c.tk);
    for (int s = 1; s <= MAX_SPLITS && (s == 1 || (tiles * s <= 2 * CUS && best.stages >= 2 * s)); ++s) {
      const int per = mm_cdiv(best.stages, s), splits = mm_cdiv(best.stages, per);
      const long blocks = tiles * splits, rest = blocks % (2 * CUS);
      float us = (float)(blocks / (2 * CUS)) * (per * c.two + c.ends);
      if (rest) us += per * (rest > CUS ? c.two : c.one) + c.ends;
      if (splits > 1) us += 2.5f + (float)M * K * 4 * (splits + 1) / 3e6f;
      if (least == 0 || us < least) {
        least = us;
        best.tile = t;
        best.splits = splits;
        best.per = per;
      }
    }
  }
  return best;
}

template <int T, class Sh>
void launch(Grad a, const Plan& p, hipStream_t st) {
  const int gm = mm_cdiv(a.M, Sh::TM), gk = mm_cdiv(a.K, Sh::TK);
  hipLaunchKernelGGL((k_mx_grad<Sh, T>), dim3((unsigned)(gm * gk), p.splits), dim3(Sh::NTHR), 0, st,
                     a, gm, gk);
}
template <int T>
void launch_t(const Grad& a, const Plan& p, hipStream_t st) {
  if (p.tile == 0) launch<T, GradTile<T, 4, 2, 2, 2>>(a, p, st);
  else if (p.tile == 1) launch<T, GradTile<T, 4, 2, 1, 1>>(a, p, st);
  else launch<T, GradTile<T, 4, 1, 1, 1>>(a, p, st);
}

// W's scales where they have to be laid out anew; the splits' sums.
struct Space {
  size_t part, total;
};
Space space_of(const Plan& p, int M, int N, int K) {
  Space s;
  const bool anew = scale_stride(K) != K / BLOCK;
  s.part = COUNTERS + (anew ? ((size_t)N * scale_stride(K) + 255) / 256 * 256 : 0);
  s.total = s.part + (p.splits > 1 ? p.splits * sum_pitch((size_t)M * K) * sizeof(float) : 0);
  if (s.total == COUNTERS) s.total = 0;
  return s;
}

}  // namespace

extern "C" size_t mm_mxfp4_gemm_backward_workspace_bytes(int M, int N, int K, int type) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return space_of(plan_of(M, N, K, type), M, N, K).total;
}

extern "C" int mm_mxfp4_gemm_backward(const void* dY, int type, int ldy, const uint32_t* W,
                                      const uint8_t* S, void* dX, int out_type, int M, int N, int K,
                                      void* ws, size_t ws_bytes, void* stream) {
  MM_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K % BLOCK == 0,
               "mm_mxfp4_gemm_backward: M=%d, N=%d, K=%d: K must be a positive multiple of %d", M, N,
               K, BLOCK);
  MM_CHECK_ARG(type >= F32 && type <= BF16 && out_type >= F32 && out_type <= BF16,
               "mm_mxfp4_gemm_backward: unknown type %d or %d", type, out_type);
  MM_CHECK_ARG(ldy >= N && ldy % (type == F32 ? 4 : 8) == 0,
               "mm_mxfp4_gemm_backward: ldy=%d: rows of dY must be whole 16-byte pieces, N=%d", ldy, N);
  MM_CHECK_ARG(M <= INT32_MAX - 127 && N < (1 << 28) && K < (1 << 28),
               "mm_mxfp4_gemm_backward: M=%d, N=%d or K=%d is too large", M, N, K);
  if (M == 0) return 0;
  MM_CHECK_ARG(dY && W && S && dX && aligned16(dY) && aligned16(W) && aligned16(S) && aligned16(dX),
               "mm_mxfp4_gemm_backward: dY, W, scales and dX must be 16-byte aligned and nothing null");
  const Plan p = plan_of(M, N, K, type);
  MM_CHECK_ARG(launch_holds((size_t)mm_cdiv(M, COSTS[p.tile].tm) * mm_cdiv(K, COSTS[p.tile].tk), 512),
               "mm_mxfp4_gemm_backward: M=%d, K=%d is too large", M, K);
  const Space sp = space_of(p, M, N, K);
  MM_CHECK_ARG(sp.total == 0 || (ws && aligned16(ws) && ws_bytes >= sp.total),
               "mm_mxfp4_gemm_backward: needs a workspace of %zu bytes, 16-byte aligned, got %zu",
               sp.total, ws_bytes);
  const hipStream_t st = (hipStream_t)stream;
  const int ks = scale_stride(K);
  if (ks != K / BLOCK) {
    uint8_t* const s = (uint8_t*)ws + COUNTERS;
    if (const int rc = launch_pad_scales(S, N, K / BLOCK, ks, s, st)) return rc;
    S = s;
  }
  float* const part = p.splits > 1 ? (float*)((char*)ws + sp.part) : nullptr;
  const Grad a{(const uint8_t*)dY, (const uint8_t*)W, S, part ? part : dX, part ? (int)F32 : out_type,
               M, N, K, ldy, ks, p.stages, p.per};
  if (type == F32) launch_t<F32>(a, p, st);
  else if (type == F16) launch_t<F16>(a, p, st);
  else launch_t<BF16>(a, p, st);
  MM_CHECK_LAUNCH("mm_mxfp4_gemm_backward");
  return part ? launch_sum(part, p.splits, (size_t)M * K, dX, out_type, st) : 0;
}
