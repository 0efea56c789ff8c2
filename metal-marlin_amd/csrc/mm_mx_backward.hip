// Input gradient of the MXFP4 product: dX[M, K] = dY[M, N] . W[N, K], W MXFP4 (mm_mx.h), straight
// through the rounding of x.
//
// The contraction runs along N, across the rows of W, whose scales change from row to row: the
// scaled matrix instructions cannot take them.  Every MXFP4 value is a bf16 number, though (2 bits
// of E2M1 and bf16 has E8M0's exponents), so weights are converted exactly, 64 rows of a stage at
// a time, into an LDS tile [n][k], from which ds_read_b64_tr_b16 takes columns as 32x32x16 bf16
// operands.  dY is bf16, or the exact sum of bf16 terms: fp16 is two of them (11 bits in 8 + 8),
// fp32 three (24 bits), each of which is multiplied: products are exact, sums fp32, rounded once.
//
// Bound by the matrix cores and LDS together; 16-bit conversions (16 per 32 weights) are small
// beside them from 64 rows of dY on.
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
// (32 of fp32).
template <int T, int WK_, int WM_, int KB_, int MB_>
struct GradTile {
  static constexpr int WK = WK_, WM = WM_, KB = KB_, MB = MB_;
  static constexpr int NWAVE = WK * WM, NTHR = NWAVE * 64;
  static constexpr int TK = WK * KB * 32, TM = WM * MB * 32;
  static constexpr int BN = 128 / kBytes<T>, STEPS = BN / 16;
  static constexpr int A = TM * 128, B = BN * TK * 2;     // bytes of a stage of dY and of W
  static constexpr int LDS = 2 * (A + B);
  static constexpr int IT = TM / 8 / NWAVE;               // copies of dY per wave and stage
  static constexpr int BLOCKS = BN * TK / 32;             // of W per stage
  static constexpr int WIT = (BLOCKS + NTHR - 1) / NTHR;  // of those per thread
  static constexpr int TERMS = T == BF16 ? 1 : (T == F16 ? 2 : 3);
  static_assert(TM % (8 * NWAVE) == 0 && NWAVE % 2 == 0, "copies per wave");
};

struct Grad {
  const uint8_t *dY, *W, *S;
  void* out;           // dX, or (split) fp32 partial sums [splits, M, K]
  int out_type, M, N, K, ldy, stages, per;   // ldy: row stride of dY; per: stages of a split
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

template <class Sh, int T>
__global__ void __launch_bounds__(Sh::NTHR) k_mx_grad(Grad a, int gm, int gk) {
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave / Sh::WM, wm = wave % Sh::WM, l32 = lane & 31, h = lane >> 5;
  // each XCD takes a stretch of tiles, row tiles innermost: they share their weights
  const int total = gm * gk, q = total >> 3, rem = total & 7, xcd = blockIdx.x & 7;
  const int lin = xcd * q + min(xcd, rem) + (int)(blockIdx.x >> 3);
  const int m0 = lin % gm * Sh::TM, k0 = lin / gm * Sh::TK;
  const int u0 = blockIdx.y * a.per, u1 = min(a.stages, u0 + a.per);
  const int kb = a.K / BLOCK, row_bytes = (a.N * kBytes<T> + 15) / 16 * 16;

  const uint8_t* src[Sh::IT];
#pragma unroll
  for (int i = 0; i < Sh::IT; ++i) {
    const int r = (i * Sh::NWAVE + wave) * 8 + lane / 8;
    src[i] = a.dY + (size_t)min(m0 + r, a.M - 1) * a.ldy * kBytes<T>;
  }
  const int at = 16 * ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7));
  auto issue = [&](int u, int st) {
#pragma unroll
    for (int i = 0; i < Sh::IT; ++i) {
      const int b = u * 128 + at;
      copy16(b < row_bytes ? src[i] + b : (const uint8_t*)mx_zeros,
             smem + st * Sh::A + (i * Sh::NWAVE + wave) * 1024);
    }
  };
  // Thread t converts blocks t, t + NTHR, .. of a stage: row t / (TK / 32), block t % (TK / 32).
  constexpr int RB = Sh::TK / 32;
  u32x4 wreg[Sh::WIT];
  uint32_t sreg[Sh::WIT];
  auto load = [&](int u) {
#pragma unroll
    for (int i = 0; i < Sh::WIT; ++i) {
      const int b = tid + i * Sh::NTHR;
      // rows past N meet zeros of dY, blocks past K are not stored
      const size_t n = min(u * Sh::BN + b / RB, a.N - 1);
      const int c = min(k0 / 32 + b % RB, kb - 1);
      wreg[i] = *(const u32x4*)(a.W + n * (a.K / 2) + c * 16);
      sreg[i] = a.S[n * kb + c];
    }
  };
  // [n][k] in 64-byte blocks, block c of row n at c ^ (n % 4): the 4 rows that a transposed read
  // takes lie in different banks.
  auto store = [&](int st) {
#pragma unroll
    for (int i = 0; i < Sh::WIT; ++i) {
      const int b = tid + i * Sh::NTHR;
      if (Sh::BLOCKS % Sh::NTHR != 0 && b >= Sh::BLOCKS) break;
      const int n = b / RB, c = b % RB;
      char* const d = smem + 2 * Sh::A + st * Sh::B + n * (Sh::TK * 2) + (c ^ (n & 3)) * 64;
      const float s = scale_of(sreg[i]);
      const uint32_t nan = sreg[i] == 255u ? 0x7fc07fc0u : 0u;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t w = wreg[i][j];
        *(u32x4*)(d + 16 * j) =
            u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 0)) | nan,
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 1)) | nan,
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 2)) | nan,
                  __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, 3)) | nan};
      }
    }
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
  auto compute = [&](int st) {
    const char* const dA = smem + st * Sh::A;
    const char* const dB = smem + 2 * Sh::A + st * Sh::B;
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
    issue(u0, 0);
    load(u0);
    store(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    int st = 0;
    for (int u = u0; u + 1 < u1; ++u) {
      issue(u + 1, st ^ 1);
      load(u + 1);
      __builtin_amdgcn_sched_barrier(0);
      compute(st);
      store(st ^ 1);
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      st ^= 1;
    }
    compute(st);
  }
  const size_t base = (size_t)blockIdx.y * a.M * a.K;      // 0 unless split
#pragma unroll
  for (int m = 0; m < Sh::MB; ++m) {
    const int mm = m0 + (wm * Sh::MB + m) * 32 + l32;
    if (mm >= a.M) continue;
#pragma unroll
    for (int k = 0; k < Sh::KB; ++k)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int kk = k0 + (wk * Sh::KB + k) * 32 + 8 * g + 4 * h;
        if (kk < a.K)                                       // K % 32 == 0: all four or none
          store4(a.out, a.out_type, base + (size_t)mm * a.K + kk,
                 f32x4{acc[k][m][4 * g], acc[k][m][4 * g + 1], acc[k][m][4 * g + 2],
                       acc[k][m][4 * g + 3]});
      }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
constexpr size_t COUNTERS = 65536;

// Splits of N: while the tiles leave CUs idle and every split keeps four stages.
struct Plan {
  int big, splits, per, stages;
};
Plan plan_of(int M, int N, int K, int type) {
  Plan p;
  const int bn = type == F32 ? 32 : 64;
  p.stages = mm_cdiv(N, bn);
  p.big = (long)mm_cdiv(M, 256) * mm_cdiv(K, 256) >= 200;
  p.splits = 1;
  if (!p.big) {
    const long tiles = (long)mm_cdiv(M, M <= 32 ? 32 : 128) * mm_cdiv(K, 128);
    p.splits = (int)std::max(1L, std::min({512 / std::max(1L, tiles), (long)p.stages / 4, 16L}));
  }
  p.per = mm_cdiv(p.stages, p.splits);
  p.splits = mm_cdiv(p.stages, p.per);
  return p;
}

template <int T, class Sh>
void launch(Grad a, const Plan& p, hipStream_t st) {
  const int gm = mm_cdiv(a.M, Sh::TM), gk = mm_cdiv(a.K, Sh::TK);
  hipLaunchKernelGGL((k_mx_grad<Sh, T>), dim3((unsigned)(gm * gk), p.splits), dim3(Sh::NTHR), 0, st,
                     a, gm, gk);
}
template <int T>
void launch_t(const Grad& a, const Plan& p, hipStream_t st) {
  if (p.big) launch<T, GradTile<T, 2, 4, 4, 2>>(a, p, st);
  else if (a.M <= 32) launch<T, GradTile<T, 4, 1, 1, 1>>(a, p, st);
  else launch<T, GradTile<T, 2, 2, 2, 2>>(a, p, st);
}

}  // namespace

extern "C" size_t mm_mxfp4_gemm_backward_workspace_bytes(int M, int N, int K, int type) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const Plan p = plan_of(M, N, K, type);
  return p.splits > 1 ? COUNTERS + (size_t)p.splits * M * K * sizeof(float) : 0;
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
  MM_CHECK_ARG(N < (1 << 28) && K < (1 << 28), "mm_mxfp4_gemm_backward: N=%d or K=%d is too large",
               N, K);
  if (M == 0) return 0;
  MM_CHECK_ARG(dY && W && S && dX && aligned16(dY) && aligned16(W) && aligned16(dX),
               "mm_mxfp4_gemm_backward: dY, W and dX must be 16-byte aligned and nothing null");
  const Plan p = plan_of(M, N, K, type);
  const size_t need = mm_mxfp4_gemm_backward_workspace_bytes(M, N, K, type);
  MM_CHECK_ARG(need == 0 || (ws && aligned16(ws) && ws_bytes >= need),
               "mm_mxfp4_gemm_backward: needs a workspace of %zu bytes, 16-byte aligned, got %zu",
               need, ws_bytes);
  const hipStream_t st = (hipStream_t)stream;
  float* const part = p.splits > 1 ? (float*)((char*)ws + COUNTERS) : nullptr;
  const Grad a{(const uint8_t*)dY, (const uint8_t*)W, S, part ? part : dX, part ? (int)F32 : out_type,
               M, N, K, ldy, p.stages, p.per};
  if (type == F32) launch_t<F32>(a, p, st);
  else if (type == F16) launch_t<F16>(a, p, st);
  else launch_t<BF16>(a, p, st);
  MM_CHECK_LAUNCH("mm_mxfp4_gemm_backward");
  return part ? launch_sum(part, p.splits, (size_t)M * K, dX, out_type, st) : 0;
}
