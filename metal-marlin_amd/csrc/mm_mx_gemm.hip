// C[M, N] = q(X) . W^T: X [M, K] fp32, fp16 or bf16 is quantized to MXFP4 (mm_mx.h), W is kept so,
// words [N, K/8] and scales [N, K/32].  The cores are in mm_mx_gemm.h.
#include "mm_mx_gemm.h"
#include "mmfp4.h"

using namespace mmmx;

namespace {

// Up to 16 rows, quantized in the kernel; grid (N / 16 NT).
template <int T, int NT, int NW>
__global__ void __launch_bounds__(NW * 64)
k_mx_skinny(const char* __restrict__ X, const uint8_t* __restrict__ W,
            const uint8_t* __restrict__ S, void* __restrict__ C, int out_type, int M, int N, int K) {
  __shared__ __attribute__((aligned(16))) float red[NW * NT * 256];
  const int lane = threadIdx.x & 63, r = lane & 15, n0 = blockIdx.x * 16 * NT;
  const char* x[1] = {X + (size_t)min(r, M - 1) * K * kBytes<T>};
  const uint8_t* xs[1] = {nullptr};
  const uint8_t *w[NT], *s[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const size_t n = min(n0 + 16 * nt + r, N - 1);
    w[nt] = W + n * (K / 2);
    s[nt] = S + n * (K / BLOCK);
  }
  f32x4 acc[1][NT];
  skinny<T, 1, NT, NW>(x, xs, w, s, K, acc);
  skinny_reduce<1, NT, NW>(acc, red, M, [&](int nn, int mm, float v) {
    if (n0 + nn < N) store1(C, out_type, (size_t)mm * N + n0 + nn, v);
  });
}

// The same for 16 MT rows a block, from codes.
template <int MT, int NT, int NW>
__global__ void __launch_bounds__(NW * 64)
k_mx_skinny_codes(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS, int kp,
                  const uint8_t* __restrict__ W, const uint8_t* __restrict__ S,
                  void* __restrict__ C, int out_type, int M, int N, int K) {
  __shared__ __attribute__((aligned(16))) float red[NW * MT * NT * 256];
  const int lane = threadIdx.x & 63, r = lane & 15;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  const char* x[MT];
  const uint8_t *xs[MT], *w[NT], *s[NT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const size_t m = min(m0 + 16 * mt + r, M - 1);
    x[mt] = (const char*)X + m * (kp / 2);
    xs[mt] = XS + m * (kp / BLOCK);
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const size_t n = min(n0 + 16 * nt + r, N - 1);
    w[nt] = W + n * (K / 2);
    s[nt] = S + n * (K / BLOCK);
  }
  f32x4 acc[MT][NT];
  skinny<CODES, MT, NT, NW>(x, xs, w, s, K, acc);
  skinny_reduce<MT, NT, NW>(acc, red, min(16 * MT, M - m0), [&](int nn, int mm, float v) {
    if (n0 + nn < N) store1(C, out_type, (size_t)(m0 + mm) * N + n0 + nn, v);
  });
}

struct DenseSrc {
  const uint8_t *W, *S, *X, *XS;
  int K, kp, n_last, m_last;
  MM_DEV uint32_t wrow(int r) const { return min(r, n_last); }
  MM_DEV uint32_t xrow(int r) const { return min(r, m_last); }
};

// Tiles are walked so that each of the 8 XCDs (blocks are dealt to them round-robin) gets one
// stretch of them, in groups of `grp` row tiles that share their weights in its L2.
MM_DEV void tile_of(int id, int gm, int gn, int grp, int& tm, int& tn) {
  const int total = gm * gn, q = total >> 3, rem = total & 7, xcd = id & 7;
  const int lin = xcd * q + min(xcd, rem) + (id >> 3);
  const int per = grp * gn, g = lin / per, first = g * grp;
  const int rows = min(grp, gm - first), in = lin - g * per;
  tm = first + in % rows;
  tn = in / rows;
}

template <class Sh>
__global__ void __launch_bounds__(Sh::NTHR)
k_mx_tile(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS, int kp,
          const uint8_t* __restrict__ W, const uint8_t* __restrict__ S, void* __restrict__ C,
          int out_type, int M, int N, int K, int gm, int gn, int grp) {
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS];
  int tm, tn;
  tile_of(blockIdx.x, gm, gn, grp, tm, tn);
  const int m0 = tm * Sh::TM, n0 = tn * Sh::TN;
  const DenseSrc src{W + (size_t)n0 * (K / 2), S + (size_t)n0 * (K / BLOCK),
                     X + (size_t)m0 * (kp / 2), XS + (size_t)m0 * (kp / BLOCK),
                     K, kp, N - 1 - n0, M - 1 - m0};
  f32x16 acc[Sh::NB][Sh::MB];
  tile_loop<Sh>(src, 0, kp / UNIT, smem, acc);
  const bool whole = N % 4 == 0;
  tile_out<Sh>(acc, [&](int n, int m, f32x4 v) {
    m += m0;
    n += n0;
    if (m >= M || n >= N) return;
    const size_t at = (size_t)m * N + n;
    if (whole) {
      store4(C, out_type, at, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < N) store1(C, out_type, at + i, v[i]);
    }
  });
}

constexpr int SKINNY_M = 16;    // rows that the kernel quantizes itself
constexpr int CODES_M = 64;     // rows that stream the weights from codes
constexpr size_t COUNTERS = 65536;   // head of every workspace: other products' arrival counters

template <int T>
void launch_skinny(const void* X, const uint32_t* W, const uint8_t* S, void* C, int out_type, int M,
                   int N, int K, hipStream_t st) {
#define MM_MX_SKINNY(NT, NW)                                                                   \
  hipLaunchKernelGGL((k_mx_skinny<T, NT, NW>), dim3(mm_cdiv(N, 16 * NT)), dim3(NW * 64), 0, st,  \
                     (const char*)X, (const uint8_t*)W, S, C, out_type, M, N, K)
  MM_MX_SKINNY(1, 8);
#undef MM_MX_SKINNY
}

template <class Sh>
void launch_tile(const uint8_t* xq, const uint8_t* xs, int kp, const uint32_t* W, const uint8_t* S,
                 void* C, int out_type, int M, int N, int K, hipStream_t st) {
  const int gm = mm_cdiv(M, Sh::TM), gn = mm_cdiv(N, Sh::TN);
  hipLaunchKernelGGL((k_mx_tile<Sh>), dim3((unsigned)(gm * gn)), dim3(Sh::NTHR), 0, st, xq, xs, kp,
                     (const uint8_t*)W, S, C, out_type, M, N, K, gm, gn, std::min(gm, 8));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" size_t mm_mxfp4_gemm_workspace_bytes(int M, int N, int K) {
  (void)N;
  if (M <= SKINNY_M || K <= 0) return 0;
  return COUNTERS + packed_bytes(M, K);
}

extern "C" int mm_mxfp4_gemm(const void* X, int type, const uint32_t* W, const uint8_t* S, void* C,
                             int out_type, int M, int N, int K, void* ws, size_t ws_bytes,
                             void* stream) {
  MM_CHECK_ARG(M >= 0 && N > 0 && K > 0 && K % BLOCK == 0,
               "mm_mxfp4_gemm: M=%d, N=%d, K=%d: K must be a positive multiple of %d", M, N, K,
               BLOCK);
  MM_CHECK_ARG(type >= F32 && type <= BF16 && out_type >= F32 && out_type <= BF16,
               "mm_mxfp4_gemm: unknown type %d or %d", type, out_type);
  if (M == 0) return 0;
  MM_CHECK_ARG(X && W && S && C && aligned16(X) && aligned16(W) && aligned16(C),
               "mm_mxfp4_gemm: X, W and C must be 16-byte aligned and nothing null");
  const size_t need = mm_mxfp4_gemm_workspace_bytes(M, N, K);
  MM_CHECK_ARG(need == 0 || (ws && aligned16(ws) && ws_bytes >= need),
               "mm_mxfp4_gemm: needs a workspace of %zu bytes, 16-byte aligned, got %zu", need,
               ws_bytes);
  const hipStream_t st = (hipStream_t)stream;
  if (M <= SKINNY_M) {
    if (type == F32) launch_skinny<F32>(X, W, S, C, out_type, M, N, K, st);
    else if (type == F16) launch_skinny<F16>(X, W, S, C, out_type, M, N, K, st);
    else launch_skinny<BF16>(X, W, S, C, out_type, M, N, K, st);
    MM_CHECK_LAUNCH("mm_mxfp4_gemm");
    return 0;
  }
  const int kp = (int)padded(K);
  uint8_t* const xq = (uint8_t*)ws + COUNTERS;
  uint8_t* const xs = xq + codes_bytes(M, K);
  if (const int rc = launch_quantize(X, type, M, K, kp, (uint32_t*)xq, xs, st)) return rc;
  if (M <= CODES_M) {
#define MM_MX_CODES(MT, NT)                                                                      \
  hipLaunchKernelGGL((k_mx_skinny_codes<MT, NT, 8>), dim3(mm_cdiv(N, 16 * NT), mm_cdiv(M, 16 * MT)), \
                     dim3(512), 0, st, xq, xs, kp, (const uint8_t*)W, S, C, out_type, M, N, K)
    if (M <= 32) MM_MX_CODES(2, 2);
    else MM_MX_CODES(4, 2);
#undef MM_MX_CODES
    MM_CHECK_LAUNCH("mm_mxfp4_gemm");
    return 0;
  }
  const long big = (long)mm_cdiv(M, 256) * mm_cdiv(N, 256);
  if (big >= 200) launch_tile<Tile<4, 2, 2, 4>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else launch_tile<Tile<2, 2, 2, 2>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  MM_CHECK_LAUNCH("mm_mxfp4_gemm");
  return 0;
}
