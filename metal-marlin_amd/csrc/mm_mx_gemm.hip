// C[M, N] = q(X) . W^T: X [M, K] fp32, fp16 or bf16 is quantized to MXFP4 (mm_mx.h), W is kept so,
// words [N, K/8] and scales [N, K/32].  The cores are in mm_mx_gemm.h.
#include <algorithm>
#include <cstdlib>

#include "mm_mx_gemm.h"
#include "mmfp4.h"

using namespace mmmx;

namespace {

// Up to 16 rows, quantized in the kernel; grid (N / 16 NT).
template <int T, int NT, int NW, int DEPTH, int U>
__global__ void __launch_bounds__(NW * 64)
k_mx_skinny(const char* __restrict__ X, const uint8_t* __restrict__ W,
            const uint8_t* __restrict__ S, void* __restrict__ C, int out_type, int M, int N, int K,
            int kp) {
  using R = Ring<NT, 0, NW, DEPTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];   // ring (later sums), scales, raw x, x
  const int lane = threadIdx.x & 63, r = lane & 15, n0 = blockIdx.x * 16 * NT, kb = K / BLOCK;
  char* const ls = lds + R::BYTES;
  char* const raw = ls + whole_kib(16 * NT * kb);
  const auto base = [=](int m) { return X + (size_t)m * K * kBytes<T>; };
  using Q = QuantizeRows<T, NW * 64, U, decltype(base)>;
  char* const lx = raw + Q::RAW;
  const Q rows{raw, lx, M, K, kp, base};
  const R ring(lds, W + (size_t)n0 * (K / 2), K, [&](int i) { return min(i, N - 1 - n0); }, nullptr,
               0, [](int) { return 0; });
  const Span sp = skinny_span<NW>(K);
  // loads come back in order: the scales and x first, the weights are the last to be needed
  scales_to_lds<NW * 64>(S + (size_t)n0 * kb, ls, 16 * NT * kb, min(16 * NT, N - n0) * kb);
  rows.first();
  skinny_begin<DEPTH>(ring, sp);
  wait_loads<R::LOADS * DEPTH>();
  rows.finish();
  block_barrier();
  const int row = min(r, M - 1);
  const LdsX x{lx + row * lds_stride(kp),
               (const uint8_t*)lx + M * lds_stride(kp) + row * (kp / BLOCK)};
  f32x4 acc[1][NT];
  skinny<1, NT, DEPTH>(ring, x, (const uint8_t*)ls + r * kb, [=](int nt) { return 16 * nt * kb; }, kb, sp, acc);
  __syncthreads();                                   // the ring has been read
  skinny_reduce<1, NT, NW>(acc, (float*)lds, M, [&](int nn, int mm, float v) {
    if (n0 + nn < N) store1(C, out_type, (size_t)mm * N + n0 + nn, v);
  });
}

// The same for 16 MT rows a block, from codes.
template <int MT, int NT, int NW, int DEPTH>
__global__ void __launch_bounds__(NW * 64)
k_mx_skinny_codes(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS, int kp,
                  const uint8_t* __restrict__ W, const uint8_t* __restrict__ S,
                  void* __restrict__ C, int out_type, int M, int N, int K) {
  using R = Ring<NT, MT, NW, DEPTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];   // ring (later sums), scales of W, of x
  const int lane = threadIdx.x & 63, r = lane & 15, kb = K / BLOCK, kbp = kp / BLOCK;
  const int n0 = blockIdx.x * 16 * NT, m0 = blockIdx.y * 16 * MT;
  static_assert(R::STAGE >= MT * NT * 1024 / DEPTH, "the waves' sums take the ring's place");
  char* const ls = lds + R::BYTES;
  char* const lx = ls + whole_kib(16 * NT * kb);
  const R ring(lds, W + (size_t)n0 * (K / 2), K, [&](int i) { return min(i, N - 1 - n0); },
               X + (size_t)m0 * (kp / 2), kp, [&](int i) { return min(i, M - 1 - m0); });
  const Span sp = skinny_span<NW>(K);
  scales_to_lds<NW * 64>(S + (size_t)n0 * kb, ls, 16 * NT * kb, min(16 * NT, N - n0) * kb);
  copy_to_lds<NW * 64>(XS + (size_t)m0 * kbp, lx, 16 * MT * kbp);
  skinny_begin<DEPTH>(ring, sp);
  wait_loads<R::LOADS * DEPTH>();
  block_barrier();
  f32x4 acc[MT][NT];
  skinny<MT, NT, DEPTH>(ring, RingX<NT>{(const uint8_t*)lx + r * kbp, 16 * kbp},
                        (const uint8_t*)ls + r * kb, [=](int nt) { return 16 * nt * kb; }, kb, sp, acc);
  __syncthreads();
  skinny_reduce<MT, NT, NW>(acc, (float*)lds, min(16 * MT, M - m0), [&](int nn, int mm, float v) {
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
  tile_loop<Sh>(src, 0, (K + UNIT - 1) / UNIT, smem, acc);
  __syncthreads();
  tile_out<Sh>(acc, smem, C, out_type, M - m0, n0, N,
               [=](int m) { return (size_t)(m0 + m) * N; });
}

constexpr int SKINNY_M = 16;    // rows that the kernel may quantize itself
constexpr int CODES_M = 64;     // rows that stream the weights from codes
constexpr size_t COUNTERS = 65536;   // head of every workspace: other products' arrival counters

// Whether the blocks quantize x themselves.  Each of them does it anew, so from about 16384 values
// on (4 rows of 4096) a launch that does it once is faster: us, in the kernel against apart,
// 4096 -> 14336 M = 4 8.8 / 10.9, M = 8 11.5 / 11.1, M = 16 17.4 / 11.1; 14336 -> 4096 M = 1
// 7.1 / 9.3, M = 2 8.4 / 9.4, M = 4 12.8 / 9.5.
bool quantizes_itself(int M, int K) { return M <= SKINNY_M && (long)M * K <= 16384 + 4096; }

template <int T, int NT, int NW, int D, int U>
void launch_skinny_as(const void* X, const uint32_t* W, const uint8_t* S, void* C, int out_type,
                      int M, int N, int K, hipStream_t st) {
  const int kp = (int)padded(K);
  const int lds = Ring<NT, 0, NW, D>::BYTES + whole_kib(16 * NT * (K / BLOCK)) +
                  U * (T == F32 ? 2 : 1) * NW * 1024 + lds_x_bytes(M, kp);
  hipLaunchKernelGGL((k_mx_skinny<T, NT, NW, D, U>), dim3(mm_cdiv(N, 16 * NT)), dim3(NW * 64), lds,
                     st, (const char*)X, (const uint8_t*)W, S, C, out_type, M, N, K, kp);
}
// Wide matrices take 32 rows of W per block of 4 waves, others, which would leave CUs idle so, 16
// rows and 8 waves: M = 1, 4096 -> 14336 6.5 us (16 rows: 7.9), 14336 -> 4096 9.0 (7.1).
template <int T>
void launch_skinny(const void* X, const uint32_t* W, const uint8_t* S, void* C, int out_type, int M,
                   int N, int K, hipStream_t st) {
  if (N >= 8192) launch_skinny_as<T, 2, 4, 2, 2>(X, W, S, C, out_type, M, N, K, st);
  else launch_skinny_as<T, 1, 8, 2, 4>(X, W, S, C, out_type, M, N, K, st);
}

template <int MT, int NT, int D>
void launch_codes(const uint8_t* xq, const uint8_t* xs, int kp, const uint32_t* W, const uint8_t* S,
                  void* C, int out_type, int M, int N, int K, hipStream_t st) {
  hipLaunchKernelGGL((k_mx_skinny_codes<MT, NT, 8, D>),
                     dim3(mm_cdiv(N, 16 * NT), mm_cdiv(M, 16 * MT)), dim3(512),
                     (Ring<NT, MT, 8, D>::BYTES + whole_kib(16 * NT * (K / BLOCK)) +
                      whole_kib(16 * MT * (kp / BLOCK))),
                     st, xq, xs, kp, (const uint8_t*)W, S, C, out_type, M, N, K);
}

template <class Sh>
void launch_tile(const uint8_t* xq, const uint8_t* xs, int kp, const uint32_t* W, const uint8_t* S,
                 void* C, int out_type, int M, int N, int K, hipStream_t st) {
  const int gm = mm_cdiv(M, Sh::TM), gn = mm_cdiv(N, Sh::TN);
  hipLaunchKernelGGL((k_mx_tile<Sh>), dim3((unsigned)(gm * gn)), dim3(Sh::NTHR), 0, st, xq, xs, kp,
                     (const uint8_t*)W, S, C, out_type, M, N, K, gm, gn, std::min(gm, 4));
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace

extern "C" size_t mm_mxfp4_gemm_workspace_bytes(int M, int N, int K) {
  (void)N;
  if (M <= 0 || K <= 0 || quantizes_itself(M, K)) return 0;
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
  MM_CHECK_ARG(X && W && S && C && aligned16(X) && aligned16(W) && aligned16(S) && aligned16(C),
               "mm_mxfp4_gemm: X, W, scales and C must be 16-byte aligned and nothing null");
  const size_t need = mm_mxfp4_gemm_workspace_bytes(M, N, K);
  MM_CHECK_ARG(need == 0 || (ws && aligned16(ws) && ws_bytes >= need),
               "mm_mxfp4_gemm: needs a workspace of %zu bytes, 16-byte aligned, got %zu", need,
               ws_bytes);
  const hipStream_t st = (hipStream_t)stream;
  if (quantizes_itself(M, K)) {
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
    if (M <= 16) launch_codes<1, 1, 1>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
    else if (M <= 32) launch_codes<2, 1, 1>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
    else launch_codes<4, 1, 1>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
    MM_CHECK_LAUNCH("mm_mxfp4_gemm");
    return 0;
  }
  const long big = (long)mm_cdiv(M, 256) * mm_cdiv(N, 256);
  static const int cfg = getenv("MX_CFG") ? atoi(getenv("MX_CFG")) : 0;
  if (cfg == 1) launch_tile<Tile<2, 2, 4, 4>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else if (cfg == 2) launch_tile<Tile<2, 2, 2, 2>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else if (cfg == 3) launch_tile<Tile<2, 2, 2, 4>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else if (cfg == 4) launch_tile<Tile<2, 2, 1, 4>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else if (cfg == 5) launch_tile<Tile<2, 4, 2, 2>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else if (big >= 200) launch_tile<Tile<4, 2, 2, 4>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  else launch_tile<Tile<2, 2, 2, 2>>(xq, xs, kp, W, S, C, out_type, M, N, K, st);
  MM_CHECK_LAUNCH("mm_mxfp4_gemm");
  return 0;
}
