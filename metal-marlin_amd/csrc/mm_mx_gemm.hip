// C[M, N] = q(X) . W^T: X [M, K] fp32, fp16 or bf16 is quantized to MXFP4 (mm_mx.h), W is kept so,
// words [N, K/8] and scales [N, K/32].  The cores are in mm_mx_gemm.h.
#include <algorithm>

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
  size_t spitch, xpitch;
  static constexpr bool BY_UNIT = true;
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

// grid (tiles, splits of K): with more than one, each split's fp32 sums go to C, sum_pitch(M * N)
// apart.
template <class Sh>
__global__ void __launch_bounds__(Sh::NTHR)
k_mx_tile(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS, int kp,
          const uint8_t* __restrict__ W, const uint8_t* __restrict__ S, void* __restrict__ C,
          int out_type, int M, int N, int K, int gm, int gn, int grp, int per) {
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS];
  int tm, tn;
  tile_of(blockIdx.x, gm, gn, grp, tm, tn);
  const int m0 = tm * Sh::TM, n0 = tn * Sh::TN;
  const DenseSrc src{W + (size_t)n0 * (K / 2), S + (size_t)n0 * 8, X + (size_t)m0 * (kp / 2),
                     XS + (size_t)m0 * 8, K, kp, N - 1 - n0, M - 1 - m0, unit_pitch(N), unit_pitch(M)};
  f32x16 acc[Sh::NB][Sh::MB];
  const int u0 = blockIdx.y * per, u1 = min((K + UNIT - 1) / UNIT, u0 + per);
  tile_loop<Sh>(src, u0, u1, smem, acc);
  __syncthreads();
  const size_t base = blockIdx.y * sum_pitch((size_t)M * N);
  tile_out<Sh>(acc, smem, C, out_type, M - m0, n0, N,
               [=](int m) { return base + (size_t)(m0 + m) * N; });
}

constexpr int SKINNY_M = 16;    // rows that the kernel may quantize itself
constexpr int CODES_M = 64;     // rows that stream the weights from codes
constexpr size_t COUNTERS = 65536;   // head of every workspace: other products' arrival counters

// Whether the blocks quantize x themselves.  Each of them does it anew, so from some number of values
// on a launch that does it once is faster: us, in the kernel against apart, 4096 -> 14336 M = 8
// 11.5 / 10.1, M = 16 17.4 / 10.4, M = 4 8.8 in the kernel; 14336 -> 4096 M = 1 7.1 / 9.2, M = 2
// 8.4 / 9.3, M = 4 12.8 / 9.3.  The border lies between 16384 and 28672 values; it is drawn at 20480,
// which costs the last M = 2 (28672) 0.9 us.
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

constexpr int CODES_WAVES = 4, CODES_DEPTH = 2, LDS_BYTES = 160 * 1024, CUS = 256;
template <int MT, int NT>
long codes_lds(int K) {
  return Ring<NT, MT, CODES_WAVES, CODES_DEPTH>::BYTES + (long)whole_kib(16 * NT * (K / BLOCK)) +
         whole_kib(16 * MT * (int)(padded(K) / BLOCK));
}
template <int MT, int NT>
void launch_codes_as(const uint8_t* xq, const uint8_t* xs, int kp, const uint32_t* W,
                     const uint8_t* S, void* C, int out_type, int M, int N, int K, hipStream_t st) {
  hipLaunchKernelGGL((k_mx_skinny_codes<MT, NT, CODES_WAVES, CODES_DEPTH>),
                     dim3(mm_cdiv(N, 16 * NT), mm_cdiv(M, 16 * MT)), dim3(CODES_WAVES * 64),
                     (codes_lds<MT, NT>(K)), st, xq, xs, kp, (const uint8_t*)W, S, C, out_type, M, N,
                     K);
}
// Up to 32 rows take 32 columns a block where 16 would make more blocks than the CUs hold at once,
// two each: us, 32 columns against 16, M = 24 4096 -> 14336 11.8 / 13.6, 4096 -> 4096 8.2 / 7.0,
// 14336 -> 4096 11.9 / 10.4.  (Eight waves and one unit ahead: 13.7, 7.7, 10.6.)
bool wide_codes(int M, int N) { return M <= 32 && N > 2 * CUS * 16; }

// Rows that stream the weights, from codes: 16, 32 or 64 a block, as long as a block's scales fit
// LDS.  More than 32 rows only while the CUs hold all blocks at once: us, streamed against tiles,
// M = 64 4096 -> 4096 9.1 / 10.8, 14336 -> 4096 14.3 / 17.5, 4096 -> 14336 24.4 / 12.3.
bool streams(int M, int N, int K) {
  if (M > CODES_M || (M > 32 && N > 2 * CUS * 16)) return false;
  const long lds = wide_codes(M, N) ? (M <= 16 ? codes_lds<1, 2>(K) : codes_lds<2, 2>(K))
                   : M <= 16        ? codes_lds<1, 1>(K)
                   : M <= 32        ? codes_lds<2, 1>(K)
                                    : codes_lds<4, 1>(K);
  return lds <= LDS_BYTES;
}

// Tiles.  A block is alone on its CU, or (64 x 64) one of two that take turns; a stage of it takes
// `stage` us and its beginning and end `ends`, measured at 65 .. 2048 rows of 14336 x 4096, 4096 x
// 14336 and 4096 x 4096.  The estimate picked the fastest tile and split of those (65, 128, 333,
// 512, 1024, 2048 rows: 14, 15, 26, 28, 42, 78 us; 17, 18, 31, 34, 50, 85; 11, 11, 14, 16, 22, 31;
// the largest tiles alone: 34 .. 78; 89 .. 103; 33 .. 39).
using Tile256 = Tile<4, 2, 2, 4, 2>;       // 256 x 256, 8 waves
using Tile128w = Tile<2, 4, 2, 2, 3>;      // 128 x 256, 8 waves
using Tile128 = Tile<4, 2, 1, 2, 4>;       // 128 x 128, 8 waves
using Tile64w = Tile<2, 4, 1, 1, 5>;       // 64 x 128, 8 waves
using Tile64 = Tile<2, 2, 1, 1, 4>;        // 64 x 64, 4 waves
struct Cost {
  int tm, tn;
  float stage, ends;
};
constexpr Cost COSTS[] = {{256, 256, 1.75f, 6.0f}, {128, 256, 1.2f, 4.0f}, {128, 128, 0.7f, 3.0f},
                          {64, 128, 0.45f, 2.5f}, {64, 64, 0.28f, 2.0f}};
constexpr int MAX_SPLITS = 8;

struct Plan {
  int tile;           // which tiles; -1: a kernel that streams the weights
  int splits, per;    // splits of K and their stages
};
// With few tiles K is split, and the splits' sums are joined by another launch: 2.5 us and their
// bytes at about 3 TB/s.
Plan plan_of(int M, int N, int K) {
  const int stages = mm_cdiv(K, UNIT);
  if (streams(M, N, K)) return Plan{-1, 1, stages};
  Plan best{0, 1, stages};
  float least = 0;
  for (int t = 0; t < 5; ++t) {
    const long tiles = (long)mm_cdiv(M, COSTS[t].tm) * mm_cdiv(N, COSTS[t].tn);
    for (int s = 1; s <= MAX_SPLITS && (s == 1 || (tiles * s <= 2 * CUS && stages >= 4 * s)); ++s) {
      const int per = mm_cdiv(stages, s), splits = mm_cdiv(stages, per);
      float us = (float)((tiles * splits + CUS - 1) / CUS) * (per * COSTS[t].stage + COSTS[t].ends);
      if (splits > 1) us += 2.5f + (float)M * N * 4 * (splits + 1) / 3e6f;
      if (least == 0 || us < least) {
        least = us;
        best = Plan{t, splits, per};
      }
    }
  }
  return best;
}

template <class Sh>
void launch_tile(const Plan& p, const uint8_t* xq, const uint8_t* xs, int kp, const uint32_t* W,
                 const uint8_t* S, void* C, int out_type, int M, int N, int K, hipStream_t st) {
  const int gm = mm_cdiv(M, Sh::TM), gn = mm_cdiv(N, Sh::TN);
  hipLaunchKernelGGL((k_mx_tile<Sh>), dim3((unsigned)(gm * gn), p.splits), dim3(Sh::NTHR), 0, st, xq,
                     xs, kp, (const uint8_t*)W, S, C, out_type, M, N, K, gm, gn,
                     std::min(gm, 4), p.per);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// x's codes and scales; for tiles W's scales by units; the splits' sums.
struct Space {
  size_t xs, scales, part, total;
};
Space space_of(const Plan& p, int M, int N, int K) {
  Space s;
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  s.xs = COUNTERS + codes_bytes(M, K);
  if (p.tile < 0) {
    s.scales = s.part = s.total = COUNTERS + up(packed_bytes(M, K));
    return s;
  }
  s.scales = s.xs + mm_cdiv(K, UNIT) * unit_pitch(M);
  s.part = s.scales + mm_cdiv(K, UNIT) * unit_pitch(N);
  s.total = s.part + (p.splits > 1 ? p.splits * sum_pitch((size_t)M * N) * sizeof(float) : 0);
  return s;
}

}  // namespace

extern "C" size_t mm_mxfp4_gemm_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || quantizes_itself(M, K)) return 0;
  return space_of(plan_of(M, N, K), M, N, K).total;
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
  // rows and columns of whole tiles are counted in 31 bits, and a launch holds the blocks that
  // stream the weights
  MM_CHECK_ARG(K < (1 << 24) && M <= INT32_MAX - 255 && N < (1 << 29),
               "mm_mxfp4_gemm: M=%d, N=%d, K=%d is too large", M, N, K);
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
  const Plan p = plan_of(M, N, K);
  const Space sp = space_of(p, M, N, K);
  uint8_t *const xq = (uint8_t*)ws + COUNTERS, *const xs = (uint8_t*)ws + sp.xs;
  if (p.tile < 0) {
    if (const int rc = launch_quantize(X, type, M, K, kp, (uint32_t*)xq, xs, st)) return rc;
    const auto run = [&](auto mt, auto nt) {
      launch_codes_as<decltype(mt)::value, decltype(nt)::value>(xq, xs, kp, W, S, C, out_type, M, N,
                                                                K, st);
    };
    constexpr std::integral_constant<int, 1> one{};
    constexpr std::integral_constant<int, 2> two{};
    if (wide_codes(M, N)) M <= 16 ? run(one, two) : run(two, two);
    else if (M <= 16) run(one, one);
    else if (M <= 32) run(two, one);
    else run(std::integral_constant<int, 4>{}, one);
    MM_CHECK_LAUNCH("mm_mxfp4_gemm");
    return 0;
  }
  const Cost& c = COSTS[p.tile];
  MM_CHECK_ARG(launch_holds((size_t)mm_cdiv(M, c.tm) * mm_cdiv(N, c.tn), 512),
               "mm_mxfp4_gemm: M=%d, N=%d is too large", M, N);
  uint8_t* const s = (uint8_t*)ws + sp.scales;
  if (const int rc = launch_quantize_units(X, type, M, K, kp, (uint32_t*)xq, xs, S, N, s, st)) return rc;
  void* const to = p.splits > 1 ? (void*)((char*)ws + sp.part) : C;
  const int to_type = p.splits > 1 ? (int)F32 : out_type;
  const auto run = [&](auto sh) {
    launch_tile<decltype(sh)>(p, xq, xs, kp, W, s, to, to_type, M, N, K, st);
  };
  switch (p.tile) {
    case 0: run(Tile256{}); break;
    case 1: run(Tile128w{}); break;
    case 2: run(Tile128{}); break;
    case 3: run(Tile64w{}); break;
    default: run(Tile64{}); break;
  }
  MM_CHECK_LAUNCH("mm_mxfp4_gemm");
  return p.splits > 1 ? launch_sum((const float*)to, p.splits, (size_t)M * N, C, out_type, st) : 0;
}
