// The experts' gated feed-forward block on MXFP4 weights (mm_mx.h) for routed tokens:
//   out[t] = sum_j p[t, j] * y,  y = q(silu(g) * u) . W_down[e]^T,  (g, u) = q(x[t]) . W_gate_up[e]^T
// with e = ids[t, j]; ids outside [0, E) contribute nothing.  Launches: the stable sort of mm_moe.hip,
// gate_up (gathers tokens; silu(g) * u in fp32 is quantized as it leaves the kernel), down, and the
// sum over a token's experts in slot order.  With many rows per expert a launch before them
// quantizes the tokens once; with few the gate_up kernel does it on the way.
//
// Both products are bound by the weights' bytes until an expert has some hundred rows.  Where the
// weights are streamed (few rows per expert on average) a block takes an expert's rows sixteen at a
// time, one sixteen after the other, and streams its part of the weights for each: once for most
// experts, but where one expert has most of the rows that expert's blocks work alone.  128 experts of
// 2048 -> 768, one per token: 64 tokens spread 35 us, all to one expert 55; 511 tokens 94 and 355,
// where 512, in tiles, take 89 and 31.
#include <algorithm>

#include "mm_mx_gemm.h"
#include "mmfp4.h"

using namespace mmmx;

namespace {

constexpr int MAX_E = 1024;

struct Rows {
  const int32_t *offsets, *sorted;   // of the sort
  int k;
};

MM_DEV float swiglu(float g, float u) { return g / (1.0f + __expf(-g)) * u; }

// Few rows per expert; grid (ip / 32, E).  A block has the 32 gate and 32 up rows of one block of
// h; its waves split K.  h: quantized rows in sorted order, ip values long, zeros behind I.
template <int T, int NW, int DEPTH, int U>
__global__ void __launch_bounds__(NW * 64)
k_mx_moe_gate_up(const char* __restrict__ X, const uint8_t* __restrict__ W,
                 const uint8_t* __restrict__ S, Rows rows, int H, int hp, int I, int ip,
                 uint32_t* __restrict__ hw, uint8_t* __restrict__ hs) {
  using R = Ring<4, 0, NW, DEPTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];   // ring (later sums), scales, x
  const int e = blockIdx.y, r0 = rows.offsets[e], r1 = rows.offsets[e + 1];
  if (r0 >= r1) return;
  const int c0 = blockIdx.x * 32, tid = threadIdx.x, lane = tid & 63, r = lane & 15;
  const int i = tid % 32, kb = H / BLOCK;            // i: this thread's column of h
  if (c0 >= I) {                                     // padding
    for (int m = r0 + tid / 32; m < r1; m += NW * 2) {
      if (i < 4) hw[(size_t)m * (ip / 8) + c0 / 8 + i] = 0;
      if (i == 4) hs[(size_t)m * (ip / 32) + c0 / 32] = 0;
    }
    return;
  }
  char* const ls = lds + R::BYTES;
  char* const raw = ls + 2 * whole_kib(32 * kb);
  const uint8_t* const we = W + (size_t)e * 2 * I * (H / 2);
  const uint8_t* const se = S + (size_t)e * 2 * I * kb;
  const R ring(lds, we, H, [&](int n) { return c0 + n % 32 + n / 32 * I; }, nullptr, 0,
               [](int) { return 0; });
  const Span sp = skinny_span<NW>(H);
  for (int m0 = r0; m0 < r1; m0 += 16) {
    const int n = min(16, r1 - m0), row = min(r, n - 1);
    const auto base = [&](int m) {
      return X + (size_t)(rows.sorted[m0 + m] / rows.k) * H * kBytes<T>;
    };
    using Q = QuantizeRows<T, NW * 64, U, decltype(base)>;
    char* const lx = raw + Q::RAW;
    const Q xrows{raw, lx, n, H, hp, base};
    if (m0 > r0) __syncthreads();                    // the sums before these have been read
    copy_to_lds<NW * 64>(se + (size_t)c0 * kb, ls, 32 * kb);
    copy_to_lds<NW * 64>(se + (size_t)(I + c0) * kb, ls + whole_kib(32 * kb), 32 * kb);
    xrows.first();
    skinny_begin<DEPTH>(ring, sp);
    wait_loads<R::LOADS * DEPTH>();
    xrows.finish();
    block_barrier();
    const LdsX x{lx + row * lds_stride(hp),
                 (const uint8_t*)lx + n * lds_stride(hp) + row * (hp / BLOCK)};
    f32x4 acc[1][4];
    skinny<1, 4, DEPTH>(ring, x, (const uint8_t*)ls + r * kb, [=](int nt) {
      return 16 * (nt % 2) * kb + (nt / 2) * whole_kib(32 * kb);
    }, kb, sp, acc);
    __syncthreads();                                 // the ring has been read
    float* const red = (float*)lds;
    skinny_park<1, 4, NW>(acc, red);
    __syncthreads();
    for (int mm = tid / 32; mm < n; mm += NW * 2) {
      const float h = swiglu(skinny_sum<1, 4, NW>(red, i, mm), skinny_sum<1, 4, NW>(red, 32 + i, mm));
      uint32_t amax = u32_of(h) & 0x7fffffffu;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) amax = max(amax, (uint32_t)__shfl_xor((int)amax, d));
      const uint32_t code = scale_code(amax);
      uint32_t word =
          __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, h, 0.0f, scale_of(code), 0) & 15u;
      word <<= 4 * (i % 8);
#pragma unroll
      for (int d = 1; d < 8; d <<= 1) word |= (uint32_t)__shfl_xor((int)word, d);
      const size_t m = m0 + mm;
      if (i % 8 == 0) hw[m * (ip / 8) + c0 / 8 + i / 8] = word;
      if (i == 0) hs[m * (ip / 32) + c0 / 32] = (uint8_t)code;
    }
  }
}

// y[row] = h[row] . W_down[e]^T; grid (H / 16 NT, E).
template <int NT, int NW, int DEPTH>
__global__ void __launch_bounds__(NW * 64)
k_mx_moe_down(const uint8_t* __restrict__ hw, const uint8_t* __restrict__ hs, int ip,
              const uint8_t* __restrict__ W, const uint8_t* __restrict__ S, Rows rows, int H, int I,
              float* __restrict__ y) {
  using R = Ring<NT, 1, NW, DEPTH>;
  extern __shared__ __attribute__((aligned(16))) char lds[];   // ring (later sums), scales of W, of h
  const int e = blockIdx.y, r0 = rows.offsets[e], r1 = rows.offsets[e + 1];
  if (r0 >= r1) return;
  const int n0 = blockIdx.x * 16 * NT, r = threadIdx.x & 15, kb = I / BLOCK, kbp = ip / BLOCK;
  char* const ls = lds + R::BYTES;
  char* const lx = ls + whole_kib(16 * NT * kb);
  const Span sp = skinny_span<NW>(I);
  for (int m0 = r0; m0 < r1; m0 += 16) {
    const R ring(lds, W + ((size_t)e * H + n0) * (I / 2), I,
                 [&](int i) { return min(i, H - 1 - n0); }, (const uint8_t*)hw, ip,
                 [&](int i) { return min(m0 + i, r1 - 1); });
    if (m0 > r0) __syncthreads();
    scales_to_lds<NW * 64>(S + ((size_t)e * H + n0) * kb, ls, 16 * NT * kb,
                           min(16 * NT, H - n0) * kb);
    copy_to_lds<NW * 64>(hs + (size_t)m0 * kbp, lx, 16 * kbp);
    skinny_begin<DEPTH>(ring, sp);
    wait_loads<R::LOADS * DEPTH>();
    block_barrier();
    f32x4 acc[1][NT];
    skinny<1, NT, DEPTH>(ring, RingX<NT>{(const uint8_t*)lx + r * kbp, 16 * kbp},
                         (const uint8_t*)ls + r * kb, [=](int nt) { return 16 * nt * kb; }, kb, sp,
                         acc);
    __syncthreads();
    skinny_reduce<1, NT, NW>(acc, (float*)lds, min(16, r1 - m0), [&](int nn, int mm, float v) {
      if (n0 + nn < H) y[(size_t)(m0 + mm) * H + n0 + nn] = v;
    });
  }
}

// Rows of x and of an expert's weights for the tile loop.  act: a wave's 64 weight rows are 32
// rows of the gate and the same 32 of up (I rows on).
struct GroupSrc {
  const uint8_t *W, *S, *X, *XS;
  int K, kp, ks;
  const int32_t* sorted;    // null: rows of x in sorted order
  int k, m0, m_last, n0, n_last, half;
  static constexpr bool BY_UNIT = false;
  MM_DEV uint32_t wrow(int r) const {
    if (half == 0) return min(n0 + r, n_last);
    return min(n0 + r / 64 * 32 + r % 32, half - 1) + (r % 64 / 32) * half;
  }
  MM_DEV uint32_t xrow(int r) const {
    const int m = min(m0 + r, m_last);
    return sorted ? sorted[m] / k : m;
  }
};

// Many rows per expert: tiles of TM rows.  The grid is an upper bound; a block finds its expert
// from the prefix sums of the experts' tiles, and those past the last one leave.
template <class Sh, bool ACT>
__global__ void __launch_bounds__(Sh::NTHR)
k_mx_moe_tile(const uint8_t* __restrict__ X, const uint8_t* __restrict__ XS, int kp,
              const uint8_t* __restrict__ W, const uint8_t* __restrict__ S, int ks, Rows rows, int E,
              int N, int K, int gn, int np, float* __restrict__ y, uint32_t* __restrict__ hw,
              uint8_t* __restrict__ hs) {
  __shared__ __attribute__((aligned(16))) char smem[Sh::LDS];
  static_assert(Sh::LDS >= (MAX_E + 1) * 4, "the prefix sums use the tiles' memory");
  static_assert(!ACT || Sh::NB == 2, "a gate and an up block per wave");
  int* const tp = (int*)smem;
  const int tid = threadIdx.x, lane = tid & 63;
  if (tid < 64) {
    int base = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int e = e0 + lane;
      int n = e < E ? (rows.offsets[e + 1] - rows.offsets[e] + Sh::TM - 1) / Sh::TM : 0;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(n, d);
        if (lane >= d) n += o;
      }
      if (e < E) tp[e + 1] = base + n;
      base += __shfl(n, 63);
    }
    if (lane == 0) tp[0] = 0;
  }
  __syncthreads();
  // each XCD takes one stretch of (row tile, column tile) pairs, column tiles innermost
  const int total = tp[E] * gn, id = blockIdx.x;
  const int q = total >> 3, rem = total & 7, xcd = id & 7;
  if (id >> 3 >= q + (xcd < rem)) return;
  const int lin = xcd * q + min(xcd, rem) + (id >> 3);
  const int tile = lin / gn;
  int lo = 0, hi = E - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (tp[mid] <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int e = __builtin_amdgcn_readfirstlane(lo);
  const int bx = __builtin_amdgcn_readfirstlane(lin - tile * gn);
  const int r1 = __builtin_amdgcn_readfirstlane(rows.offsets[e + 1]);
  const int m0 = __builtin_amdgcn_readfirstlane(rows.offsets[e] + (tile - tp[e]) * Sh::TM);
  __syncthreads();
  const int half = ACT ? N / 2 : 0, n0 = bx * (ACT ? Sh::TN / 2 : Sh::TN);
  const GroupSrc src{W + (size_t)e * N * (K / 2), S + (size_t)e * N * ks, X, XS, K, kp, ks,
                     ACT ? rows.sorted : nullptr, rows.k, m0, r1 - 1, n0, N - 1, half};
  f32x16 acc[Sh::NB][Sh::MB];
  if (!ACT || n0 < half) tile_loop<Sh>(src, 0, (K + UNIT - 1) / UNIT, smem, acc);
  if constexpr (!ACT) {
    __syncthreads();
    tile_out<Sh>(acc, smem, y, F32, r1 - m0, n0, N,
                 [=](int m) { return (size_t)(m0 + m) * N; });
  } else {
    // A block of h is 16 values in each of lanes l and l + 32: n = 8 g + 4 h + i.
    const int wave = tid >> 6, wm = wave / Sh::WN, wn = wave % Sh::WN, l32 = lane & 31;
    const int c0 = n0 + 32 * wn;
    const bool pad = c0 >= half;
#pragma unroll
    for (int mb = 0; mb < Sh::MB; ++mb) {
      float h[16];
      uint32_t amax = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        h[i] = pad ? 0.0f : swiglu(acc[0][mb][i], acc[1][mb][i]);
        amax = max(amax, u32_of(h[i]) & 0x7fffffffu);
      }
      amax = max(amax, (uint32_t)__shfl_xor((int)amax, 32));
      const uint32_t code = scale_code(amax);
      const float s = scale_of(code);
      uint32_t d[2] = {0, 0};                        // halves of words 0, 1 and 2, 3
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        d[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[g], h[8 * g], h[8 * g + 1], s, 0);
        d[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[g], h[8 * g + 2], h[8 * g + 3], s, 1);
        d[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[g], h[8 * g + 4], h[8 * g + 5], s, 2);
        d[g] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d[g], h[8 * g + 6], h[8 * g + 7], s, 3);
      }
      const uint32_t o0 = (uint32_t)__shfl_xor((int)d[0], 32);
      const uint32_t o1 = (uint32_t)__shfl_xor((int)d[1], 32);
      const int m = m0 + (wm * Sh::MB + mb) * 32 + l32;
      if (lane < 32 && m < r1 && c0 < np) {
        *(u32x4*)(hw + (size_t)m * (np / 8) + c0 / 8) =
            u32x4{(d[0] & 0xffffu) | o0 << 16, d[0] >> 16 | (o0 & 0xffff0000u),
                  (d[1] & 0xffffu) | o1 << 16, d[1] >> 16 | (o1 & 0xffff0000u)};
        hs[(size_t)m * (np / 32) + c0 / 32] = (uint8_t)code;
      }
    }
  }
}

// out[t] = sum over j of p[t, j] * y[inverse[t, j]], in slot order; rows past the valid ones are
// those of ids outside [0, E).  y is fp32: rounded to out's type it would add an error as large as
// out's own rounding.
template <int T>
__global__ void __launch_bounds__(256)
k_mx_moe_combine(const float* __restrict__ y, const float* __restrict__ probs,
                 const int32_t* __restrict__ inverse, const int32_t* __restrict__ valid, int k,
                 int H, void* __restrict__ out) {
  const size_t t = blockIdx.x;
  const int nv = *valid;
  for (int c = threadIdx.x * 8; c < H; c += 256 * 8) {
    float sum[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    for (int j = 0; j < k; ++j) {
      const int row = inverse[t * k + j];
      if (row >= nv) continue;
      const float p = probs[t * k + j];
      const f32x4 v[2] = {*(const f32x4*)(y + (size_t)row * H + c),
                          *(const f32x4*)(y + (size_t)row * H + c + 4)};
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[i] += p * v[i / 4][i % 4];
    }
    store4(out, T, t * H + c, f32x4{sum[0], sum[1], sum[2], sum[3]});
    store4(out, T, t * H + c + 4, f32x4{sum[4], sum[5], sum[6], sum[7]});
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
size_t up(size_t n) { return (n + 255) / 256 * 256; }

// Whether an expert's rows are taken in tiles: from 4 of them on average (128 experts, T = 64: 93
// us streamed; T = 128 116), or where 16 rows of x, or an expert's scales, do not fit LDS.
bool takes_tiles(long rows, int E, int H, int I) {
  return rows >= 4L * E || I > 65536 || lds_x_bytes(16, (int)padded(H)) > 65536;
}

template <int T>
void launch_gate_up(const void* X, const uint8_t* W, const uint8_t* S, Rows rows, int R, int E,
                    int H, int I, uint32_t* hw, uint8_t* hs, hipStream_t st) {
  constexpr int NW = 4, DEPTH = 1, U = 2;
  const int hp = (int)padded(H), ip = (int)padded(I);
  const int lds = Ring<4, 0, NW, DEPTH>::BYTES + 2 * whole_kib(32 * (H / BLOCK)) +
                  U * (T == F32 ? 2 : 1) * NW * 1024 + lds_x_bytes(std::min(16, R), hp);
  hipLaunchKernelGGL((k_mx_moe_gate_up<T, NW, DEPTH, U>), dim3(ip / 32, E), dim3(NW * 64), lds, st,
                     (const char*)X, W, S, rows, H, hp, I, ip, hw, hs);
}

struct Scratch {
  size_t sort, xq, gs, ds, hq, y, total;
};
Scratch scratch_of(int T, int k, int E, int H, int I) {
  const size_t R = (size_t)T * k;
  const bool tiles = takes_tiles((long)R, E, H, I);
  const auto anew = [&](size_t rows, int K) {      // scales that the tiles take from a copy
    return tiles && scale_stride(K) != K / BLOCK ? up(rows * scale_stride(K)) : 0;
  };
  Scratch s;
  s.sort = 0;
  s.xq = up((E + 1 + 2 * R) * sizeof(int32_t));
  s.gs = s.xq + (tiles ? up(packed_bytes(T, H)) : 0);
  s.ds = s.gs + anew((size_t)E * 2 * I, H);
  s.hq = s.ds + anew((size_t)E * H, I);
  s.y = s.hq + up(packed_bytes(R, I));
  s.total = s.y + up(R * H * sizeof(float));
  return s;
}

}  // namespace

extern "C" size_t mm_moe_mlp_mxfp4_scratch_bytes(int T, int k, int E, int H, int I) {
  if (T <= 0 || k <= 0 || E <= 0 || H <= 0 || I <= 0) return 0;
  return scratch_of(T, k, E, H, I).total;
}

extern "C" int mm_moe_mlp_mxfp4(const void* X, int type, const void* expert_ids, int ids_i64,
                                const float* probs, int T, int k, int E, int H, int I,
                                const uint32_t* Wgu, const uint8_t* Sgu, const uint32_t* Wdn,
                                const uint8_t* Sdn, void* scratch, size_t scratch_bytes, void* out,
                                void* stream) {
  MM_CHECK_ARG(T >= 0 && k > 0 && E > 0 && E <= MAX_E,
               "mm_moe_mlp_mxfp4: T=%d, k=%d, E=%d: k > 0 and at most %d experts", T, k, E, MAX_E);
  MM_CHECK_ARG(H > 0 && I > 0 && H % BLOCK == 0 && I % BLOCK == 0,
               "mm_moe_mlp_mxfp4: H=%d, I=%d must be positive multiples of %d", H, I, BLOCK);
  MM_CHECK_ARG(type >= F32 && type <= BF16, "mm_moe_mlp_mxfp4: unknown type %d", type);
  MM_CHECK_ARG((long long)T * k < (1LL << 28), "mm_moe_mlp_mxfp4: T*k=%lld is too large",
               (long long)T * k);
  if (T == 0) return 0;
  MM_CHECK_ARG(X && expert_ids && probs && Wgu && Sgu && Wdn && Sdn && out && aligned16(X) &&
                   aligned16(Wgu) && aligned16(Wdn) && aligned16(Sgu) && aligned16(Sdn) &&
                   aligned16(out),
               "mm_moe_mlp_mxfp4: X, weights, scales and out must be 16-byte aligned and nothing null");
  const Scratch sc = scratch_of(T, k, E, H, I);
  MM_CHECK_ARG(scratch && aligned16(scratch) && scratch_bytes >= sc.total,
               "mm_moe_mlp_mxfp4: needs %zu bytes of scratch, 16-byte aligned, got %zu", sc.total,
               scratch_bytes);
  const int R = T * k, hp = (int)padded(H), ip = (int)padded(I);
  // the tile loop's row offsets within one expert's weights, the tokens and h
  MM_CHECK_ARG((size_t)2 * I * (H / 2) < ((size_t)1 << 32) && (size_t)H * (I / 2) < ((size_t)1 << 32) &&
                   (size_t)T * (hp / 2) < ((size_t)1 << 32) && (size_t)R * (ip / 2) < ((size_t)1 << 32),
               "mm_moe_mlp_mxfp4: one expert's words, the tokens' or h's reach 4 GiB");
  char* const base = (char*)scratch;
  int32_t* const offsets = (int32_t*)(base + sc.sort);
  int32_t *const sorted = offsets + E + 1, *const inverse = sorted + R;
  const hipStream_t st = (hipStream_t)stream;
  if (const int rc = ids_i64 ? mm_moe_sort_i64((const int64_t*)expert_ids, T, k, E, offsets, sorted,
                                               inverse, stream)
                             : mm_moe_sort((const int32_t*)expert_ids, T, k, E, offsets, sorted,
                                           inverse, stream))
    return rc;
  const Rows rows{offsets, sorted, k};
  uint32_t* const hw = (uint32_t*)(base + sc.hq);
  uint8_t* const hs = (uint8_t*)hw + codes_bytes(R, I);
  float* const y = (float*)(base + sc.y);
  const uint8_t *gw = (const uint8_t*)Wgu, *dw = (const uint8_t*)Wdn;
  if (takes_tiles(R, E, H, I)) {
    uint8_t* const xq = (uint8_t*)base + sc.xq;
    uint8_t* const xs = xq + codes_bytes(T, H);
    if (const int rc = launch_quantize(X, type, T, H, hp, (uint32_t*)xq, xs, st)) return rc;
    // 64 x 128: three blocks share a CU.  us of both products, 1000 tokens of 128 experts of 2048 ->
    // 768: 71 + 43; of 128 x 128 73 + 47, with rings of three 76 + 51, of 64 x 256 104 + 54.
    using Sh = Tile<2, 2, 1, 2>;
    const uint8_t *gs = Sgu, *ds = Sdn;
    if (scale_stride(H) != H / BLOCK) {
      uint8_t* const s = (uint8_t*)base + sc.gs;
      if (const int rc = launch_pad_scales(gs, (size_t)E * 2 * I, H / BLOCK, scale_stride(H), s, st))
        return rc;
      gs = s;
    }
    if (scale_stride(I) != I / BLOCK) {
      uint8_t* const s = (uint8_t*)base + sc.ds;
      if (const int rc = launch_pad_scales(ds, (size_t)E * H, I / BLOCK, scale_stride(I), s, st))
        return rc;
      ds = s;
    }
    const long tiles = (R + Sh::TM - 1) / Sh::TM + std::min(E, R);
    const int g1 = mm_cdiv(ip, Sh::TN / 2), g2 = mm_cdiv(H, Sh::TN);
    MM_CHECK_ARG(launch_holds(tiles * std::max(g1, g2) + 7, Sh::NTHR), "mm_moe_mlp_mxfp4: too many tiles");
    hipLaunchKernelGGL((k_mx_moe_tile<Sh, true>), dim3((unsigned)((tiles * g1 + 7) / 8 * 8)),
                       dim3(Sh::NTHR), 0, st, xq, xs, hp, gw, gs, scale_stride(H), rows, E, 2 * I, H, g1, ip,
                       nullptr, hw, hs);
    hipLaunchKernelGGL((k_mx_moe_tile<Sh, false>), dim3((unsigned)((tiles * g2 + 7) / 8 * 8)),
                       dim3(Sh::NTHR), 0, st, (const uint8_t*)hw, hs, ip, dw, ds, scale_stride(I), rows, E, H, I,
                       g2, 0, y, nullptr, nullptr);
  } else {
    if (type == F32) launch_gate_up<F32>(X, gw, Sgu, rows, R, E, H, I, hw, hs, st);
    else if (type == F16) launch_gate_up<F16>(X, gw, Sgu, rows, R, E, H, I, hw, hs, st);
    else launch_gate_up<BF16>(X, gw, Sgu, rows, R, E, H, I, hw, hs, st);
    using Rg = Ring<2, 1, 4, 1>;
    hipLaunchKernelGGL((k_mx_moe_down<2, 4, 1>), dim3(mm_cdiv(H, 32), E), dim3(256),
                       (Rg::BYTES + whole_kib(32 * (I / BLOCK)) + whole_kib(16 * (ip / BLOCK))), st,
                       (const uint8_t*)hw, hs, ip, dw, Sdn, rows, H, I, y);
  }
#define MM_MX_COMBINE(T)                                                                         \
  hipLaunchKernelGGL((k_mx_moe_combine<T>), dim3(T_), dim3(256), 0, st, y, probs,     \
                     inverse, offsets + E, k, H, out)
  const int T_ = T;
  if (type == F32) MM_MX_COMBINE(F32);
  else if (type == F16) MM_MX_COMBINE(F16);
  else MM_MX_COMBINE(BF16);
#undef MM_MX_COMBINE
  MM_CHECK_LAUNCH("mm_moe_mlp_mxfp4");
  return 0;
}
