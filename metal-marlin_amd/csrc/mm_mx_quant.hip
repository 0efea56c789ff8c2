// MXFP4 quantization and its inverse (mm_mx.h has the format).
//
// Both are bound by HBM: b bytes in and 17/32 out per value, or the reverse.  Four lanes share a
// block of 32, eight values each, so that a wave reads 1 KiB (16-bit types; 2 KiB of fp32) in one
// stretch and writes 256 bytes of words in one; the block's largest magnitude is two lane
// exchanges.  A lane's 8 values become one word in four conversions.
#include "mm_mx.h"
#include "mmfp4.h"

using namespace mmmx;

namespace {

constexpr int QT = 256, QU = 4;    // threads; groups of 8 values per thread, loaded together

// Scales that are to lie by units, 8 of each row side by side: x's own (pitch != 0: the bytes from
// unit to unit), and in blocks from `first` on those S of a matrix of n rows of kb, 64 rows by 16
// units a block (a wave reads 64 pieces of 8 bytes and writes 512 bytes in one; the lines that it
// reads serve all 16 units).  Zeros behind kb.
struct Units {
  size_t pitch;
  const uint8_t* S;
  uint8_t* to;
  size_t to_pitch;
  int n, units;
  uint32_t first, across;       // across: blocks that share 64 rows
};
MM_DEV void scales_by_units(const Units& g, int kb) {
  const uint32_t id = blockIdx.x - g.first;
  const int row = (int)(id / g.across) * 64 + (threadIdx.x & 63);
  const int u0 = (int)(id % g.across) * 16 + (threadIdx.x >> 6);
  if (row >= g.n) return;
  const uint8_t* const s = g.S + (size_t)row * kb;
  u32x2 v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int at = (u0 + 4 * i) * 8;
    v[i] = u32x2{0, 0};
    if (kb % 8 == 0) {
      if (at < kb) v[i] = *(const u32x2*)(s + at);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (at + j < kb) v[i][j / 4] |= (uint32_t)s[at + j] << (8 * (j % 4));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (u0 + 4 * i < g.units) *(u32x2*)(g.to + (u0 + 4 * i) * g.to_pitch + (size_t)row * 8) = v[i];
}

// A wave takes QU * 16 blocks that lie side by side in the padded rows: kp / 32 blocks a row, of
// which the first K / 32 are x's and the others zeros.  PAD = false: kp == K, all one row.
template <int T, bool PAD, bool UNITS>
__global__ void __launch_bounds__(QT)
k_mx_quantize(const char* __restrict__ x, size_t blocks, int kb, int kbp,
              uint32_t* __restrict__ words, uint8_t* __restrict__ scales, Units g) {
  static_assert(PAD || !UNITS, "rows are told apart");
  if constexpr (UNITS)
    if (blockIdx.x >= g.first) return scales_by_units(g, kb);
  const int lane = threadIdx.x & 63, sub = lane & 3;
  const size_t wave = (size_t)blockIdx.x * (QT / 64) + (threadIdx.x >> 6);
  const size_t b0 = wave * (QU * 16) + lane / 4;
  Vals<T> v[QU];
  bool live[QU];
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    const size_t b = b0 + 16 * u;
    size_t src = b;
    live[u] = b < blocks;
    if constexpr (PAD) {
      const size_t row = b / (uint32_t)kbp;
      const int at = (int)(b - row * kbp);
      live[u] = live[u] && at < kb;
      src = row * kb + at;
    }
    v[u] = live[u] ? load8<T>(x + (src * BLOCK + 8 * sub) * kBytes<T>) : zero8<T>();
  }
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    const size_t b = b0 + 16 * u;
    uint32_t m = amax8<T>(v[u]);
    m = max(m, (uint32_t)__shfl_xor((int)m, 1));
    m = max(m, (uint32_t)__shfl_xor((int)m, 2));
    const uint32_t code = scale_code(amax_bits<T>(m));
    if (b < blocks) {
      words[b * 4 + sub] = pack8<T>(v[u], scale_of(code));
      if (sub == 0) {
        size_t at = b;
        if constexpr (UNITS) {
          const size_t row = b / (uint32_t)kbp;
          const int c = (int)(b - row * kbp);
          if (c >= 8 * g.units) continue;
          at = (size_t)(c / 8) * g.pitch + row * 8 + c % 8;
        }
        scales[at] = (uint8_t)code;
      }
    }
  }
}

// One word per lane and step: 8 values of type T.
template <int T>
__global__ void __launch_bounds__(QT)
k_mx_dequantize(const uint32_t* __restrict__ words, const uint8_t* __restrict__ scales, size_t n,
                char* __restrict__ out) {
  const size_t i0 = (size_t)blockIdx.x * (QT * QU) + threadIdx.x;
  uint32_t w[QU], c[QU];
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    const size_t i = min(i0 + QT * u, n - 1);
    w[u] = words[i];
    c[u] = scales[i / 4];
  }
#pragma unroll
  for (int u = 0; u < QU; ++u) {
    const size_t i = i0 + QT * u;
    if (i >= n) return;
    const float s = scale_of(c[u]);
    const bool nan = c[u] == 255u;
    char* o = out + i * 8 * kBytes<T>;
    if constexpr (T == BF16) {   // exact, to the ends of the range
      u32x4 r = {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[u], s, 3))};
      if (nan) r = u32x4{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u};
      *(u32x4*)o = r;
    } else {
      f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 0),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 1),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 2),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 3)};
      if (nan)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = f32x2{__builtin_nanf(""), __builtin_nanf("")};
      if constexpr (T == F32) {
        *(f32x4*)o = f32x4{p[0].x, p[0].y, p[1].x, p[1].y};
        *(f32x4*)(o + 16) = f32x4{p[2].x, p[2].y, p[3].x, p[3].y};
      } else {                   // rounded once from the exact fp32 value
        *(f16x8*)o = f16x8{(f16)p[0].x, (f16)p[0].y, (f16)p[1].x, (f16)p[1].y,
                           (f16)p[2].x, (f16)p[2].y, (f16)p[3].x, (f16)p[3].y};
      }
    }
  }
}

__global__ void __launch_bounds__(QT)
k_mx_pad_scales(const uint8_t* __restrict__ s, size_t n, int kb, int ks, uint32_t* __restrict__ out) {
  const size_t i = (size_t)blockIdx.x * QT + threadIdx.x;      // four scales
  if (i >= n) return;
  const size_t row = i / (uint32_t)(ks / 4);
  const int c = (int)(i - row * (ks / 4)) * 4;
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (c + j < kb) w |= (uint32_t)s[row * kb + c + j] << (8 * j);
  out[i] = w;
}

// Each split's n sums begin at a multiple of 4.
__global__ void __launch_bounds__(QT)
k_mx_sum(const float* __restrict__ part, int splits, size_t n, void* __restrict__ out, int type) {
  const size_t i = ((size_t)blockIdx.x * QT + threadIdx.x) * 4, pitch = (n + 3) / 4 * 4;
  if (i >= n) return;
  f32x4 v = *(const f32x4*)(part + i);
  for (int s = 1; s < splits; ++s) v += *(const f32x4*)(part + (size_t)s * pitch + i);
  if (i + 4 <= n) {
    store4(out, type, i, v);
  } else {
    for (int j = 0; i + j < n; ++j) store1(out, type, i + j, v[j]);
  }
}

constexpr size_t PER = QT / 4 * QU;      // MX blocks per thread block

template <int T>
void quantize_t(const void* x, size_t rows, int K, size_t kp, uint32_t* words, uint8_t* scales,
                Units g, hipStream_t stream) {
  const int kb = K / BLOCK, kbp = (int)(kp / BLOCK);
  const size_t blocks = rows * kbp;
  const uint32_t own = (uint32_t)((blocks + PER - 1) / PER);
  if (g.pitch) {
    g.first = own;
    g.across = (g.units + 15) / 16;
    hipLaunchKernelGGL((k_mx_quantize<T, true, true>), dim3(own + (g.n + 63) / 64 * g.across), dim3(QT),
                       0, stream, (const char*)x, blocks, kb, kbp, words, scales, g);
  } else if (kb == kbp) {
    hipLaunchKernelGGL((k_mx_quantize<T, false, false>), dim3(own), dim3(QT), 0, stream,
                       (const char*)x, blocks, kb, kbp, words, scales, g);
  } else {
    hipLaunchKernelGGL((k_mx_quantize<T, true, false>), dim3(own), dim3(QT), 0, stream,
                       (const char*)x, blocks, kb, kbp, words, scales, g);
  }
}
int quantize(const void* x, int type, size_t rows, int K, size_t kp, uint32_t* words, uint8_t* scales,
             const Units& g, hipStream_t stream) {
  const size_t own = (rows * (kp / BLOCK) + PER - 1) / PER;
  MM_CHECK_ARG(launch_holds(own + ((size_t)g.n + 63) / 64 * ((g.units + 15) / 16), QT),
               "MXFP4 quantization: %zu rows of %d are too many", rows, K);
  if (type == F32) quantize_t<F32>(x, rows, K, kp, words, scales, g, stream);
  else if (type == F16) quantize_t<F16>(x, rows, K, kp, words, scales, g, stream);
  else quantize_t<BF16>(x, rows, K, kp, words, scales, g, stream);
  MM_CHECK_LAUNCH("MXFP4 quantization");
  return 0;
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// MX blocks that one launch takes: each has one thread.
static_assert(PER == QT, "a thread per block");
constexpr size_t MAX_BLOCKS = ((size_t)1 << 32) - 2 * QT;

}  // namespace

int mmmx::launch_quantize(const void* x, int type, size_t rows, int K, size_t kp, uint32_t* words,
                          uint8_t* scales, hipStream_t stream) {
  return quantize(x, type, rows, K, kp, words, scales, Units{}, stream);
}

int mmmx::launch_quantize_units(const void* x, int type, size_t rows, int K, size_t kp,
                                uint32_t* words, uint8_t* scales, const uint8_t* S, size_t N,
                                uint8_t* units, hipStream_t stream) {
  const Units g{unit_pitch(rows), S, units, unit_pitch(N), (int)N, (K + 255) / 256, 0, 0};
  return quantize(x, type, rows, K, kp, words, scales, g, stream);
}

int mmmx::launch_pad_scales(const uint8_t* s, size_t rows, int kb, int ks, uint8_t* out,
                            hipStream_t stream) {
  const size_t n = rows * (ks / 4);
  MM_CHECK_ARG(launch_holds((n + QT - 1) / QT, QT), "MXFP4 scales: %zu rows of %d are too many", rows,
               kb);
  hipLaunchKernelGGL(k_mx_pad_scales, dim3((unsigned)((n + QT - 1) / QT)), dim3(QT), 0, stream, s, n,
                     kb, ks, (uint32_t*)out);
  MM_CHECK_LAUNCH("MXFP4 scales");
  return 0;
}

int mmmx::launch_sum(const float* part, int splits, size_t n, void* out, int type,
                     hipStream_t stream) {
  hipLaunchKernelGGL(k_mx_sum, dim3((unsigned)(((n + 3) / 4 + QT - 1) / QT)), dim3(QT), 0, stream, part,
                     splits, n, out, type);
  MM_CHECK_LAUNCH("MXFP4 partial sums");
  return 0;
}

extern "C" int mm_mxfp4_quantize(const void* X, int type, long long rows, int K, uint32_t* words,
                                 uint8_t* scales, void* stream) {
  MM_CHECK_ARG(rows >= 0 && K > 0 && K % BLOCK == 0,
               "mm_mxfp4_quantize: rows=%lld, K=%d: K must be a positive multiple of %d", rows, K,
               BLOCK);
  MM_CHECK_ARG(type >= F32 && type <= BF16, "mm_mxfp4_quantize: unknown type %d", type);
  if (rows == 0) return 0;
  MM_CHECK_ARG((size_t)rows <= MAX_BLOCKS / (K / BLOCK), "mm_mxfp4_quantize: too many values");
  MM_CHECK_ARG(X && words && scales && aligned16(X) && aligned16(words),
               "mm_mxfp4_quantize: X and words must be 16-byte aligned and not null");
  return launch_quantize(X, type, (size_t)rows, K, K, words, scales, (hipStream_t)stream);
}

extern "C" int mm_mxfp4_dequantize(const uint32_t* words, const uint8_t* scales, long long rows,
                                   int K, void* out, int type, void* stream) {
  MM_CHECK_ARG(rows >= 0 && K > 0 && K % BLOCK == 0,
               "mm_mxfp4_dequantize: rows=%lld, K=%d: K must be a positive multiple of %d", rows, K,
               BLOCK);
  MM_CHECK_ARG(type >= F32 && type <= BF16, "mm_mxfp4_dequantize: unknown type %d", type);
  if (rows == 0) return 0;
  MM_CHECK_ARG((size_t)rows <= MAX_BLOCKS / (K / BLOCK), "mm_mxfp4_dequantize: too many values");
  MM_CHECK_ARG(words && scales && out && ((uintptr_t)words & 3) == 0 && aligned16(out),
               "mm_mxfp4_dequantize: out must be 16-byte aligned and nothing null");
  const size_t n = (size_t)rows * K / 8;
  const dim3 grid((unsigned)((n + QT * QU - 1) / (QT * QU)));
  const hipStream_t st = (hipStream_t)stream;
  if (type == F32)
    hipLaunchKernelGGL((k_mx_dequantize<F32>), grid, dim3(QT), 0, st, words, scales, n, (char*)out);
  else if (type == F16)
    hipLaunchKernelGGL((k_mx_dequantize<F16>), grid, dim3(QT), 0, st, words, scales, n, (char*)out);
  else
    hipLaunchKernelGGL((k_mx_dequantize<BF16>), grid, dim3(QT), 0, st, words, scales, n,
                       (char*)out);
  MM_CHECK_LAUNCH("mm_mxfp4_dequantize");
  return 0;
}
