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

// A wave takes QU * 16 blocks that lie side by side in the padded rows: kp / 32 blocks a row, of
// which the first K / 32 are x's and the others zeros.  PAD = false: kp == K, all one row.
template <int T, bool PAD>
__global__ void __launch_bounds__(QT)
k_mx_quantize(const char* __restrict__ x, size_t blocks, int kb, int kbp,
              uint32_t* __restrict__ words, uint8_t* __restrict__ scales) {
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
      if (sub == 0) scales[b] = (uint8_t)code;
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

template <int T>
void quantize_t(const void* x, size_t rows, int K, size_t kp, uint32_t* words, uint8_t* scales,
                hipStream_t stream) {
  const int kb = K / BLOCK, kbp = (int)(kp / BLOCK);
  const size_t blocks = rows * kbp, per = QT / 4 * QU;
  const dim3 grid((unsigned)((blocks + per - 1) / per));
  if (kb == kbp)
    hipLaunchKernelGGL((k_mx_quantize<T, false>), grid, dim3(QT), 0, stream, (const char*)x, blocks,
                       kb, kbp, words, scales);
  else
    hipLaunchKernelGGL((k_mx_quantize<T, true>), grid, dim3(QT), 0, stream, (const char*)x, blocks,
                       kb, kbp, words, scales);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Blocks that one launch takes: a grid has at most 2^31 - 1 thread blocks of 256 MX blocks.
constexpr size_t MAX_BLOCKS = (size_t)1 << 38;

}  // namespace

int mmmx::launch_quantize(const void* x, int type, size_t rows, int K, size_t kp, uint32_t* words,
                          uint8_t* scales, hipStream_t stream) {
  if (type == F32) quantize_t<F32>(x, rows, K, kp, words, scales, stream);
  else if (type == F16) quantize_t<F16>(x, rows, K, kp, words, scales, stream);
  else quantize_t<BF16>(x, rows, K, kp, words, scales, stream);
  MM_CHECK_LAUNCH("MXFP4 quantization");
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
