// Microscaled 4-bit floating point (MXFP4, the OCP microscaling format's FP4 type): blocks of 32
// values along K share one power of two, E8M0 code c = 2^(c - 127), and every value is E2M1.
//   words  uint32 [rows, K/8]   word j holds values 8j..8j+7 of its row in bits 4i..4i+3
//   scales uint8  [rows, K/32]  255: the block holds a NaN or an infinity and stands for NaNs
// A block with largest magnitude a is scaled by 2^(floor(log2 a) - 2), at least 2^-127; values
// are rounded to nearest, ties to the even code, and saturate at 6 (which those of [7, 8) times
// the scale need).  Both steps are exact but for that rounding: the scale only moves exponents.
//
// gfx950 multiplies such blocks directly: v_mfma_scale_f32_32x32x64_f8f6f4 (and 16x16x128) takes
// 16 bytes, one block of a row, and one scale byte per lane, so a row's words need no rearranging,
// and a NaN scale gives NaNs whatever the codes are.  Conversions are v_cvt_scalef32_pk_*, which
// take the scale as an fp32 power of two, 2^-127 included.
#pragma once

#include "mm_common.h"

namespace mmmx {

typedef __bf16 bf16;
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 32;            // values that share a scale
constexpr int UNIT = 256;            // k of one step of the products: 128 bytes of a row's words
enum Type { F32 = 0, F16 = 1, BF16 = 2 };

MM_DEV uint32_t u32_of(float f) { return __builtin_bit_cast(uint32_t, f); }
MM_DEV float f32_of(uint32_t u) { return __builtin_bit_cast(float, u); }

// By value: a bit cast of a vector's element itself reads element 0.
MM_DEV f16x2 as_f16x2(uint32_t u) { return __builtin_bit_cast(f16x2, u); }
MM_DEV bf16x2 as_bf16x2(uint32_t u) { return __builtin_bit_cast(bf16x2, u); }

// E8M0 code of a block from the fp32 bits of its largest magnitude.
MM_DEV uint32_t scale_code(uint32_t amax_bits) {
  const uint32_t e = amax_bits >> 23;
  return e == 255u ? 255u : (e > 2u ? e - 2u : 0u);
}
// 2^(code - 127); code 255 gives an infinity.
MM_DEV float scale_of(uint32_t code) { return f32_of(code ? code << 23 : 0x00400000u); }

// Eight values of one row as they are loaded.
template <int T>
struct Vals {
  u32x4 v;
};
template <>
struct Vals<F32> {
  f32x4 v[2];
};
template <int T>
constexpr int kBytes = T == F32 ? 4 : 2;

template <int T>
MM_DEV Vals<T> load8(const void* p) {
  return *(const Vals<T>*)p;
}
template <int T>
MM_DEV Vals<T> zero8() {
  return Vals<T>{};
}

// The largest magnitude, as bits that order as magnitudes do (NaN last): 16 of them for the
// 16-bit types.
template <int T>
MM_DEV uint32_t amax8(const Vals<T>& x) {
  if constexpr (T == F32) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, u32_of(x.v[i / 4][i % 4]) & 0x7fffffffu);
    return m;
  } else {
    u16x2 m = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x.v[i] & 0x7fff7fffu));
    return max((uint32_t)m.x, (uint32_t)m.y);
  }
}
template <int T>
MM_DEV uint32_t amax_bits(uint32_t m) {
  if constexpr (T == F32) return m;
  if constexpr (T == BF16) return m << 16;
  return u32_of((float)__builtin_bit_cast(f16, (uint16_t)m));
}

// Eight values to one word of codes.
template <int T>
MM_DEV uint32_t pack8(const Vals<T>& x, float scale) {
  uint32_t w = 0;
  if constexpr (T == F32) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.v[0][0], x.v[0][1], scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.v[0][2], x.v[0][3], scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.v[1][0], x.v[1][1], scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x.v[1][2], x.v[1][3], scale, 3);
  } else if constexpr (T == F16) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, as_f16x2(x.v[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, as_f16x2(x.v[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, as_f16x2(x.v[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, as_f16x2(x.v[3]), scale, 3);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_bf16x2(x.v[0]), scale, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_bf16x2(x.v[1]), scale, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_bf16x2(x.v[2]), scale, 2);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, as_bf16x2(x.v[3]), scale, 3);
  }
  return w;
}

// One block held by one lane.
template <int T>
MM_DEV u32x4 pack_block(const Vals<T> (&x)[4], uint32_t& code) {
  uint32_t m = amax8<T>(x[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) m = max(m, amax8<T>(x[i]));
  code = scale_code(amax_bits<T>(m));
  const float s = scale_of(code);
  return u32x4{pack8<T>(x[0], s), pack8<T>(x[1], s), pack8<T>(x[2], s), pack8<T>(x[3], s)};
}

MM_DEV i32x8 operand(u32x4 v) {
  return i32x8{(int)v.x, (int)v.y, (int)v.z, (int)v.w, 0, 0, 0, 0};
}
// D[16 x 16] += A[16 x 128] . B[16 x 128]^T: lane l holds block l / 16 of row l % 16, and rows
// 4 (l / 16) + i of column l % 16 of D.  SA, SB: which byte of sa, sb is the scale.
template <int SA, int SB>
MM_DEV f32x4 mfma16(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(a), operand(b), c, 4, 4, SA,
                                                          (int)sa, SB, (int)sb);
}
// D[32 x 32] += A[32 x 64] . B[32 x 64]^T: lane l holds block l / 32 of row l % 32, and rows
// 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32 of D.
template <int SA, int SB>
MM_DEV f32x16 mfma32(u32x4 a, uint32_t sa, u32x4 b, uint32_t sb, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(operand(a), operand(b), c, 4, 4, SA,
                                                         (int)sa, SB, (int)sb);
}

MM_DEV uint16_t to16(int type, float v) {
  return type == F16 ? __builtin_bit_cast(uint16_t, (f16)v)
                     : __builtin_bit_cast(uint16_t, (bf16)v);
}
// One result, rounded once.
MM_DEV void store1(void* C, int type, size_t i, float v) {
  if (type == F32) ((float*)C)[i] = v;
  else ((uint16_t*)C)[i] = to16(type, v);
}
// Four results that lie side by side at an index divisible by 4.
MM_DEV void store4(void* C, int type, size_t i, f32x4 v) {
  if (type == F32) {
    *(f32x4*)((float*)C + i) = v;
    return;
  }
  const u32x2 p = {to16(type, v[0]) | (uint32_t)to16(type, v[1]) << 16,
                   to16(type, v[2]) | (uint32_t)to16(type, v[3]) << 16};
  *(u32x2*)((uint16_t*)C + i) = p;
}

// A launch has fewer than 2^32 threads along an axis.
inline bool launch_holds(size_t blocks, size_t threads) {
  return blocks < ((size_t)1 << 32) / threads;
}

inline const char* type_name(int t) {
  return t == F32 ? "fp32" : (t == F16 ? "fp16" : (t == BF16 ? "bf16" : "?"));
}

// Quantized rows in a workspace: words [rows, kp/8] and scales [rows, kp/32], kp = K padded to a
// multiple of 512 with zeros, so that a row's scales are whole 16-byte pieces; behind the last row
// there is room for the scales of 63 more, which kernels may read and never use.
inline size_t padded(int K) { return ((size_t)K + 511) / 512 * 512; }
inline size_t codes_bytes(size_t rows, int K) { return rows * padded(K) / 2; }
inline size_t packed_bytes(size_t rows, int K) {
  return codes_bytes(rows, K) + (rows + 63) * padded(K) / BLOCK;
}
// x [rows, K] of `type` to words and scales whose rows are kp values long (kp >= K, zeros behind
// K).
int launch_quantize(const void* x, int type, size_t rows, int K, size_t kp, uint32_t* words,
                    uint8_t* scales, hipStream_t stream);

// The same for tiles, which take scales by units of 256 values, 8 of each row side by side and
// unit_pitch(rows) from unit to unit (there is room for the rows of whole tiles); in the same
// launch the scales S of the weights [N, K] go to `units` in that order.
inline __host__ __device__ size_t unit_pitch(size_t rows) { return (rows + 255) / 256 * 2048; }
int launch_quantize_units(const void* x, int type, size_t rows, int K, size_t kp, uint32_t* words,
                          uint8_t* scales, const uint8_t* S, size_t N, uint8_t* units,
                          hipStream_t stream);

// Rows of `kb` scales to rows of `ks` >= kb, zeros behind: where kb is no multiple of 4, the tiles,
// which copy four at a time, take such a copy.
inline int scale_stride(int K) { return K / BLOCK % 4 == 0 ? K / BLOCK : (K / BLOCK + 3) / 4 * 4; }
int launch_pad_scales(const uint8_t* s, size_t rows, int kb, int ks, uint8_t* out, hipStream_t stream);

// out[i] = sum over s of part[s][i], in order, rounded once; part[s] begins s * sum_pitch(n) on.
__host__ __device__ inline size_t sum_pitch(size_t n) { return (n + 3) / 4 * 4; }
int launch_sum(const float* part, int splits, size_t n, void* out, int type, hipStream_t stream);

}  // namespace mmmx
