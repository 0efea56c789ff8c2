// Low-rank adapters of many requests beside a shared projection, and their gradients:
//   out[t] = base[t] + s_a (x[t] A_a^T) B_a^T,   a = ids[t]   (no adapter: out = base)
//   H = s x A^T, dH = s dy B;   dx = dx_base + dH A,   dA_a = sum dH[t]^T x[t],
//   dB_a = sum dy[t]^T H[t]     over the tokens t of adapter a
// with A [L, r, K], B [L, N, r], s = scale * scaling[a] (scaling fp32 [L], or none).
//
// Few tokens: every token on its own, two launches of fp32 dot products (k_vec_down,
// k_vec_up).  Otherwise the tokens are sorted by adapter (mm_moe_sort) and cut into tiles
// of 32 of one adapter:
//   k_down   H of a tile, over the whole width: 16x16x32 MFMAs, the width split over the
//            waves and over blocks.  The block that finishes a tile leaves a record of it:
//            H as hi + lo in the operands' type, under one power of two per tile that puts
//            the tile's largest value in [2^14, 2^15): 16 (bf16) or 22 (fp16) bits of H
//            reach the second product, whatever its size.  The record has H by token and
//            by rank, the operand orders of the two kernels that follow.
//   k_up     out of a tile: MFMAs over [hi | lo] of 16 ranks at a time.
//   k_wgrad  dA_a or dB_a: MFMAs over the 32 tokens of a tile, tile after tile.
// All sums are fp32 and in a fixed order.  All three kernels stream activations that are
// read once (x, dy) or read and written once (out): HBM bounds them, the factors stay in L2.
#include <algorithm>

#include "mm_common.h"
#include "mmfp4.h"

namespace {

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
// Rows of any width start at any even address.
typedef u16x4 u16x4_any __attribute__((aligned(2)));
typedef u16x8 u16x8_any __attribute__((aligned(2)));

constexpr int LO_TM = 32;               // tokens per tile
constexpr int LO_NT = 256;              // threads per block
constexpr int LO_COLS = 256;            // columns per block of k_up and k_wgrad: 64 a wave
// Arrival counters at the head of the workspace, where every entry point has them.
constexpr size_t LO_COUNTER_BYTES = (size_t)16384 * sizeof(uint32_t);

// T: 1 fp16, 2 bf16 (the type codes of the C ABI).
template <int T>
MM_DEV float to_f32(uint16_t v) {
  if constexpr (T == 1) return (float)__builtin_bit_cast(f16, v);
  else return __builtin_bit_cast(float, (uint32_t)v << 16);
}
template <int T>
MM_DEV uint16_t from_f32(float v) {   // to nearest even
  if constexpr (T == 1) return __builtin_bit_cast(uint16_t, (f16)v);
  else return __builtin_bit_cast(uint16_t, (bf16)v);
}
template <int T>
MM_DEV f32x4 mfma(u16x8 a, u16x8 b, f32x4 c) {
  if constexpr (T == 1)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// n of 8 (4) values from p on, zeros behind them; n <= 0 reads nothing.
MM_DEV u16x8 load8(const uint16_t* p, int n) {
  if (n >= 8) return *(const u16x8_any*)p;
  u16x8 v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 7; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
MM_DEV u16x4 load4(const uint16_t* p, int n) {
  if (n >= 4) return *(const u16x4_any*)p;
  u16x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
MM_DEV void store4(uint16_t* p, u16x4 v, int n) {
  if (n >= 4) {
    *(u16x4_any*)p = v;
    return;
  }
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) p[i] = v[i];
}
// Eight rows of four values -> four columns of eight (the MFMA operand of each column).
MM_DEV void transpose84(const u16x4 (&v)[8], u16x8 (&o)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const u32x2 a = __builtin_bit_cast(u32x2, v[2 * p]), b = __builtin_bit_cast(u32x2, v[2 * p + 1]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t x = __builtin_amdgcn_perm(b[j >> 1], a[j >> 1],
                                               (j & 1) ? 0x07060302u : 0x05040100u);
      o[j][2 * p] = (uint16_t)x;
      o[j][2 * p + 1] = (uint16_t)(x >> 16);
    }
  }
}

// ---------------------------------------------------------------------------
// Tokens sorted by adapter: group e (e < L: adapter e; e == L: none) holds sorted rows
// [first(e), first(e + 1)); order maps them to tokens.  offsets == nullptr: one adapter
// for all tokens, in their own order.
// ---------------------------------------------------------------------------
struct Groups {
  const int *offsets, *order;
  int T, L;
  MM_DEV int first(int e) const {
    if (offsets == nullptr) return e == 0 ? 0 : T;
    return e <= L ? offsets[e] : T;
  }
  MM_DEV int token(int row) const { return order != nullptr ? order[row] : row; }
};

struct Scaling {
  const float* p;
  float scale;
  MM_DEV float at(int e) const { return p != nullptr ? scale * p[e] : scale; }
};

struct Tile {
  int e, row0, rows;   // group, first sorted row, rows; e < 0: no such tile
};
// Tile b of the groups' tiles, counted group by group over `ngroups` groups.  Every lane
// of the wave takes part.
MM_DEV Tile find_tile(const Groups& gs, int ngroups, int b) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int e0 = 0; e0 < ngroups; e0 += 64) {
    const int e = e0 + lane;
    const int f = e < ngroups ? gs.first(e) : 0, l = e < ngroups ? gs.first(e + 1) : 0;
    const int n = mm_cdiv(l - f, LO_TM);
    int inc = n;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(inc, d);
      if (lane >= d) inc += v;
    }
    const uint64_t hit = __ballot(base + inc > b);
    if (hit != 0) {
      const int src = __builtin_ctzll(hit);
      const int k = b - base - __shfl(inc - n, src);
      const int row0 = __shfl(f, src) + k * LO_TM;
      return Tile{e0 + src, row0, min(LO_TM, __shfl(l, src) - row0)};
    }
    base += __shfl(inc, 63);
  }
  return Tile{-1, 0, 0};
}
// Number of tiles of the groups before e.
MM_DEV int tiles_before(const Groups& gs, int e) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int i = lane; i < e; i += 64) n += mm_cdiv(gs.first(i + 1) - gs.first(i), LO_TM);
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d);
  return n;
}

// The records of a launch's tiles; rp ranks (of a chunk) each, nrc chunks.
struct Records {
  uint16_t* by_token;   // [tile][chunk][hi, lo][32][rp]
  uint16_t* by_rank;    // [tile][chunk][hi, lo][rp][32]
  float* scale;         // [tile][chunk]: H = scale * (hi + lo)
  int* tokens;          // [tile][32], the last one repeated behind the tile's rows
  int rp, nrc;
};

// Hand-off of a split sum (k_mid's): every block of the split stores its partial with sc1
// accesses (coherent across the XCDs' L2s), waits until they are performed, and bumps the
// counter; true in the block that arrives last, which leaves the counter at zero.
MM_DEV bool last_of(uint32_t* counter, int n, uint32_t* s_last) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0) {
    const uint32_t prev =
        __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    *s_last = prev == (uint32_t)n - 1u;
    if (*s_last) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *s_last != 0;
}

// ---------------------------------------------------------------------------
// k_down.  One launch does up to two problems (H from x and A, dH from dy and B); block
// (tile, split, problem x rank chunk).  CR: the factor is [C, r] (B), else [r, C] (A).
// Wave w of a block takes every fourth pair of 32-wide steps of the block's range.
// ---------------------------------------------------------------------------
struct DownProblem {
  const uint16_t *V, *W;   // activations [T, C], factors
  int C, ks, per;          // width, splits, 64-wide step pairs per split
  Records rec;
  float* part;             // [tile][chunk][ks][32 * rp]
  uint32_t* counters;      // [tile][chunk]
  int by_token, by_rank;   // which records are wanted
};

template <int T, bool CR, int RT>
MM_DEV void down_tile(const DownProblem& p, const Groups& gs, const Scaling& scaling, int r,
                      int chunk, float* lds) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const int b = blockIdx.x;
  const Tile t = find_tile(gs, gs.L, b);
  if (t.e < 0) return;
  const int r0 = chunk * RP;
  const uint16_t* W = p.W + (size_t)t.e * r * p.C;
  const uint16_t* v[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    v[i] = p.V + (size_t)gs.token(t.row0 + min(16 * i + c, t.rows - 1)) * p.C;
  f32x4 acc[2][RT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < RT; ++k) acc[i][k] = f32x4{0, 0, 0, 0};
  const int pairs = mm_cdiv(p.C, 64);
  const int p_end = min(pairs, ((int)blockIdx.y + 1) * p.per);
  for (int pr = blockIdx.y * p.per + wave; pr < p_end; pr += 4) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int k0 = 64 * pr + 32 * s + 8 * q, left = p.C - k0;
      u16x8 x[2], w[RT];
#pragma unroll
      for (int i = 0; i < 2; ++i) x[i] = load8(v[i] + k0, left);
#pragma unroll
      for (int k = 0; k < RT; ++k) {
        const int rank = min(r0 + 16 * k + c, r - 1);
        if constexpr (!CR) {
          w[k] = load8(W + (size_t)rank * p.C + k0, left);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            w[k][i] = i < left ? W[(size_t)(k0 + i) * r + rank] : (uint16_t)0;
        }
      }
      // D rows: ranks 4q + i, columns: tokens c
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) acc[i][k] = mfma<T>(w[k], x[i], acc[i][k]);
    }
  }
  // Sum over the waves: lds[wave][token][rank].
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < RT; ++k)
      *(f32x4*)(lds + (wave * LO_TM + 16 * i + c) * RP + 16 * k + 4 * q) = acc[i][k];
  __syncthreads();
  constexpr int PER = LO_TM * RP / 4 / LO_NT > 0 ? LO_TM * RP / 4 / LO_NT : 1;   // f32x4 a thread
  constexpr int ITEMS = LO_TM * RP / 4;
  __shared__ uint32_t s_last;
  __shared__ float s_max[4];
  f32x4 h[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * LO_NT;
    h[k] = f32x4{0, 0, 0, 0};
    if (it < ITEMS)
#pragma unroll
      for (int w = 0; w < 4; ++w) h[k] += *(const f32x4*)(lds + w * LO_TM * RP + 4 * it);
  }
  const int slot = b * p.rec.nrc + chunk;
  if (p.ks > 1) {
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(p.part + (size_t)slot * p.ks * (LO_TM * RP));
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int it = threadIdx.x + k * LO_NT;
      if (it < ITEMS) store_agent_x4(prs, 16u * (uint32_t)(blockIdx.y * ITEMS + it), h[k]);
    }
    if (!last_of(p.counters + slot, p.ks, &s_last)) return;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int it = min((int)threadIdx.x + k * LO_NT, ITEMS - 1);
      h[k] = f32x4{0, 0, 0, 0};
      for (int z0 = 0; z0 < p.ks; z0 += 4) {
        f32x4 ld[4];
#pragma unroll
        for (int z = 0; z < 4; ++z)
          ld[z] = load_agent_x4(prs, 16u * (uint32_t)(min(z0 + z, p.ks - 1) * ITEMS + it));
#pragma unroll
        for (int z = 0; z < 4; ++z)
          if (z0 + z < p.ks) h[k] += ld[z];
      }
    }
  }
  // The record.  Ranks and rows past the last are zero.
  const float s = scaling.at(t.e);
  float m = 0.0f;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * LO_NT, row = 4 * it / RP, rank = 4 * it % RP;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[k][i] = row < t.rows && r0 + rank + i < r ? h[k][i] * s : 0.0f;
      m = fmaxf(m, fabsf(h[k][i]));
    }
  }
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  if (lane == 0) s_max[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  int ex = 0;
  if (m > 0.0f && m < __builtin_inff()) {
    (void)frexpf(m, &ex);                      // m = f * 2^ex, f in [0.5, 1)
    ex = max(-110, min(110, 15 - ex));
  }
  const float up = ldexpf(1.0f, ex);
  uint16_t* bt = p.rec.by_token + (size_t)slot * 2 * LO_TM * RP;
  uint16_t* br = p.rec.by_rank + (size_t)slot * 2 * LO_TM * RP;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * LO_NT, row = 4 * it / RP, rank = 4 * it % RP;
    if (it >= ITEMS) continue;
    u16x4 hi, lo;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v = h[k][i] * up;
      hi[i] = from_f32<T>(v);
      const float f = to_f32<T>(hi[i]);
      lo[i] = __builtin_isfinite(f) ? from_f32<T>(v - f) : (uint16_t)0;
    }
    if (p.by_token) {
      *(u16x4*)(bt + row * RP + rank) = hi;
      *(u16x4*)(bt + LO_TM * RP + row * RP + rank) = lo;
    }
    if (p.by_rank)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        br[(rank + i) * LO_TM + row] = hi[i];
        br[LO_TM * RP + (rank + i) * LO_TM + row] = lo[i];
      }
  }
  if (threadIdx.x == 0) p.rec.scale[slot] = ldexpf(1.0f, -ex);
  if (chunk == 0 && threadIdx.x < LO_TM)
    p.rec.tokens[b * LO_TM + threadIdx.x] = gs.token(t.row0 + min((int)threadIdx.x, t.rows - 1));
}

template <int T, int RT>
__global__ void __launch_bounds__(LO_NT)
k_down(DownProblem p0, DownProblem p1, Groups gs, Scaling scaling, int r) {
  __shared__ __attribute__((aligned(16))) float lds[4 * LO_TM * 16 * RT];
  const int nrc = p0.rec.nrc;
  const bool second = (int)blockIdx.z >= nrc;
  if ((int)blockIdx.y >= (second ? p1.ks : p0.ks)) return;
  if (!second) down_tile<T, false, RT>(p0, gs, scaling, r, blockIdx.z, lds);
  else down_tile<T, true, RT>(p1, gs, scaling, r, blockIdx.z - nrc, lds);
}

// ---------------------------------------------------------------------------
// k_up.  Block (tile, 256 columns): wave: 64 columns, lane (c, q): columns 4c .. 4c + 3 of
// tokens 4q + i of both halves of the tile.  CR: the factor is [C, r] (B), else [r, C] (A).
// BT: the base's type (0: no base, zeros).  Group L (no adapter) copies the base.
// ---------------------------------------------------------------------------
template <int T, bool CR, int RT, int BT>
__global__ void __launch_bounds__(LO_NT)
k_up(const uint16_t* __restrict__ W, const uint16_t* base, uint16_t* out, int C, int r,
     Groups gs, Records rec) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const int b = blockIdx.x, n0 = blockIdx.y * LO_COLS + wave * 64 + 4 * c;
  const Tile t = find_tile(gs, gs.L + 1, b);
  if (t.e < 0) return;
  const bool none = t.e >= gs.L;
  if (none && base == out) return;
  const int left = C - n0;
  u16x4 bv[2][4];
  size_t at[2][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      at[i][k] = (size_t)gs.token(t.row0 + min(16 * i + 4 * q + k, t.rows - 1)) * C + n0;
      if constexpr (BT != 0) bv[i][k] = load4(base + at[i][k], left);
      else bv[i][k] = u16x4{0, 0, 0, 0};
    }
  f32x4 sum[2][4];   // [half][column j]: tokens 4q + i
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = f32x4{0, 0, 0, 0};
  if (!none) {
    W += (size_t)t.e * r * C;
    for (int ch = 0; ch < rec.nrc; ++ch) {
      const size_t slot = (size_t)b * rec.nrc + ch;
      const uint16_t* H = rec.by_token + slot * 2 * LO_TM * RP + (q >> 1) * LO_TM * RP + 8 * (q & 1);
      f32x4 acc[2][4];
#pragma unroll
      for (int k = 0; k < RT; ++k) {
        const int rank = ch * RP + 16 * k + 8 * (q & 1);   // the first of this lane's eight
        u16x8 w[4], hv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) hv[i] = *(const u16x8*)(H + (16 * i + c) * RP + 16 * k);
        if constexpr (CR) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            w[j] = load8(W + (size_t)min(n0 + j, C - 1) * r + rank, r - rank);
        } else {
          u16x4 rows[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            rows[i] = load4(W + (size_t)min(rank + i, r - 1) * C + n0, left);
          transpose84(rows, w);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = mfma<T>(hv[i], w[j], k == 0 ? f32x4{0, 0, 0, 0} : acc[i][j]);
      }
      const float f = rec.scale[slot];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) sum[i][j] += f * acc[i][j];
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (16 * i + 4 * q + k >= t.rows) continue;
      u16x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        o[j] = from_f32<T>(BT != 0 ? to_f32<BT != 0 ? BT : T>(bv[i][k][j]) + sum[i][j][k]
                                   : sum[i][j][k]);
      store4(out + at[i][k], o, left);
    }
}

// ---------------------------------------------------------------------------
// k_wgrad.  Up to two problems: dA_a [r, K] from dH and x, dB_a [N, r] from H and dy.
// Block (256 columns, adapter, problem x chunk x split): wave: 64 columns, all tiles of its
// share of the adapter's.  D rows: ranks 4q + i, columns 4c + j.
// ---------------------------------------------------------------------------
struct GradProblem {
  const uint16_t* V;    // [T, C]
  uint16_t* G;          // [L, r, C] or, CR, [L, C, r]
  int C, ks;
  Records rec;
  float* part;          // [adapter][chunk][column block][ks][LO_COLS * rp]
  uint32_t* counters;   // [adapter][chunk][column block]
};

template <int T, bool CR, int RT>
MM_DEV void wgrad_tile(const GradProblem& p, const Groups& gs, int r, int chunk, int split) {
  constexpr int RP = 16 * RT;
  __shared__ uint32_t s_last;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const int e = blockIdx.y, n0 = blockIdx.x * LO_COLS + wave * 64 + 4 * c, left = p.C - n0;
  if ((int)blockIdx.x * LO_COLS >= p.C) return;
  const int nt = mm_cdiv(gs.first(e + 1) - gs.first(e), LO_TM);
  const int per = mm_cdiv(nt, p.ks), tb = tiles_before(gs, e);
  const int t_beg = tb + split * per, t_end = tb + min(nt, (split + 1) * per);
  f32x4 sum[RT][4];
#pragma unroll
  for (int k = 0; k < RT; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[k][j] = f32x4{0, 0, 0, 0};
  for (int b = t_beg; b < t_end; ++b) {
    const i32x4 t0 = *(const i32x4*)(p.rec.tokens + b * LO_TM + 8 * q);
    const i32x4 t1 = *(const i32x4*)(p.rec.tokens + b * LO_TM + 8 * q + 4);
    u16x4 rows[8];
    u16x8 w[4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      rows[i] = load4(p.V + (size_t)(i < 4 ? t0[i & 3] : t1[i & 3]) * p.C + n0, left);
    transpose84(rows, w);
    const size_t slot = (size_t)b * p.rec.nrc + chunk;
    const uint16_t* H = p.rec.by_rank + slot * 2 * LO_TM * RP + c * LO_TM + 8 * q;
    const float f = p.rec.scale[slot];
#pragma unroll
    for (int k = 0; k < RT; ++k) {
      const u16x8 hi = *(const u16x8*)(H + 16 * k * LO_TM);
      const u16x8 lo = *(const u16x8*)(H + LO_TM * RP + 16 * k * LO_TM);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sum[k][j] += f * mfma<T>(hi, w[j], mfma<T>(lo, w[j], f32x4{0, 0, 0, 0}));
    }
  }
  if (p.ks > 1) {
    const int slot = (e * p.rec.nrc + chunk) * mm_cdiv(p.C, LO_COLS) + blockIdx.x;
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(p.part + (size_t)slot * p.ks * (LO_COLS * RP));
    auto at = [&](int z, int k, int j) {
      return 16u * (uint32_t)(((z * RT + k) * 4 + j) * LO_NT + threadIdx.x);
    };
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) store_agent_x4(prs, at(split, k, j), sum[k][j]);
    if (!last_of(p.counters + slot, p.ks, &s_last)) return;
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[k][j] = f32x4{0, 0, 0, 0};
        for (int z0 = 0; z0 < p.ks; z0 += 4) {
          f32x4 ld[4];
#pragma unroll
          for (int z = 0; z < 4; ++z) ld[z] = load_agent_x4(prs, at(min(z0 + z, p.ks - 1), k, j));
#pragma unroll
          for (int z = 0; z < 4; ++z)
            if (z0 + z < p.ks) sum[k][j] += ld[z];
        }
      }
  }
  uint16_t* G = p.G + (size_t)e * r * p.C;
#pragma unroll
  for (int k = 0; k < RT; ++k) {
    const int rank = chunk * RP + 16 * k + 4 * q;
    if constexpr (CR) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u16x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = from_f32<T>(sum[k][j][i]);
        if (j < left) store4(G + (size_t)(n0 + j) * r + rank, o, r - rank);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        u16x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = from_f32<T>(sum[k][j][i]);
        if (rank + i < r) store4(G + (size_t)(rank + i) * p.C + n0, o, left);
      }
    }
  }
}

template <int T, int RT>
__global__ void __launch_bounds__(LO_NT)
k_wgrad(GradProblem pa, GradProblem pb, Groups gs, int r) {
  const int nrc = pa.rec.nrc, za = nrc * pa.ks;
  const int z = blockIdx.z;
  if (z < za) wgrad_tile<T, false, RT>(pa, gs, r, z / pa.ks, z % pa.ks);
  else wgrad_tile<T, true, RT>(pb, gs, r, (z - za) / pb.ks, (z - za) % pb.ks);
}

// ---------------------------------------------------------------------------
// Few tokens.  k_vec_down: block (token, RG ranks), the width over 256 threads; H fp32
// [T, r].  k_vec_up: block (256 columns, token), a column per thread.
// ---------------------------------------------------------------------------
struct Ids {
  const void* p;   // nullptr: adapter 0
  int wide, L;     // int64 ids
  MM_DEV int at(int t) const {   // the token's adapter, or -1
    if (p == nullptr) return 0;
    const int64_t a = wide ? ((const int64_t*)p)[t] : ((const int32_t*)p)[t];
    return a >= 0 && a < L ? (int)a : -1;
  }
};

template <int T, int RG>
__global__ void __launch_bounds__(LO_NT)
k_vec_down(const uint16_t* __restrict__ X, const uint16_t* __restrict__ A, Ids ids,
           Scaling scaling, float* __restrict__ H, int K, int r) {
  __shared__ float red[4][RG];
  const int t = blockIdx.y, r0 = blockIdx.x * RG, a = ids.at(t);
  if (a < 0) return;   // k_vec_up does not read this row
  const uint16_t* x = X + (size_t)t * K;
  const uint16_t* w = A + (size_t)a * r * K;
  float acc[RG];
#pragma unroll
  for (int i = 0; i < RG; ++i) acc[i] = 0.0f;
#pragma unroll 2
  for (int k = 8 * threadIdx.x; k < K; k += 8 * LO_NT) {
    const u16x8 xv = load8(x + k, K - k);
    u16x8 wv[RG];
#pragma unroll
    for (int i = 0; i < RG; ++i) wv[i] = load8(w + (size_t)min(r0 + i, r - 1) * K + k, K - k);
#pragma unroll
    for (int i = 0; i < RG; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[i] += to_f32<T>(xv[j]) * to_f32<T>(wv[i][j]);
  }
#pragma unroll
  for (int i = 0; i < RG; ++i) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) acc[i] += __shfl_xor(acc[i], d);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][i] = acc[i];
  }
  __syncthreads();
  const int i = threadIdx.x;
  if (i < RG && r0 + i < r)
    H[(size_t)t * r + r0 + i] = scaling.at(a) * (red[0][i] + red[1][i] + red[2][i] + red[3][i]);
}

template <int T, int BT>
__global__ void __launch_bounds__(LO_NT)
k_vec_up(const float* __restrict__ H, const uint16_t* __restrict__ B, Ids ids,
         const uint16_t* base, uint16_t* out, int N, int r) {
  const int t = blockIdx.y, n = blockIdx.x * LO_NT + threadIdx.x, a = ids.at(t);
  if (n >= N) return;
  const size_t at = (size_t)t * N + n;
  float v = to_f32<BT>(base[at]);
  if (a >= 0) {
    const uint16_t* w = B + ((size_t)a * N + n) * r;
    const float* h = H + (size_t)t * r;
    float s = 0.0f;
    for (int k = 0; k < r; k += 8) {
      const u16x8 wv = load8(w + k, r - k);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < r) s += h[k + j] * to_f32<T>(wv[j]);
    }
    v += s;
  }
  out[at] = from_f32<T>(v);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
constexpr int LO_VEC_TOKENS = 64;   // up to here k_vec_*
// Sums are split over blocks while a launch has fewer than these: two a CU.  A split
// launch therefore has fewer arrival counters than this in use per problem.
constexpr int LO_SPLIT_BELOW = 512;

int rank_tiles(int r) { return r <= 16 ? 1 : (r <= 32 ? 2 : 4); }

struct LoraPlan {
  int rt, rp, nrc, tiles;          // tiles: upper bound of the adapters' tiles
  size_t sort, rec[2], part, total;
};

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

int down_split(int tiles, int nrc, int C) {
  const int pairs = mm_cdiv(C, 64);
  int ks = 1;
  while (tiles * nrc * ks < LO_SPLIT_BELOW && pairs / (2 * ks) >= 8) ks *= 2;
  return ks;
}
int wgrad_split(int T, int L, int nrc, int C) {
  const long blocks = (long)mm_cdiv(C, LO_COLS) * L * nrc;
  const int most = std::max(1, mm_cdiv(T, LO_TM) / 4);
  int ks = 1;
  while (blocks * ks < LO_SPLIT_BELOW && ks * 2 <= most && ks < 32) ks *= 2;
  return ks;
}

size_t record_bytes(const LoraPlan& p) {
  const size_t h = (size_t)p.tiles * p.nrc * 2 * LO_TM * p.rp * 2;
  return 2 * align256(h) + align256((size_t)p.tiles * p.nrc * 4) +
         align256((size_t)p.tiles * LO_TM * 4);
}
Records record_at(const LoraPlan& p, char* at) {
  const size_t h = align256((size_t)p.tiles * p.nrc * 2 * LO_TM * p.rp * 2);
  Records r{};
  r.by_token = (uint16_t*)at;
  r.by_rank = (uint16_t*)(at + h);
  r.scale = (float*)(at + 2 * h);
  r.tokens = (int*)(at + 2 * h + align256((size_t)p.tiles * p.nrc * 4));
  r.rp = p.rp;
  r.nrc = p.nrc;
  return r;
}

// Workspace: counters, the sort's arrays, the records of both problems, partial sums (of
// k_down and then of k_wgrad, one after the other in the same memory).
LoraPlan plan_lora(int T, int K, int N, int r, int L, bool backward) {
  LoraPlan p{};
  p.rt = rank_tiles(r);
  p.rp = 16 * p.rt;
  p.nrc = mm_cdiv(r, p.rp);
  p.tiles = T / LO_TM + std::min(L, T);
  p.sort = LO_COUNTER_BYTES;
  p.rec[0] = p.sort + align256(((size_t)L + 1 + 2 * (size_t)T) * 4);
  p.rec[1] = p.rec[0] + record_bytes(p);
  p.part = p.rec[1] + (backward ? record_bytes(p) : 0);
  const size_t tile = (size_t)p.tiles * p.nrc * LO_TM * p.rp * 4;
  size_t part = tile * down_split(p.tiles, p.nrc, K);
  if (backward) {
    part += tile * down_split(p.tiles, p.nrc, N);
    const size_t col = (size_t)L * p.nrc * LO_COLS * p.rp * 4;
    part = std::max(part, col * (mm_cdiv(K, LO_COLS) * (size_t)wgrad_split(T, L, p.nrc, K) +
                                 mm_cdiv(N, LO_COLS) * (size_t)wgrad_split(T, L, p.nrc, N)));
  }
  p.total = p.part + align256(part);
  return p;
}

int check_common(const char* who, int type, int T, int K, int N, int r, int L, const void* ids,
                 int ids64) {
  MM_CHECK_ARG(type == 1 || type == 2, "%s: type=%d must be 1 (fp16) or 2 (bf16)", who, type);
  MM_CHECK_ARG(T >= 0 && K > 0 && N > 0 && r > 0 && L > 0,
               "%s: bad shape T=%d K=%d N=%d rank=%d adapters=%d", who, T, K, N, r, L);
  MM_CHECK_ARG(ids == nullptr || ids64 == 0 || ids64 == 1, "%s: ids64=%d must be 0 or 1", who,
               ids64);
  MM_CHECK_ARG(ids != nullptr || L == 1, "%s: %d adapters need ids", who, L);
  MM_CHECK_ARG(L <= 1024, "%s: at most 1024 adapters, got %d", who, L);
  MM_CHECK_ARG((long)mm_cdiv(N, LO_COLS) <= 65535 && (long)mm_cdiv(K, LO_COLS) <= 65535,
               "%s: K=%d, N=%d exceed %ld columns", who, K, N, 65535L * LO_COLS);
  return 0;
}

// Sorts the tokens by adapter (none needed for a single adapter without ids).
int make_groups(const char* who, const LoraPlan& p, const void* ids, int ids64, int T, int L,
                void* ws, void* stream, Groups* gs) {
  *gs = Groups{nullptr, nullptr, T, L};
  if (ids == nullptr) return 0;
  int32_t* off = (int32_t*)((char*)ws + p.sort);
  int32_t* order = off + L + 1;
  int32_t* inverse = order + T;
  const int rc = ids64 ? mm_moe_sort_i64((const int64_t*)ids, T, 1, L, off, order, inverse, stream)
                       : mm_moe_sort((const int32_t*)ids, T, 1, L, off, order, inverse, stream);
  gs->offsets = off;
  gs->order = order;
  return rc;
}

#define MM_LORA_RT(F, ...)                    \
  switch (p.rt) {                             \
    case 1: F(1, __VA_ARGS__); break;         \
    case 2: F(2, __VA_ARGS__); break;         \
    default: F(4, __VA_ARGS__); break;        \
  }

}  // namespace

extern "C" size_t mm_lora_workspace_bytes(int T, int K, int N, int r, int L, int backward) {
  if (T <= 0 || K <= 0 || N <= 0 || r <= 0 || L <= 0) return LO_COUNTER_BYTES;
  if (!backward && T <= LO_VEC_TOKENS) return LO_COUNTER_BYTES + (size_t)T * r * 4;
  return plan_lora(T, K, N, r, L, backward != 0).total;
}

extern "C" int mm_lora_add(const uint16_t* x, int type, const uint16_t* base, int base_type,
                           uint16_t* out, const uint16_t* A, const uint16_t* B, const void* ids,
                           int ids64, const float* scaling, float scale, int T, int K, int N,
                           int r, int L, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "mm_lora_add";
  if (const int rc = check_common(who, type, T, K, N, r, L, ids, ids64)) return rc;
  MM_CHECK_ARG(base_type == 1 || (base_type == 2 && type == 2),
               "%s: base_type=%d must be 1 (fp16) or the type of x", who, base_type);
  MM_CHECK_ARG(base != out || base_type == type, "%s: in place needs a base of the type of x",
               who);
  if (T == 0) return 0;
  const size_t need = mm_lora_workspace_bytes(T, K, N, r, L, 0);
  MM_CHECK_ARG(ws != nullptr && ws_bytes >= need,
               "%s: workspace of %zu bytes is smaller than the %zu required", who, ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  const Scaling sc{scaling, scale};
  if (T <= LO_VEC_TOKENS) {
    float* H = (float*)((char*)ws + LO_COUNTER_BYTES);
    const Ids id{ids, ids64, L};
    // Fewer ranks a block while that leaves CUs idle.
#define MM_VEC_DOWN(TV, RG)                                                                    \
  hipLaunchKernelGGL((k_vec_down<TV, RG>), dim3(mm_cdiv(r, RG), T), dim3(LO_NT), 0, st, x, A, id, \
                     sc, H, K, r)
    if (T * r <= 512) { if (type == 1) MM_VEC_DOWN(1, 2); else MM_VEC_DOWN(2, 2); }
    else { if (type == 1) MM_VEC_DOWN(1, 4); else MM_VEC_DOWN(2, 4); }
#undef MM_VEC_DOWN
    MM_CHECK_LAUNCH(who);
#define MM_VEC_UP(TV, BV)                                                                      \
  hipLaunchKernelGGL((k_vec_up<TV, BV>), dim3(mm_cdiv(N, LO_NT), T), dim3(LO_NT), 0, st, H, B, id, \
                     base, out, N, r)
    if (type == 1) MM_VEC_UP(1, 1);
    else if (base_type == 1) MM_VEC_UP(2, 1);
    else MM_VEC_UP(2, 2);
#undef MM_VEC_UP
    MM_CHECK_LAUNCH(who);
    return 0;
  }
  const LoraPlan p = plan_lora(T, K, N, r, L, false);
  Groups gs;
  if (const int rc = make_groups(who, p, ids, ids64, T, L, ws, stream, &gs)) return rc;
  const Records rec = record_at(p, (char*)ws + p.rec[0]);
  const int ks = down_split(p.tiles, p.nrc, K);
  const DownProblem d{x, A, K, ks, mm_cdiv(mm_cdiv(K, 64), ks), rec, (float*)((char*)ws + p.part),
                      (uint32_t*)ws, 1, 0};
#define MM_DOWN(RTV, TV)                                                                       \
  hipLaunchKernelGGL((k_down<TV, RTV>), dim3(p.tiles, ks, p.nrc), dim3(LO_NT), 0, st, d, d, gs, \
                     sc, r)
  if (type == 1) { MM_LORA_RT(MM_DOWN, 1) } else { MM_LORA_RT(MM_DOWN, 2) }
  MM_CHECK_LAUNCH(who);
  // group L (tokens without an adapter) has tiles of its own
  const dim3 grid(p.tiles + (ids != nullptr ? mm_cdiv(T, LO_TM) : 0), mm_cdiv(N, LO_COLS));
#define MM_UP(RTV, TV, BV)                                                                     \
  hipLaunchKernelGGL((k_up<TV, true, RTV, BV>), grid, dim3(LO_NT), 0, st, B, base, out, N, r, gs, rec)
  if (type == 1) { MM_LORA_RT(MM_UP, 1, 1) }
  else if (base_type == 1) { MM_LORA_RT(MM_UP, 2, 1) }
  else { MM_LORA_RT(MM_UP, 2, 2) }
#undef MM_UP
#undef MM_DOWN
  MM_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int mm_lora_backward(const uint16_t* dy, const uint16_t* x, int type,
                                const uint16_t* A, const uint16_t* B, const void* ids, int ids64,
                                const float* scaling, float scale, const uint16_t* dx_base,
                                uint16_t* dx, uint16_t* dA, uint16_t* dB, int T, int K, int N,
                                int r, int L, void* ws, size_t ws_bytes, void* stream) {
  const char* who = "mm_lora_backward";
  if (const int rc = check_common(who, type, T, K, N, r, L, ids, ids64)) return rc;
  MM_CHECK_ARG(T > 0, "%s: no tokens (the gradients are zeros)", who);
  const size_t need = mm_lora_workspace_bytes(T, K, N, r, L, 1);
  MM_CHECK_ARG(ws != nullptr && ws_bytes >= need,
               "%s: workspace of %zu bytes is smaller than the %zu required", who, ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  const Scaling sc{scaling, scale};
  const LoraPlan p = plan_lora(T, K, N, r, L, true);
  Groups gs;
  if (const int rc = make_groups(who, p, ids, ids64, T, L, ws, stream, &gs)) return rc;
  const Records rx = record_at(p, (char*)ws + p.rec[0]), ry = record_at(p, (char*)ws + p.rec[1]);
  float* part = (float*)((char*)ws + p.part);
  uint32_t* counters = (uint32_t*)ws;
  const int kx = down_split(p.tiles, p.nrc, K), ky = down_split(p.tiles, p.nrc, N);
  const size_t tile = (size_t)p.tiles * p.nrc * LO_TM * p.rp;
  const DownProblem px{x, A, K, kx, mm_cdiv(mm_cdiv(K, 64), kx), rx, part, counters, 0, 1};
  const DownProblem py{dy, B, N, ky, mm_cdiv(mm_cdiv(N, 64), ky), ry, part + tile * kx,
                       counters + LO_SPLIT_BELOW, 1, 1};
#define MM_DOWN(RTV, TV)                                                                       \
  hipLaunchKernelGGL((k_down<TV, RTV>), dim3(p.tiles, std::max(kx, ky), 2 * p.nrc), dim3(LO_NT), \
                     0, st, px, py, gs, sc, r)
  if (type == 1) { MM_LORA_RT(MM_DOWN, 1) } else { MM_LORA_RT(MM_DOWN, 2) }
#undef MM_DOWN
  MM_CHECK_LAUNCH(who);
  const int ca = mm_cdiv(K, LO_COLS), cb = mm_cdiv(N, LO_COLS);
  const int ga = wgrad_split(T, L, p.nrc, K), gb = wgrad_split(T, L, p.nrc, N);
  const GradProblem pa{x, dA, K, ga, ry, part, counters};
  const GradProblem pb{dy, dB, N, gb, rx, part + (size_t)L * p.nrc * ca * ga * LO_COLS * p.rp,
                       counters + LO_SPLIT_BELOW};
#define MM_WGRAD(RTV, TV)                                                                      \
  hipLaunchKernelGGL((k_wgrad<TV, RTV>), dim3(std::max(ca, cb), L, p.nrc * (ga + gb)),           \
                     dim3(LO_NT), 0, st, pa, pb, gs, r)
  if (type == 1) { MM_LORA_RT(MM_WGRAD, 1) } else { MM_LORA_RT(MM_WGRAD, 2) }
#undef MM_WGRAD
  MM_CHECK_LAUNCH(who);
  const dim3 grid(p.tiles + (ids != nullptr ? mm_cdiv(T, LO_TM) : 0), ca);
#define MM_UP(RTV, TV, BV)                                                                     \
  hipLaunchKernelGGL((k_up<TV, false, RTV, BV>), grid, dim3(LO_NT), 0, st, A, dx_base, dx, K, r, \
                     gs, ry)
  if (dx_base != nullptr) {
    if (type == 1) { MM_LORA_RT(MM_UP, 1, 1) } else { MM_LORA_RT(MM_UP, 2, 2) }
  } else {
    if (type == 1) { MM_LORA_RT(MM_UP, 1, 0) } else { MM_LORA_RT(MM_UP, 2, 0) }
  }
#undef MM_UP
  MM_CHECK_LAUNCH(who);
  return 0;
}
