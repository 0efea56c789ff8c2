// Low-rank adapters of many requests beside a shared projection, and their gradients:
//   out[t] = base[t] + s_a (x[t] A_a^T) B_a^T,   a = ids[t]   (no adapter: out = base)
//   H = s x A^T, dH = s dy B;   dx = dx_base + dH A,   dA_a = sum dH[t]^T x[t],
//   dB_a = sum dy[t]^T H[t]     over the tokens t of adapter a
// with A [L, r, K], B [L, N, r], s = scale * scaling[a] (scaling fp32 [L], or none).
//
// Few tokens: every token on its own, one launch of fp32 dot products (k_vec) or two
// (k_vec_down, k_vec_up).  Otherwise the tokens are sorted by adapter and cut into tiles of 64
// of one adapter (k_plan, or up to 2048 tokens each block of k_down for its own tile), and
//   k_down   H of a tile, over the whole width: 16x16x32 MFMAs, the width split over the
//            waves and over blocks.  The block that finishes a tile leaves a record of it:
//            H as hi + lo in the operands' type, under a power of two that puts the largest
//            value in [2^14, 2^15), so that 16 (bf16) or 22 (fp16) bits of H reach the second
//            product.  The record has H by token and by rank, the operand orders of the two
//            kernels that follow: by token each token has a power of two of its own (in fp16
//            another request's large values would cost it bits), by rank, where the tokens
//            of a tile are summed, the tile has one.
//   up       out of a tile: MFMAs over [hi | lo] of 16 ranks at a time.
//   wgrad    dA_a or dB_a: MFMAs over 32 tokens at a time, tile after tile; the tiles are shared
//            out over a block's waves, or a wave has them all where an adapter has few tokens.
// All sums are fp32 and in a fixed order.  They stream activations, the factors stay in L2: the
// forward reads x and the base once and writes out; the backward reads x and dy twice, in k_down
// and in wgrad (one pass over dy could give dH and dB, were H there before it).  HBM bounds long
// batches, the latency of the chain sort, loads, hand-off short ones.
#include <algorithm>
#include <type_traits>

#include "mm_common.h"
#include "mmfp4.h"

namespace {

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
// Rows of any width start at any even address.
typedef u16x4 u16x4_any __attribute__((aligned(2)));
typedef u16x8 u16x8_any __attribute__((aligned(2)));

constexpr int LO_TM = 64;               // tokens per tile
constexpr int LO_NT = 256;              // threads per block of the dot products, up and wgrad
constexpr int LO_DW = 8;                // waves of a k_down block
constexpr int LO_UP_COLS = 256;         // columns per block of up: 64 a wave
constexpr int LO_WG_COLS = 64;          // columns per block of wgrad
constexpr int LO_MAX_ADAPTERS = 1024;
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
// The same where the caller knows that all are there: a guard costs a branch and a wait for
// every load before it, so the kernels have a form of each for whole pieces.
template <bool WHOLE>
MM_DEV u16x4 ld4(const uint16_t* p, int n) {
  if constexpr (WHOLE) return *(const u16x4_any*)p;
  else return load4(p, n);
}
template <bool WHOLE>
MM_DEV void st4(uint16_t* p, u16x4 v, int n) {
  if constexpr (WHOLE) *(u16x4_any*)p = v;
  else store4(p, v, n);
}

// The same of fp32 rows, which start at any multiple of four bytes.
typedef f32x4 f32x4_any __attribute__((aligned(4)));
template <bool WHOLE>
MM_DEV f32x4 ld4f(const float* p, int n) {
  if (WHOLE || n >= 4) return *(const f32x4_any*)p;
  f32x4 v = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 3; ++i)
    if (i < n) v[i] = p[i];
  return v;
}
template <bool WHOLE>
MM_DEV void st4f(float* p, f32x4 v, int n) {
  if (WHOLE || n >= 4) {
    *(f32x4_any*)p = v;
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
// Tokens sorted by adapter, and the tiles: tile b has `rows` tokens of group e (e < L:
// adapter e; e == L: no adapter; e < 0: no such tile), listed in tokens[64 b ..], the last one
// repeated behind them.  tiles == nullptr: one adapter for all tokens, as they come.
// ---------------------------------------------------------------------------
struct TileInfo {
  int e, rows;
};
struct Plan {
  const TileInfo* tiles;
  const int *tokens, *first;   // first[e]: first tile of group e
  int T, L;
  MM_DEV TileInfo tile(int b) const {
    if (tiles == nullptr)
      return LO_TM * b < T ? TileInfo{0, min(LO_TM, T - LO_TM * b)} : TileInfo{-1, 0};
    return tiles[b];
  }
  MM_DEV int first_tile(int e) const {
    if (tiles == nullptr) return e == 0 ? 0 : mm_cdiv(T, LO_TM);
    return first[e];
  }
  // Tokens at[k] of tile b (the list does not wait for the tile's entry).
  template <int N>
  MM_DEV void get(int b, const int (&at)[N], int (&tok)[N]) const {
    if (tiles != nullptr) {
#pragma unroll
      for (int k = 0; k < N; ++k) tok[k] = tokens[LO_TM * b + at[k]];
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k) tok[k] = min(LO_TM * b + at[k], T - 1);
    }
  }
};

struct Scaling {
  const float* p;
  float scale;
  MM_DEV float at(int e) const { return p != nullptr ? scale * p[e] : scale; }
};

struct Ids {
  const void* p;   // nullptr: adapter 0
  int wide, L;     // int64 ids
  MM_DEV int64_t raw(int t) const { return wide ? ((const int64_t*)p)[t] : ((const int32_t*)p)[t]; }
  MM_DEV int at(int t) const {   // the token's adapter, or -1
    if (p == nullptr) return 0;
    const int64_t a = raw(t);
    return a >= 0 && a < L ? (int)a : -1;
  }
};

// Stable counting sort of the tokens by group in one block, and the tile table.  Each wave
// counts and places its own stretch of the tokens, 64 at a time; requests lie one after
// another, so that a step mostly has one or two groups.  Latency bounds it: the ids of eight
// steps are loaded together and kept for the second pass (up to 8192 tokens).
constexpr int PL_NT = 1024, PL_NW = PL_NT / 64, PL_HOLD = 8;
__global__ void __launch_bounds__(PL_NT)
k_plan(Ids ids, int T, int max_tiles, TileInfo* __restrict__ tiles, int* __restrict__ tokens,
       int* __restrict__ first) {
  __shared__ int cnt[PL_NW][LO_MAX_ADAPTERS + 1];
  __shared__ int rows_of[LO_MAX_ADAPTERS + 2], tile0[LO_MAX_ADAPTERS + 2];   // rows, first tile
  __shared__ int last[LO_MAX_ADAPTERS + 1];                               // last token
  __shared__ int wsum[PL_NW];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int G = ids.L + 1;
  const int steps = mm_cdiv(T, 64 * PL_NW), t0 = wave * steps * 64 + lane;   // per wave
  int hold[PL_HOLD];
  auto load = [&](int s0) {
    int64_t raw[PL_HOLD];
#pragma unroll
    for (int i = 0; i < PL_HOLD; ++i) raw[i] = ids.raw(min(t0 + 64 * (s0 + i), T - 1));
#pragma unroll
    for (int i = 0; i < PL_HOLD; ++i)
      hold[i] = s0 + i < steps && t0 + 64 * (s0 + i) < T
                    ? (raw[i] >= 0 && raw[i] < ids.L ? (int)raw[i] : ids.L)
                    : -1;                     // no token
  };
  load(0);
  for (int i = tid; i < PL_NW * G; i += PL_NT) cnt[i / G][i % G] = 0;
  __syncthreads();
  for (int s0 = 0; s0 < steps; s0 += PL_HOLD) {
    if (s0 > 0) load(s0);
#pragma unroll
    for (int i = 0; i < PL_HOLD; ++i) {
      const int g = hold[i], g0 = __builtin_amdgcn_readfirstlane(g);
      const uint64_t live = __ballot(g >= 0);
      if (live == 0) continue;
      if (__ballot(g == g0) == live) {
        if (lane == 0) atomicAdd(&cnt[wave][g0], __popcll(live));
      } else if (g >= 0) {
        atomicAdd(&cnt[wave][g], 1);
      }
    }
  }
  __syncthreads();
  // Groups 2 tid and 2 tid + 1: rows of each wave in front of one another, then both scans.
  int n[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int g = 2 * tid + k;
    if (g >= G) continue;
#pragma unroll
    for (int w = 0; w < PL_NW; ++w) {
      const int c = cnt[w][g];
      cnt[w][g] = n[k];
      n[k] += c;
    }
    rows_of[g] = n[k];                           // the group's rows
  }
  const int nt = mm_cdiv(n[0], LO_TM) + mm_cdiv(n[1], LO_TM);
  int it = nt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int b = __shfl_up(it, d);
    if (lane >= d) it += b;
  }
  if (lane == 63) wsum[wave] = it;
  __syncthreads();
  int b = it - nt;
  for (int w = 0; w < wave; ++w) b += wsum[w];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int g = 2 * tid + k;
    if (g > G) continue;                      // entry G: the end
    tile0[g] = b;
    first[g] = b;
    b += mm_cdiv(n[k], LO_TM);
  }
  __syncthreads();
  const int total = tile0[G];
  for (int i = tid; i < max_tiles; i += PL_NT) {
    TileInfo t = {-1, 0};
    if (i < total) {
      int lo = 0, hi = G;                     // tile0[lo] <= i < tile0[hi]
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (tile0[mid] <= i) lo = mid;
        else hi = mid;
      }
      t = TileInfo{lo, min(LO_TM, rows_of[lo] - (i - tile0[lo]) * LO_TM)};
    }
    tiles[i] = t;
  }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int s0 = 0; s0 < steps; s0 += PL_HOLD) {
    if (steps > PL_HOLD) load(s0);
#pragma unroll
    for (int i = 0; i < PL_HOLD; ++i) {
      const int g = hold[i], t = t0 + 64 * (s0 + i);
      uint64_t left = __ballot(g >= 0);
      while (left != 0) {
        const int src = __builtin_ctzll(left);
        const int g0 = __builtin_amdgcn_readlane(g, src);
        const uint64_t m = __ballot(g == g0);
        volatile int* next = &cnt[wave][g0];  // read by all lanes, moved on by one
        const int at = *next;
        if (lane == src) *next = at + __popcll(m);
        if ((m >> lane) & 1) {
          const int row = at + __popcll(m & below);   // of the group
          tokens[LO_TM * tile0[g0] + row] = t;
          if (row == rows_of[g0] - 1) last[g0] = t;
        }
        left &= ~m;
      }
    }
  }
  __syncthreads();
  for (int g = wave; g < G; g += PL_NW) {
    const int i = rows_of[g] + lane;
    if (i < LO_TM * mm_cdiv(rows_of[g], LO_TM)) tokens[LO_TM * tile0[g] + i] = last[g];
  }
}

// The same for up to DP_TOKENS tokens, by each block of k_down for its own tile: a launch less,
// and a pass over the ids costs a block less than the launch.  Block (b, 0, 0) also leaves tile
// b's entry and list, and block 0 the first tiles, for the kernels that follow.
// us, a launch of its own / this: forward of 256 tokens of 4 adapters, 4096 -> 4096, rank 16
// 17.9 / 15.1; 2000 tokens 26.7 / 24.5; 1111 tokens, 14336 -> 4096, rank 64 41.9 / 39.0; backward
// of 777 tokens, 2048 -> 5632, rank 8 23.9 / 20.8; with several blocks to a CU the other way, 128
// tokens of 8 adapters, 4096 -> 14336, rank 64, 71.6 / 74.5; 4000 tokens no gain.
constexpr int DP_NT = 64 * LO_DW, DP_HOLD = 4, DP_TOKENS = DP_NT * DP_HOLD;
struct PlanOut {
  Ids ids;             // ids.p == nullptr: the plan is there
  TileInfo* tiles;
  int *tokens, *first;
};
MM_DEV TileInfo own_tile(const PlanOut& o, int T, int b, bool write, int* cnt, int* list) {
  __shared__ int wsum[LO_DW], found[3];        // group, first row, rows
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int L = o.ids.L, G = L + 1;
  const int steps = mm_cdiv(T, DP_NT), t0 = wave * steps * 64 + lane;
  int64_t raw[DP_HOLD];
  int hold[DP_HOLD];
#pragma unroll
  for (int i = 0; i < DP_HOLD; ++i)
    raw[i] = i < steps ? o.ids.raw(min(t0 + 64 * i, T - 1)) : -1;
  for (int i = tid; i < LO_DW * G; i += DP_NT) cnt[i] = 0;
  if (tid == 0) found[0] = -1;
#pragma unroll
  for (int i = 0; i < DP_HOLD; ++i)
    hold[i] = i < steps && t0 + 64 * i < T ? (raw[i] >= 0 && raw[i] < L ? (int)raw[i] : L) : -1;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < DP_HOLD; ++i) {
    const int g = hold[i], g0 = __builtin_amdgcn_readfirstlane(g);
    const uint64_t live = __ballot(g >= 0);
    if (live == 0) continue;
    if (__ballot(g == g0) == live) {
      if (lane == 0) atomicAdd(&cnt[wave * G + g0], __popcll(live));
    } else if (g >= 0) {
      atomicAdd(&cnt[wave * G + g], 1);
    }
  }
  __syncthreads();
  constexpr int PER = (LO_MAX_ADAPTERS + 2 + DP_NT - 1) / DP_NT;   // groups of a thread, entry G
  int n[PER], nt = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    n[k] = 0;
    if (PER * tid + k < G)
#pragma unroll
      for (int w = 0; w < LO_DW; ++w) n[k] += cnt[w * G + PER * tid + k];
    nt += mm_cdiv(n[k], LO_TM);
  }
  int at = nt;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int v = __shfl_up(at, d);
    if (lane >= d) at += v;
  }
  if (lane == 63) wsum[wave] = at;
  __syncthreads();
  at -= nt;
  for (int w = 0; w < wave; ++w) at += wsum[w];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int g = PER * tid + k, tiles = mm_cdiv(n[k], LO_TM);
    if (write && b == 0 && g <= G) o.first[g] = at;
    if (b >= at && b < at + tiles) {
      found[0] = g;
      found[1] = (b - at) * LO_TM;
      found[2] = min(LO_TM, n[k] - found[1]);
    }
    at += tiles;
  }
  __syncthreads();
  const TileInfo t{found[0], found[0] < 0 ? 0 : found[2]};
  if (write && tid == 0) o.tiles[b] = t;
  if (t.e < 0) return t;
  int row = -found[1];
  for (int w = 0; w < wave; ++w) row += cnt[w * G + t.e];
#pragma unroll
  for (int i = 0; i < DP_HOLD; ++i) {
    const uint64_t m = __ballot(hold[i] == t.e);
    const int mine = row + __popcll(m & (((uint64_t)1 << lane) - 1));
    if (hold[i] == t.e && mine >= 0 && mine < LO_TM) list[mine] = t0 + 64 * i;
    row += __popcll(m);
  }
  __syncthreads();
  if (tid < LO_TM) {
    const int token = list[min(tid, t.rows - 1)];
    if (write) o.tokens[LO_TM * b + tid] = token;
    if (tid >= t.rows) list[tid] = token;
  }
  __syncthreads();
  return t;
}

// The records of a launch's tiles; rp ranks (of a chunk) each, nrc chunks.
struct Records {
  uint16_t* by_token;   // [tile][chunk][hi, lo][64][rp]
  uint16_t* by_rank;    // [tile][chunk][hi, lo][rp][64]
  float* token_scale;   // [tile][chunk][64]: H of a token = token_scale * (hi + lo) by token
  float* scale;         // [tile][chunk]: H = scale * (hi + lo) by rank
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
// Wave w of a block takes every eighth pair of 32-wide steps of the block's range.  Rows of
// 16 that hold no token are skipped.
// ---------------------------------------------------------------------------
struct DownProblem {
  const uint16_t *V, *W;   // activations [T, C], factors
  int C, ks, per;          // width, splits, 64-wide step pairs per split
  Records rec;
  float* part;             // [tile][chunk][ks][64 * rp]
  uint32_t* counters;      // [tile][chunk]
  int by_token, by_rank;   // which records are wanted
  const float* row_mul;    // [T] or nullptr: factors of the tokens' dy, taken into H and dH
};

// LDS of a wave: its pair's activations, 64 rows of 128 bytes, 16-byte piece (row, p) at
// row * 8 + (p ^ ((row >> 1) & 7)); then the factors, 16 * RT rows laid out the same, or (CR) 64
// rows of 16 * RT ranks and 16 bytes.  A load of a whole row's 128 bytes by 8 lanes is one
// request; straight into the operands' layout, 64 bytes a row, it is two, and those are what a
// CU has a limited number of in flight (117 MB of dy 33 us so, 3.5 TB/s).
template <int RT>
constexpr int down_lds_wave() { return LO_TM * 128 + 64 * (32 * RT + 16); }

// Tokens at[k] of tile b: of own_tile's list in LDS, or of the plan.
template <int N>
MM_DEV void tokens_of(const Plan& plan, const int* list, int b, const int (&at)[N],
                      int (&tok)[N]) {
  if (list == nullptr) {
    plan.get(b, at, tok);
    return;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) tok[k] = list[at[k]];
}

template <int T, bool CR, int RT, int NR>
MM_DEV void down_sum(const DownProblem& p, const Plan& plan, const int* list, int b, int e,
                     int r, int r0, char* lds, f32x4 (&acc)[4][RT]) {
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint16_t* W = p.W + (size_t)e * r * p.C;
  const int beg = blockIdx.y * p.per, end = min(p.C / 64, beg + p.per);   // whole pairs
  constexpr int WROW = 32 * RT + 16;   // CR: bytes of a factor row in LDS
  char* xs = lds + wave * down_lds_wave<RT>();
  char* ws = xs + LO_TM * 128;
  if (!CR || r % 8 == 0) {
    constexpr int NX = 2 * NR, NW = 2 * RT;   // load instructions of a pair
    const uint16_t* v[NX];
    int at[NX], tok[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) at[i] = 8 * i + (lane >> 3);
    tokens_of(plan, list, b, at, tok);
#pragma unroll
    for (int i = 0; i < NX; ++i) v[i] = p.V + (size_t)tok[i] * p.C + 8 * (lane & 7);
    uint32_t woff[NW], wlds[NW];   // element offset of the lane's pieces at k = 0, place in LDS
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      if constexpr (!CR) {
        const int row = 8 * i + (lane >> 3);
        woff[i] = (uint32_t)min(r0 + row, r - 1) * p.C + 8 * (lane & 7);
        wlds[i] = row * 128 + ((lane & 7) ^ ((row >> 1) & 7)) * 16;
      } else {
        const int n = (64 * i + lane) / (2 * RT), piece = (64 * i + lane) % (2 * RT);
        woff[i] = (uint32_t)n * r + min(r0 + 8 * piece, r - 8);
        wlds[i] = n * WROW + piece * 16;
      }
    }
    struct Stage {
      u16x8 x[NX], w[NW];
    };
    auto load = [&](Stage& o, int pr) {
#pragma unroll
      for (int i = 0; i < NX; ++i) o.x[i] = *(const u16x8_any*)(v[i] + 64 * pr);
      const uint16_t* w = W + (size_t)64 * pr * (CR ? r : 1);
#pragma unroll
      for (int i = 0; i < NW; ++i) o.w[i] = *(const u16x8_any*)(w + woff[i]);
    };
    // Through the wave's own LDS (no barrier) into the operands' order.  D rows: ranks
    // 4q + i, columns: tokens c.
    auto park = [&](const Stage& o) {
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        const int row = 8 * i + (lane >> 3);
        *(u16x8*)(xs + row * 128 + ((lane & 7) ^ ((row >> 1) & 7)) * 16) = o.x[i];
      }
#pragma unroll
      for (int i = 0; i < NW; ++i) *(u16x8*)(ws + wlds[i]) = o.w[i];
    };
    auto multiply = [&]() {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        u16x8 x[NR], w[RT];
#pragma unroll
        for (int i = 0; i < NR; ++i)
          x[i] = *(const u16x8*)(xs + (16 * i + c) * 128 + ((4 * s + q) ^ ((c >> 1) & 7)) * 16);
#pragma unroll
        for (int k = 0; k < RT; ++k) {
          if constexpr (!CR) {
            w[k] = *(const u16x8*)(ws + (16 * k + c) * 128 + ((4 * s + q) ^ ((c >> 1) & 7)) * 16);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              w[k][i] = *(const uint16_t*)(ws + (32 * s + 8 * q + i) * WROW + (16 * k + c) * 2);
          }
        }
#pragma unroll
        for (int i = 0; i < NR; ++i)
#pragma unroll
          for (int k = 0; k < RT; ++k) acc[i][k] = mfma<T>(w[k], x[i], acc[i][k]);
      }
    };
    // A pair (with up to 32 ranks two) is on its way while one is multiplied; behind the last
    // it is the last again.
    constexpr int SETS = RT == 4 ? 1 : 2;
    const int np = beg + wave < end ? (end - beg - wave + LO_DW - 1) / LO_DW : 0;
    auto pair = [&](int n) { return beg + wave + LO_DW * min(n, np - 1); };
    if (np > 0) {
      Stage set[SETS];
#pragma unroll
      for (int d = 0; d < SETS; ++d) load(set[d], pair(d));
      for (int n = 0; n < np; n += SETS) {
#pragma unroll
        for (int d = 0; d < SETS; ++d) {
          if (n + d >= np) break;
          park(set[d]);
          __builtin_amdgcn_sched_barrier(0);   // or the loads sink to where they are used
          load(set[d], pair(n + d + SETS));
          __builtin_amdgcn_sched_barrier(0);
          multiply();
        }
      }
    }
  }
  // What is left of a width that is no multiple of 64; all of it where the rows of B are not
  // made of 16-byte pieces: straight into the operands.
  const uint16_t* v[NR];
  int at[NR], tok[NR];
#pragma unroll
  for (int i = 0; i < NR; ++i) at[i] = 16 * i + c;
  tokens_of(plan, list, b, at, tok);
#pragma unroll
  for (int i = 0; i < NR; ++i) v[i] = p.V + (size_t)tok[i] * p.C;
  const int direct_end = min(mm_cdiv(p.C, 64), beg + p.per);
  for (int pr = beg + wave; pr < direct_end; pr += LO_DW) {
    if (pr < p.C / 64 && (!CR || r % 8 == 0)) continue;
    for (int s = 0; s < 2; ++s) {
      const int k0 = 64 * pr + 32 * s + 8 * q, left = p.C - k0;
#pragma unroll
      for (int k = 0; k < RT; ++k) {
        const int rank = min(r0 + 16 * k + c, r - 1);
        u16x8 w;
        if constexpr (!CR) {
          w = load8(W + (size_t)rank * p.C + k0, left);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = i < left ? W[(size_t)(k0 + i) * r + rank] : (uint16_t)0;
        }
#pragma unroll
        for (int i = 0; i < NR; ++i) acc[i][k] = mfma<T>(w, load8(v[i] + k0, left), acc[i][k]);
      }
    }
  }
}

template <int T, bool CR, int RT>
MM_DEV void down_tile(const DownProblem& p, const Plan& plan, const int* list, TileInfo t,
                      const Scaling& scaling, int r, int chunk, float* lds) {
  constexpr int RP = 16 * RT, NT = 64 * LO_DW, ITEMS = LO_TM * RP / 4;   // f32x4 items
  constexpr int PER = ITEMS / NT > 0 ? ITEMS / NT : 1;                   // per thread
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, q = lane >> 4;
  const int b = blockIdx.x, r0 = chunk * RP;
  f32x4 acc[4][RT];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int k = 0; k < RT; ++k) acc[i][k] = f32x4{0, 0, 0, 0};
  if (t.rows > 32) down_sum<T, CR, RT, 4>(p, plan, list, b, t.e, r, r0, (char*)lds, acc);
  else if (t.rows > 16) down_sum<T, CR, RT, 2>(p, plan, list, b, t.e, r, r0, (char*)lds, acc);
  else down_sum<T, CR, RT, 1>(p, plan, list, b, t.e, r, r0, (char*)lds, acc);
  __syncthreads();   // every wave is done with its staging area
  // Sum over the waves, half of them at a time: lds[wave % 4][token][rank].
  uint32_t* s_last = (uint32_t*)(lds + 4 * LO_TM * RP);
  float* s_max = lds + 4 * LO_TM * RP + 4;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    if (wave / 4 == half)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) {
          f32x4* at = (f32x4*)(lds + ((wave & 3) * LO_TM + 16 * i + c) * RP + 16 * k + 4 * q);
          *at = half == 0 ? acc[i][k] : *at + acc[i][k];
        }
    __syncthreads();
  }
  f32x4 h[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * NT;
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
      const int it = threadIdx.x + k * NT;
      if (it < ITEMS) store_agent_x4(prs, 16u * (uint32_t)(blockIdx.y * ITEMS + it), h[k]);
    }
    if (!last_of(p.counters + slot, p.ks, s_last)) return;
#pragma unroll
    for (int k = 0; k < PER; ++k) h[k] = f32x4{0, 0, 0, 0};
    for (int z0 = 0; z0 < p.ks; z0 += 8) {
      f32x4 ld[8][PER];
#pragma unroll
      for (int z = 0; z < 8; ++z)
#pragma unroll
        for (int k = 0; k < PER; ++k)
          ld[z][k] = load_agent_x4(prs, 16u * (uint32_t)(min(z0 + z, p.ks - 1) * ITEMS +
                                                        min((int)threadIdx.x + k * NT, ITEMS - 1)));
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (z0 + z < p.ks)
#pragma unroll
          for (int k = 0; k < PER; ++k) h[k] += ld[z][k];
    }
  }
  // The record.  Ranks and rows past the last are zero.  The RP / 4 threads of a token lie side
  // by side.  A non-finite token leaves the others their bits.
  const float s = scaling.at(t.e);
  float m = 0.0f;
  int row_ex[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * NT, row = 4 * it / RP, rank = 4 * it % RP;
    float rm = 0.0f, f = s;
    if (p.row_mul != nullptr) {
      const int at[1] = {min(row, LO_TM - 1)};
      int token[1];
      tokens_of(plan, list, b, at, token);
      f *= p.row_mul[token[0]];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      h[k][i] = row < t.rows && r0 + rank + i < r ? h[k][i] * f : 0.0f;
      const float a = fabsf(h[k][i]);
      rm = a < __builtin_inff() ? fmaxf(rm, a) : rm;
    }
#pragma unroll
    for (int d = RP / 8; d > 0; d >>= 1) rm = fmaxf(rm, __shfl_xor(rm, d));
    row_ex[k] = carry_exponent(rm);
    m = fmaxf(m, rm);
  }
  int ex = 0;
  if (p.by_rank) {
#pragma unroll
    for (int d = 32; d > RP / 8; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (lane == 0) s_max[wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < LO_DW; ++w) m = fmaxf(m, s_max[w]);
    ex = carry_exponent(m);
    if (threadIdx.x == 0) p.rec.scale[slot] = ldexpf(1.0f, -ex);
  }
  uint16_t* bt = p.rec.by_token + (size_t)slot * 2 * LO_TM * RP;
  uint16_t* br = p.rec.by_rank + (size_t)slot * 2 * LO_TM * RP;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int it = threadIdx.x + k * NT, row = 4 * it / RP, rank = 4 * it % RP;
    if (it >= ITEMS) continue;
    auto split = [&](int e, u16x4& hi, u16x4& lo) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = ldexpf(h[k][i], e);
        hi[i] = from_f32<T>(v);
        const float f = to_f32<T>(hi[i]);
        lo[i] = __builtin_isfinite(f) ? from_f32<T>(v - f) : (uint16_t)0;
      }
    };
    u16x4 hi, lo;
    if (p.by_token) {
      split(row_ex[k], hi, lo);
      *(u16x4*)(bt + row * RP + rank) = hi;
      *(u16x4*)(bt + LO_TM * RP + row * RP + rank) = lo;
      if (rank == 0) p.rec.token_scale[(size_t)slot * LO_TM + row] = ldexpf(1.0f, -row_ex[k]);
    }
    if (p.by_rank) {
      split(ex, hi, lo);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        br[(rank + i) * LO_TM + row] = hi[i];
        br[LO_TM * RP + (rank + i) * LO_TM + row] = lo[i];
      }
    }
  }
}

template <int T, int RT>
__global__ void __launch_bounds__(64 * LO_DW)
k_down(DownProblem p0, DownProblem p1, Plan plan, PlanOut own, Scaling scaling, int r) {
  constexpr int SUM = 4 * LO_TM * 16 * RT + 4 + LO_DW, STAGE = LO_DW * down_lds_wave<RT>() / 4;
  static_assert(LO_DW * (LO_MAX_ADAPTERS + 1) <= STAGE, "own_tile's counts");
  __shared__ __attribute__((aligned(16))) float lds[SUM > STAGE ? SUM : STAGE];
  const int nrc = p0.rec.nrc;
  const bool second = (int)blockIdx.z >= nrc;
  if ((int)blockIdx.y >= (second ? p1.ks : p0.ks)) return;
  __shared__ int list[LO_TM];
  const int* own_list = nullptr;
  TileInfo t;
  if (own.ids.p != nullptr) {
    t = own_tile(own, plan.T, blockIdx.x, blockIdx.y == 0 && blockIdx.z == 0, (int*)lds, list);
    own_list = list;
  } else {
    t = plan.tile(blockIdx.x);
  }
  if (t.e < 0 || t.e >= plan.L) return;
  if (!second) down_tile<T, false, RT>(p0, plan, own_list, t, scaling, r, blockIdx.z, lds);
  else down_tile<T, true, RT>(p1, plan, own_list, t, scaling, r, blockIdx.z - nrc, lds);
}

// ---------------------------------------------------------------------------
// up.  Block (tile, 256 columns): wave: 64 columns, lane (c, q): columns 4c .. 4c + 3 of
// tokens 16 i + 4 q + k.  CR: the factor is [C, r] (B), else [r, C] (A).  BT: the base's
// type (0: no base, zeros), BT_F32: base (or none) and out are fp32.  Group L (no adapter)
// copies the base.
// ---------------------------------------------------------------------------
constexpr int BT_F32 = 3;
struct UpProblem {
  const uint16_t* W;
  const void* base;
  void* out;
  int C;
  Records rec;
};

template <int T, bool CR, int RT, int BT, bool WHOLE>
MM_DEV void up_rows(const UpProblem& p, const Plan& plan, TileInfo t, int r, int b, int col0) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int C = p.C, n0 = col0 + 4 * c;
  const bool none = t.e >= plan.L;
  const int left = C - n0;
  const Records& rec = p.rec;
  const uint16_t* W = p.W + (none ? 0 : (size_t)t.e * r * C);
  // The bases of all rows are on their way before anything else.
  constexpr int NR = LO_TM / 16;
  typename std::conditional<BT == BT_F32, f32x4, u16x4>::type bv[NR * 4];
  int at[NR * 4], token[NR * 4];
#pragma unroll
  for (int i = 0; i < NR * 4; ++i) at[i] = 16 * (i / 4) + 4 * q + i % 4;
  plan.get(b, at, token);
#pragma unroll
  for (int i = 0; i < NR * 4; ++i) {
    const size_t from = (size_t)token[i] * C + n0;
    if constexpr (BT == BT_F32)
      bv[i] = p.base != nullptr ? ld4f<WHOLE>((const float*)p.base + from, left) : f32x4{0, 0, 0, 0};
    else if constexpr (BT != 0) bv[i] = ld4<WHOLE>((const uint16_t*)p.base + from, left);
    else bv[i] = u16x4{0, 0, 0, 0};
  }
  constexpr int NI = 2;   // blocks of 16 rows at a time (all four take the registers of a wave)
  u16x8 w[RT][4];
#pragma unroll
  for (int i0 = 0; i0 < NR; i0 += NI) {
    if (16 * i0 >= t.rows) break;
    f32x4 sum[NI][4];     // [16 rows][column j]: tokens 4q + k
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) sum[i][j] = f32x4{0, 0, 0, 0};
    for (int ch = 0; ch < (none ? 0 : rec.nrc); ++ch) {
      const size_t slot = (size_t)b * rec.nrc + ch;
      const uint16_t* H = rec.by_token + slot * 2 * LO_TM * RP + (q >> 1) * LO_TM * RP +
                          (16 * i0 + c) * RP + 8 * (q & 1);
      f32x4 f[NI];   // of tokens 4q + k
#pragma unroll
      for (int i = 0; i < NI; ++i)
        f[i] = *(const f32x4*)(rec.token_scale + slot * LO_TM + 16 * (i0 + i) + 4 * q);
      u16x8 hv[NI][RT];
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int k = 0; k < RT; ++k) hv[i][k] = *(const u16x8*)(H + 16 * i * RP + 16 * k);
      if (i0 == 0 || rec.nrc > 1) {
#pragma unroll
        for (int k = 0; k < RT; ++k) {
          const int rank = ch * RP + 16 * k + 8 * (q & 1);   // the first of this lane's eight
          if constexpr (CR) {
            // ranks past the last: any, the record has zeros there
#pragma unroll
            for (int j = 0; j < 4; ++j)
              w[k][j] = WHOLE ? *(const u16x8_any*)(W + (size_t)(n0 + j) * r + min(rank, r - 8))
                              : load8(W + (size_t)min(n0 + j, C - 1) * r + rank, r - rank);
          } else {
            u16x4 rows[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              rows[i] = ld4<WHOLE>(W + (size_t)min(rank + i, r - 1) * C + n0, left);
            transpose84(rows, w[k]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int k = 0; k < RT; ++k) acc = mfma<T>(hv[i][k], w[k][j], acc);
          sum[i][j] += f[i] * acc;
        }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = 4 * (i0 + i) + k;
        if (16 * (i0 + i) + 4 * q + k >= t.rows) continue;
        const size_t to = (size_t)token[row] * C + n0;
        if constexpr (BT == BT_F32) {
          f32x4 o = bv[row];
#pragma unroll
          for (int j = 0; j < 4; ++j) o[j] += sum[i][j][k];
          st4f<WHOLE>((float*)p.out + to, o, left);
        } else {
          u16x4 o;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            o[j] = from_f32<T>(BT != 0 ? to_f32<BT != 0 ? BT : T>(bv[row][j]) + sum[i][j][k]
                                       : sum[i][j][k]);
          st4<WHOLE>((uint16_t*)p.out + to, o, left);
        }
      }
  }
}

template <int T, bool CR, int RT, int BT>
MM_DEV void up_tile(const UpProblem& p, const Plan& plan, int r, int b, int colblock) {
  const TileInfo t = plan.tile(b);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col0 = colblock * LO_UP_COLS + wave * 64;
  if (t.e < 0 || (t.e >= plan.L && p.base == p.out) || col0 >= p.C) return;
  if (col0 + 64 <= p.C && (!CR || r % 8 == 0))
    up_rows<T, CR, RT, BT, true>(p, plan, t, r, b, col0);
  else
    up_rows<T, CR, RT, BT, false>(p, plan, t, r, b, col0);
}

template <int T, int RT, int BT>
__global__ void __launch_bounds__(LO_NT)
k_up(UpProblem p, Plan plan, int r) {
  up_tile<T, true, RT, BT>(p, plan, r, blockIdx.x, blockIdx.y);
}

// ---------------------------------------------------------------------------
// wgrad.  Up to two problems: dA_a [r, K] from dH and x, dB_a [N, r] from H and dy.  Block
// (64 columns, adapter, problem x chunk x split): its waves take every fourth 32 tokens of
// the adapter's tiles in its share and add up in LDS.  D rows: ranks 4q + i, columns 4c + j.
// ---------------------------------------------------------------------------
struct GradProblem {
  const uint16_t* V;    // [T, C]
  void* G;              // [L, r, C] or, CR, [L, C, r]; fp32 or the operands' type
  int C, ks, f32;
  int wide;             // every wave has 64 columns of its own and all of the adapter's tokens
  Records rec;
  float* part;          // [adapter][chunk][column block][ks][64 * rp]
  uint32_t* counters;   // [adapter][chunk][column block]

  MM_DEV int cols() const { return mm_cdiv(C, wide ? 4 * LO_WG_COLS : LO_WG_COLS); }
  // n of four adjacent values of the gradient.
  template <int T>
  MM_DEV void store(size_t at, f32x4 v, bool whole, int n) const {
    if (f32) {
      float* o = (float*)G + at;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) o[i] = v[i];
      return;
    }
    u16x4 o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = from_f32<T>(v[i]);
    if (whole) *(u16x4_any*)((uint16_t*)G + at) = o;
    else store4((uint16_t*)G + at, o, n);
  }
};

// sum[k][j]: ranks 16 k + 4 q + i of column n0 + j, over the steps st, st + stride, .. < s_end of
// 32 tokens each, from the adapter's first tile tb on.
template <int T, int RT, bool WHOLE>
MM_DEV void wgrad_sum(const GradProblem& p, const Plan& plan, int n0, int tb, int chunk, int st,
                      int stride, int s_end, f32x4 (&sum)[RT][4]) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4, left = p.C - n0;
#pragma unroll
  for (int k = 0; k < RT; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[k][j] = f32x4{0, 0, 0, 0};
  // Tokens two steps ahead, their rows and the records one step ahead (the last again).
  struct Step {
    u16x4 rows[8];
    u16x8 hi[RT], lo[RT];
    float f;
  };
  int token[8];
  auto find = [&](int st) {
    int at[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) at[i] = 32 * (st & 1) + 8 * q + i;
    plan.get(tb + (st >> 1), at, token);
  };
  auto load = [&](Step& o, int st) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o.rows[i] = ld4<WHOLE>(p.V + (size_t)token[i] * p.C + n0, left);
    const size_t slot = (size_t)(tb + (st >> 1)) * p.rec.nrc + chunk;
    const uint16_t* H =
        p.rec.by_rank + slot * 2 * LO_TM * RP + c * LO_TM + 32 * (st & 1) + 8 * q;
#pragma unroll
    for (int k = 0; k < RT; ++k) {
      o.hi[k] = *(const u16x8*)(H + 16 * k * LO_TM);
      o.lo[k] = *(const u16x8*)(H + LO_TM * RP + 16 * k * LO_TM);
    }
    o.f = p.rec.scale[slot];
  };
  auto multiply = [&](const Step& o) {
    u16x8 w[4];
    transpose84(o.rows, w);
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        sum[k][j] += o.f * mfma<T>(o.hi[k], w[j], mfma<T>(o.lo[k], w[j], f32x4{0, 0, 0, 0}));
  };
  Step even, odd;
  if (st < s_end) {
    const int last = s_end - 1;
    find(st);
    load(even, st);
    find(min(st + stride, last));
    while (true) {
      load(odd, min(st + stride, last));
      find(min(st + 2 * stride, last));
      __builtin_amdgcn_sched_barrier(0);
      multiply(even);
      if ((st += stride) >= s_end) break;
      load(even, min(st + stride, last));
      find(min(st + 2 * stride, last));
      __builtin_amdgcn_sched_barrier(0);
      multiply(odd);
      if ((st += stride) >= s_end) break;
    }
  }
}

template <int T, bool CR, int RT, bool WHOLE>
MM_DEV void wgrad_tile(const GradProblem& p, const Plan& plan, int r, int colblock, int e,
                       int chunk, int split, f32x4* lds) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int n0 = colblock * LO_WG_COLS + 4 * c, left = p.C - n0;
  const int tb = plan.first_tile(e), nt = plan.first_tile(e + 1) - tb;
  const int steps = 2 * nt, per = mm_cdiv(steps, p.ks);
  f32x4 sum[RT][4];
  wgrad_sum<T, RT, WHOLE>(p, plan, n0, tb, chunk, split * per + wave, 4,
                          min(steps, (split + 1) * per), sum);
  // lds[wave][k, j][lane]; wave w then owns columns j = w of every rank tile.
  uint32_t* s_last = (uint32_t*)(lds + 4 * RT * 4 * 64);
#pragma unroll
  for (int k = 0; k < RT; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) lds[((wave * RT + k) * 4 + j) * 64 + lane] = sum[k][j];
  __syncthreads();
  f32x4 own[RT];
#pragma unroll
  for (int k = 0; k < RT; ++k) {
    own[k] = lds[(k * 4 + wave) * 64 + lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) own[k] += lds[((w * RT + k) * 4 + wave) * 64 + lane];
  }
  if (p.ks > 1) {
    const int slot = (e * p.rec.nrc + chunk) * mm_cdiv(p.C, LO_WG_COLS) + colblock;
    const __amdgpu_buffer_rsrc_t prs = mm_rsrc(p.part + (size_t)slot * p.ks * (LO_WG_COLS * RP));
    auto at = [&](int z, int k) { return 16u * (uint32_t)((z * RT + k) * LO_NT + threadIdx.x); };
#pragma unroll
    for (int k = 0; k < RT; ++k) store_agent_x4(prs, at(split, k), own[k]);
    if (!last_of(p.counters + slot, p.ks, s_last)) return;
#pragma unroll
    for (int k = 0; k < RT; ++k) own[k] = f32x4{0, 0, 0, 0};
    for (int z0 = 0; z0 < p.ks; z0 += 8) {
      f32x4 ld[8][RT];
#pragma unroll
      for (int z = 0; z < 8; ++z)
#pragma unroll
        for (int k = 0; k < RT; ++k) ld[z][k] = load_agent_x4(prs, at(min(z0 + z, p.ks - 1), k));
#pragma unroll
      for (int z = 0; z < 8; ++z)
        if (z0 + z < p.ks)
#pragma unroll
          for (int k = 0; k < RT; ++k) own[k] += ld[z][k];
    }
  } else {
    __syncthreads();
  }
  // Wave w holds column 4c + w, ranks 4q + i.  dB has the ranks of a column side by side;
  // dA, columns side by side, goes through LDS once more.
  const size_t G = (size_t)e * r * p.C;
  if constexpr (CR) {
#pragma unroll
    for (int k = 0; k < RT; ++k) {
      const int rank = chunk * RP + 16 * k + 4 * q;
      if (wave < left) p.store<T>(G + (size_t)(n0 + wave) * r + rank, own[k], false, r - rank);
    }
  } else {
    float* tr = (float*)lds;   // [rank][64 columns]
#pragma unroll
    for (int k = 0; k < RT; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        tr[(16 * k + 4 * q + i) * LO_WG_COLS + 4 * c + wave] = own[k][i];
    __syncthreads();
    for (int it = threadIdx.x; it < RP * LO_WG_COLS / 4; it += LO_NT) {
      const int rank = it / (LO_WG_COLS / 4), col = 4 * (it % (LO_WG_COLS / 4));
      const f32x4 v = *(const f32x4*)(tr + rank * LO_WG_COLS + col);
      const int n = colblock * LO_WG_COLS + col;
      if (chunk * RP + rank < r)
        p.store<T>(G + (size_t)(chunk * RP + rank) * p.C + n, v, WHOLE, p.C - n);
    }
  }
}

// The same where an adapter has few tokens: a wave takes all of them, for 64 columns of its own.
template <int T, bool CR, int RT, bool WHOLE>
MM_DEV void wgrad_wave(const GradProblem& p, const Plan& plan, int r, int col0, int e,
                       int chunk) {
  constexpr int RP = 16 * RT;
  const int lane = threadIdx.x & 63, n0 = col0 + 4 * (lane & 15), q = lane >> 4;
  const int tb = plan.first_tile(e), nt = plan.first_tile(e + 1) - tb;
  f32x4 sum[RT][4];
  wgrad_sum<T, RT, WHOLE>(p, plan, n0, tb, chunk, 0, 1, 2 * nt, sum);
  const size_t G = (size_t)e * r * p.C;
#pragma unroll
  for (int k = 0; k < RT; ++k) {
    const int rank = chunk * RP + 16 * k + 4 * q;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if constexpr (CR) {
        if (n0 + i < p.C) p.store<T>(G + (size_t)(n0 + i) * r + rank, sum[k][i], false, r - rank);
      } else if (rank + i < r) {
        p.store<T>(G + (size_t)(rank + i) * p.C + n0,
                   f32x4{sum[k][0][i], sum[k][1][i], sum[k][2][i], sum[k][3][i]}, WHOLE, p.C - n0);
      }
  }
}

// The backward pass behind k_down: dA's blocks, dB's, then dx's.  They do not depend on one
// another, and one launch lets them fill one another's gaps.
// 256 registers, so that two waves share a SIMD: rank 64 by itself takes 309 (backward of 1111
// tokens, 14336 -> 4096, rank 64 105 us; 85 so, with 10 of them spilled, nearly all outside the loops).
template <int T, int RT, int BT>
__global__ void __launch_bounds__(LO_NT, 2)
k_back(GradProblem pa, GradProblem pb, UpProblem pu, Plan plan, int r, int na, int nb) {
  __shared__ __attribute__((aligned(16))) f32x4 lds[4 * RT * 4 * 64 + 1];
  const int nrc = pa.rec.nrc;
  int b = blockIdx.x;
  if (b < na + nb) {
    const GradProblem& p = b < na ? pa : pb;
    const int cols = p.cols(), first = b < na ? 0 : na;
    b -= first;
    const int cb = b % cols, e = b / cols % plan.L, z = b / cols / plan.L;
    if (p.wide) {
      const int col0 =
          (4 * cb + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * LO_WG_COLS;
      if (col0 >= p.C) return;
      const bool whole = col0 + LO_WG_COLS <= p.C;
#define MM_WGRAD(CR, P)                                                       \
  if (whole) wgrad_wave<T, CR, RT, true>(P, plan, r, col0, e, z);              \
  else wgrad_wave<T, CR, RT, false>(P, plan, r, col0, e, z)
      if (first == 0 && (int)blockIdx.x < na) {
        MM_WGRAD(false, pa);
      } else {
        MM_WGRAD(true, pb);
      }
#undef MM_WGRAD
      return;
    }
    const bool whole = (cb + 1) * LO_WG_COLS <= p.C;
#define MM_WGRAD(CR, P)                                                                     \
  if (whole) wgrad_tile<T, CR, RT, true>(P, plan, r, cb, e, z / P.ks, z % P.ks, lds);        \
  else wgrad_tile<T, CR, RT, false>(P, plan, r, cb, e, z / P.ks, z % P.ks, lds)
    if (first == 0 && (int)blockIdx.x < na) {
      MM_WGRAD(false, pa);
    } else {
      MM_WGRAD(true, pb);
    }
#undef MM_WGRAD
    return;
  }
  b -= na + nb;
  const int cols = mm_cdiv(pu.C, LO_UP_COLS);
  up_tile<T, false, RT, BT>(pu, plan, r, b / cols, b % cols);
}

// ---------------------------------------------------------------------------
// Few tokens, and so few factors that every block may read its adapter's A itself: one
// launch.  Block (512 columns, token): its waves take the ranks in pairs and leave H in LDS,
// then a thread has a column, whose factors were on their way meanwhile.
// ---------------------------------------------------------------------------
constexpr int VE_NT = 512, VE_RANKS = 128;
template <int T, int BT>
__global__ void __launch_bounds__(VE_NT)
k_vec(const uint16_t* __restrict__ X, const uint16_t* __restrict__ A,
      const uint16_t* __restrict__ B, Ids ids, Scaling scaling, const uint16_t* base,
      uint16_t* out, int K, int N, int r) {
  __shared__ float h[VE_RANKS];
  const int t = blockIdx.y, n = blockIdx.x * VE_NT + threadIdx.x, a = ids.at(t);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const size_t at = (size_t)t * N + min(n, N - 1);
  float v = to_f32<BT>(base[at]);
  if (a >= 0) {
    const uint16_t* w = B + ((size_t)a * N + min(n, N - 1)) * r;
    const u16x8 w0 = load8(w, r), w1 = load8(w + 8, r - 8);
    const uint16_t* x = X + (size_t)t * K;
    for (int r0 = 2 * wave; r0 < r; r0 += 2 * (VE_NT / 64)) {
      const uint16_t* a0 = A + ((size_t)a * r + r0) * K;
      const uint16_t* a1 = A + ((size_t)a * r + min(r0 + 1, r - 1)) * K;
      float s0 = 0.0f, s1 = 0.0f;
      auto add = [&](u16x8 xv, u16x8 p, u16x8 q) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float f = to_f32<T>(xv[j]);
          s0 += f * to_f32<T>(p[j]);
          s1 += f * to_f32<T>(q[j]);
        }
      };
      int k = 8 * lane;
      for (; k + 3 * 512 + 8 <= K; k += 4 * 512) {
        u16x8 xv[4], p[4], q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          xv[i] = *(const u16x8_any*)(x + k + 512 * i);
          p[i] = *(const u16x8_any*)(a0 + k + 512 * i);
          q[i] = *(const u16x8_any*)(a1 + k + 512 * i);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) add(xv[i], p[i], q[i]);
      }
      for (; k < K; k += 512) add(load8(x + k, K - k), load8(a0 + k, K - k), load8(a1 + k, K - k));
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) {
        s0 += __shfl_xor(s0, d);
        s1 += __shfl_xor(s1, d);
      }
      if (lane == 0) {
        h[r0] = s0 * scaling.at(a);
        if (r0 + 1 < r) h[r0 + 1] = s1 * scaling.at(a);
      }
    }
    __syncthreads();
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if (j < r) s += h[j] * to_f32<T>(w0[j]);
      if (j + 8 < r) s += h[j + 8] * to_f32<T>(w1[j]);
    }
    for (int k = 16; k < r; k += 8) {
      const u16x8 wv = load8(w + k, r - k);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < r) s += h[k + j] * to_f32<T>(wv[j]);
    }
    v += s;
  }
  if (n < N) out[at] = from_f32<T>(v);
}

// ---------------------------------------------------------------------------
// Few tokens, two launches.  k_vec_down: block (token, RG ranks), the width over 256 threads;
// H fp32 [T, r].  k_vec_up: block (256 columns, token), a column per thread.
// ---------------------------------------------------------------------------
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
// Whether every token goes on its own (k_vec*) rather than in tiles of its adapter: two time
// models, us.  On its own a token reads its factors itself, at about 5 TB/s whether from L2 or
// HBM; by tiles there are three launches and a tile per adapter in use, at most L.  Measured,
// on their own / by tiles: 64 tokens of 64 adapters, 4096 -> 4096, rank 16 8.7 / 35; 64 of 8,
// 4096 -> 14336, rank 64 37 / 29; 32 of 32, 14336 -> 4096, rank 64 19 / 42; 128 of 8, 4096 ->
// 4096, rank 16 12 / 16.
bool tokens_alone(int T, int K, int N, int r, int L) {
  if (T > 4096) return false;
  const double factors = 2e-6 * r * ((double)K + N), used = std::min(L, T);
  const double alone = 6 + T * factors / 5;
  const double tiles = 16 + 0.3 * used * mm_cdiv(r, 64) + used * factors / 3.5 +
                       2e-6 * T * (K + 2.0 * N) / 4;
  return alone < tiles;
}
// No sum of a launch with this many blocks per problem is split: a split launch therefore has
// fewer arrival counters than this in use per problem.
constexpr int LO_SPLIT_BELOW = 512;

int rank_tiles(int r) { return r <= 16 ? 1 : (r <= 32 ? 2 : 4); }

struct LoraPlan {
  int rt, rp, nrc;
  int tiles;                       // upper bound of the adapters' tiles
  int all;                         // with those of the tokens without one
  int kx, ky, per;                 // splits of k_down over K and (backward) N, pairs of each
  size_t tokens, first, rec[2], part, total;   // byte offsets; the tile table comes first
};

size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// A k_down block costs about 8 us besides its sums (launch, lists, the hand-off) and one fits
// a CU, so the widths of the launch are cut into equal ranges, as many as fill the CUs once,
// of at least a pair per wave.  us, splits 1 / 2 / 4 / 8 / 16: forward of 1111 tokens, K =
// 14336, rank 64 71 / 55 / 45 / 43 / 52; 4096, 14336, 16 68 / 52 / 43 / 48 / 57; backward of
// 8192 tokens, 4096, 4096 96 / 101 / 108 / 122 / 142.
int down_range(long tiles, int pairs) {
  return std::max(LO_DW, (int)((tiles * pairs + 255) / 256));
}
// Whether a wave of wgrad takes all of an adapter's tokens: where they are few, and the blocks
// still a fair number.  us, backward, four waves an adapter and 64 columns / a wave: 1000 tokens of
// 64 adapters, 4096 -> 4096, rank 16 54.9 / 38.2; 2000 of 16 37.9 / 32.8; 512 of 4, rank 64 40.7 /
// 33.8; 4000 of 1000 771 / 452; the other way 2000 of 4, rank 16 33.0 / 35.0, 128 of 1 15.1 / 16.1.
bool wgrad_wide(int T, int L, int nrc, int C) {
  return T / 32 / L <= 4 && (long)mm_cdiv(C, 4 * LO_WG_COLS) * L * nrc >= 64;
}

// Splits of an adapter's tokens: while a wave has more than 16 steps of 32 on average.  us,
// splits 1 / 2 / 4: backward of 4096 tokens 113 / 104 / 107, 2048 of 2 adapters 81 / 90 / 100.
int wgrad_split(int T, int L, int nrc, int C) {
  if (wgrad_wide(T, L, nrc, C)) return 1;
  const long blocks = (long)mm_cdiv(C, LO_WG_COLS) * L * nrc;
  int ks = 1;
  while (blocks * ks < LO_SPLIT_BELOW && T / 32 / L / (4 * ks) > 16) ks *= 2;
  return ks;
}

size_t record_bytes(const LoraPlan& p) {
  const size_t h = (size_t)p.tiles * p.nrc * 2 * LO_TM * p.rp * 2;
  const size_t n = (size_t)p.tiles * p.nrc;
  return 2 * align256(h) + n * LO_TM * 4 + align256(n * 4);
}
Records record_at(const LoraPlan& p, char* at) {
  const size_t h = align256((size_t)p.tiles * p.nrc * 2 * LO_TM * p.rp * 2);
  float* scales = (float*)(at + 2 * h);
  return Records{(uint16_t*)at, (uint16_t*)(at + h), scales,
                 scales + (size_t)p.tiles * p.nrc * LO_TM, p.rp, p.nrc};
}

// Bytes of a problem's partial sums: `sums` of them if each is split, none otherwise.
size_t part_bytes(size_t sums, int ks) { return ks > 1 ? sums * ks : 0; }
size_t down_part(const LoraPlan& p, int ks) {
  return part_bytes((size_t)p.tiles * p.nrc * LO_TM * p.rp * 4, ks);
}
size_t wgrad_part(const LoraPlan& p, int T, int L, int C) {
  return part_bytes((size_t)L * p.nrc * mm_cdiv(C, LO_WG_COLS) * LO_WG_COLS * p.rp * 4,
                    wgrad_split(T, L, p.nrc, C));
}

// Workspace: counters, the plan, the records of both problems, partial sums (of k_down and
// then of wgrad, one after the other in the same memory).
LoraPlan plan_lora(int T, int K, int N, int r, int L, bool backward) {
  LoraPlan p{};
  p.rt = rank_tiles(r);
  p.rp = 16 * p.rt;
  p.nrc = mm_cdiv(r, p.rp);
  p.tiles = T / LO_TM + std::min(L, T);
  p.all = T / LO_TM + std::min(L + 1, T);
  p.tokens = LO_COUNTER_BYTES + align256((size_t)p.all * sizeof(TileInfo));
  p.first = p.tokens + align256((size_t)p.all * LO_TM * 4);
  p.rec[0] = p.first + align256(((size_t)L + 2) * 4);
  p.rec[1] = p.rec[0] + record_bytes(p);
  p.part = p.rec[1] + (backward ? record_bytes(p) : 0);
  const int px = mm_cdiv(K, 64), py = backward ? mm_cdiv(N, 64) : 0;
  p.per = down_range((long)p.tiles * p.nrc, px + py);
  p.kx = mm_cdiv(px, p.per);
  p.ky = mm_cdiv(py, p.per);
  size_t part = down_part(p, p.kx) + down_part(p, p.ky);
  if (backward) part = std::max(part, wgrad_part(p, T, L, K) + wgrad_part(p, T, L, N));
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
  MM_CHECK_ARG(L <= LO_MAX_ADAPTERS, "%s: at most %d adapters, got %d", who, LO_MAX_ADAPTERS, L);
  MM_CHECK_ARG(T <= (1 << 24) && K <= (1 << 24) && N <= (1 << 24) && r <= (1 << 12),
               "%s: T=%d, K=%d, N=%d or rank=%d is too large", who, T, K, N, r);
  // an adapter's factors are addressed with 32 bits
  MM_CHECK_ARG((long)r * K < (1L << 31) && (long)r * N < (1L << 31),
               "%s: rank=%d times K=%d or N=%d is too large", who, r, K, N);
  return 0;
}

// The tokens sorted by adapter: by a launch, by k_down's blocks (`own`), or as they come (a
// single adapter without ids).
int make_plan(const char* who, const LoraPlan& p, const void* ids, int ids64, int T, int L,
              void* ws, hipStream_t st, Plan* plan, PlanOut* own) {
  *plan = Plan{nullptr, nullptr, nullptr, T, L};
  *own = PlanOut{};
  if (ids == nullptr) return 0;
  const PlanOut o{Ids{ids, ids64, L}, (TileInfo*)((char*)ws + LO_COUNTER_BYTES),
                  (int*)((char*)ws + p.tokens), (int*)((char*)ws + p.first)};
  *plan = Plan{o.tiles, o.tokens, o.first, T, L};
  if (T <= DP_TOKENS) {
    *own = o;
    return 0;
  }
  hipLaunchKernelGGL(k_plan, dim3(1), dim3(PL_NT), 0, st, o.ids, T, p.all, o.tiles, o.tokens,
                     o.first);
  MM_CHECK_LAUNCH(who);
  return 0;
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
  if (!backward && tokens_alone(T, K, N, r, L)) return LO_COUNTER_BYTES + (size_t)T * r * 4;
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
  if (tokens_alone(T, K, N, r, L)) {
    float* H = (float*)((char*)ws + LO_COUNTER_BYTES);
    const Ids id{ids, ids64, L};
    // One launch while a block's read of A (at 50 GB/s and CU) costs less than a launch.  us,
    // one / two launches: 1 token, 4096 -> 4096, rank 16 4.8 / 7.2; 8 tokens 5.1 / 8.0; 32
    // tokens, 4096 -> 6144 9.5 / 8.0; 1 token, 14336 -> 4096, rank 64 29 / 9.4.
    const long a_bytes = 2L * r * K;
    if (r <= VE_RANKS && a_bytes <= 256 << 10 && mm_cdiv(N, VE_NT) * T * a_bytes <= 24L << 20) {
#define MM_VEC(TV, BV)                                                                         \
  hipLaunchKernelGGL((k_vec<TV, BV>), dim3(mm_cdiv(N, VE_NT), T), dim3(VE_NT), 0, st, x, A, B, id, \
                     sc, base, out, K, N, r)
      if (type == 1) MM_VEC(1, 1);
      else if (base_type == 1) MM_VEC(2, 1);
      else MM_VEC(2, 2);
#undef MM_VEC
      MM_CHECK_LAUNCH(who);
      return 0;
    }
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
  Plan plan;
  PlanOut own;
  if (const int rc = make_plan(who, p, ids, ids64, T, L, ws, st, &plan, &own)) return rc;
  const int down_tiles = own.ids.p != nullptr ? p.all : p.tiles;
  const Records rec = record_at(p, (char*)ws + p.rec[0]);
  const int ks = p.kx;
  const DownProblem d{x, A, K, ks, p.per, rec, (float*)((char*)ws + p.part),
                      (uint32_t*)ws, 1, 0, nullptr};
#define MM_DOWN(RTV, TV)                                                                       \
  hipLaunchKernelGGL((k_down<TV, RTV>), dim3(down_tiles, ks, p.nrc), dim3(64 * LO_DW), 0, st, d,  \
                     d, plan, own, sc, r)
  if (type == 1) { MM_LORA_RT(MM_DOWN, 1) } else { MM_LORA_RT(MM_DOWN, 2) }
  MM_CHECK_LAUNCH(who);
  const UpProblem u{B, base, out, N, rec};
  const dim3 grid(p.all, mm_cdiv(N, LO_UP_COLS));
#define MM_UP(RTV, TV, BV) \
  hipLaunchKernelGGL((k_up<TV, RTV, BV>), grid, dim3(LO_NT), 0, st, u, plan, r)
  if (type == 1) { MM_LORA_RT(MM_UP, 1, 1) }
  else if (base_type == 1) { MM_LORA_RT(MM_UP, 2, 1) }
  else { MM_LORA_RT(MM_UP, 2, 2) }
#undef MM_UP
#undef MM_DOWN
  MM_CHECK_LAUNCH(who);
  return 0;
}

// wide: dx_base and dx are fp32, else of the type of x.
static int lora_backward(const char* who, const uint16_t* dy, const float* row_mul,
                         const uint16_t* x, int type, const uint16_t* A, const uint16_t* B,
                         const void* ids, int ids64, const float* scaling, float scale, bool wide,
                         const void* dx_base, void* dx, void* dA, void* dB, int grad_type, int T,
                         int K, int N, int r, int L, void* ws, size_t ws_bytes, void* stream) {
  if (const int rc = check_common(who, type, T, K, N, r, L, ids, ids64)) return rc;
  MM_CHECK_ARG(grad_type == 0 || grad_type == type,
               "%s: grad_type=%d must be 0 (fp32) or the type of x", who, grad_type);
  MM_CHECK_ARG(T > 0, "%s: no tokens (the gradients are zeros)", who);
  const size_t need = mm_lora_workspace_bytes(T, K, N, r, L, 1);
  MM_CHECK_ARG(ws != nullptr && ws_bytes >= need,
               "%s: workspace of %zu bytes is smaller than the %zu required", who, ws_bytes, need);
  hipStream_t st = (hipStream_t)stream;
  const Scaling sc{scaling, scale};
  const LoraPlan p = plan_lora(T, K, N, r, L, true);
  Plan plan;
  PlanOut own;
  if (const int rc = make_plan(who, p, ids, ids64, T, L, ws, st, &plan, &own)) return rc;
  const int down_tiles = own.ids.p != nullptr ? p.all : p.tiles;
  const Records rx = record_at(p, (char*)ws + p.rec[0]), ry = record_at(p, (char*)ws + p.rec[1]);
  char* part = (char*)ws + p.part;
  uint32_t* counters = (uint32_t*)ws;
  const int kx = p.kx, ky = p.ky;
  const DownProblem px{x, A, K, kx, p.per, rx, (float*)part, counters, 0, 1, row_mul};
  const DownProblem py{dy, B, N, ky, p.per, ry, (float*)(part + down_part(p, kx)),
                       counters + LO_SPLIT_BELOW, 1, 1, row_mul};
#define MM_DOWN(RTV, TV)                                                                       \
  hipLaunchKernelGGL((k_down<TV, RTV>), dim3(down_tiles, std::max(kx, ky), 2 * p.nrc),             \
                     dim3(64 * LO_DW), 0, st, px, py, plan, own, sc, r)
  if (type == 1) { MM_LORA_RT(MM_DOWN, 1) } else { MM_LORA_RT(MM_DOWN, 2) }
#undef MM_DOWN
  MM_CHECK_LAUNCH(who);
  const bool wa = wgrad_wide(T, L, p.nrc, K), wb = wgrad_wide(T, L, p.nrc, N);
  const int ca = mm_cdiv(K, wa ? 4 * LO_WG_COLS : LO_WG_COLS);
  const int cb = mm_cdiv(N, wb ? 4 * LO_WG_COLS : LO_WG_COLS);
  const int ga = wgrad_split(T, L, p.nrc, K), gb = wgrad_split(T, L, p.nrc, N);
  const GradProblem pa{x, dA, K, ga, grad_type == 0, wa, ry, (float*)part, counters};
  const GradProblem pb{dy, dB, N, gb, grad_type == 0, wb, rx,
                       (float*)(part + wgrad_part(p, T, L, K)), counters + LO_SPLIT_BELOW};
  const UpProblem pu{A, dx_base, dx, K, ry};
  const long na = (long)ca * L * p.nrc * ga, nb = (long)cb * L * p.nrc * gb;
  const long nu = (long)p.all * mm_cdiv(K, LO_UP_COLS);
  MM_CHECK_ARG(na + nb + nu < 0x7fffffffL, "%s: K=%d, N=%d with %d adapters is too large", who, K,
               N, L);
#define MM_BACK(RTV, TV, BV)                                                                   \
  hipLaunchKernelGGL((k_back<TV, RTV, BV>), dim3((unsigned)(na + nb + nu)), dim3(LO_NT), 0, st, pa, \
                     pb, pu, plan, r, (int)na, (int)nb)
  if (wide) {
    MM_LORA_RT(MM_BACK, 1, BT_F32)
  } else if (dx_base != nullptr) {
    if (type == 1) { MM_LORA_RT(MM_BACK, 1, 1) } else { MM_LORA_RT(MM_BACK, 2, 2) }
  } else {
    if (type == 1) { MM_LORA_RT(MM_BACK, 1, 0) } else { MM_LORA_RT(MM_BACK, 2, 0) }
  }
#undef MM_BACK
  MM_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int mm_lora_backward(const uint16_t* dy, const uint16_t* x, int type,
                                const uint16_t* A, const uint16_t* B, const void* ids, int ids64,
                                const float* scaling, float scale, const uint16_t* dx_base,
                                uint16_t* dx, void* dA, void* dB, int grad_type, int T, int K,
                                int N, int r, int L, void* ws, size_t ws_bytes, void* stream) {
  return lora_backward("mm_lora_backward", dy, nullptr, x, type, A, B, ids, ids64, scaling, scale,
                       false, dx_base, dx, dA, dB, grad_type, T, K, N, r, L, ws, ws_bytes, stream);
}

extern "C" int mm_lora_backward_f32(const uint16_t* dy, const float* row_mul, const uint16_t* x,
                                    const uint16_t* A, const uint16_t* B, const void* ids,
                                    int ids64, const float* scaling, float scale,
                                    const float* dx_base, float* dx, void* dA, void* dB,
                                    int grad_type, int T, int K, int N, int r, int L, void* ws,
                                    size_t ws_bytes, void* stream) {
  const char* who = "mm_lora_backward_f32";
  MM_CHECK_ARG((((uintptr_t)row_mul | (uintptr_t)dx_base | (uintptr_t)dx) & 3) == 0,
               "%s: row_mul, dx_base and dx must be 4-byte aligned", who);
  return lora_backward(who, dy, row_mul, x, 1, A, B, ids, ids64, scaling, scale, true, dx_base, dx,
                       dA, dB, grad_type, T, K, N, r, L, ws, ws_bytes, stream);
}
