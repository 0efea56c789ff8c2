// Cores of the MXFP4 products, shared by the dense and the grouped (experts') kernels:
//   D[n, m] = sum_k W[n, k] x[m, k], W and x both MXFP4 (mm_mx.h), fp32 sums.
// The weights are the matrix instruction's first operand, so a lane holds consecutive n of one m.
#pragma once

#include <type_traits>
#include <utility>

#include "mm_mx.h"

namespace mmmx {

template <class F, int... I>
MM_DEV void static_for(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
MM_DEV void repeat(F&& f) {
  static_for(f, std::make_integer_sequence<int, N>{});
}

// ---------------------------------------------------------------------------
// Few rows: bound by the weights' bytes.  NW waves share out the units of 256 k; a lane's 16-byte
// loads are the matrix operand as it lies in memory (a 16-row tile's 1 KiB per instruction), so
// weights go from HBM to the matrix cores without LDS.  The 16 rows of x per instruction are
// quantized in registers by every wave for its own k (a lane holds whole blocks: no exchange), or
// come as codes (T == CODES, rows padded to whole units).
// ---------------------------------------------------------------------------
template <int T, int MT>
struct XUnit {
  Vals<T> v[MT][2][4];
};
template <int MT>
struct XUnit<CODES, MT> {
  u32x4 v[MT][2];
  uint8_t s[MT][2];
};
template <int NT>
struct WUnit {
  u32x4 v[NT][2];
  uint8_t s[NT][2];
};

MM_DEV u32x4 load_once(const uint8_t* p) {   // weights: each is read once per launch
  return __builtin_nontemporal_load((const u32x4*)p);
}

// x: this lane's row of each 16-row tile; xs: its scales (CODES).  w, s: its weight rows.
// acc[mt][nt][i] is D[16 nt + 4 (lane / 16) + i, 16 mt + lane % 16].
template <int T, int MT, int NT, int NW>
MM_DEV void skinny(const char* const (&x)[MT], const uint8_t* const (&xs)[MT],
                   const uint8_t* const (&w)[NT], const uint8_t* const (&s)[NT], int K,
                   f32x4 (&acc)[MT][NT]) {
  const int lane = threadIdx.x & 63, q = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kb = K / BLOCK, units = K / UNIT;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0, 0, 0, 0};
  // b: this lane's block of the instruction
  auto load_w = [&](int b, int j, bool live, WUnit<NT>& o) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      o.v[nt][j] = live ? load_once(w[nt] + (size_t)b * 16) : u32x4{0, 0, 0, 0};
      o.s[nt][j] = live ? s[nt][b] : (uint8_t)0;
    }
  };
  auto load_x = [&](int b, int j, bool live, XUnit<T, MT>& o) {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      if constexpr (T == CODES) {
        o.v[mt][j] = *(const u32x4*)(x[mt] + (size_t)b * 16);    // padded: always there
        o.s[mt][j] = xs[mt][b];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          o.v[mt][j][i] =
              live ? load8<T>(x[mt] + ((size_t)b * BLOCK + 8 * i) * kBytes<T>) : zero8<T>();
      }
    }
  };
  auto compute = [&](const WUnit<NT>& wu, const XUnit<T, MT>& xu) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        u32x4 xv;
        uint32_t xc;
        if constexpr (T == CODES) {
          xv = xu.v[mt][j];
          xc = xu.s[mt][j];
        } else {
          xv = pack_block<T>(xu.v[mt][j], xc);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          acc[mt][nt] = mfma16<0, 0>(wu.v[nt][j], wu.s[nt][j], xv, xc, acc[mt][nt]);
      }
  };
  int u = wave;
  if (u < units) {
    WUnit<NT> wu;
    XUnit<T, MT> xu;
#pragma unroll
    for (int j = 0; j < 2; ++j) load_w(8 * u + 4 * j + q, j, true, wu);
#pragma unroll
    for (int j = 0; j < 2; ++j) load_x(8 * u + 4 * j + q, j, true, xu);
    for (; u + NW < units; u += NW) {
      WUnit<NT> wn;
      XUnit<T, MT> xn;
#pragma unroll
      for (int j = 0; j < 2; ++j) load_w(8 * (u + NW) + 4 * j + q, j, true, wn);
#pragma unroll
      for (int j = 0; j < 2; ++j) load_x(8 * (u + NW) + 4 * j + q, j, true, xn);
      compute(wu, xu);
      wu = wn;
      xu = xn;
    }
    compute(wu, xu);
  }
  if (K % UNIT != 0 && wave == units % NW) {   // the last blocks, fewer than 8
    WUnit<NT> wu;
    XUnit<T, MT> xu;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int b = 8 * units + 4 * j + q;
      load_w(b, j, b < kb, wu);
      load_x(b, j, b < kb, xu);
    }
    compute(wu, xu);
  }
}

// Sums of the waves: every wave parks its tiles, then fn(nn, mm, sum) gets D[nn, mm] of the
// 16 NT x rows block, each from one thread, summed in wave order.
template <int MT, int NT, int NW, class F>
MM_DEV void skinny_reduce(const f32x4 (&acc)[MT][NT], float* red, int rows, F&& fn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f32x4* mine = (f32x4*)red + (size_t)wave * MT * NT * 64 + lane;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mine[(mt * NT + nt) * 64] = acc[mt][nt];
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * NT * rows; o += NW * 64) {
    const int mm = o / (16 * NT), nn = o % (16 * NT);
    const int at = (((mm / 16) * NT + nn / 16) * 64 + (nn % 16 / 4) * 16 + mm % 16) * 4 + nn % 4;
    float sum = red[at];
#pragma unroll
    for (int v = 1; v < NW; ++v) sum += red[v * MT * NT * 256 + at];
    fn(nn, mm, sum);
  }
}

// ---------------------------------------------------------------------------
// More rows: tiles of TM x-rows by TN weight rows, bound by the matrix cores and LDS.  A stage is
// one unit of 256 k: 128 bytes of every row, copied global -> LDS directly in 16-byte pieces, the
// next stage while this one is multiplied.  Piece p of row r lies at p ^ (r / 2 % 8), so that the
// 16 rows that an operand read takes at once spread over all banks.  The 8 scales per row go
// through registers.  Each wave owns 32 NB x 32 MB of the tile.
// Rows of x are padded to whole units with zeros; what a weight row's last stage reads behind K
// is some of its own blocks, times those zeros.
// ---------------------------------------------------------------------------
typedef __attribute__((address_space(3))) void* lds_ptr;
MM_DEV void copy16(const void* src, void* lds_uniform) {
  __builtin_amdgcn_global_load_lds(src, (lds_ptr)lds_uniform, 16, 0, 0);
}

template <int WM_, int WN_, int MB_, int NB_>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MB = MB_, NB = NB_;
  static constexpr int NTHR = WM * WN * 64, NWAVE = WM * WN;
  static constexpr int TM = WM * MB * 32, TN = WN * NB * 32, ROWS = TM + TN;
  static constexpr int STAGE = ROWS * 128, SSTAGE = ROWS * 8;
  static constexpr int LDS = 2 * (STAGE + SSTAGE);
  static constexpr int IT = ROWS / 8 / NWAVE;          // 1 KiB copies per wave and stage
  static constexpr int SIT = (ROWS + NTHR - 1) / NTHR; // scale rows per thread
  static_assert(ROWS % (8 * NWAVE) == 0, "copies per wave");
  static_assert(TN % 8 == 0 && TM % 8 == 0, "a copy's rows are all of W or all of x");
};

// The 8 scales from `at` on, of `blocks` >= 8; those behind the end are zero.
MM_DEV u32x2 load_scales(const uint8_t* p, int at, int blocks) {
  u32x2 v;
  __builtin_memcpy(&v, p + min(at, blocks - 8), 8);    // one load, whatever its alignment
  return v;
}
MM_DEV u32x2 shift_scales(u32x2 v, int at, int blocks) {
  const uint64_t q = (uint64_t)v.y << 32 | v.x;
  const uint64_t r = q >> (8 * max(0, at + 8 - blocks));
  return u32x2{(uint32_t)r, (uint32_t)(r >> 32)};
}

// Stages [u0, u1) into acc.  src: W, S, X, XS (the bases of the weights' and x's words and
// scales), K and kp (values per row of W and of x), wrow(r) and xrow(r): the row, counted from
// those bases, of row r of the tile; every one must be readable, and rows times K / 2 or kp / 2
// stay below 2^32.
template <class Sh, class Src>
MM_DEV void tile_loop(const Src& src, int u0, int u1, char* smem, f32x16 (&acc)[Sh::NB][Sh::MB]) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / Sh::WN, wn = wave % Sh::WN, l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int n = 0; n < Sh::NB; ++n)
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[n][m][i] = 0.0f;
  if (u0 >= u1) return;

  uint32_t off[Sh::IT];
#pragma unroll
  for (int i = 0; i < Sh::IT; ++i) {
    const int r0 = (i * Sh::NWAVE + wave) * 8, r = r0 + lane / 8;
    off[i] = r0 < Sh::TN ? src.wrow(r) * (uint32_t)(src.K / 2)
                         : src.xrow(r - Sh::TN) * (uint32_t)(src.kp / 2);
  }
  static_assert(Sh::NWAVE % 2 == 0, "a lane's pieces lie alike in all its copies");
  const int at = 16 * ((lane & 7) ^ ((wave * 4 + (lane >> 4)) & 7));
  auto issue = [&](int u, int st) {
#pragma unroll
    for (int i = 0; i < Sh::IT; ++i) {
      const bool isw = (i * Sh::NWAVE + wave) * 8 < Sh::TN;
      const uint8_t* const base = (isw ? src.W : src.X) + (size_t)u * 128;
      const int left = (isw ? src.K : src.kp) / 2 - 16 - u * 128;
      copy16(base + (off[i] + (uint32_t)min(at, left)),
             smem + st * Sh::STAGE + (i * Sh::NWAVE + wave) * 1024);
    }
  };
  const uint8_t* scale[Sh::SIT];
  int blocks[Sh::SIT];
#pragma unroll
  for (int i = 0; i < Sh::SIT; ++i) {
    const int r = min(tid + i * Sh::NTHR, Sh::ROWS - 1);
    const bool isw = r < Sh::TN;
    blocks[i] = (isw ? src.K : src.kp) / BLOCK;
    scale[i] = isw ? src.S + (size_t)src.wrow(r) * blocks[i]
                   : src.XS + (size_t)src.xrow(r - Sh::TN) * blocks[i];
  }
  u32x2 sc[Sh::SIT];
  auto load_sc = [&](int u) {
#pragma unroll
    for (int i = 0; i < Sh::SIT; ++i) sc[i] = load_scales(scale[i], 8 * u, blocks[i]);
  };
  auto store_sc = [&](int u, int st) {
#pragma unroll
    for (int i = 0; i < Sh::SIT; ++i) {
      const int r = tid + i * Sh::NTHR;
      if (Sh::ROWS % Sh::NTHR == 0 || r < Sh::ROWS)
        *(u32x2*)(smem + 2 * Sh::STAGE + st * Sh::SSTAGE + r * 8) =
            shift_scales(sc[i], 8 * u, blocks[i]);
    }
  };
  auto compute = [&](int st) {
    const char* const d = smem + st * Sh::STAGE;
    const char* const s = smem + 2 * Sh::STAGE + st * Sh::SSTAGE;
    u32x2 sw[Sh::NB], sx[Sh::MB];
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n)
      sw[n] = *(const u32x2*)(s + ((wn * Sh::NB + n) * 32 + l32) * 8) >> (uint32_t)(8 * h);
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
      sx[m] = *(const u32x2*)(s + (Sh::TN + (wm * Sh::MB + m) * 32 + l32) * 8) >> (uint32_t)(8 * h);
    // The operands of a quarter are read while the quarter before it is multiplied.
    u32x4 a[2][Sh::NB], b[2][Sh::MB];
    auto read = [&](int j, u32x4 (&av)[Sh::NB], u32x4 (&bv)[Sh::MB]) {
      const int p = 16 * ((2 * j + h) ^ ((l32 >> 1) & 7));
#pragma unroll
      for (int n = 0; n < Sh::NB; ++n)
        av[n] = *(const u32x4*)(d + ((wn * Sh::NB + n) * 32 + l32) * 128 + p);
#pragma unroll
      for (int m = 0; m < Sh::MB; ++m)
        bv[m] = *(const u32x4*)(d + (Sh::TN + (wm * Sh::MB + m) * 32 + l32) * 128 + p);
    };
    read(0, a[0], b[0]);
    repeat<4>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < 3) read(j + 1, a[(j + 1) & 1], b[(j + 1) & 1]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < Sh::NB; ++n)
#pragma unroll
        for (int m = 0; m < Sh::MB; ++m)
          acc[n][m] = mfma32<j % 2 * 2, j % 2 * 2>(a[j & 1][n], sw[n][j / 2], b[j & 1][m],
                                                   sx[m][j / 2], acc[n][m]);
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  issue(u0, 0);
  if (src.K >= UNIT) {
    load_sc(u0);
    store_sc(u0, 0);
  } else {                        // one stage, fewer than 8 blocks in a row of W
#pragma unroll
    for (int i = 0; i < Sh::SIT; ++i) {
      const int r = tid + i * Sh::NTHR;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (r < Sh::ROWS)
          smem[2 * Sh::STAGE + r * 8 + c] = c < blocks[i] ? (char)scale[i][c] : (char)0;
    }
  }
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  int st = 0;
  for (int u = u0; u + 1 < u1; ++u) {
    issue(u + 1, st ^ 1);
    load_sc(u + 1);
    __builtin_amdgcn_sched_barrier(0);
    compute(st);
    store_sc(u + 1, st ^ 1);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    st ^= 1;
  }
  compute(st);
}

// fn(n, m, v): v[0..3] are D[n..n+3, m] of the tile, n a multiple of 4.
template <class Sh, class F>
MM_DEV void tile_out(const f32x16 (&acc)[Sh::NB][Sh::MB], F&& fn) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int wm = wave / Sh::WN, wn = wave % Sh::WN, l32 = lane & 31, h = lane >> 5;
#pragma unroll
  for (int m = 0; m < Sh::MB; ++m)
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        fn((wn * Sh::NB + n) * 32 + 8 * g + 4 * h, (wm * Sh::MB + m) * 32 + l32,
           f32x4{acc[n][m][4 * g], acc[n][m][4 * g + 1], acc[n][m][4 * g + 2], acc[n][m][4 * g + 3]});
}

}  // namespace mmmx
