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

typedef __attribute__((address_space(3))) void* lds_ptr;
// 16 bytes per lane straight to LDS, the lanes' pieces side by side from lds_uniform on.
MM_DEV void copy16(const void* src, void* lds_uniform) {
  __builtin_amdgcn_global_load_lds(src, (lds_ptr)lds_uniform, 16, 0, 0);
}
MM_DEV void copy4(const void* src, void* lds_uniform) {
  __builtin_amdgcn_global_load_lds(src, (lds_ptr)lds_uniform, 4, 0, 0);
}
// Waits until at most N vector memory operations are in flight.
template <int N>
MM_DEV void wait_loads() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
  __builtin_amdgcn_sched_barrier(0);
}

// Stores to LDS beside copies to other parts of it: the compiler has a store of its own wait for
// all copies in flight, which may be to the same place for all that it knows.  stores_done()
// before what relies on them.
MM_DEV uint32_t lds_at(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
MM_DEV void lds_store4(void* p, uint32_t v) {
  asm volatile("ds_write_b32 %0, %1" ::"v"(lds_at(p)), "v"(v) : "memory");
}
MM_DEV void lds_store16(void* p, u32x4 v) {
  asm volatile("ds_write_b128 %0, %1" ::"v"(lds_at(p)), "v"(v) : "memory");
}
MM_DEV void lds_store1(void* p, uint32_t v) {
  asm volatile("ds_write_b8 %0, %1" ::"v"(lds_at(p)), "v"(v) : "memory");
}
MM_DEV void stores_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// A barrier that waits for no copy in flight (__syncthreads waits for them all).
MM_DEV void block_barrier() {
  stores_done();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Nothing moves across this, loads of LDS least of all.
MM_DEV void in_order() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// ---------------------------------------------------------------------------
// Few rows: bound by the weights' bytes.  The NW waves of a block share out the units of 256 k.
// A wave copies its units' rows global -> LDS, 128 bytes of 8 rows per instruction (a matrix
// operand taken straight from memory would ask for 64 bytes of 16 rows, and a CU then gets 13
// GB/s where it gets 29 from whole lines), DEPTH units ahead, in a ring of its own: it waits for
// its own loads only, never for another wave.  Piece p of row r lies at p ^ (r / 2 % 8): the 16
// rows that an operand read takes at once spread over all banks.
// The rows are 16 NT of W, then (XT > 0) 16 XT of x's codes.
// ---------------------------------------------------------------------------
template <int NT, int XT, int NW, int DEPTH>
struct Ring {
  static constexpr int ROWS = 16 * (NT + XT), LOADS = ROWS / 8, STAGE = ROWS * 128;
  static constexpr int BYTES = NW * DEPTH * STAGE;
  static_assert(LOADS * (DEPTH - 1) < 64, "loads in flight");
  static_assert(STAGE >= NT * 1024, "the waves' sums take its place");
  uint32_t off[LOADS];
  const uint8_t *W, *X;
  char* mine;
  int k;               // bytes per row of W

  // wrow(r), xrow(r): the row, from W and X on, of row r of the tile.
  template <class WRow, class XRow>
  MM_DEV Ring(char* lds, const uint8_t* w, int K, WRow&& wrow, const uint8_t* x, int kp, XRow&& xrow)
      : W(w), X(x), k(K / 2) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    mine = lds + wave * DEPTH * STAGE;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int r = i * 8 + lane / 8;
      off[i] = i < 2 * NT ? wrow(r) * (uint32_t)k : xrow(r - 16 * NT) * (uint32_t)(kp / 2);
    }
  }
  MM_DEV void issue(int u, int d) const {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int at = 16 * ((lane & 7) ^ (4 * (i & 1) + (lane >> 4)));
      // behind K the row's last piece, which meets zeros of x
      if (i < 2 * NT) at = min(at, k - 16 - u * 128);
      copy16((i < 2 * NT ? W : X) + (size_t)u * 128 + (off[i] + (uint32_t)at),
             mine + d * STAGE + i * 1024);
    }
  }
  // Blocks 4 j + lane / 16 of row 16 t + lane % 16, t counting the weights' tiles, then x's.
  MM_DEV u32x4 operand(int d, int t, int j) const {
    const int lane = threadIdx.x & 63, r = lane & 15, p = (4 * j + (lane >> 4)) ^ (r >> 1);
    return *(const u32x4*)(mine + d * STAGE + (16 * t + r) * 128 + p * 16);
  }
};

// Bytes to LDS by the whole block, 16 per lane and copy: the last piece again where a wave has
// lanes to spare, so dst has room for whole KiB.  bytes a multiple of 16, both ends aligned so.
template <int NTHR>
MM_DEV void copy_to_lds(const uint8_t* src, char* dst, int bytes) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int b = wave * 1024; b < bytes; b += NTHR * 16)
    copy16(src + min(b + lane * 16, bytes - 16), dst + b);
}
constexpr int whole_kib(int bytes) { return (bytes + 1023) / 1024 * 1024; }

// Scales of rows that lie side by side, of whose `bytes` the first `valid` are there: copied, or,
// for the last rows of W, stored byte by byte (before any copy is in flight).
template <int NTHR>
MM_DEV void scales_to_lds(const uint8_t* src, char* dst, int bytes, int valid) {
  if (valid == bytes) {
    copy_to_lds<NTHR>(src, dst, bytes);
  } else {
    for (int i = threadIdx.x; i < bytes; i += NTHR) dst[i] = i < valid ? (char)src[i] : (char)0;
  }
}

// Rows of x in LDS, `lds_stride` bytes of codes each (an odd number of 16-byte pieces:
// consecutive rows in different banks), then their scales.
constexpr int lds_stride(int kp) { return kp / 2 + 16; }
__host__ __device__ constexpr int lds_x_bytes(int rows, int kp) {
  return rows * (lds_stride(kp) + kp / BLOCK);
}

// Exchange within groups of four lanes.
MM_DEV uint32_t quad_max(uint32_t m) {
  m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true));
  return max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true));
}

// The block quantizes `rows` <= 16 rows of K values into LDS, zeros from K to kp, U pieces of 8
// values per thread and batch, four lanes to a block of 32.  The values come through LDS as well
// (raw: raw_bytes of it): a value in a register would be waited for together with every copy in
// flight.  A lane reads what it copied itself.
// base(m): where row m begins.  first() issues the first batch; finish() expects it there and
// leaves no copy in flight if there are more.
template <int T, int NTHR, int U, class Base>
struct QuantizeRows {
  static constexpr int PARTS = T == F32 ? 2 : 1;
  static constexpr int RAW = U * PARTS * NTHR * 16;
  char *raw, *out;
  int rows, K, kp;
  Base base;
  // row and column (in pieces) of piece p; exact for the few rows there are
  MM_DEV void place(int p, int& m, int& c) const {
    const int w = kp / 8;
    m = (int)(((float)p + 0.5f) * (1.0f / (float)w));
    c = p - m * w;
  }
  MM_DEV void issue(int p0) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      int m, c;
      place(p0 + i * NTHR + threadIdx.x, m, c);
      const char* src = base(min(m, rows - 1)) + (size_t)min(c, K / 8 - 1) * 8 * kBytes<T>;
#pragma unroll
      for (int h = 0; h < PARTS; ++h)
        copy16(src + 16 * h, raw + ((i * PARTS + h) * (NTHR / 64) + wave) * 1024);
    }
  }
  MM_DEV void store(int p0) const {
    const int stride = lds_stride(kp);
    char* const scales = out + rows * stride;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      int m, c;
      place(p0 + i * NTHR + threadIdx.x, m, c);
      Vals<T> v;
      if constexpr (T == F32) {
        v.v[0] = *(const f32x4*)(raw + (2 * i * NTHR + threadIdx.x) * 16);
        v.v[1] = *(const f32x4*)(raw + ((2 * i + 1) * NTHR + threadIdx.x) * 16);
      } else {
        v.v = *(const u32x4*)(raw + (i * NTHR + threadIdx.x) * 16);
      }
      if (c >= K / 8) v = zero8<T>();
      const uint32_t code = scale_code(amax_bits<T>(quad_max(amax8<T>(v))));
      const uint32_t w = pack8<T>(v, scale_of(code));
      if (m < rows) {
        lds_store4(out + m * stride + c * 4, w);
        if ((c & 3) == 0) lds_store1(scales + m * (kp / BLOCK) + c / 4, code);
      }
    }
  }
  MM_DEV void first() const { issue(0); }
  MM_DEV void finish() const {
    store(0);
    for (int p = U * NTHR; p < rows * (kp / 8); p += U * NTHR) {
      stores_done();                                 // and reads: raw is free again
      issue(p);
      wait_loads<0>();
      store(p);
    }
    stores_done();
  }
};

// A block's weights' scales in LDS, and x there or in the ring.
struct LdsX {
  const char* codes;       // of this lane's row
  const uint8_t* scales;
  template <class R>
  MM_DEV void get(const R&, int, int, int, int b, u32x4& v, uint32_t& c) const {
    v = *(const u32x4*)(codes + b * 16);
    c = scales[b];
  }
};
template <int NT>
struct RingX {
  const uint8_t* scales;   // of this lane's row of the first tile, in LDS
  int tile;                // bytes from tile to tile
  template <class R>
  MM_DEV void get(const R& ring, int d, int mt, int j, int b, u32x4& v, uint32_t& c) const {
    v = ring.operand(d, NT + mt, j);
    c = scales[mt * tile + b];
  }
};

// This wave's units; those of the first DEPTH are issued by skinny_begin.
struct Span {
  int beg, end;
};
template <int NW>
MM_DEV Span skinny_span(int K) {
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int units = (K + UNIT - 1) / UNIT, upw = (units + NW - 1) / NW;
  return {min(units, wave * upw), min(units, wave * upw + upw)};
}
// Always DEPTH of them, the last one again where the wave has fewer: what is loaded before can
// then be waited for by counting.
template <int DEPTH, class R>
MM_DEV void skinny_begin(const R& ring, Span sp) {
#pragma unroll
  for (int d = 0; d < DEPTH; ++d) ring.issue(max(0, min(sp.beg + d, sp.end - 1)), d);
  __builtin_amdgcn_sched_barrier(0);
}
// ws: the scales in LDS of this lane's row of the first weight tile, woff(nt) bytes before tile
// nt's.  acc[mt][nt][i] is D[16 nt + 4 (lane / 16) + i, 16 mt + lane % 16].
template <int MT, int NT, int DEPTH, class R, class X, class WOff>
MM_DEV void skinny(const R& ring, const X& x, const uint8_t* ws, WOff&& woff, int kb, Span sp,
                   f32x4 (&acc)[MT][NT]) {
  const int q = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) acc[mt][nt] = f32x4{0, 0, 0, 0};
  for (int u0 = sp.beg; u0 < sp.end; u0 += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d) {
      const int u = u0 + d;
      if (u >= sp.end) break;
      if (u + DEPTH <= sp.end) wait_loads<R::LOADS * (DEPTH - 1)>();
      else wait_loads<0>();
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int b = 8 * u + 4 * j + q, bw = min(b, kb - 1);
        u32x4 wv[NT];
        uint32_t wc[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          wv[nt] = ring.operand(d, nt, j);
          wc[nt] = ws[woff(nt) + bw];
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          u32x4 xv;
          uint32_t xc;
          x.get(ring, d, mt, j, b, xv, xc);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            acc[mt][nt] = mfma16<0, 0>(wv[nt], wc[nt], xv, xc, acc[mt][nt]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      if (u + DEPTH < sp.end) {
        stores_done();                               // reads of what is overwritten, that is
        ring.issue(u + DEPTH, d);
      }
    }
  }
}

// Sums of the waves: every wave parks its tiles, then fn(nn, mm, sum) gets D[nn, mm] of the
// 16 NT x rows block, each from one thread, summed in wave order.
template <int MT, int NT, int NW>
MM_DEV void skinny_park(const f32x4 (&acc)[MT][NT], float* red) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  f32x4* mine = (f32x4*)red + (size_t)wave * MT * NT * 64 + lane;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) mine[(mt * NT + nt) * 64] = acc[mt][nt];
}
template <int MT, int NT, int NW>
MM_DEV float skinny_sum(const float* red, int nn, int mm) {
  const int at = (((mm / 16) * NT + nn / 16) * 64 + (nn % 16 / 4) * 16 + mm % 16) * 4 + nn % 4;
  float sum = red[at];
#pragma unroll
  for (int v = 1; v < NW; ++v) sum += red[v * MT * NT * 256 + at];
  return sum;
}
template <int MT, int NT, int NW, class F>
MM_DEV void skinny_reduce(const f32x4 (&acc)[MT][NT], float* red, int rows, F&& fn) {
  skinny_park<MT, NT, NW>(acc, red);
  __syncthreads();
  for (int o = threadIdx.x; o < 16 * NT * rows; o += NW * 64) {
    const int mm = o / (16 * NT), nn = o % (16 * NT);
    fn(nn, mm, skinny_sum<MT, NT, NW>(red, nn, mm));
  }
}

// ---------------------------------------------------------------------------
// More rows: tiles of TM x-rows by TN weight rows, bound by the matrix cores and LDS.  A stage is
// one unit of 256 k: 128 bytes and 8 scales of every row, copied global -> LDS directly into a
// ring of S stages, S - 1 of them ahead of the one that is multiplied.  Piece p of row r lies at
// p ^ (r / 2 % 8), so that the 16 rows that an operand read takes at once spread over all banks.
// Each wave owns 32 NB x 32 MB of the tile.
// Rows of x are padded to whole units with zeros; what a weight row's last stage reads behind K
// is some of its own blocks, times those zeros.
// ---------------------------------------------------------------------------
template <int WM_, int WN_, int MB_, int NB_, int S_ = 2>
struct Tile {
  static constexpr int WM = WM_, WN = WN_, MB = MB_, NB = NB_, S = S_;
  static constexpr int NTHR = WM * WN * 64, NWAVE = WM * WN;
  static constexpr int TM = WM * MB * 32, TN = WN * NB * 32, ROWS = TM + TN;
  static constexpr int STAGE = ROWS * 128;
  static constexpr int SW = (TN + 127) / 128, SX = (TM + 127) / 128;   // KiB of scales of a stage
  static constexpr int SSTAGE = (SW + SX) * 1024;
  static constexpr int LDS = S * (STAGE + SSTAGE);
  static constexpr int IT = ROWS / 8 / NWAVE;            // 1 KiB copies per wave and stage
  static_assert(ROWS % (8 * NWAVE) == 0 && NWAVE % 2 == 0, "copies per wave");
  static_assert(TN % 32 == 0 && TM % 32 == 0, "a copy's rows are all of W or all of x");
};

// Stages [u0, u1) into acc.  src: W, S, X, XS (the bases of the weights' and x's words and
// scales), K and kp (values per row of W and of x), wrow(r) and xrow(r): the row, counted from
// those bases, of row r of the tile; every one must be readable, and rows times K / 2 or kp / 2
// stay below 2^32.  Scales: Src::BY_UNIT: those of a unit lie together, 8 of each row, spitch and
// xpitch bytes from unit to unit, readable for all rows of the tile.
// Else rows of ks scales of W, a multiple of 4, and of kp / 32 of x: each of them is a line of
// memory for 8 bytes, which cost as much as the words (4096 x 14336, 128 rows, tiles of 64 x 128:
// 34.3 us, 28.5 without any scales).
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

  constexpr int PIECES = Src::BY_UNIT ? Sh::SW + Sh::SX : Sh::ROWS / 32;    // copies of scales
  constexpr int SIT = (PIECES + Sh::NWAVE - 1) / Sh::NWAVE, COPIES = Sh::IT + SIT;
  static_assert(COPIES * (Sh::S - 2) < 64, "copies in flight");
  uint32_t off[Sh::IT], soff[SIT];
#pragma unroll
  for (int i = 0; i < Sh::IT; ++i) {
    const int r0 = (i * Sh::NWAVE + wave) * 8, r = r0 + lane / 8;
    off[i] = r0 < Sh::TN ? src.wrow(r) * (uint32_t)(src.K / 2)
                         : src.xrow(r - Sh::TN) * (uint32_t)(src.kp / 2);
  }
#pragma unroll
  for (int i = 0; i < SIT; ++i) {          // waves to spare copy the last piece again
    const int c = min(i * Sh::NWAVE + wave, PIECES - 1);
    if constexpr (Src::BY_UNIT) {
      soff[i] = c < Sh::SW ? min(c * 1024 + lane * 16, Sh::TN * 8 - 16)
                           : min((c - Sh::SW) * 1024 + lane * 16, Sh::TM * 8 - 16);
    } else {
      const int r = c * 32 + lane / 2;
      soff[i] = c * 32 < Sh::TN ? src.wrow(r) * (uint32_t)src.ks
                                : src.xrow(r - Sh::TN) * (uint32_t)(src.kp / BLOCK);
    }
  }
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
    char* const to = smem + Sh::S * Sh::STAGE + st * Sh::SSTAGE;
#pragma unroll
    for (int i = 0; i < SIT; ++i) {
      const int c = min(i * Sh::NWAVE + wave, PIECES - 1);
      if constexpr (Src::BY_UNIT) {
        copy16((c < Sh::SW ? src.S + (size_t)u * src.spitch : src.XS + (size_t)u * src.xpitch) + soff[i],
               to + c * 1024);
      } else {
        const bool isw = c * 32 < Sh::TN;
        const int left = (isw ? src.ks : src.kp / BLOCK) - 4 - u * 8;
        copy4((isw ? src.S : src.XS) + u * 8 + (soff[i] + (uint32_t)min(4 * (lane & 1), left)),
              to + (isw ? c * 256 : Sh::SW * 1024 + (c - Sh::TN / 32) * 256));
      }
    }
  };
  // Deep rings are for few blocks: one on a CU, with registers to spare.  A stage's operands are
  // read whole while the stage before is multiplied, so that a wave waits for LDS and for the others
  // only where the copies are late.
  if constexpr (Sh::S > 2) {
    u32x4 a[2][4][Sh::NB], b[2][4][Sh::MB];
    u32x2 sw[2][Sh::NB], sx[2][Sh::MB];
    auto read = [&](int st, auto to_) {
      constexpr int to = decltype(to_)::value;
      const char* const s = smem + Sh::S * Sh::STAGE + st * Sh::SSTAGE;
      const char* const d = smem + st * Sh::STAGE;
#pragma unroll
      for (int n = 0; n < Sh::NB; ++n)
        sw[to][n] = *(const u32x2*)(s + ((wn * Sh::NB + n) * 32 + l32) * 8);
#pragma unroll
      for (int m = 0; m < Sh::MB; ++m)
        sx[to][m] = *(const u32x2*)(s + Sh::SW * 1024 + ((wm * Sh::MB + m) * 32 + l32) * 8);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int p = 16 * ((2 * j + h) ^ ((l32 >> 1) & 7));
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n)
          a[to][j][n] = *(const u32x4*)(d + ((wn * Sh::NB + n) * 32 + l32) * 128 + p);
#pragma unroll
        for (int m = 0; m < Sh::MB; ++m)
          b[to][j][m] = *(const u32x4*)(d + (Sh::TN + (wm * Sh::MB + m) * 32 + l32) * 128 + p);
      }
    };
    auto multiply = [&](auto of_) {
      constexpr int of = decltype(of_)::value;
      u32x2 w[Sh::NB], x[Sh::MB];
#pragma unroll
      for (int n = 0; n < Sh::NB; ++n) w[n] = sw[of][n] >> (uint32_t)(8 * h);
#pragma unroll
      for (int m = 0; m < Sh::MB; ++m) x[m] = sx[of][m] >> (uint32_t)(8 * h);
      repeat<4>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
#pragma unroll
        for (int n = 0; n < Sh::NB; ++n)
#pragma unroll
          for (int m = 0; m < Sh::MB; ++m)
            acc[n][m] = mfma32<j % 2 * 2, j % 2 * 2>(a[of][j][n], w[n][j / 2], b[of][j][m],
                                                     x[m][j / 2], acc[n][m]);
      });
      in_order();
    };
#pragma unroll
    for (int d = 0; d < Sh::S; ++d) issue(min(u0 + d, u1 - 1), d);
    wait_loads<COPIES * (Sh::S - 1)>();
    block_barrier();
    read(0, std::integral_constant<int, 0>{});
    int st = 0, u = u0;
    // One stage: what it reads of the next is not waited for before the next one's turn.
    auto step = [&](auto of_) {
      constexpr int of = decltype(of_)::value;
      stores_done();                        // this stage's operands are in registers
      wait_loads<COPIES * (Sh::S - 2)>();
      block_barrier();
      issue(min(u + Sh::S, u1 - 1), st);
      st = st + 1 == Sh::S ? 0 : st + 1;
      read(st, std::integral_constant<int, 1 - of>{});
      in_order();
      multiply(of_);
      ++u;
    };
#pragma unroll 1
    for (; u + 2 < u1;) {
      step(std::integral_constant<int, 0>{});
      step(std::integral_constant<int, 1>{});
    }
    if (u + 1 < u1) {
      step(std::integral_constant<int, 0>{});
      multiply(std::integral_constant<int, 1>{});
    } else {
      multiply(std::integral_constant<int, 0>{});
    }
    wait_loads<0>();
    return;
  }
  // Operands of quarter j (64 k) of a stage, and the lane's scales of a whole stage (half h's in
  // every second byte from byte 0 on).
  u32x4 a[2][Sh::NB], b[2][Sh::MB];
  u32x2 sw[Sh::NB], sx[Sh::MB];
  auto read = [&](int st, int j, int to) {
    const char* const d = smem + st * Sh::STAGE;
    const int p = 16 * ((2 * j + h) ^ ((l32 >> 1) & 7));
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n)
      a[to][n] = *(const u32x4*)(d + ((wn * Sh::NB + n) * 32 + l32) * 128 + p);
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
      b[to][m] = *(const u32x4*)(d + (Sh::TN + (wm * Sh::MB + m) * 32 + l32) * 128 + p);
  };
  auto read_sc = [&](int st) {
    const char* const s = smem + Sh::S * Sh::STAGE + st * Sh::SSTAGE;
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n)
      sw[n] = *(const u32x2*)(s + ((wn * Sh::NB + n) * 32 + l32) * 8) >> (uint32_t)(8 * h);
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m)
      sx[m] = *(const u32x2*)(s + Sh::SW * 1024 + ((wm * Sh::MB + m) * 32 + l32) * 8) >> (uint32_t)(8 * h);
  };
  // Quarter j; `between` runs after its first products: what it reads is not waited for by them.
  auto multiply = [&](auto jc, const u32x2 (&w)[Sh::NB], const u32x2 (&x)[Sh::MB], auto&& between) {
    constexpr int j = decltype(jc)::value;
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n) {
#pragma unroll
      for (int m = 0; m < Sh::MB; ++m)
        acc[n][m] = mfma32<j % 2 * 2, j % 2 * 2>(a[j & 1][n], w[n][j / 2], b[j & 1][m], x[m][j / 2],
                                                 acc[n][m]);
      if (n == 0) {
        in_order();
        between();
        in_order();
      }
    }
    in_order();
  };
  // Quarters 0 to 2 of a stage, each while the next one's operands are read.
  auto quarters = [&](int st) {
    repeat<3>([&](auto jc) {
      constexpr int j = decltype(jc)::value;
      multiply(jc, sw, sx, [&] { read(st, j + 1, (j + 1) & 1); });
    });
  };
  // Past the last stage that one again, and nobody reads it: the copies in flight can be counted,
  // and no branch lets the compiler move the multiplications of a stage behind it.
#pragma unroll
  for (int d = 0; d < Sh::S; ++d) issue(min(u0 + d, u1 - 1), d);
  wait_loads<COPIES * (Sh::S - 1)>();
  block_barrier();
  read_sc(0);
  read(0, 0, 0);
  int st = 0;
#pragma unroll 1
  for (int u = u0; u + 1 < u1; ++u) {
    quarters(st);
    // Once every wave has the last operands of this stage in registers, its memory goes to the
    // stage S further on; the last quarter is multiplied while the next stage's first is read.
    wait_loads<COPIES * (Sh::S - 2)>();
    block_barrier();
    issue(min(u + Sh::S, u1 - 1), st);
    u32x2 w[Sh::NB], x[Sh::MB];
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n) w[n] = sw[n];
#pragma unroll
    for (int m = 0; m < Sh::MB; ++m) x[m] = sx[m];
    st = st + 1 == Sh::S ? 0 : st + 1;
    multiply(std::integral_constant<int, 3>{}, w, x, [&] {
      read_sc(st);
      read(st, 0, 0);
    });
  }
  quarters(st);
  multiply(std::integral_constant<int, 3>{}, sw, sx, [] {});
  wait_loads<0>();
}

// The tile's results to C, row m of which begins at row_at(m) (row m of the tile, an index into C),
// columns n0 .. N: through LDS, 32 rows of a wave at a time, so that stores are whole lines (a
// lane holds 4 results of a row, and stores of those took a sixth of the time of a large
// product: 2048 x 14336 x 4096 93 us, 77 without them).  Every wave of the block has to be done
// with the tile's memory.  rows: rows of the tile that are there.
template <class Sh, class RowAt>
MM_DEV void tile_out(const f32x16 (&acc)[Sh::NB][Sh::MB], char* smem, void* C, int type, int rows,
                     int n0, int N, RowAt&& row_at) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / Sh::WN, wn = wave % Sh::WN, l32 = lane & 31, h = lane >> 5;
  constexpr int COLS = Sh::NB * 32;
  const int size = type == F32 ? 4 : 2, pitch = COLS * size + 16;
  static_assert(Sh::NWAVE * 32 * (COLS * 4 + 16) <= Sh::LDS, "the waves' rows take the tile's place");
  char* const mine = smem + wave * 32 * (COLS * 4 + 16);
  const int c0 = n0 + wn * COLS, cols = min(COLS, N - c0);
  if (cols <= 0) return;
  const bool whole = N * size % 16 == 0;      // pieces of 16 bytes lie whole and aligned
#pragma unroll
  for (int m = 0; m < Sh::MB; ++m) {
    const int m0 = (wm * Sh::MB + m) * 32;
    if (m0 >= rows) break;
    stores_done();                            // and the reads of the rows before
#pragma unroll
    for (int n = 0; n < Sh::NB; ++n)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 v = {acc[n][m][4 * g], acc[n][m][4 * g + 1], acc[n][m][4 * g + 2],
                         acc[n][m][4 * g + 3]};
        store4(mine + l32 * pitch, type, n * 32 + 8 * g + 4 * h, v);
      }
    stores_done();
    const int rn = min(32, rows - m0);
    if (whole) {
      const int per = cols * size / 16;       // pieces per row
      for (int p = lane; p < 32 * (COLS * size / 16); p += 64) {
        const int r = p / (COLS * size / 16), c = p % (COLS * size / 16);
        if (r < rn && c < per)
          *(u32x4*)((char*)C + (row_at(m0 + r) + c0) * size + 16 * c) =
              *(const u32x4*)(mine + r * pitch + 16 * c);
      }
    } else {
      for (int p = lane; p < 32 * COLS; p += 64) {
        const int r = p / COLS, c = p % COLS;
        if (r >= rn || c >= cols) continue;
        const size_t at = row_at(m0 + r) + c0 + c;
        if (type == F32) ((float*)C)[at] = *(const float*)(mine + r * pitch + 4 * c);
        else ((uint16_t*)C)[at] = *(const uint16_t*)(mine + r * pitch + 2 * c);
      }
    }
  }
}

}  // namespace mmmx
