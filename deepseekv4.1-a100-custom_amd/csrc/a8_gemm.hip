// Products of 8-bit activations with block-scaled FP8 weights, and the gated product of a feed-forward:
//   linear: y[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]) + residual[m, n]
//   gated:  y[m, n] = act(min(g, limit)) clamp(u, -limit, limit),  g = sum_k x wg, u = sum_k x wu
// x and y: A8 (a8_core.h), y also bf16; w: e4m3 codes [N, K] and E8M0 scales per [32 x 32] block (dsv41/w8.py:39-60).
// Both operands keep their bytes: the block-scaled matrix instructions take the codes and the scales of 32 k of a row as
// they are.  A lane's 32 codes of such an instruction (R = 16 or 32 rows, KI = 128 or 64 k, lane group g = lane / R) are
// k 16 g .. 16 g + 15 and KI / 2 + 16 g .. KI / 2 + 16 g + 15, and the scale it gives is that of k 32 g .. 32 g + 31.
// The instruction adds its products with about 2^-16 of relative error (measured 1.5e-5 in the 2-norm at every K, random
// in sign), well below half a step of bf16 (2^-9 of a value) or of e4m3; outputs are therefore bf16 or A8, not fp32.
// Sums over k are fp32, in a fixed order.
//
// The weights are the instruction's row operand: a lane ends with 4 adjacent columns of a row of y.
#include <type_traits>

#include "a8_core.h"

namespace {

struct A8Args {
  const uint8_t *x, *xs;      // codes [M, K], scales [ceil(K / 128)][M][4]
  const uint8_t *w, *ws;      // codes [N, K], scales [ceil(N / 32), Kc]
  const uint8_t *w2, *ws2;    // the up weights of a gated product
  int M, N, K, Kc, Kc2;
  A8Epi e;
  int mtiles, ntiles;
  int words;                  // weight scales in whole words: K % 128 == 0, rows 4-byte aligned
  int splits, kslice;         // K slices of kslice steps of 128 k; more than one: partials
  float* part;                // [splits][M][ldp], ldp = ceil(N / 32) * 32 (gated: twice, up behind gate)
  long ldp;
};

DSV41_DEV i32x8_t a8_operand(uint4 lo, uint4 hi) {
  return i32x8_t{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}
// (scales in the lowest byte)
DSV41_DEV f32x4_t a8_mfma16(i32x8_t a, i32x8_t b, f32x4_t c, int sa, int sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, sa, 0, sb);
}

// ------------------------------------------------------------------------------------------------ few rows
// Up to 16 MT rows: a stream of the weights.  A workgroup has 16 CT output columns, its waves take the steps of 128 k in
// turn (wave v: steps v, v + waves, ...), so that together they read whole rows in order; sums meet in LDS.  The weights
// go from memory into the instruction's registers, a step ahead; x comes from the L2, in the same lanes.
template <int MT, int CT, bool GATED>
__global__ void __launch_bounds__(512) a8_stream_kernel(const A8Args a) {
  extern __shared__ __align__(16) float red[];  // [waves][WT * MT][64 lanes][4]
  constexpr int WT = GATED ? 2 * CT : CT;       // weight tiles of 16 rows: gate tiles, then up tiles
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, nw = blockDim.x >> 6;
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * CT;
  const int steps = (a.K + 127) / 128, last = a.K / 32 - 1;
  const uint8_t *wp[WT], *sp[WT], *xp[MT], *xsp[MT];
#pragma unroll
  for (int t = 0; t < WT; ++t) {
    const int n = min(n0 + 16 * (t % CT) + l16, a.N - 1);  // (columns past N repeat the last and are not stored)
    const bool up = GATED && t >= CT;
    wp[t] = (up ? a.w2 : a.w) + (long)n * a.K;
    sp[t] = up ? a.ws2 + (long)(n >> 5) * a.Kc2 : a.ws + (long)(n >> 5) * a.Kc;
  }
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    const int m = min(16 * t + l16, a.M - 1);
    xp[t] = a.x + (long)m * a.K;
    xsp[t] = a.xs + 4l * m + g;
  }
  struct Step {
    uint4 w[WT][2], x[MT][2];
    int ws[WT], xs[MT];
  };
  auto load = [&](int s, Step& o) {
    const int k = min(s, steps - 1) * 128;
    const int p = k + 16 * g < a.K ? k + 16 * g : k, q = k + 64 + 16 * g < a.K ? k + 64 + 16 * g : k;
    const int b = min(k / 32 + g, last);
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      o.w[t][0] = *(const uint4*)(wp[t] + p);
      o.w[t][1] = *(const uint4*)(wp[t] + q);
      o.ws[t] = sp[t][b];
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      o.x[t][0] = *(const uint4*)(xp[t] + p);
      o.x[t][1] = *(const uint4*)(xp[t] + q);
      o.xs[t] = xsp[t][(long)(k / 128) * a.M * 4];
    }
  };
  f32x4_t acc[WT][MT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  auto mul = [&](int s, Step& o) {
    if (s * 128 + 128 > a.K) {  // K ends inside this step: codes past it are zero on both sides
      const bool p = s * 128 + 16 * g < a.K, q = s * 128 + 64 + 16 * g < a.K;
      const uint4 z = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int t = 0; t < WT; ++t) {
        if (!p) o.w[t][0] = z;
        if (!q) o.w[t][1] = z;
        if (s * 4 + g > last) o.ws[t] = 127;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (!p) o.x[t][0] = z;
        if (!q) o.x[t][1] = z;
      }
    }
#pragma unroll
    for (int j = 0; j < MT; ++j)
#pragma unroll
      for (int i = 0; i < WT; ++i)
        acc[i][j] = a8_mfma16(a8_operand(o.w[i][0], o.w[i][1]), a8_operand(o.x[j][0], o.x[j][1]), acc[i][j], o.ws[i],
                              o.xs[j]);
  };
  Step s0, s1;
  load(wave, s0);
#pragma unroll 1
  for (int s = wave; s < steps; s += 2 * nw) {
    load(s + nw, s1);
    mul(s, s0);
    if (s + nw < steps) {
      load(s + 2 * nw, s0);
      mul(s + nw, s1);
    }
  }
  // lane (l16, g): row l16 of x, columns 4 g .. 4 g + 3 of the tile
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *(f32x4_t*)(red + (((long)wave * WT + i) * MT + j) * 256 + lane * 4) = acc[i][j];
  __syncthreads();
  constexpr int QN = 2 * CT;  // lanes of a row: 8 columns each
  for (int t = tid; t < QN * 16 * MT; t += blockDim.x) {  // (in whole quads of lanes: a block of 32 columns with CT 2)
    const int c = t % QN, m = t / QN, n = n0 + 8 * c;
    const float* p = red + ((c >> 1) * MT + (m >> 4)) * 256 + ((c & 1) * 32 + (m & 15)) * 4;  // the next 4: lanes on 16
    const bool live = m < a.M && n < a.N;
    const uint4 res = a8_res8(a.e, m, n);
    const A8x8 bias = a8_bias8(a.e, n);
    A8x8 y, u;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = u.v[i] = 0.0f;
    for (int w = 0; w < nw; ++w) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        y.v[i] += p[w * (WT * MT * 256) + (i >> 2) * 64 + (i & 3)];
        if constexpr (GATED) u.v[i] += p[(w * WT + CT) * MT * 256 + (i >> 2) * 64 + (i & 3)];
      }
    }
    if constexpr (GATED) a8_gated8(a.e, y, u);
    else a8_linear8(a.e, y, bias, res);
    a8_store8(a.e, y, m, n, live);
  }
}

// ------------------------------------------------------------------------------------------------ tiles
// Direct-to-LDS load of 16 (4) bytes a lane from base + off to lds_addr + 16 (4) i; callers wait with vmcnt counts.
DSV41_DEV void a8_dma16(const void* base, uint32_t off, uint32_t lds_addr) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds_addr);
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(m) : "memory", "m0");
}
DSV41_DEV void a8_dma4(const void* base, uint32_t off, uint32_t lds_addr) {
  const uint32_t m = __builtin_amdgcn_readfirstlane(lds_addr);
  asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "s"(m) : "memory", "m0");
}

constexpr int kA8Strip = 4;
constexpr int kA8SliceSteps = 128;  // a K slice's steps of 128 k at most: its weight scales are held in LDS

// Output of a wave's ROWS x OCW block of sums from LDS (fp32, row stride LD bytes): rolled, so that bias, activation and
// quantisation stand there once (unrolled over the accumulators they were 100 KB of code); the residual of U passes is
// loaded before any of them is stored.
template <int ROWS, int LD, int OCW, bool GATED>
DSV41_DEV void a8_wave_out(const A8Args& a, const uint8_t* s, int m0, int n0) {
  constexpr int QN = OCW / 8, RP = 64 / QN, PASSES = ROWS / RP, U = PASSES < 8 ? PASSES : 8;  // lanes of a row, rows of a pass
  static_assert(ROWS % RP == 0 && PASSES % U == 0, "whole passes");
  const int lane = threadIdx.x & 63, c = lane % QN * 8, n = n0 + c;
  s += (lane / QN) * LD + (GATED ? (c / 32 * 64 + c % 32) * 4 : c * 4);
  const A8x8 bias = a8_bias8(a.e, n);
#pragma unroll 1
  for (int r0 = 0; r0 < ROWS; r0 += U * RP) {
    uint4 res[U];
    if constexpr (!GATED) {
#pragma unroll
      for (int k = 0; k < U; ++k) res[k] = a8_res8(a.e, m0 + r0 + k * RP + lane / QN, n);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int m = m0 + r0 + k * RP + lane / QN;
      const uint8_t* p = s + (r0 + k * RP) * LD;
      A8x8 y = *(const A8x8*)p, u = y;
      if constexpr (GATED) u = *(const A8x8*)(p + 128);
      if (a.splits > 1) {
        float* o = a.part + ((long)blockIdx.y * a.M + m) * a.ldp + n;
        if (m < a.M && n < (a.N + 31) / 32 * 32) {
          *(A8x8*)o = y;
          if constexpr (GATED) *(A8x8*)(o + a.ldp / 2) = u;
        }
      } else {
        if constexpr (GATED) a8_gated8(a.e, y, u);
        else a8_linear8(a.e, y, bias, res[k]);
        a8_store8(a.e, y, m, n, m < a.M && n < a.N);
      }
    }
  }
}

// BM rows of x by BN rows of weights in WM x WN waves of (BM / WM) x (BN / WN); stages of 128 k through NBUF LDS buffers.
// A gated tile has BN / 2 output columns: of a wave's 32-row weight blocks the even ones are gate rows, the odd ones the
// up rows of the same columns.
template <int BM, int BN, int WM, int WN, int NBUF, bool GATED>
__global__ void __launch_bounds__(64 * WM * WN) a8_tile_kernel(const A8Args a) {
  constexpr int NT = 64 * WM * WN;
  constexpr int MT = BM / WM / 16, CT = BN / WN / 16;  // 16-row blocks of a wave
  constexpr int XB = BM * 128, WB = BN * 128, SB = (BM < 64 ? 64 : BM) * 4, STAGE = XB + WB + SB;
  constexpr int XL = XB / 16 / NT, WL = WB / 16 / NT, LPT = XL + WL + 1;  // loads per thread and stage
  constexpr int OC = GATED ? BN / 2 : BN;                                 // output columns
  // A stage is MT steps: x block t with the CT weight blocks.  x of a step is read AHEAD steps before, across the stage's
  // end too: the barrier stands in step ENTER, where the first of the next stage is read.  A weight block is read for the
  // next stage behind its last product.
    constexpr int RING = MT >= 4 ? 4 : 2, AHEAD = RING / 2, ENTER = MT - AHEAD;
  // A stage's loads are issued between the products from that barrier on, in the first POS of the MT CT places; FIRST of
  // them fall into the stage in which they begin.
  constexpr int POS = MT * CT * 3 / 4;
  constexpr auto upto = [](int z) constexpr { return z >= POS ? LPT : z * LPT / POS; };
  constexpr int FIRST = upto(AHEAD * CT);
  static_assert(XL * NT * 16 == XB && WL * NT * 16 == WB && MT * WM * 16 == BM && CT * WN * 16 == BN, "tile shape");
  static_assert(!GATED || CT % 4 == 0, "gate and up blocks in pairs");
  static_assert(MT % RING == 0, "ring");
  static_assert((NBUF - 2) * LPT + FIRST < 64, "vmcnt immediate");
  __shared__ __align__(16) uint8_t buf[NBUF * STAGE];
  __shared__ __align__(16) uint8_t scl[BN / 32][kA8SliceSteps * 4 + 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int wm = wave / WN, wn = wave - wm * WN;
  // contiguous tile ranges per XCD, in strips of kA8Strip row tiles: the tiles that run on an XCD together share rows and
  // weights in its L2
  const int per = gridDim.x / kXcds;
  const int id = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
  if (id >= a.mtiles * a.ntiles) return;
  const int strip = id / (kA8Strip * a.ntiles), sm = min(kA8Strip, a.mtiles - strip * kA8Strip);
  const int in = id - strip * kA8Strip * a.ntiles;
  const int m0 = (strip * kA8Strip + in % sm) * BM, n0 = in / sm * OC;
  const int s0 = blockIdx.y * a.kslice;
  const int nk = min(a.K / 128 - s0, a.kslice);  // whole stages of the slice
  const int tail = a.K / 128 < s0 + a.kslice ? a.K % 128 : 0;  // k behind them, in the slice of that step

  // weight row r of the tile: output column (from n0) and matrix
  auto column = [&](int r) { return GATED ? (r / 64) * 32 + (r & 31) : r; };
  auto is_up = [&](int r) { return GATED && (r & 32) != 0; };
  const uint8_t* xb = a.x + (long)m0 * a.K + s0 * 128l;
  const uint8_t* wb = a.w + (long)n0 * a.K + s0 * 128l;
  const uint8_t* wb2 = GATED ? a.w2 + (long)n0 * a.K + s0 * 128l : nullptr;
  const uint8_t* xsb = a.xs + ((long)s0 * a.M + m0) * 4;
  // Load u of a thread brings 16 bytes of row u NT / 8 + tid / 8 (rows past the end repeat the last and are not stored).
  // Chunk c of a 128-byte row r sits at c ^ (r & 7): the 8 lanes of an LDS read cycle (8 rows, one chunk) then hit 8
  // different 16-byte bank groups.
  const int r0 = tid >> 3, ch = ((tid & 7) ^ (r0 & 7)) * 16;
  const int xlim = a.M - 1 - m0, wlim = a.N - 1 - n0;
  const int sr = min((wave % (SB / 256)) * 64 + lane, BM - 1);
  const uint32_t so = (uint32_t)min(sr, xlim) * 4;
  const uint32_t lds0 = lds_addr_of(buf);
  const uint32_t ldsw = lds0 + (uint32_t)wave * 1024, ldss = lds0 + XB + WB + (uint32_t)(wave % (SB / 256)) * 256;
  const int klast = a.K - s0 * 128 - 16;  // the last 16 codes of a row, from the slice's start
  uint32_t xo[XL], wo[WL];
#pragma unroll
  for (int u = 0; u < XL; ++u) xo[u] = (uint32_t)min(u * (NT / 8) + r0, xlim) * (uint32_t)a.K;
#pragma unroll
  for (int u = 0; u < WL; ++u) wo[u] = (uint32_t)min(column(u * (NT / 8) + r0), wlim) * (uint32_t)a.K;
  // Load q of stage kt (past the last: the last again, into a buffer that is read no more, so that counts stay the same)
  auto dma = [&](int kt, int b, int q) {
    const uint32_t l = (uint32_t)(b * STAGE);
    const uint32_t k = (uint32_t)min(kt * 128 + ch, klast);  // (chunks past K load the last one and are zeroed below)
    if (q < XL) {
      a8_dma16(xb, xo[q] + k, ldsw + l + q * NT * 16);
    } else if (q < XL + WL) {  // (a wave's 8 rows are of one matrix)
      const int u = q - XL;
      a8_dma16(is_up(u * (NT / 8) + wave * 8) ? wb2 : wb, wo[u] + k, ldsw + l + XB + u * NT * 16);
    } else {
      a8_dma4(xsb + (long)kt * a.M * 4, so, ldss + l);
    }
  };
  {  // the slice's weight scales
    const int nb = (a.N + 31) / 32, kb = (nk * 128 + tail) / 32;
    auto scales = [&](int b) {
      const int row = min((n0 + column(b * 32)) / 32, nb - 1);
      return (is_up(b * 32) ? a.ws2 + (long)row * a.Kc2 : a.ws + (long)row * a.Kc) + s0 * 4;
    };
    if (a.words) {  // whole words: by direct loads, ahead of the stages'
      for (int b = wave; b < BN / 32; b += WM * WN)
        for (int c = 0; c < nk; c += 64)
          a8_dma4(scales(b), (uint32_t)min(c + lane, nk - 1) * 4, lds_addr_of(&scl[b][0]) + c * 4);
    } else {  // by bytes, 127 behind the last
      for (int b = wave; b < BN / 32; b += WM * WN) {
        const uint8_t* p = scales(b);
        for (int k = lane; k < (nk + 1) * 4; k += 64) scl[b][k] = k < kb ? p[k] : 127;
      }
    }
  }
#pragma unroll
  for (int p = 0; p < NBUF; ++p)
#pragma unroll
    for (int q = 0; q < (p < NBUF - 1 ? LPT : FIRST); ++q) dma(max(min(p, nk - 1), 0), p, q);

  f32x4_t acc[MT][CT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int xr = wm * (BM / WM) + l16, wr = wn * (BN / WN) + l16;  // (16-row steps keep the swizzle's row bits)
  const int c0 = (g ^ (l16 & 7)) * 16, c1 = c0 ^ 64;                // chunks g and 4 + g
  auto operand = [&](const uint8_t* p) { return a8_operand(*(const uint4*)(p + c0), *(const uint4*)(p + c1)); };
  // The next stage has landed for every wave (`later` younger loads may not have), and every wave has read this one.
  auto enter = [&](auto later) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(decltype(later)::value));
    lds_barrier();
  };
  i32x8_t xf[RING], wf[CT];
  int xs[RING], ws[CT];  // (bytes: a shift of a word would wait for it where it is read)
  auto fetch_w = [&](int j, int kt, int b) {
    wf[j] = operand(buf + b * STAGE + XB + (wr + 16 * j) * 128);
    ws[j] = scl[wn * (CT / 2) + j / 2][kt * 4 + g];  // (kt may be one past the slice: the row is longer)
  };
  auto fetch_x = [&](int t, int b) {
    const uint8_t* st = buf + b * STAGE;
    xf[t % RING] = operand(st + (xr + 16 * t) * 128);
    xs[t % RING] = st[XB + WB + (xr + 16 * t) * 4 + g];
  };
  if (nk > 0) {
    int bi = 0;
    enter(std::integral_constant<int, (NBUF - 2) * LPT + FIRST>{});
#pragma unroll
    for (int j = 0; j < CT; ++j) fetch_w(j, 0, 0);
#pragma unroll
    for (int t = 0; t < AHEAD; ++t) fetch_x(t, 0);
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {  // (what the last stage reads and loads ahead is the last again, and not used)
      const int b0 = bi;
      bi = bi + 1 == NBUF ? 0 : bi + 1;
      const int bp = b0 == 0 ? NBUF - 1 : b0 - 1;
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t < ENTER) {
          fetch_x(t + AHEAD, b0);
        } else {
          if (t == ENTER) enter(std::integral_constant<int, (NBUF - 2) * LPT>{});
          fetch_x(t - ENTER, bi);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          acc[t][j] = a8_mfma16(wf[j], xf[t % RING], acc[t][j], ws[j], xs[t % RING]);
          if (t == MT - 1) fetch_w(j, kt + 1, bi);
          const int z = (t < ENTER ? t + AHEAD : t - ENTER) * CT + j;
#pragma unroll
          for (int q = upto(z); q < upto(z + 1); ++q) dma(min(t < ENTER ? kt + NBUF - 1 : kt + NBUF, nk - 1), t < ENTER ? bp : b0, q);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  lds_barrier();  // every wave has read its last stage, and no load is on its way
  if (tail) {     // K ends inside a stage of its own: zeros behind it
#pragma unroll
    for (int q = 0; q < LPT; ++q) dma(nk, 0, q);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
    lds_barrier();
    for (int e = tid; e < (BM + BN) * 8; e += NT)
      if ((e & 7) * 16 >= tail) *(uint4*)(buf + (e >> 3) * 128 + (((e & 7) ^ ((e >> 3) & 7)) * 16)) = make_uint4(0, 0, 0, 0);
    lds_barrier();
#pragma unroll
    for (int j = 0; j < CT; ++j) fetch_w(j, nk, 0);
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      fetch_x(t, 0);
#pragma unroll
      for (int j = 0; j < CT; ++j) acc[t][j] = a8_mfma16(wf[j], xf[t % RING], acc[t][j], ws[j], xs[t % RING]);
    }
    lds_barrier();
  }

  // A lane (l16, g) has row l16, columns 4 g .. 4 g + 3 of a block: PM blocks of rows at a time through the wave's part of
  // the LDS (rows padded by 16 bytes: 8 lanes write 8 different bank groups)
  constexpr int LD = BN / WN * 4 + 16;
  constexpr int PM = MT * 16 * LD * WM * WN <= NBUF * STAGE ? MT : MT * 8 * LD * WM * WN <= NBUF * STAGE ? MT / 2 : MT / 4;
  static_assert(PM * 16 * LD * WM * WN <= NBUF * STAGE && MT % PM == 0 && PM % 2 == 0, "output staging");
  uint8_t* own = buf + wave * (PM * 16 * LD);
#pragma unroll
  for (int p = 0; p < MT; p += PM) {
#pragma unroll
    for (int i = 0; i < PM; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j) *(f32x4_t*)(own + (16 * i + l16) * LD + (16 * j + 4 * g) * 4) = acc[p + i][j];
    a8_wave_out<PM * 16, LD, OC / WN, GATED>(a, own, m0 + wm * (BM / WM) + 16 * p, n0 + wn * (OC / WN));
  }
}

// The K slices' partials summed in slice order and finished: 8 columns a thread, 4 adjacent lanes a block of 32.
template <bool GATED>
__global__ void __launch_bounds__(256) a8_sum_kernel(const A8Args a) {
  const int q = (a.N + 31) / 32 * 4;  // threads of a row
  const long t = (long)blockIdx.x * 256 + threadIdx.x;
  const long m = t / q;
  const int n = (int)(t - m * q) * 8;
  const bool live = m < a.M && n < a.N;
  A8x8 y, u;
#pragma unroll
  for (int i = 0; i < 8; ++i) y.v[i] = u.v[i] = 0.0f;
  if (live) {
    const uint4 res = a8_res8(a.e, (int)m, n);
    const A8x8 bias = a8_bias8(a.e, n);
    const float* p = a.part + m * a.ldp + n;
#pragma unroll 4
    for (int s = 0; s < a.splits; ++s) {
      const A8x8 v = *(const A8x8*)(p + (long)s * a.M * a.ldp);
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] += v.v[i];
      if constexpr (GATED) {
        const A8x8 w = *(const A8x8*)(p + (long)s * a.M * a.ldp + a.ldp / 2);
#pragma unroll
        for (int i = 0; i < 8; ++i) u.v[i] += w.v[i];
      }
    }
    if constexpr (GATED) a8_gated8(a.e, y, u);
    else a8_linear8(a.e, y, bias, res);
  }
  a8_store8(a.e, y, (int)m, n, live);
}

// ------------------------------------------------------------------------------------------------ plan
constexpr int kCus = 256;
struct A8Plan {
  int rows;  // 0: the stream
  int cols;  // weight rows of a tile (stream: output columns of a workgroup)
  int splits, kslice, waves;
};

A8Plan a8_plan(int M, int N, int K, bool gated) {
  const int steps = (K + 127) / 128;
  A8Plan p{0, 32, 1, steps, 8};
  if (M <= 32) {
    if (!gated && M <= 16 && N % 32 != 0) p.cols = 16;
    return p;
  }
  p.rows = M <= 64 ? 64 : M <= 2048 ? 128 : 256;
  p.cols = M <= 2048 ? 128 : 256;
  const long tiles = (long)((M + p.rows - 1) / p.rows) * ((N * (gated ? 2l : 1l) + p.cols - 1) / p.cols);
  int s = (int)(2 * kCus / tiles);
  s = s < 1 ? 1 : s > steps / 2 ? (steps / 2 < 1 ? 1 : steps / 2) : s;
  const int least = (steps + kA8SliceSteps - 1) / kA8SliceSteps;
  if (s < least) s = least;
  p.kslice = (steps + s - 1) / s;
  p.splits = (steps + p.kslice - 1) / p.kslice;
  return p;
}

long a8_ldp(int N, bool gated) { return (long)(N + 31) / 32 * 32 * (gated ? 2 : 1); }

long a8_workspace(int M, int N, int K, bool gated) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const A8Plan p = a8_plan(M, N, K, gated);
  return p.rows == 0 || p.splits == 1 ? 0 : (long)p.splits * M * a8_ldp(N, gated) * 4;
}

template <bool GATED>
int a8_run(A8Args& a, void* ws, long ws_bytes, hipStream_t st) {
  if (a.M == 0 || a.N == 0) return 0;
  if (a.M < 0 || a.N < 0 || a.K <= 0 || a.K % 32 != 0 || a.Kc < a.K / 32 || (GATED && a.Kc2 < a.K / 32))
    return (int)hipErrorInvalidValue;
  if (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.w2) & 15 || (uintptr_t)a.xs & 3) return (int)hipErrorInvalidValue;
  if (a.e.act < kActNone || a.e.act > kActGeluTanh || !(a.e.limit >= 0.0f)) return (int)hipErrorInvalidValue;
  if (!a.e.out && (!a.e.oa8 || !a.e.os8 || a.N % 32 != 0 || (uintptr_t)a.e.oa8 & 15)) return (int)hipErrorInvalidValue;
  a.e.M = a.M;
  a.e.N = a.N;
  a.e.vec = a.N % 8 == 0 && (((uintptr_t)a.e.out | (uintptr_t)a.e.res) & 15) == 0;
  a.words = a.K % 128 == 0 && ((a.Kc | a.Kc2 | (uintptr_t)a.ws | (uintptr_t)a.ws2) & 3) == 0;
  const A8Plan p = a8_plan(a.M, a.N, a.K, GATED);
  a.splits = p.splits;
  a.kslice = p.kslice;
  if (p.rows == 0) {
    const dim3 g((unsigned)((a.N + p.cols - 1) / p.cols)), b((unsigned)(64 * p.waves));
    const int mt = a.M <= 16 ? 1 : 2;
    const size_t lds = (size_t)p.waves * (p.cols / 16) * (GATED ? 2 : 1) * mt * 1024;
    if (p.cols == 16) {
      if constexpr (!GATED) a8_stream_kernel<1, 1, false><<<g, b, lds, st>>>(a);
    } else if (mt == 1) {
      a8_stream_kernel<1, 2, GATED><<<g, b, lds, st>>>(a);
    } else {
      a8_stream_kernel<2, 2, GATED><<<g, b, lds, st>>>(a);
    }
    DSV41_CHECK_LAUNCH();
    return 0;
  }
  if (p.splits > 1) {
    a.ldp = a8_ldp(a.N, GATED);
    a.part = (float*)ws;
    if (!ws || ((uintptr_t)ws & 15) != 0 || ws_bytes < a8_workspace(a.M, a.N, a.K, GATED)) return (int)hipErrorInvalidValue;
  }
  const int oc = GATED ? p.cols / 2 : p.cols;
  a.mtiles = (a.M + p.rows - 1) / p.rows;
  a.ntiles = (a.N + oc - 1) / oc;
  const dim3 g((unsigned)((a.mtiles * a.ntiles + kXcds - 1) / kXcds * kXcds), (unsigned)p.splits);
  if (p.rows == 64) a8_tile_kernel<64, 128, 2, 2, 2, GATED><<<g, 256, 0, st>>>(a);
  else if (p.rows == 128) a8_tile_kernel<128, 128, 2, 2, 2, GATED><<<g, 256, 0, st>>>(a);
  else a8_tile_kernel<256, 256, 2, 4, 2, GATED><<<g, 512, 0, st>>>(a);
  DSV41_CHECK_LAUNCH();
  if (p.splits > 1) {
    const long t = (long)a.M * ((a.N + 31) / 32 * 4);
    a8_sum_kernel<GATED><<<(unsigned)((t + 255) / 256), 256, 0, st>>>(a);
    DSV41_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" {

long dsv41_a8_workspace_bytes(int M, int N, int K, int gated) { return a8_workspace(M, N, K, gated != 0); }

int dsv41_linear_a8(const void* a8, const void* s8, const void* w8, const void* ws8, int M, int N, int K, int Kc,
                    const void* bias, int bias_f32, int act, const void* residual, void* out, void* out_a8,
                    void* out_s8, void* ws, long ws_bytes, void* stream) {
  A8Args a{};
  a.x = (const uint8_t*)a8;
  a.xs = (const uint8_t*)s8;
  a.w = (const uint8_t*)w8;
  a.ws = (const uint8_t*)ws8;
  a.M = M;
  a.N = N;
  a.K = K;
  a.Kc = Kc;
  a.e.bias = bias;
  a.e.bias_f32 = bias_f32;
  a.e.act = act;
  a.e.res = (const uint16_t*)residual;
  a.e.out = (uint16_t*)out;
  a.e.oa8 = (uint8_t*)out_a8;
  a.e.os8 = (uint8_t*)out_s8;
  return a8_run<false>(a, ws, ws_bytes, (hipStream_t)stream);
}

int dsv41_gated_a8(const void* a8, const void* s8, const void* wg8, const void* wgs8, const void* wu8,
                   const void* wus8, int M, int N, int K, int Kcg, int Kcu, int act, float limit, void* out,
                   void* out_a8, void* out_s8, void* ws, long ws_bytes, void* stream) {
  A8Args a{};
  a.x = (const uint8_t*)a8;
  a.xs = (const uint8_t*)s8;
  a.w = (const uint8_t*)wg8;
  a.ws = (const uint8_t*)wgs8;
  a.w2 = (const uint8_t*)wu8;
  a.ws2 = (const uint8_t*)wus8;
  a.M = M;
  a.N = N;
  a.K = K;
  a.Kc = Kcg;
  a.Kc2 = Kcu;
  a.e.act = act;
  a.e.limit = limit;
  a.e.out = (uint16_t*)out;
  a.e.oa8 = (uint8_t*)out_a8;
  a.e.os8 = (uint8_t*)out_s8;
  if (!wu8 || !wus8) return (int)hipErrorInvalidValue;
  return a8_run<true>(a, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
