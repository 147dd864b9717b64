// Products of 8-bit activations with block-scaled FP8 weights, and the gated product of a feed-forward:
//   linear: y[m, n] = act(sum_k x[m, k] w[n, k] + bias[n]) + residual[m, n]
//   gated:  y[m, n] = act(min(g, limit)) clamp(u, -limit, limit),  g = sum_k x wg, u = sum_k x wu
// x and y: A8 (a8_core.h), y also bf16; w: e4m3 codes [N, K] and E8M0 scales per [32 x 32] block (dsv41/w8.py:39-60).
// Both operands keep their bytes up to the registers, where code times scale becomes bf16: exact (in bf16's range, past
// which a value is infinite), and so are the bf16 matrix units' products; sums over k are fp32, in a fixed order (8.8e-8 of
// relative error in the 2-norm at 5120 k, 1.2e-7 at 8192).  A lane's 32 codes of 128 k (16 rows; lane group g = lane / 16)
// are k 32 g .. 32 g + 31: one scale.
// The fp8 matrix instructions, block-scaled or not, take the bytes as they are at twice the rate, but drop what lies some
// 2^-17 below an instruction's largest product: 1.5e-5 in the 2-norm for normal values, 4.5e-5 with a few large channels,
// and where two large products cancel, all of the result.  That is not a sum in 32 bits, so they are not used (with them
// 4096 x 5120 x 8192 took 161 us a pass for 301, gated 4096 x 2 x 8192 x 5120 290 for 541; up to 130 rows 3 % less).
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
  int mtiles, ntiles, first;  // tiles: of the columns from `first` on
  int words;                  // weight scales in whole words: K % 128 == 0, rows 4-byte aligned
};

DSV41_DEV float a8_e8m0(int s) {
  return s == 255 ? __builtin_nanf("") : s ? __int_as_float(s << 23) : __int_as_float(0x00400000);
}
// 8 codes (two words) times their scale, exact in bf16.
DSV41_DEV uint4 a8_decode(uint32_t a, uint32_t b, float sc) {
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, sc, true)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, false)),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, sc, true)));
}

// ------------------------------------------------------------------------------------------------ few rows
// 16 MT rows by 16 CT output columns a workgroup: a stream of the weights.  Its NW waves take the steps of 128 k in turn
// (wave v: steps v, v + NW, ...), so that together they read whole rows in order, each through a ring of D steps in LDS
// that only it fills and reads: no barrier until the sums meet, and D steps of loads on the way in every wave.  (Loads
// into registers a step ahead were 16 us where this is 11: 24 rows of 1280 k, 32768 columns.)
constexpr int kStreamMaxK = 32768;  // (the weight scales of all of K are held in LDS)

template <int MT, int CT, int NW, int D, bool GATED>
__global__ void __launch_bounds__(64 * NW) a8_stream_kernel(const A8Args a) {
  constexpr int WT = GATED ? 2 * CT : CT;  // weight tiles of 16 rows: gate tiles, then up tiles
  constexpr int STEP = (WT + MT) * 2048 + 256, LPS = 2 * (WT + MT) + 1;
  constexpr int RING = NW * D * STEP, SUMS = NW * WT * MT * 1024;
  static_assert((D - 1) * LPS < 64, "vmcnt immediate");
  __shared__ __align__(16) uint8_t lds[RING > SUMS ? RING : SUMS];
  __shared__ __align__(16) uint8_t scl[GATED ? 2 : 1][kStreamMaxK / 32];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16 * CT, m0 = blockIdx.y * 16 * MT;
  const int steps = (a.K + 127) / 128;
  const int mine = (steps - wave + NW - 1) / NW;  // this wave's steps (none where K is short)
  // 16 bytes of row (lane / 8) of 8: chunk c of a 128-byte row r sits at c ^ (r & 7)
  const int r8 = lane >> 3, ch = ((lane & 7) ^ r8) * 16;
  uint32_t wo[WT][2], xo[MT][2];
#pragma unroll
  for (int t = 0; t < WT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u)  // (columns past N repeat the last and are not stored)
      wo[t][u] = (uint32_t)min(16 * (t % CT) + 8 * u + r8, a.N - 1 - n0) * (uint32_t)a.K;
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int u = 0; u < 2; ++u) xo[t][u] = (uint32_t)min(16 * t + 8 * u + r8, a.M - 1 - m0) * (uint32_t)a.K;
  const uint8_t* wb = a.w + (long)n0 * a.K;
  const uint8_t* wb2 = GATED ? a.w2 + (long)n0 * a.K : nullptr;
  const uint8_t* xb = a.x + (long)m0 * a.K;
  const uint8_t* xsb = a.xs + 4l * m0;
  const uint32_t so = (uint32_t)min(min(lane, 16 * MT - 1), a.M - 1 - m0) * 4;
  uint8_t* ring = lds + wave * (D * STEP);
  const uint32_t ring0 = lds_addr_of(lds) + (uint32_t)wave * (D * STEP);
  auto issue = [&](int i, int b) {  // step i of this wave (past the last: the last again, not used) into slot b
    const int s = min(wave + i * NW, steps - 1);
    const uint32_t k = (uint32_t)min(s * 128 + ch, a.K - 16);  // (chunks past K load the last one and are zeroed below)
    const uint32_t l = ring0 + (uint32_t)(b * STEP);
#pragma unroll
    for (int t = 0; t < WT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) lds_dma16_off(GATED && t >= CT ? wb2 : wb, wo[t][u] + k, l + t * 2048 + u * 1024);
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int u = 0; u < 2; ++u) lds_dma16_off(xb, xo[t][u] + k, l + (WT + t) * 2048 + u * 1024);
    lds_dma4_off(xsb + (long)s * a.M * 4, so, l + (WT + MT) * 2048);
  };
  {  // the weight scales of the columns' block, in whole words or by bytes
    const int row = n0 >> 5, nb = a.K / 32;
    for (int q = wave; q < (GATED ? 2 : 1); q += NW) {
      const uint8_t* p = q ? a.ws2 + (long)row * a.Kc2 : a.ws + (long)row * a.Kc;
      if (a.words)
        for (int c = 0; c < nb / 4; c += 64)
          lds_dma4_off(p, (uint32_t)min(c + lane, nb / 4 - 1) * 4, lds_addr_of(&scl[q][0]) + c * 4);
      else
        for (int k = lane; k < nb; k += 64) scl[q][k] = p[k];
    }
  }
#pragma unroll
  for (int i = 0; i < D - 1; ++i) issue(i, i);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm((D - 1) * LPS));  // the scales are there (they were first)
  lds_barrier();

  f32x4_t acc[WT][MT];
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
  const int c0 = (2 * g) ^ (l16 & 7), c1 = c0 ^ 1;  // a lane's two chunks
  const int last = a.K / 32 - 1;
  int bi = 0;
#pragma unroll 1
  for (int i = 0; i < mine; ++i) {
    issue(i + D - 1, bi == 0 ? D - 1 : bi - 1);
    __builtin_amdgcn_s_waitcnt(vmcnt_imm((D - 1) * LPS));
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    uint8_t* st = ring + bi * STEP;
    const int s = wave + i * NW;
    if (s * 128 + 128 > a.K) {  // K ends inside this step: zeros from there on
      const int first = (a.K - s * 128) / 16;
      for (int e = lane; e < (WT + MT) * 128; e += 64)
        if ((e & 7) >= first) *(uint4*)(st + (e >> 3) * 128 + (((e & 7) ^ ((e >> 3) & 7)) * 16)) = make_uint4(0, 0, 0, 0);
    }
    auto operand = [&](int t, uint4& p, uint4& q) {
      const uint8_t* r = st + t * 2048 + l16 * 128;
      p = *(const uint4*)(r + c0 * 16);
      q = *(const uint4*)(r + c1 * 16);
    };
    const int blk = min(4 * s + g, last);  // (behind the last: any scale that is a number, the codes are zero)
    int ws[GATED ? 2 : 1], xs[MT];
    ws[0] = scl[0][blk];
    if constexpr (GATED) ws[1] = scl[1][blk];
#pragma unroll
    for (int j = 0; j < MT; ++j) xs[j] = st[(WT + MT) * 2048 + (16 * j + l16) * 4 + (blk & 3)];
    uint4 x[MT][2];
#pragma unroll
    for (int j = 0; j < MT; ++j) operand(WT + j, x[j][0], x[j][1]);
    uint4 xd[MT][4];
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const float sc = a8_e8m0(xs[j]);
#pragma unroll
      for (int h = 0; h < 4; ++h)
        xd[j][h] = h & 1 ? a8_decode(x[j][h >> 1].z, x[j][h >> 1].w, sc) : a8_decode(x[j][h >> 1].x, x[j][h >> 1].y, sc);
    }
#pragma unroll
    for (int t = 0; t < WT; ++t) {
      const float sc = a8_e8m0(ws[t / CT]);
      uint4 c[2];
      operand(t, c[0], c[1]);
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const uint4 w = h & 1 ? a8_decode(c[h >> 1].z, c[h >> 1].w, sc) : a8_decode(c[h >> 1].x, c[h >> 1].y, sc);
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[t][j] = mfma_bf16_16x16x32(w, xd[j][h], acc[t][j]);
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this slot is read: the next issue may fill it
    bi = bi + 1 == D ? 0 : bi + 1;
  }
  // lane (l16, g): row l16 of x, columns 4 g .. 4 g + 3 of the tile
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));
  lds_barrier();  // no load is on its way into the LDS, and every wave has read its last step
  float* red = (float*)lds;  // [waves][WT * MT][64 lanes][4]
#pragma unroll
  for (int i = 0; i < WT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *(f32x4_t*)(red + ((wave * WT + i) * MT + j) * 256 + lane * 4) = acc[i][j];
  __syncthreads();
  constexpr int QN = 2 * CT;  // lanes of a row: 8 columns each
  for (int t = tid; t < QN * 16 * MT; t += 64 * NW) {  // (in whole quads of lanes: a block of 32 columns with CT 2)
    const int c = t % QN, r = t / QN, m = m0 + r, n = n0 + 8 * c;
    const float* p = red + ((c >> 1) * MT + (r >> 4)) * 256 + ((c & 1) * 32 + (r & 15)) * 4;  // the next 4: lanes on 16
    const bool live = m < a.M && n < a.N;
    const uint4 res = a8_res8(a.e, m, n);
    const A8x8 bias = a8_bias8(a.e, n);
    A8x8 y, u;
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] = u.v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
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
constexpr int kA8Strip = 4;
constexpr int kTileMaxK = 16384;  // (the weight scales of a tile are held in LDS)

// Output of a wave's ROWS x OCW block of sums from LDS (fp32, row stride LD bytes), not from the accumulators: unrolled over
// those, bias, activation and quantisation were 100 KB of code.  The residual is loaded before any of it is stored.
template <int ROWS, int LD, int OCW, bool GATED>
DSV41_DEV void a8_wave_out(const A8Args& a, const uint8_t* s, int m0, int n0) {
  constexpr int QN = OCW / 8, RP = 64 / QN, PASSES = ROWS / RP;  // lanes of a row, rows of a pass
  static_assert(64 % QN == 0 && ROWS % RP == 0 && PASSES <= 8, "whole passes, residuals in registers");
  static_assert(!GATED || OCW == 32, "a gate block and its up block");
  const int lane = threadIdx.x & 63, c = lane % QN * 8, n = n0 + c, m = m0 + lane / QN;
  s += lane / QN * LD + c * 4;
  const A8x8 bias = a8_bias8(a.e, n);
  uint4 res[PASSES];
  if constexpr (!GATED) {
#pragma unroll
    for (int k = 0; k < PASSES; ++k) res[k] = a8_res8(a.e, m + k * RP, n);
  }
#pragma unroll
  for (int k = 0; k < PASSES; ++k) {
    const uint8_t* p = s + k * RP * LD;
    A8x8 y = *(const A8x8*)p, u = y;
    if constexpr (GATED) u = *(const A8x8*)(p + 128);
    if constexpr (GATED) a8_gated8(a.e, y, u);
    else a8_linear8(a.e, y, bias, res[k]);
    a8_store8(a.e, y, m + k * RP, n, m + k * RP < a.M && n < a.N);
  }
}

// BM rows of x by BN rows of weights in WM x WN waves of (BM / WM) x (BN / WN); stages of 128 k through NBUF LDS buffers.
// Bound: the bf16 matrix units under load.  256 x 256, gated 4096 x 2 x 8192 x 5120: 523 us, 1.31 PFLOP/s (a library bf16
// product of 8192^3: 1.24); a wave's 96 decoding conversions of a half stand beside 64 products of 16 cycles.  Smaller tiles
// decode more a product: 128 x 128, a wave of 32 x 64, 0.87.
// A gated tile has BN / 2 output columns: of a wave's 32-row weight blocks the even ones are gate rows, the odd ones the
// up rows of the same columns.
template <int BM, int BN, int WM, int WN, int NBUF, bool GATED>
__global__ void __launch_bounds__(64 * WM * WN) a8_tile_kernel(const A8Args a) {
  constexpr int NT = 64 * WM * WN;
  constexpr int MT = BM / WM / 16, CT = BN / WN / 16;  // 16-row blocks of a wave
  constexpr int XB = BM * 128, WB = BN * 128, SB = BM * 4, STAGE = XB + WB + SB;
  constexpr int XL = XB / 16 / NT, WL = WB / 16 / NT, LPT = XL + WL + 1;  // loads per thread and stage
  constexpr int OC = GATED ? BN / 2 : BN;                                 // output columns
  // A stage is two halves (a lane's first and second 16 of its 32 codes) of MT steps each: 16 rows of x with the CT weight
  // blocks.  The codes of a step are read two steps before it, across the stage's end too, and decoded one step before; the
  // barrier stands in step ENTER, where the first of the next stage is read.  A half's weights are read in the step before
  // the last of the half in front of it and decoded behind its last products.
  constexpr int S = 2 * MT, ENTER = S - 2;
  // A stage's loads are issued between the products from that barrier on, in the first POS of the S CT places; FIRST of
  // them fall into the stage in which they begin.
  constexpr int POS = S * CT * (NBUF == 2 ? 3 : 6) / 8;
  constexpr auto upto = [](int z) constexpr { return z >= POS ? LPT : z * LPT / POS; };
  constexpr int FIRST = upto(2 * CT);
  static_assert(XL * NT * 16 == XB && WL * NT * 16 == WB && MT * WM * 16 == BM && CT * WN * 16 == BN, "tile shape");
  static_assert(!GATED || CT % 4 == 0, "gate and up blocks in pairs");
  static_assert(MT >= 2 && BM % 64 == 0, "two steps a half, scales of 64 rows a wave");
  static_assert((NBUF - 2) * LPT + FIRST < 64, "vmcnt immediate");
  __shared__ __align__(16) uint8_t buf[NBUF * STAGE];
  __shared__ __align__(16) uint8_t scl[BN / 32][kTileMaxK / 32 + 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int wm = wave / WN, wn = wave - wm * WN;
  // contiguous tile ranges per XCD, in strips of kA8Strip row tiles: the tiles that run on an XCD together share rows and
  // weights in its L2
  const int per = gridDim.x / kXcds;
  const int id = (blockIdx.x % kXcds) * per + blockIdx.x / kXcds;
  if (id >= a.mtiles * a.ntiles) return;  // (the grid is a multiple of the XCDs)
  const int strip = id / (kA8Strip * a.ntiles), sm = min(kA8Strip, a.mtiles - strip * kA8Strip);
  const int in = id - strip * kA8Strip * a.ntiles;
  const int m0 = (strip * kA8Strip + in % sm) * BM, n0 = a.first + in / sm * OC;
  const int nk = a.K / 128, tail = a.K % 128;  // whole stages, and the k behind them

  // weight row r of the tile: output column (from n0) and matrix
  auto column = [&](int r) { return GATED ? (r / 64) * 32 + (r & 31) : r; };
  auto is_up = [&](int r) { return GATED && (r & 32) != 0; };
  const uint8_t* xb = a.x + (long)m0 * a.K;
  const uint8_t* wb = a.w + (long)n0 * a.K;
  const uint8_t* wb2 = GATED ? a.w2 + (long)n0 * a.K : nullptr;
  const uint8_t* xsb = a.xs + 4l * m0;
  // Load u of a thread brings 16 bytes of row u NT / 8 + tid / 8 (rows past the end repeat the last and are not stored).
  // Chunk c of a 128-byte row r sits at c ^ (r & 7): the 8 lanes of an LDS read cycle (8 rows, one chunk) then hit 8
  // different 16-byte bank groups.
  const int r0 = tid >> 3, ch = ((tid & 7) ^ (r0 & 7)) * 16;
  const int xlim = a.M - 1 - m0, wlim = a.N - 1 - n0;
  const uint32_t so = (uint32_t)min((wave % (SB / 256)) * 64 + lane, xlim) * 4;
  const uint32_t lds0 = lds_addr_of(buf);
  const uint32_t ldsw = lds0 + (uint32_t)wave * 1024, ldss = lds0 + XB + WB + (uint32_t)(wave % (SB / 256)) * 256;
  const int klast = a.K - 16;  // the last 16 codes of a row
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
      lds_dma16_off(xb, xo[q] + k, ldsw + l + q * NT * 16);
    } else if (q < XL + WL) {  // (a wave's 8 rows are of one matrix)
      const int u = q - XL;
      lds_dma16_off(is_up(u * (NT / 8) + wave * 8) ? wb2 : wb, wo[u] + k, ldsw + l + XB + u * NT * 16);
    } else {
      lds_dma4_off(xsb + (long)kt * a.M * 4, so, ldss + l);
    }
  };
  {  // the tile's weight scales
    const int nb = (a.N + 31) / 32, kb = a.K / 32;
    auto scales = [&](int b) {
      const int row = min((n0 + column(b * 32)) / 32, nb - 1);
      return (is_up(b * 32) ? a.ws2 + (long)row * a.Kc2 : a.ws + (long)row * a.Kc);
    };
    if (a.words) {  // whole words: by direct loads, ahead of the stages'
      for (int b = wave; b < BN / 32; b += WM * WN)
        for (int c = 0; c < nk; c += 64)
          lds_dma4_off(scales(b), (uint32_t)min(c + lane, nk - 1) * 4, lds_addr_of(&scl[b][0]) + c * 4);
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
  const int c0 = ((2 * g) ^ (l16 & 7)) * 16;                        // chunk 2 g; 2 g + 1 sits at c0 ^ 16
  // The next stage has landed for every wave (`later` younger loads may not have), and every wave has read this one.
  auto enter = [&](auto later) {
    __builtin_amdgcn_s_waitcnt(vmcnt_imm(decltype(later)::value));
    lds_barrier();
  };
  uint4 xq[2], wq[CT], xd[2][2], wd[CT][2];  // codes as read; decoded
  int xs[2], ws[CT / 2];                     // scale bytes
  float wsc[CT / 2];
  auto read_x = [&](int u, int b) {
    const uint8_t* st = buf + b * STAGE;
    xq[u & 1] = *(const uint4*)(st + (xr + 16 * (u % MT)) * 128 + (c0 ^ (u / MT * 16)));
    xs[u & 1] = st[XB + WB + (xr + 16 * (u % MT)) * 4 + g];
  };
  auto read_w = [&](int half, int kt, int b) {
#pragma unroll
    for (int j = 0; j < CT; ++j) wq[j] = *(const uint4*)(buf + b * STAGE + XB + (wr + 16 * j) * 128 + (c0 ^ (half * 16)));
    if (half == 0) {
#pragma unroll
      for (int j = 0; j < CT / 2; ++j) ws[j] = scl[wn * (CT / 2) + j][kt * 4 + g];  // (kt: to one past the last, in the row)
    }
  };
  auto decode_x = [&](int u) {
    const float sc = a8_e8m0(xs[u & 1]);
    xd[u & 1][0] = a8_decode(xq[u & 1].x, xq[u & 1].y, sc);
    xd[u & 1][1] = a8_decode(xq[u & 1].z, xq[u & 1].w, sc);
  };
  auto decode_w = [&](int j) {
    wd[j][0] = a8_decode(wq[j].x, wq[j].y, wsc[j / 2]);
    wd[j][1] = a8_decode(wq[j].z, wq[j].w, wsc[j / 2]);
  };
  auto scales_w = [&] {
#pragma unroll
    for (int j = 0; j < CT / 2; ++j) wsc[j] = a8_e8m0(ws[j]);
  };
  auto product = [&](int u, int j) {
    acc[u % MT][j] = mfma_bf16_16x16x32(wd[j][0], xd[u & 1][0], acc[u % MT][j]);
    acc[u % MT][j] = mfma_bf16_16x16x32(wd[j][1], xd[u & 1][1], acc[u % MT][j]);
  };
  if (nk > 0) {
    int bi = 0;
    enter(std::integral_constant<int, (NBUF - 2) * LPT + FIRST>{});
    read_w(0, 0, 0);
    read_x(0, 0);
    read_x(1, 0);
    scales_w();
#pragma unroll
    for (int j = 0; j < CT; ++j) decode_w(j);
    decode_x(0);
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {  // (what the last stage reads and loads ahead is the last again, and not used)
      const int b0 = bi;
      bi = bi + 1 == NBUF ? 0 : bi + 1;
      const int bp = b0 == 0 ? NBUF - 1 : b0 - 1;
#pragma unroll
      for (int u = 0; u < S; ++u) {
        if (u == ENTER) enter(std::integral_constant<int, (NBUF - 2) * LPT>{});
        if (u % MT == MT - 2) read_w(u < MT ? 1 : 0, u < MT ? kt : kt + 1, u < MT ? b0 : bi);
        read_x((u + 2) % S, u < ENTER ? b0 : bi);
        __builtin_amdgcn_sched_barrier(0);
        if (u == S - 1) scales_w();
#pragma unroll
        for (int j = 0; j < CT; ++j) {
          product(u, j);
          if (j == 0) decode_x((u + 1) % S);
          if (u % MT == MT - 1) decode_w(j);
          const int z = (u < ENTER ? u + 2 : u - ENTER) * CT + j;
#pragma unroll
          for (int q = upto(z); q < upto(z + 1); ++q)
            dma(min(u < ENTER ? kt + NBUF - 1 : kt + NBUF, nk - 1), u < ENTER ? bp : b0, q);
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
    for (int u = 0; u < S; ++u) {
      if (u % MT == 0) {
        read_w(u / MT, nk, 0);
        if (u == 0) scales_w();
#pragma unroll
        for (int j = 0; j < CT; ++j) decode_w(j);
      }
      read_x(u, 0);
      xs[u & 1] = buf[XB + WB + (xr + 16 * (u % MT)) * 4 + min(g, tail / 32 - 1)];  // (bytes behind the last may be anything)
      decode_x(u);
#pragma unroll
      for (int j = 0; j < CT; ++j) product(u, j);
    }
    lds_barrier();
  }

  // A lane (l16, g) has row l16, columns 4 g .. 4 g + 3 of a block: PM blocks of rows at a time through the wave's part of
  // the LDS (rows padded by 16 bytes: 8 lanes write 8 different bank groups)
  constexpr int LD = BN / WN * 4 + 16;
  constexpr int ROOM = NBUF * STAGE / (16 * LD * WM * WN);  // blocks of rows a wave has LDS for
  constexpr int PM = ROOM >= MT ? MT : ROOM >= MT / 2 ? MT / 2 : MT / 4;
  static_assert(PM > 0 && PM <= ROOM && MT % PM == 0, "output staging");
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

// ------------------------------------------------------------------------------------------------ plan
// Up to 32 rows: the stream of one row block.  16 columns a workgroup (one token, 8192 k, 5120 columns 10.8 us
// against 13.3 of 32) unless the output is in blocks of 32 or there are columns enough to fill the card twice over (32768
// columns of 1280 k 10.5 against 9.1 us, in workgroups of 2 waves, 10.3 in 4); 8 waves where a workgroup of 4 to every CU
// would leave half of them idle (512 columns of 5120 k 5.3 against 6.1 us).
// More rows: the least of the estimates below, microseconds (fitted to whole rounds of 640 to 8192 k; 33 to 4096 rows of
// the layer's widths: within a tenth of the fastest kernel but for a few places between two rounds).  Of estimates within
// half a microsecond of the least, which is as well as they are known, the one that reads the fewest operand bytes.
// Streams of 32, 48 and 64 rows and the smallest tile at 5120 k and 2048 columns, us: 64 rows 9.3, 11.1, 12.8, 36; 130 rows
// 12.4, 11.5, 13.4, 37; 500 rows 24.1, 31.5, 25.7, 38.  A stream's blocks of rows read the weights again (3.1 TB/s, half
// of each reading after the first from the caches): 64 rows of 8192 columns and 8192 k 34 us in two blocks of 32 rows and
// 23 in one of 64.
// A tile with rows and columns exchanged is as fast (64 x 128, 64 x 256, 128 x 256: within 3 %).  One round of 256 x 256
// and one of 128 x 128 for the columns behind it: 4096 rows of 5120 columns, 8192 k 293 us for 323 in 2 rounds of 192 x 256.
constexpr int kCus = 256;
constexpr int kMaxRows = 0x7fffff00;  // (a workgroup's rows are counted to its end)
enum A8Kernel {
  kStream16, kStream32, kStream48, kStream64,
  kTile128x64, kTile128x128, kTile256x128, kTile192x256, kTile256x256
};
struct A8Plan {
  A8Kernel kernel;
  int rows, cols, waves;  // a workgroup's rows of x, weight rows, and (streams) waves
};
struct A8Parts {
  A8Plan plan, rest;
  int columns;  // output columns on `plan`, and from there on those on `rest`
};

A8Parts a8_plan(int M, int N, int K, bool gated, bool a8_out) {
  if (M <= 32) {
    const bool wide = N > 16384;
    const int cols = a8_out || wide || (M > 16 && gated) ? 32 : 16;
    const A8Plan p{M <= 16 ? kStream16 : kStream32, M <= 16 ? 16 : 32, cols,
                   wide ? 2 : M <= 16 && cols == 16 && N <= 16 * kCus / 2 ? 8 : 4};
    return A8Parts{p, p, N};
  }
  struct Cost {
    A8Plan plan;
    float fixed, step;  // us of a round of kCus workgroups: launch, first loads and output; 128 k
    int least;          // rounds at least (2: two workgroups a CU at once)
  };
  const Cost linear[] = {
      {{kStream32, 32, 32, 4}, 3.5f, 0.159f, 1},
      {{kStream32, 32, 32, 4}, 1.9f, 0.120f, 2},
      {{kStream48, 48, 32, 4}, 3.6f, 0.203f, 1},
      {{kStream64, 64, 32, 4}, 4.0f, 0.250f, 1},
      {{kTile128x64, 128, 64, 4}, 5.7f, 0.877f, 1},
      {{kTile128x64, 128, 64, 4}, 3.4f, 0.690f, 2},
      {{kTile128x128, 128, 128, 8}, 7.2f, 1.335f, 1},
      {{kTile256x128, 256, 128, 8}, 10.5f, 2.110f, 1},
      {{kTile192x256, 192, 256, 8}, 13.1f, 2.800f, 1},
      {{kTile256x256, 256, 256, 8}, 16.4f, 3.520f, 1},
  };
  const Cost gates[] = {  // (two 32-row streams do not fit a CU's LDS: 102400 bytes each)
      {{kStream32, 32, 64, 4}, 4.0f, 0.250f, 1},
      {{kStream48, 48, 64, 4}, 4.4f, 0.312f, 1},
      {{kStream64, 64, 64, 4}, 5.0f, 0.372f, 1},
      {{kTile128x64, 128, 64, 4}, 4.3f, 0.940f, 1},
      {{kTile128x64, 128, 64, 4}, 2.4f, 0.703f, 2},
      {{kTile128x128, 128, 128, 8}, 5.0f, 1.360f, 1},
      {{kTile256x128, 256, 128, 8}, 7.0f, 2.160f, 1},
      {{kTile192x256, 192, 256, 8}, 8.7f, 2.810f, 1},
      {{kTile256x256, 256, 256, 8}, 11.3f, 3.520f, 1},
  };
  const Cost* const costs = gated ? gates : linear;
  const int n_costs = gated ? sizeof(gates) / sizeof(Cost) : sizeof(linear) / sizeof(Cost);
  const float steps = (float)((K + 127) / 128);
  const long wr = gated ? 2 : 1;
  struct Estimate {
    float us, bytes;  // bytes: operands read, a k
  };
  auto estimate = [&](const Cost& c, long n) {
    const long rows = (M + c.plan.rows - 1l) / c.plan.rows, cols = (n * wr + c.plan.cols - 1) / c.plan.cols;
    const float rounds = fmaxf((float)((rows * cols + kCus - 1) / kCus), (float)c.least), weights = (float)(n * wr);
    float us = rounds * (c.fixed + steps * c.step);
    if (c.plan.kernel < kTile128x64) us = fmaxf(us, weights * (float)K * (0.5f + 0.5f * (float)rows) / 3.1e6f);
    return Estimate{us, weights * (float)rows + (float)M * (float)cols};
  };
  // The plan of n columns on one kernel (`any`, or a tile kernel), and its estimate
  auto choose = [&](long n, bool any, A8Plan* plan) {
    float best = 1e30f;
    auto open = [&](const Cost& c) {  // (a stream's row blocks are the grid's y)
      return c.plan.kernel >= kTile128x64 ? K <= kTileMaxK : any && (M + c.plan.rows - 1l) / c.plan.rows <= 65535;
    };
    for (int i = 0; i < n_costs; ++i)
      if (open(costs[i])) best = fminf(best, estimate(costs[i], n).us);
    Estimate least{best, 1e30f};
    for (int i = 0; i < n_costs; ++i) {
      const Estimate e = estimate(costs[i], n);
      if (!open(costs[i]) || e.us > best + 0.5f) continue;
      if (e.bytes > least.bytes || (e.bytes == least.bytes && e.us >= least.us)) continue;
      least = e;
      *plan = costs[i].plan;
    }
    return least.us;
  };
  A8Parts p{linear[3].plan, linear[3].plan, N};
  float best = choose(N, true, &p.plan);
  // Or the columns that fill whole rounds of a tile kernel, and a second launch for the others
  if (K <= kTileMaxK) {
    for (int i = 0; i < n_costs; ++i) {
      const Cost& c = costs[i];
      if (c.plan.kernel < kTile128x64) continue;
      const long rows = (M + c.plan.rows - 1l) / c.plan.rows, per = c.plan.cols / wr, rounds = rows * (N / per) / kCus;
      const long columns = rounds * kCus / rows * per;
      if (rounds < c.least || columns == 0 || columns >= N) continue;
      A8Plan rest;
      const float us = (float)rounds * (c.fixed + steps * c.step) + choose(N - columns, false, &rest);
      if (us < 0.97f * best) {
        best = us;
        p = A8Parts{c.plan, rest, (int)columns};
      }
    }
  }
  return p;
}

// Columns first .. end - 1 by the kernel of p.
template <bool GATED>
int a8_launch(A8Args& a, const A8Plan& p, int first, int end, hipStream_t st) {
  // (a plan's columns are the output's up to 32 rows, the weights' rows above)
  const long oc = GATED && a.M > 32 ? p.cols / 2 : p.cols;
  a.mtiles = (int)((a.M + p.rows - 1l) / p.rows);
  a.first = first;
  a.ntiles = (int)((end - first + oc - 1l) / oc);
  const bool tile = p.kernel >= kTile128x64;
  const long tiles = ((long)a.mtiles * a.ntiles + kXcds - 1) / kXcds * kXcds, threads = 64 * p.waves;
  if ((tile ? tiles : a.ntiles) * threads > 0xffffffffl || (!tile && a.mtiles > 65535)) return (int)hipErrorInvalidValue;
  const dim3 gs((unsigned)a.ntiles, (unsigned)a.mtiles), gt((unsigned)tiles);
  switch (p.kernel) {
    case kStream16:
      if (p.cols == 16 && p.waves == 8) a8_stream_kernel<1, 1, 8, 2, GATED><<<gs, 512, 0, st>>>(a);
      else if (p.cols == 16) a8_stream_kernel<1, 1, 4, 2, GATED><<<gs, 256, 0, st>>>(a);
      else if (p.waves == 2) a8_stream_kernel<1, 2, 2, 2, GATED><<<gs, 128, 0, st>>>(a);
      else a8_stream_kernel<1, 2, 4, 2, GATED><<<gs, 256, 0, st>>>(a);
      break;
    case kStream32:
      if (p.cols == 16) {
        if constexpr (!GATED) a8_stream_kernel<2, 1, 4, 2, false><<<gs, 256, 0, st>>>(a);
      } else if (p.waves == 2) {
        a8_stream_kernel<2, 2, 2, 2, GATED><<<gs, 128, 0, st>>>(a);
      } else {
        a8_stream_kernel<2, 2, 4, 2, GATED><<<gs, 256, 0, st>>>(a);
      }
      break;
    case kStream48: a8_stream_kernel<3, 2, 4, 2, GATED><<<gs, 256, 0, st>>>(a); break;
    case kStream64: a8_stream_kernel<4, 2, 4, 2, GATED><<<gs, 256, 0, st>>>(a); break;
    case kTile128x64: a8_tile_kernel<128, 64, 4, 1, 3, GATED><<<gt, 256, 0, st>>>(a); break;
    case kTile128x128: a8_tile_kernel<128, 128, 4, 2, 3, GATED><<<gt, 512, 0, st>>>(a); break;
    case kTile256x128: a8_tile_kernel<256, 128, 4, 2, 3, GATED><<<gt, 512, 0, st>>>(a); break;
    case kTile192x256: a8_tile_kernel<192, 256, 2, 4, 2, GATED><<<gt, 512, 0, st>>>(a); break;
    case kTile256x256: a8_tile_kernel<256, 256, 2, 4, 2, GATED><<<gt, 512, 0, st>>>(a); break;
  }
  DSV41_CHECK_LAUNCH();
  return 0;
}

template <bool GATED>
int a8_run(A8Args& a, hipStream_t st) {
  if (a.M == 0 || a.N == 0) return 0;
  if (a.M < 0 || a.N < 0 || a.M > kMaxRows || a.N > kMaxRows || a.K <= 0 || a.K % 32 != 0 || a.K > kStreamMaxK ||
      a.Kc < a.K / 32 || (GATED && a.Kc2 < a.K / 32))
    return (int)hipErrorInvalidValue;
  if (!a.x || !a.xs || !a.w || !a.ws || (GATED && (!a.w2 || !a.ws2))) return (int)hipErrorInvalidValue;
  if (((uintptr_t)a.x | (uintptr_t)a.w | (uintptr_t)a.w2) & 15 || (uintptr_t)a.xs & 3) return (int)hipErrorInvalidValue;
  if (a.e.act < kActNone || a.e.act > kActGeluTanh || !(a.e.limit >= 0.0f)) return (int)hipErrorInvalidValue;
  if (!a.e.out && (!a.e.oa8 || !a.e.os8 || a.N % 32 != 0 || (uintptr_t)a.e.oa8 & 15)) return (int)hipErrorInvalidValue;
  a.e.M = a.M;
  a.e.N = a.N;
  a.e.vec = a.N % 8 == 0 && (((uintptr_t)a.e.out | (uintptr_t)a.e.res) & 15) == 0;
  a.words = a.K % 128 == 0 && ((a.Kc | a.Kc2 | (uintptr_t)a.ws | (uintptr_t)a.ws2) & 3) == 0;
  const A8Parts p = a8_plan(a.M, a.N, a.K, GATED, a.e.out == nullptr);
  const int rc = a8_launch<GATED>(a, p.plan, 0, p.columns, st);
  return rc != 0 || p.columns == a.N ? rc : a8_launch<GATED>(a, p.rest, p.columns, a.N, st);
}

}  // namespace

extern "C" {

int dsv41_a8_plan(int M, int N, int K, int gated, int a8_out, int rest) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const A8Parts p = a8_plan(M, N, K, gated != 0, a8_out != 0);
  const A8Plan& k = rest ? p.rest : p.plan;
  if (rest && p.columns == N) return 0;
  return (k.kernel >= kTile128x64 ? 1 << 30 : 0) | k.rows << 16 | k.cols << 4 | k.waves;
}

int dsv41_linear_a8(const void* a8, const void* s8, const void* w8, const void* ws8, int M, int N, int K, int Kc,
                    const void* bias, int bias_f32, int act, const void* residual, void* out, void* out_a8,
                    void* out_s8, void* stream) {
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
  return a8_run<false>(a, (hipStream_t)stream);
}

int dsv41_gated_a8(const void* a8, const void* s8, const void* wg8, const void* wgs8, const void* wu8,
                   const void* wus8, int M, int N, int K, int Kcg, int Kcu, int act, float limit, void* out,
                   void* out_a8, void* out_s8, void* stream) {
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
  return a8_run<true>(a, (hipStream_t)stream);
}

}  // extern "C"
