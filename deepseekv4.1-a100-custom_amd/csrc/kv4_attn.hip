// Sparse attention over window rows (bf16) and selected rows of the paged 4-bit cache.
//
// One workgroup of four waves: one query row, 16 heads, a run of 64-key tiles (first the window's, then the cache's).
// Each wave scores 16 of a tile's keys: S^T = K Q^T by 16x16x32 MFMAs, the keys' fragments straight from memory into
// registers -- lane (key l % 16, quarter l / 16) holds 128 consecutive values of its key, 64 bytes of codes, which are
// the operands of 16 k steps if Q is held in the same order.  The decoded rows go to LDS once, as the values; then each
// wave multiplies the tile's probabilities by 128 of the 512 value columns, O^T += V^T P^T.
//
// Decoding is exact in fp16 (E2M1 times e4m3 has 6 significand bits), two packed instructions for two values; Q in fp16,
// each head scaled by a power of two, is exact too, but for values under 2^-28 of their head's largest (off by 2^-39 of it
// at most, a logit by less than fp32's own rounding of a sum with that one).  Window rows have bf16's range, so they stay
// in bf16.
// Sums, the softmax's maximum and sum and O are fp32; the reference maximum moves only for a score 2^8 above it; the
// probabilities are rounded to fp16 (2^-11 of each; bf16 for window rows, whose values need its range: 2^-8), the operand type
// of the products, and the output once, after the rotation.
// Of a cache's rows the reference is 2^7 under the maximum, so that the largest probability is 2^7 to 2^15 and fp16's last
// bit, 2^-24, is 2^-31 of it or less: n keys of a long flat rest are off by n 2^-32 of the peak's weight together (with the
// maximum as the reference weights under 2^-25 were lost, 2^18 of them 0.5 % of the numerator).
//
// Whole rows go to LDS by direct loads, a row a wave and load: a lane's own 16 bytes of 16 rows are 64 requests a load (Q and
// window rows so, with their reads ahead: a prompt of 2 x 301 queries 62.7 us for 77.7).  Codes come that way all the same, 4 loads a tile: the
// LDS has no room for them beside the values of two workgroups, and an exchange of lanes costs what it saves.
//
// What bounds it.  A step of single tokens: latency.  Four sequences of 2048 selected rows and 64 heads of 576 read 4 MB
// and take 17.3 us in a graph, of them 4.0 us for joining the splits; one sequence of 300 rows of 512 10.8 us.  Prompts
// of few heads: the writes of the decoded rows to LDS (13 cycles a wave's kilobyte, 840 a tile and workgroup) and the
// chain of a tile's phases, 4300 cycles beside another workgroup (602 query rows of 512 + 128 keys, 20 heads of 512:
// 62.7 us).  32 heads a workgroup halve the decoding but leave one workgroup a CU (97 us when 16 heads took 83).
#include <type_traits>

#include "kv4_attn_core.h"

namespace {

constexpr float kLow = 7.0f;  // the reference of fp16 probabilities under the maximum, in powers of two

template <int DQK>
__global__ void __launch_bounds__(256, 2) kv4_attn_kernel(const Kv4AttnArgs a) {
  constexpr int TS = DQK == 576 ? 2 : 0;   // k steps of the last 64 columns
  constexpr int RB = kv4_row_bytes(DQK);
  __shared__ __align__(1024) uint8_t s_v[64 * 1024];
  __shared__ __align__(16) uint8_t s_p[16 * 128];
  __shared__ __align__(16) float s_m[16 * 4];

  // The head groups of a (row, split) read the same rows of the cache: eight workgroups apart they share an XCD's L2.
  const int b = blockIdx.x, units = a.R * a.nsplit, full = units & ~7;
  const int n8 = b < full * a.groups ? 8 : units - full;
  const int in = b < full * a.groups ? b % (8 * a.groups) : b - full * a.groups;
  const int u0 = (b < full * a.groups ? b / (8 * a.groups) * 8 : full) + in % n8;
  const int hg = in / n8, sp = u0 % a.nsplit, r = u0 / a.nsplit;
  const int h0 = hg * 16;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int slot = r / a.rows_per_slot;
  const long seq = a.seq ? a.seq[slot] : slot;
  const long pos = a.pos ? a.pos[r] : 0;
  const int t0 = sp * a.chunk, t1 = min(t0 + a.chunk, a.tiles);

  const int key = wave * 16 + l16;  // this lane's key of a tile

  typedef const __attribute__((address_space(1))) uint8_t* row_t;
  row_t none = (row_t)g_kv4_none;  // (its address read once)
  asm volatile("" : "+s"(none));

  auto get16 = [](row_t p) { return __builtin_bit_cast(uint4, *(const __attribute__((address_space(1))) u32x4*)p); };
  auto get8 = [](row_t p) { return __builtin_bit_cast(uint2, *(const __attribute__((address_space(1))) u32x2*)p); };

  // the row of the window that this lane's key of tile u is, nullptr: none; by its index where there is a list
  const bool ring = !a.widx;
  const long pmax = ring && a.pmax ? a.pmax[r] : 0, plim = ring && a.plim ? a.plim[r] : pos;
  auto listed = [&](int u) { return ring || a.wt == 0 ? -1 : a.widx[(long)r * a.wt + min(u * 64 + key, a.wt - 1)]; };
  auto window = [&](int u, int i) -> row_t {
    const int j = u * 64 + key;
    bool there;
    if (ring) {  // slot j of the ring holds the newest position of its residue
      i = j;
      int d = (int)(pmax - j) % a.win_rows;  // (positions fit in 31 bits)
      if (d < 0) d += a.win_rows;
      const long held = pmax - d;
      there = j < a.win_rows && held >= 0 && held <= plim && pos - held < a.win_rows && seq >= 0 && seq < a.win_slots;
    } else {
      there = j < a.wt && i >= 0 && i < a.win_rows;
    }
    return there ? (row_t)(a.win + (ring ? seq : (long)slot) * a.win_sstride + (long)i * DQK) : nullptr;
  };
  // the cache's rows
  const int* const ids = a.idx + (long)r * a.t;
  const long rows = (long)a.map.cols << a.map.shift;
  const bool known = seq >= 0 && seq < a.map.slots;
  const int* const pages = a.map.table + (known ? seq : 0) * a.map.cols;
  // the way to this lane's key of tile u (where the list ends, the last entry's, which source() then leaves out)
  auto index = [&](int u) { return ids[min((u - a.wtiles) * 64 + key, a.t - 1)]; };
  auto page = [&](int i) { return pages[i >= 0 && i < rows ? i >> a.map.shift : 0]; };
  auto source = [&](int u, int i, int p) -> row_t {
    const bool there = known && u < t1 && (u - a.wtiles) * 64 + key < a.t && i >= 0 && i < rows;
    return there && (unsigned)p < (unsigned)a.map.pages ? (row_t)(a.pool + kv4_offset(a.map, p, i, RB)) : nullptr;
  };
  const uint32_t v_base = lds_addr_of(s_v), p_base = lds_addr_of(s_p), m_base = lds_addr_of(s_m);
  // this lane's unit 0 of its key's row, and its place in the transpose reads of key g * 8 + l16 / 4; the other units, and
  // the keys 4 further, are an XOR away
  const uint32_t v_put = v_base + key * 1024 + 256 * g + (v_swizzle(key) << 4);
  const uint32_t v_get = v_base + (g * 8 + (l16 >> 2)) * 1024 + wave * 256 +
                         ((((l16 & 3) >> 1) | ((l16 >> 2) << 1 ^ (g & 1) << 3)) << 4) + (l16 & 1) * 8;

  // The way to the first rows, two loads deep, is gone before Q is asked for.
  int t = t0;
  const int first = max(t0, a.wtiles);
  const bool cached = first < t1 && a.t > 0;
  const int wend = min(t1, a.wtiles);
  int w0 = -1, w1 = -1, i0 = -1, i1 = -1;
  if (t < wend) {
    w0 = listed(t);
    w1 = listed(t + 1);
  }
  if (cached) {
    i0 = index(first);
    i1 = index(first + 1);
  }

  // Q: head l % 16, quarter l / 16 of the 512 columns, in k steps of 8.  A lane's own 16 bytes of 16 rows would be 64
  // requests a load, so whole rows (of bf16, Q's and the window's) go to LDS by direct loads, in the values' places.
  const int h = h0 + l16;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int head = wave * 4 + j;
    lds_dma16_off(a.q + r * a.q_rstride + (long)min(h0 + head, a.H - 1) * DQK, (lane ^ v_swizzle(head)) << 4, v_base + head * 1024);
  }
  uint4 q[16 + TS];
  const uint16_t* const qrow = a.q + r * a.q_rstride + (long)min(h, a.H - 1) * DQK;
#pragma unroll
  for (int k = 0; k < TS; ++k) q[16 + k] = *(const uint4*)(qrow + 512 + 16 * g + 8 * k);
  uint4 code[4];
  uint2 sc, tail;
  uint32_t tsc = 0;
  auto load = [&](row_t row) {
    row_t p = row ? row : none;
#pragma unroll
    for (int k = 0; k < 4; ++k) code[k] = get16(p + 64 * g + 16 * k);
    sc = get8(p + 256 + 8 * g);
    if (TS) {
      tail = get8(p + 288 + 8 * g);
      tsc = p[320 + g];
    }
  };
  row_t row = nullptr;
  int p1 = -1, i2 = -1;
  if (cached) {
    row = source(first, i0, page(i0));
    load(row);
    // (a tile ahead of its rows the page, two ahead the index, asked for behind the rows' loads: nothing waits for them)
    p1 = page(i1);
    i2 = index(first + 2);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  lds_barrier();
#pragma unroll
  for (int k = 0; k < 16; ++k)
    q[k] = __builtin_bit_cast(uint4, *(__attribute__((address_space(3))) u32x4*)(
                                         (v_base + l16 * 1024 + 256 * g + (v_swizzle(l16) << 4)) ^ k << 4));
  f32x4_t o[8];
  float m = -__builtin_inff(), l = 0.0f, cq = a.scale;
#pragma unroll
  for (int c = 0; c < 8; ++c) o[c] = f32x4_t{0, 0, 0, 0};

  const uint32_t p_put = p_base + l16 * 128 + (((wave * 2 + (g >> 1)) ^ (l16 & 7)) << 4) + (g & 1) * 8;

  // the softmax of a tile's scores and the product with its values in LDS
  auto attend = [&](f32x4_t& s, bool valid, auto f16) {
    constexpr bool F16 = decltype(f16)::value;
    constexpr float kUnder = F16 ? kLow : 0.0f;  // what the reference is under the maximum that it was taken from
    const uint32_t mask = (uint32_t)(__ballot(valid) & 0xffffu) >> (4 * g);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = (mask >> i & 1) ? s[i] * cq : -__builtin_inff();
    float mx = row_max4(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
    if (g == 0) *(__attribute__((address_space(3))) float*)(m_base + (l16 * 4 + wave) * 4) = mx;
    // the probabilities by the reference as it stands; where the tile then turns out to move it, once more
    float p[4];
    auto probabilities = [&]() {
      const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
      for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(s[i] - ref);
      const uint2 pk = F16 ? make_uint2(pack_f16(p[0], p[1]), pack_f16(p[2], p[3]))
                           : make_uint2(pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3]));
      *(__attribute__((address_space(3))) uint64_t*)p_put = (uint64_t)pk.y << 32 | pk.x;
    };
    probabilities();
    lds_barrier();
    const f32x4_t w = *(__attribute__((address_space(3))) f32x4_t*)(m_base + l16 * 16);
    mx = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
    if (__any(mx > m + (8.0f + kUnder))) {  // (alike in every wave: all have the same maxima)
      const float to = fmaxf(m, mx - kUnder);
      const float f = to > m ? __builtin_amdgcn_exp2f(m - to) : 1.0f;
      m = to;
      l *= f;
#pragma unroll
      for (int c = 0; c < 8; ++c) o[c] *= f;
      probabilities();
      lds_barrier();
    }
    l += (p[0] + p[1]) + (p[2] + p[3]);
    uint32_t va = v_get;
    asm volatile("" : "+v"(va));  // (addresses computed anew: as the loops' invariants they would fill the registers)
    auto values = [&](int i) {  // of column block i % 8, keys 32 (i / 8) ..
      const int c = i % 8, at = i / 8 * 32768;
      const uint2 lo = lds_read_tr((va ^ ((2 * c) << 4)) + at), hi = lds_read_tr((va ^ ((2 * c + 1) << 4)) + 4096 + at);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    // (reads five products ahead, pinned: the compiler kept one or two in flight, and more than 15 wait for one another)
    constexpr int kAhead = 4;
    uint4 pb[2], v[16];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
      pb[kk] = __builtin_bit_cast(
          uint4, *(__attribute__((address_space(3))) u32x4*)(p_base + l16 * 128 + (((kk * 4 + g) ^ (l16 & 7)) << 4)));
#pragma unroll
    for (int i = 0; i < kAhead; ++i) v[i] = values(i);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (i + kAhead < 16) v[i + kAhead] = values(i + kAhead);
      o[i % 8] = F16 ? mfma_f16_16x16x32(v[i], pb[i / 8], o[i % 8]) : mfma_bf16_16x16x32(v[i], pb[i / 8], o[i % 8]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto put_v = [&](uint32_t to, int k, uint4 x) {
    *(__attribute__((address_space(3))) u32x4*)(to ^ k << 4) = __builtin_bit_cast(u32x4, x);
  };

  // ---- window rows
#pragma unroll 1
  for (; t < wend; ++t) {
    const row_t wrow = window(t, w0);
    const bool valid = wrow != nullptr;
    const uint64_t src = (uint64_t)(valid ? wrow : none);
    lds_barrier();  // (the last tile's values have been read)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint64_t p = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(src >> 32), j) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)src, j);
      lds_dma16_lane((const void*)p, (lane ^ v_swizzle(j)) << 4, v_base + (wave * 16 + j) * 1024);
    }
    uint4 x[16 + TS];
#pragma unroll
    for (int k = 0; k < TS; ++k) x[16 + k] = get16((row_t)src + 1024 + 32 * g + 16 * k);
    w0 = w1;
    w1 = listed(t + 2);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a wave reads its own keys' rows)
    auto part = [&](int k) { x[k] = __builtin_bit_cast(uint4, *(__attribute__((address_space(3))) u32x4*)(v_put ^ k << 4)); };
    f32x4_t s = {0, 0, 0, 0}, s2 = s;
    constexpr int kAhead = 6;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) part(k);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int k = 0; k < 16 + TS; ++k) {
      if (k + kAhead < 16) part(k + kAhead);
      if (k & 1)
        s2 = mfma_bf16_16x16x32(x[k], q[k], s2);
      else
        s = mfma_bf16_16x16x32(x[k], q[k], s);
      __builtin_amdgcn_sched_barrier(0);
    }
    s += s2;
    attend(s, valid, std::false_type{});
  }

  // ---- rows of the cache
  if (cached) {
    // Q to fp16: each head scaled by the power of two that brings its largest value to 2^14 or more, so that heads far under
    // fp16's normal numbers keep their bits; the scores are multiplied by its inverse
    typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
    u16x2_t top2{0, 0};
#pragma unroll
    for (int k = 0; k < 16 + TS; ++k) {
      const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
#pragma unroll
      for (int i = 0; i < 4; ++i)
        top2 = __builtin_elementwise_max(top2, __builtin_bit_cast(u16x2_t, w[i] & 0x7fff7fffu));
    }
    const uint32_t most = max((int)top2[0], (int)top2[1]);  // (a NaN's bits are above an infinity's; both are scaled)
    const float top = row_max4(__uint_as_float(min(most, 0x7f80u) << 16));
    // (an infinity leaves zeros and infinities: its head's result is NaN; 2^126 at most: subnormal bf16 is then exact)
    const int e = max(min(((__float_as_int(top) >> 23) & 255) - 127, 127) - 14, -126);
    const float down = pow2i(-e);
    cq *= pow2i(e);
    m -= kLow;  // (the window's reference is its maximum)
    l *= pow2i((int)kLow);
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] *= pow2i((int)kLow);
#pragma unroll
    for (int k = 0; k < 16 + TS; ++k) {
      const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
      uint32_t f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f[i] = pack_f16(__uint_as_float(w[i] << 16) * down, __uint_as_float(w[i] & 0xffff0000u) * down);
      q[k] = make_uint4(f[0], f[1], f[2], f[3]);
    }
#pragma unroll 1
    for (; t < t1; ++t) {
      const h16x2_t s01 = kv4_scales<false>(sc.x), s23 = kv4_scales<true>(sc.x);
      const h16x2_t s45 = kv4_scales<false>(sc.y), s67 = kv4_scales<true>(sc.y);
      const _Float16 sv[9] = {s01[0], s01[1], s23[0], s23[1], s45[0], s45[1], s67[0], s67[1], kv4_scales<false>(tsc)[0]};
      f32x4_t s = {0, 0, 0, 0};
      lds_barrier();
      uint32_t to = v_put;
      asm volatile("" : "+v"(to));
#pragma unroll
      for (int k = 0; k < 16 + TS; ++k) {
        const uint32_t w[4] = {code[(k / 4) % 4].x, code[(k / 4) % 4].y, code[(k / 4) % 4].z, code[(k / 4) % 4].w};
        const uint4 x = kv4_values(k < 16 ? w[k % 4] : (k == 16 ? tail.x : tail.y), sv[k / 2]);
        if (k < 16) put_v(to, k, x);
        s = mfma_f16_16x16x32(x, q[k], s);
      }
      const bool valid = row != nullptr;
      row = source(t + 1, i1, p1);
      load(row);
      // (moved here: the compiler's move at the loop's end, of the value then on its way, would wait for it)
      asm volatile("v_mov_b32 %0, %1" : "=&v"(i1) : "v"(i2));
      p1 = page(i1);
      i2 = index(t + 3);
      attend(s, valid, std::true_type{});
    }
  }

  // ---- sums of the waves' keys, output
  lds_barrier();
  l = row_sum4(l);
  if (g == 0) *(__attribute__((address_space(3))) float*)(m_base + (l16 * 4 + wave) * 4) = l;
  lds_barrier();
  const f32x4_t w = *(__attribute__((address_space(3))) f32x4_t*)(m_base + l16 * 16);
  l = (w[0] + w[1]) + (w[2] + w[3]);
  if (h >= a.H) return;
  if (a.nsplit > 1) {
    const long at = ((long)r * a.H + h) * a.nsplit + sp;
    if (wave == 0 && g == 0) *(float2*)(a.part + 512L * a.R * a.H * a.nsplit + 2 * at) = make_float2(m, l);
    float* dst = a.part + at * 512 + wave * 128 + 4 * g;
#pragma unroll
    for (int c = 0; c < 8; ++c) *(float4*)(dst + 16 * c) = make_float4(o[c][0], o[c][1], o[c][2], o[c][3]);
  } else {
    const float den = l + exp2f(a.sink[h] * kLog2e - m);
    const float inv = m == -__builtin_inff() ? 0.0f : 1.0f / den;  // (no key: zeros)
    uint16_t* dst = a.out + ((long)r * a.H + h) * 512 + wave * 128 + 4 * g;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      *(uint2*)(dst + 16 * c) = finish4(a, pos, wave * 128 + 16 * c + 4 * g,
                                        make_float4(o[c][0] * inv, o[c][1] * inv, o[c][2] * inv, o[c][3] * inv));
  }
}

// The splits of a (row, head), in order: one workgroup of 128 lanes, four columns each.
__global__ void __launch_bounds__(128) kv4_combine_kernel(const Kv4AttnArgs a) {
  const int r = blockIdx.x / a.H, h = blockIdx.x % a.H;
  const long at = ((long)r * a.H + h) * a.nsplit;
  const float* ml = a.part + 512L * a.R * a.H * a.nsplit + 2 * at;
  const float* src = a.part + at * 512 + 4 * threadIdx.x;
  float4 v[12];  // (twelve splits' loads in flight, the first before their maxima are known; the sums go in order)
  float2 st[12];
  auto load = [&](int s0) {
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      const int s = min(s0 + i, a.nsplit - 1);
      st[i] = *(const float2*)(ml + 2 * s);
      v[i] = *(const float4*)(src + 512L * s);
    }
  };
  load(0);
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < 12; ++i) m = fmaxf(m, st[i].x);
#pragma unroll 8
  for (int s = 12; s < a.nsplit; ++s) m = fmaxf(m, ml[2 * s]);
  const float ref = m == -__builtin_inff() ? 0.0f : m;  // (no key: zeros, but a NaN stays one)
  float den = exp2f(a.sink[h] * kLog2e - ref);
  float4 o = make_float4(0, 0, 0, 0);
  for (int s0 = 0;;) {
#pragma unroll
    for (int i = 0; i < 12; ++i) {
      if (s0 + i < a.nsplit) {
        const float w = exp2f(st[i].x - ref);
        den += w * st[i].y;
        o = make_float4(o.x + w * v[i].x, o.y + w * v[i].y, o.z + w * v[i].z, o.w + w * v[i].w);
      }
    }
    if ((s0 += 12) >= a.nsplit) break;
    load(s0);
  }
  const float inv = m == -__builtin_inff() ? 0.0f : 1.0f / den;
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  *(uint2*)(a.out + ((long)r * a.H + h) * 512 + 4 * threadIdx.x) =
      finish4(a, a.pos ? a.pos[r] : 0, 4 * threadIdx.x, o);
}

constexpr int kMost = 0x7fffffff - 4096;  // entries of a list, which are counted on past its end in 32 bits

struct Plan {
  bool many;  // the cache's rows decoded first
  int wtiles, tiles, nsplit, chunk, groups;
  long list, rows, part;  // bytes of the workspace
};

Plan plan_of(int R, int H, int wt, int t, int dim, long rows) {
  Plan p{};
  // Decoding first, then the bf16 kernel of 64 heads a workgroup, pays with more than half of them (512 query rows of 2048
  // keys: 64 heads 183 us for 303, 33 heads 180 for 229, 32 heads 180 for 158), from 2^18 keys of 16 heads each on (602
  // query rows of 512 keys: 64 heads 99 us for 118, 48 and 33 heads 96 for 94; 150 rows, 64 heads 37.3 for 41.6, 33 heads 35.7
  // for 27.8; 32 rows of 2048 39.6 for 40.6, 16 of them 36.7 for 27.5) and with each row of the cache listed four times.
  // (rows: what the tables have room for, whether or not pages are there: how many are is known on the device alone.)
  // (From 16 query rows on the bf16 kernel joins its splits by a kernel of its own; its grid ends at 65535.)
  p.groups = (H + 15) / 16;
  p.many = rows > 0 && H > 32 && R >= 16 && R <= 65528 && (long)R * t * p.groups >= 1L << 18 && (long)R * t >= 4 * rows &&
           (long)wt + t <= kMost;
  if (p.many) {
    p.list = ((long)R * (wt + t) * 4 + 255) & ~255L;
    p.rows = (rows * dim * 2 + 255) & ~255L;
    p.part = dsv41_attn_workspace_bytes(R, H, wt + t, 512, 0);
    return p;
  }
  p.wtiles = (wt + 63) / 64;
  p.tiles = p.wtiles + (t + 63) / 64;
  if (p.tiles == 0) p.tiles = 1;  // (no key at all: zeros)
  // Splits until each of the card's CUs has a workgroup, two where one would have more than 12 tiles: before, two cost more
  // in partial results than they hide (64 heads, 34 tiles: 4 sequences 17.3 us and 20.0, 16 27.1 and 29.0, 32 41.8 and 37.9).
  // Of more than 16 tiles no split has a single one (1 sequence 14.7 us for 16.2; 10 tiles 11.7 for 10.8).
  const long units = (long)R * p.groups, most = p.tiles > 16 ? (p.tiles + 1) / 2 : p.tiles;
  long ns = (256 + units - 1) / units;
  if (p.tiles > 12 * ns) ns = (512 + units - 1) / units;
  if (ns > most) ns = most;
  p.chunk = (int)((p.tiles + ns - 1) / ns);
  p.nsplit = (p.tiles + p.chunk - 1) / p.chunk;
  p.part = p.nsplit > 1 ? 4L * R * H * p.nsplit * 514 : 0;
  return p;
}

// Batch rows b of a prompt, 0: single tokens.
int run(Kv4AttnArgs& a, int dqk, int b, float scale, void* ws, long ws_bytes, hipStream_t st) {
  const long rows = b > 0 ? (long)b * a.map.cols << a.map.shift : 0;
  const Plan p = plan_of(a.R, a.H, a.pos ? a.win_rows : a.wt, a.t, dqk, rows);
  const long need = p.list + p.rows + p.part;
  if (need > 0 && (!ws || ((uintptr_t)ws & 15) || ws_bytes < need)) return (int)hipErrorInvalidValue;
  void* const part = (char*)ws + p.list + p.rows;
  if (p.many) {
    const long l = (long)a.wt + a.t, n = rows / b, pages = rows >> a.map.shift;
    if (a.win_rows + n >= (1L << 31) || !kv4_grid_ok(pages + a.R)) return (int)hipErrorInvalidValue;
    int* const list = (int*)ws;
    void* const table = (char*)ws + p.list;
    kv4_unpack_launch(a, dqk, b, table, list, st);
    DSV41_CHECK_LAUNCH();
    if (a.win_rows > 0)
      return dsv41_sparse_attn_kv2(a.q, a.win, table, a.sink, list, a.out, b, a.rows_per_slot, a.H, dqk, 512, a.win_rows,
                                   a.win_sstride, (int)n, n * dqk, (int)l, l, scale, 0, part, p.part, st);
    return dsv41_sparse_attn(a.q, table, a.sink, list, a.out, b, a.rows_per_slot, a.H, dqk, 512, (int)n, n * dqk, (int)l,
                             scale, 0, part, p.part, st);
  }
  a.scale = scale * kLog2e;
  a.wtiles = p.wtiles;
  a.tiles = p.tiles;
  a.nsplit = p.nsplit;
  a.chunk = p.chunk;
  a.groups = p.groups;
  a.part = (float*)part;
  if (!kv4_grid_ok((long)a.R * a.groups * a.nsplit) || (p.nsplit > 1 && !kv4_grid_ok((long)a.R * a.H))) return (int)hipErrorInvalidValue;
  const unsigned grid = (unsigned)((long)a.R * a.groups * a.nsplit);
  if (dqk == 512)
    kv4_attn_kernel<512><<<grid, 256, 0, st>>>(a);
  else
    kv4_attn_kernel<576><<<grid, 256, 0, st>>>(a);
  DSV41_CHECK_LAUNCH();
  if (a.nsplit > 1) {
    kv4_combine_kernel<<<a.R * a.H, 128, 0, st>>>(a);
    DSV41_CHECK_LAUNCH();
  }
  return 0;
}

bool attn_ok(const Kv4AttnArgs& a, const dsv41_kv4* c) {
  return kv4_ok(c) && a.q && a.H > 0 && a.sink && a.out && a.t >= 0 && a.t <= kMost && a.wt <= kMost && a.win_rows <= kMost &&
         (a.t == 0 || a.idx) &&
         (((uintptr_t)a.q | (uintptr_t)a.win | (uintptr_t)a.out) & 15) == 0 && a.win_sstride % 8 == 0;
}

}  // namespace

extern "C" {

long dsv41_kv4_attn_workspace_bytes(const dsv41_kv4* c, int R, int H, int wt, int t, int b) {
  if (R <= 0 || H <= 0 || wt < 0 || t < 0 || wt > kMost || t > kMost) return 0;
  const Plan p = plan_of(R, H, wt, t, c->dim, (long)b * c->cols * c->page);
  return p.list + p.rows + p.part;
}

int dsv41_sattn4(const dsv41_kv4* c, const void* q, const void* kv_win, long win_sstride, int win_slots, int win,
                 const int* idx, int t, const long* pos, const long* seq, const long* pmax, const long* plim,
                 const float* sink, const float* cos_t, const float* sin_t, long n_pos, int rd, float scale, void* out,
                 int B, int h, void* ws, long ws_bytes, void* stream) {
  if (B <= 0) return B < 0 ? (int)hipErrorInvalidValue : 0;
  Kv4AttnArgs a{};
  a.q = (const uint16_t*)q;
  a.R = B;
  a.H = h;
  a.win = (const uint16_t*)kv_win;
  a.win_sstride = win_sstride;
  a.win_rows = win;
  a.win_slots = win_slots;
  a.idx = idx;
  a.t = t;
  a.rows_per_slot = 1;
  a.seq = seq;
  a.pos = pos;
  a.pmax = pmax;
  a.plim = plim;
  a.sink = sink;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.n_pos = n_pos;
  a.rd = rd;
  a.out = (uint16_t*)out;
  if (!attn_ok(a, c) || !kv_win || win <= 0 || !pos || !seq || !pmax || rd < 0 || rd > 512 || rd % 4 ||
      (rd > 0 && (!cos_t || !sin_t)))
    return (int)hipErrorInvalidValue;
  a.q_rstride = (long)h * c->dim;
  a.pool = (const uint8_t*)c->pool;
  a.map = kv4_map(*c);
  return run(a, c->dim, 0, scale, ws, ws_bytes, (hipStream_t)stream);
}

int dsv41_sparse_attn4(const dsv41_kv4* c, const void* q, const void* kv, long kv_bstride, int n_kv, const int* widx,
                       int wt, const int* idx, int t, const long* seq, const float* sink, float scale, void* out, int b,
                       int s, int h, void* ws, long ws_bytes, void* stream) {
  if (b <= 0 || s <= 0) return b < 0 || s < 0 ? (int)hipErrorInvalidValue : 0;
  if ((long)b * s >= (1L << 31)) return (int)hipErrorInvalidValue;
  Kv4AttnArgs a{};
  a.q = (const uint16_t*)q;
  a.R = b * s;
  a.H = h;
  a.win = (const uint16_t*)kv;
  a.win_sstride = kv_bstride;
  a.win_rows = n_kv;
  a.widx = widx;
  a.wt = wt;
  a.idx = idx;
  a.t = t;
  a.rows_per_slot = s;
  a.seq = seq;
  a.sink = sink;
  a.out = (uint16_t*)out;
  if (!attn_ok(a, c) || wt < 0 || n_kv < 0 || (wt > 0 && (!kv || !widx))) return (int)hipErrorInvalidValue;
  a.q_rstride = (long)h * c->dim;
  a.pool = (const uint8_t*)c->pool;
  a.map = kv4_map(*c);
  return run(a, c->dim, b, scale, ws, ws_bytes, (hipStream_t)stream);
}

}  // extern "C"
