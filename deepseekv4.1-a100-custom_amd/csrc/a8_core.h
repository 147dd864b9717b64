// Shared pieces of the 8-bit activation operators (a8_norm.hip, a8_gemm.hip): the block quantisation and the epilogue.
//
// An activation in 8 bits ("A8", the twin of the W8 weights) is, per row and 32 values v,
//   s = 2^ceil(log2(max(amax, 1e-4) / 448)),  q = e4m3(v / s)  (nearest, ties to even),
// the grid of fake_quant_fp8 (dsv41/quant.py:45-72) held as bytes.  Codes are [rows, K], every 16 of a row in the weights'
// byte order (position p holds k = kPermK[p], dsv41/w8.py:23), so that a product pairs them with no move; scales are E8M0
// bytes [ceil(K / 128)][rows][4] (blocks 4 c .. 4 c + 3 of a row in one 32-bit word: what the matrix kernels load of a
// row for 128 k, rows adjacent), 127 where K ends inside a word.  A block with an infinity or a NaN has scale 255, the
// NaN of E8M0, and NaN codes.
#pragma once
#include "common.h"

namespace {

// ---- block quantisation
// The E8M0 byte of a block whose largest |v| has the bits `top` (an fp32 as a signed integer: NaN > Inf > finite).
// a / 448 <= 2^e  <=>  a <= 1.75 * 2^(e + 8), so the exponent comes from the bits alone.
DSV41_DEV int a8_scale(int top) {
  if (top >= 0x7f800000) return 255;
  top = max(top, __float_as_int(1e-4f));
  return (top >> 23) - 8 + ((top & 0x7fffff) > 0x600000 ? 1 : 0);
}
// The reciprocal of such a scale, a power of two: 105 <= byte <= 247 (255: unused).
DSV41_DEV float a8_inv(int byte) { return __int_as_float((254 - min(byte, 253)) << 23); }
DSV41_DEV int a8_abs_bits(float v) { return __float_as_int(v) & 0x7fffffff; }
// Four values to codes; |v * inv| <= 448 by the choice of the scale.  bad: the block is NaN.
DSV41_DEV uint32_t a8_pack4(float a, float b, float c, float d, float inv, bool bad) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * inv, b * inv, 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(c * inv, d * inv, w, true);
  return bad ? 0x7f7f7f7fu : (uint32_t)w;
}
template <int CTRL>
DSV41_DEV int dpp_movi(int v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, false);
}

typedef __bf16 a8_bf2_t __attribute__((ext_vector_type(2)));
DSV41_DEV uint32_t a8_bf16x2(float a, float b) {  // nearest, ties to even
  return __builtin_bit_cast(uint32_t, a8_bf2_t{(__bf16)a, (__bf16)b});
}

// ---- activations
constexpr int kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3, kActGeluTanh = 4;

// e^x: the argument's rounding makes it |x| 2^-24 off (5e-6 at the ends of the range), far below half a step of the
// outputs, bf16 and e4m3.
DSV41_DEV float a8_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// silu(v) = v / (1 + e^-v); gelu_tanh(v) = v / (1 + e^(-2 c (v + 0.044715 v^3))), c = sqrt(2 / pi): 1/2 (1 + tanh z) is
// 1 / (1 + e^-2z).  gelu(v) = v Phi(v), Phi(-a) = e^(-a^2 / 2) R(1 / (1 + 0.35 a)): R a polynomial of degree 7 fitted to
// erfcx(a / sqrt 2) / 2 over a <= 14 for the relative error (3.1e-7), so that the tail keeps its digits.
template <int act>
DSV41_DEV float a8_act(float v) {
  if (act == kActRelu) return v < 0.0f ? 0.0f : v;  // (NaN stays)
  if (act == kActSilu || act == kActGeluTanh) {
    const float z = act == kActSilu ? v : v * __builtin_fmaf(0.07135481283f, v * v, 1.595769122f);
    return v * __builtin_amdgcn_rcpf(1.0f + a8_exp(-z));
  }
  if (act == kActGelu) {
    const float a = fabsf(v), t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f));
    float r = 0.04894096404f;
    r = __builtin_fmaf(r, t, -0.2021136582f);
    r = __builtin_fmaf(r, t, 0.2406320274f);
    r = __builtin_fmaf(r, t, -0.01701612398f);
    r = __builtin_fmaf(r, t, 0.1559579968f);
    r = __builtin_fmaf(r, t, 0.1333560497f);
    r = __builtin_fmaf(r, t, 0.1402702034f);
    r = __builtin_fmaf(r, t, -2.730727283e-5f);
    r *= a8_exp(-0.5f * a * a);
    return v * (v < 0.0f ? r : 1.0f - r);
  }
  return v;
}

// ---- epilogue: y = act(sum + bias) + residual, or act(min(gate, limit)) * clamp(up, -limit, limit)
// A lane has 8 adjacent columns of a row, n % 8 == 0: 16 bytes of bf16, 8 of codes, a quarter of a block.
struct A8Epi {
  const void* bias;  // [N] or null
  int bias_f32;
  const uint16_t* res;  // bf16 [M, N] or null
  int act;
  float limit;        // gated products: > 0 clamps
  uint16_t* out;      // bf16 [M, N], or null:
  uint8_t *oa8, *os8; // codes [M, N] and scales
  int M, N;
  int vec;            // rows of out and res in whole 16-byte units
};
struct alignas(16) A8x8 {
  float v[8];
};

DSV41_DEV void a8_unpack8(uint4 q, float (&v)[8]) {
  const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(u[i] << 16);
    v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
  }
}
DSV41_DEV uint4 a8_pack8(const float (&v)[8]) {
  return make_uint4(a8_bf16x2(v[0], v[1]), a8_bf16x2(v[2], v[3]), a8_bf16x2(v[4], v[5]), a8_bf16x2(v[6], v[7]));
}
// Columns n .. n + 7 of the bias, 0 behind the last and without one.
DSV41_DEV A8x8 a8_bias8(const A8Epi& e, int n) {
  A8x8 b;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    b.v[i] = !e.bias || n + i >= e.N ? 0.0f : e.bias_f32 ? ((const float*)e.bias)[n + i] : bf2f(((const uint16_t*)e.bias)[n + i]);
  return b;
}
// The residual's columns n .. n + 7 of row m, as loaded (a conversion here would wait for it).
DSV41_DEV uint4 a8_res8(const A8Epi& e, int m, int n) {
  uint4 q = make_uint4(0, 0, 0, 0);
  if (!e.res || m >= e.M || n >= e.N) return q;
  const uint16_t* r = e.res + (long)m * e.N + n;
  if (e.vec) return *(const uint4*)r;
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (n + i < e.N) u[i >> 1] |= (uint32_t)r[i] << (16 * (i & 1));
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <int ACT>
DSV41_DEV void a8_act8(A8x8& y) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y.v[i] = a8_act<ACT>(y.v[i]);
}
// (one branch for the 8 of them)
DSV41_DEV void a8_act8(A8x8& y, int act) {
  if (act == kActSilu) a8_act8<kActSilu>(y);
  else if (act == kActRelu) a8_act8<kActRelu>(y);
  else if (act == kActGelu) a8_act8<kActGelu>(y);
  else if (act == kActGeluTanh) a8_act8<kActGeluTanh>(y);
}
DSV41_DEV void a8_linear8(const A8Epi& e, A8x8& y, const A8x8& bias, uint4 res) {
#pragma unroll
  for (int i = 0; i < 8; ++i) y.v[i] += bias.v[i];
  a8_act8(y, e.act);
  if (e.res) {
    float r[8];
    a8_unpack8(res, r);
#pragma unroll
    for (int i = 0; i < 8; ++i) y.v[i] += r[i];
  }
}
DSV41_DEV void a8_gated8(const A8Epi& e, A8x8& g, A8x8& u) {
  if (e.limit > 0.0f) {  // (comparisons, not fminf: a NaN stays)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g.v[i] = g.v[i] > e.limit ? e.limit : g.v[i];
      u.v[i] = u.v[i] > e.limit ? e.limit : u.v[i] < -e.limit ? -e.limit : u.v[i];
    }
  }
  a8_act8(g, e.act);
#pragma unroll
  for (int i = 0; i < 8; ++i) g.v[i] *= u.v[i];
}

DSV41_DEV long a8_scale_at(int M, int m, int block) { return ((long)(block >> 2) * M + m) * 4 + (block & 3); }
// The bytes behind the last block of a row whose K ends inside a scale word: 127, written with the last block's.
DSV41_DEV void a8_store_scale(const A8Epi& e, int m, int block, int byte) {
  uint8_t* s = e.os8 + a8_scale_at(e.M, m, block);
  *s = (uint8_t)byte;
  if (block == e.N / 32 - 1)
    for (int b = (block & 3) + 1; b < 4; ++b) *++s = 127;
}

// The codes of a lane's 8 of 16 values in the byte order's words {0 1 8 9} {2 3 10 11} {4 5 12 13} {6 7 14 15}: the even
// lane has 0..7 and gets the first two words, the odd one 8..15 and the last two; one exchange with the neighbour.
DSV41_DEV uint2 a8_words(uint32_t lo, uint32_t hi, bool odd) {
  const uint32_t got = (uint32_t)dpp_movi<0xB1>((int)(odd ? lo : hi));
  const uint32_t p = odd ? got : lo, q = odd ? hi : got;
  return make_uint2((p & 0xffffu) | (q << 16), (p >> 16) | (q & 0xffff0000u));
}
// Codes and scale byte of 8 of a block's 32 values, the block in 4 adjacent lanes (all of them must call it).
DSV41_DEV uint2 a8_quant8(const float (&v)[8], bool odd, int* scale) {
  float top = 0.0f;  // (the maximum that keeps a NaN)
#pragma unroll
  for (int i = 0; i < 8; ++i) top = __builtin_elementwise_maximum(top, fabsf(v[i]));
  int t = __float_as_int(top) & 0x7fffffff;
  t = max(t, dpp_movi<0xB1>(t));
  t = max(t, dpp_movi<0x4E>(t));
  const int s = a8_scale(t);
  const float inv = a8_inv(s);
  *scale = s;
  return a8_words(a8_pack4(v[0], v[1], v[2], v[3], inv, s == 255), a8_pack4(v[4], v[5], v[6], v[7], inv, s == 255), odd);
}

// A lane's 8 columns n .. n + 7 of row m to the output.  Every lane of a wave calls it; live: m < M and n < N.
DSV41_DEV void a8_store8(const A8Epi& e, const A8x8& y, int m, int n, bool live) {
  if (e.out) {
    if (!live) return;
    uint16_t* o = e.out + (long)m * e.N + n;
    const uint4 q = a8_pack8(y.v);
    if (e.vec) {
      *(uint4*)o = q;
    } else {
      const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < e.N) o[i] = (uint16_t)(u[i >> 1] >> (16 * (i & 1)));
    }
    return;
  }
  int s;
  const uint2 w = a8_quant8(y.v, (n >> 3) & 1, &s);
  if (!live) return;
  *(uint2*)(e.oa8 + (long)m * e.N + n) = w;
  if ((n & 31) == 0) a8_store_scale(e, m, n >> 5, s);
}

}  // namespace
