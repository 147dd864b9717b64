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

// exp(x) to about 2 ulp: 2^(x log2 e) with the product's rounding error carried into the result.
DSV41_DEV float a8_exp(float x) {
  const float t = x * kLog2e;
  const float lo = __builtin_fmaf(x, kLog2e, -t) + x * 1.925963033e-8f;  // (log2 e = kLog2e + 1.92596e-8)
  const float e = __builtin_amdgcn_exp2f(t);
  return fabsf(t) < 126.0f ? __builtin_fmaf(e, lo * 0.6931471806f, e) : e;  // (beyond: e is or nears 0 or infinity)
}
// silu(v) = v / (1 + e^-v); gelu_tanh(v) = v / (1 + e^(-2 c (v + 0.044715 v^3))), c = sqrt(2 / pi): 1/2 (1 + tanh z) is
// 1 / (1 + e^-2z).  gelu(v) = v Phi(v), Phi(-a) = e^(-a^2 / 2) R(1 / (1 + 0.35 a)): R a polynomial of degree 7 fitted to
// erfcx(a / sqrt 2) / 2 over a <= 14 for the relative error (3.1e-7), so that the tail keeps its digits.
DSV41_DEV float a8_act(float v, int act) {
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
struct A8Epi {
  const void* bias;  // [N] or null
  int bias_f32;
  const uint16_t* res;  // bf16 [M, N] or null
  int act;
  float limit;        // gated products: > 0 clamps
  uint16_t* out;      // bf16 [M, N], or null:
  uint8_t *oa8, *os8; // codes [M, N] and scales
  int M, N;
  int vec;            // N % 4 == 0, out / res 8-byte aligned, fp32 bias 16-byte
};

DSV41_DEV float a8_gate(const A8Epi& e, float g, float u) {
  if (e.limit > 0.0f) {  // (comparisons, not fminf: a NaN stays)
    g = g > e.limit ? e.limit : g;
    u = u > e.limit ? e.limit : u < -e.limit ? -e.limit : u;
  }
  return a8_act(g, e.act) * u;
}

// Columns n .. n + 3 of row m (m < M), bias, activation and residual applied.
template <bool GATED>
DSV41_DEV f32x4_t a8_finish4(const A8Epi& e, f32x4_t v, f32x4_t u, int m, int n) {
  if constexpr (GATED) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a8_gate(e, v[i], u[i]);
    return v;
  }
  const bool whole = e.vec && n < e.N;
  if (e.bias) {
    if (whole && e.bias_f32) {
      v += *(const f32x4_t*)((const float*)e.bias + n);
    } else if (whole) {
      const uint2 b = *(const uint2*)((const uint16_t*)e.bias + n);
      v += f32x4_t{__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                   __uint_as_float(b.y & 0xffff0000u)};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < e.N) v[i] += e.bias_f32 ? ((const float*)e.bias)[n + i] : bf2f(((const uint16_t*)e.bias)[n + i]);
    }
  }
  if (e.act != kActNone) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a8_act(v[i], e.act);
  }
  if (e.res) {
    const uint16_t* r = e.res + (long)m * e.N + n;
    if (whole) {
      const uint2 b = *(const uint2*)r;
      v += f32x4_t{__uint_as_float(b.x << 16), __uint_as_float(b.x & 0xffff0000u), __uint_as_float(b.y << 16),
                   __uint_as_float(b.y & 0xffff0000u)};
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (n + i < e.N) v[i] += bf2f(r[i]);
    }
  }
  return v;
}

DSV41_DEV void a8_store4(const A8Epi& e, f32x4_t v, int m, int n) {
  uint16_t* o = e.out + (long)m * e.N + n;
  if (e.vec && n < e.N) {
    *(uint2*)o = make_uint2(a8_bf16x2(v[0], v[1]), a8_bf16x2(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < e.N) o[i] = (uint16_t)a8_bf16x2(v[i], 0.0f);
  }
}

DSV41_DEV long a8_scale_at(int M, int m, int block) { return ((long)(block >> 2) * M + m) * 4 + (block & 3); }
// The bytes behind the last block of a row whose K ends inside a scale word: 127, written with the last block's.
DSV41_DEV void a8_store_scale(const A8Epi& e, int m, int block, int byte) {
  uint8_t* s = e.os8 + a8_scale_at(e.M, m, block);
  *s = (uint8_t)byte;
  if (block == e.N / 32 - 1)
    for (int b = (block & 3) + 1; b < 4; ++b) *++s = 127;
}

// Codes and scale of a block of 32 columns held by 8 adjacent lanes (lane a: columns 4 a .. 4 a + 3 from n).  Every lane
// of the group must call it; valid is the group's.  In the byte order a lane's first two codes and those of the lane two
// on are one word, its last two and theirs another: lane a of four writes word 2 (a & 1) + (a >> 1).
DSV41_DEV void a8_store_block8(const A8Epi& e, f32x4_t v, int m, int n, bool valid) {
  int top = max(max(a8_abs_bits(v[0]), a8_abs_bits(v[1])), max(a8_abs_bits(v[2]), a8_abs_bits(v[3])));
  top = max(top, dpp_movi<0xB1>(top));
  top = max(top, dpp_movi<0x4E>(top));
  top = max(top, dpp_movi<0x141>(top));
  const int s = a8_scale(top);
  const uint32_t c = a8_pack4(v[0], v[1], v[2], v[3], a8_inv(s), s == 255);
  const uint32_t p = (uint32_t)dpp_movi<0x4E>((int)c);  // lane a ^ 2
  const int a = (n >> 2) & 3;
  const uint32_t w = a < 2 ? (c & 0xffffu) | (p << 16) : (p >> 16) | (c & 0xffff0000u);
  if (!valid) return;
  *(uint32_t*)(e.oa8 + (long)m * e.N + (n & ~15) + 4 * (2 * (a & 1) + (a >> 1))) = w;
  if (((n >> 2) & 7) == 0) a8_store_scale(e, m, n >> 5, s);
}

}  // namespace
