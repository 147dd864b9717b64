// Rows of the paged 4-bit cache: written (rope, 4-bit grid, packed into the row's page) and read back as bf16.
//
// One wave a row: lane l holds values 8 l .. 8 l + 7 (one 16-byte load), so a group of 16 is a lane pair, the codes of
// a lane are one dword and a row's codes one 256-byte store; lanes 0-7 take the last 64 values of rows of 576 too.
#include "kv4_core.h"

namespace {

struct RowsArgs {
  const uint16_t* x;
  long x_rstride;
  const long* seq;
  const long* row;
  long n;
  int ratio;
  const float* cos_t;
  const float* sin_t;
  long n_pos;
  int rd;
  uint8_t* pool;
  Kv4Table map;
  const int* refs;
  int* err;
  uint16_t* out;
};

// The grid's scale of 16 values and the codes of this lane's eight.  bf16 values over a 4-bit significand often lie on a
// border of the grid, where the even code is right, so a quotient may not be off there.  Quotients are products with a
// reciprocal (two fp32 roundings) rounded to bf16: one that is a border comes out as the border, which has 3 bits (the
// scale's 5); any other is at least 2^-8 of itself away from one -- two integers of at most 8 bits that differ -- and bf16
// moves it by 2^-9.  The conversions round to even and saturate: the scale at 448, the codes at 6.  A group with an
// infinity or a NaN reads back as NaN (scale 0x7f).
DSV41_DEV uint32_t kv4_encode(const float* v, uint8_t* scale) {
  float a = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    a = fmaxf(a, fabsf(v[i]));
    bad |= !(fabsf(v[i]) < __builtin_inff());
  }
  a = group_max(bad ? __builtin_inff() : a, 2);
  const float t = round_bf16(fminf(fmaxf(a, 6.0f * 0.001953125f) * (1.0f / 6.0f), 448.0f));
  const int byte = __builtin_amdgcn_cvt_pk_fp8_f32(t, t, 0, false);
  const float inv = __builtin_amdgcn_rcpf(__builtin_amdgcn_cvt_f32_fp8(byte, 0));
  const bool nan = !(a < __builtin_inff());
  *scale = nan ? 0x7f : (uint8_t)byte;
  typedef __bf16 b16x2_t __attribute__((ext_vector_type(2)));
  uint32_t codes = 0;
#define DSV41_PAIR(i)                                                                                                  \
  codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(                                                                   \
      codes, b16x2_t{(__bf16)fmaf(v[2 * i], inv, 0.0f), (__bf16)fmaf(v[2 * i + 1], inv, 0.0f)}, 1.0f, i)
  DSV41_PAIR(0);  // (plus zero: -0 has the code of 0)
  DSV41_PAIR(1);
  DSV41_PAIR(2);
  DSV41_PAIR(3);
#undef DSV41_PAIR
  return nan ? 0 : codes;
}

// Eight values of a row from element e on: bf16, the last rd columns rotated.  The rotation's products are exact in 64
// bits, so the value before bf16's rounding is off by 2^-53 of its terms at most.
DSV41_DEV void kv4_load(const uint4 raw, int e, int dim, const RowsArgs& a, long pos, float* v) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = __uint_as_float(w[i] << 16);
    v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    const int at = e + 2 * i - (dim - a.rd);
    if (at >= 0) {
      const long j = pos * (a.rd / 2) + (at >> 1);
      const double c = a.cos_t[j], s = a.sin_t[j], p = v[2 * i], q = v[2 * i + 1];
      v[2 * i] = round_bf16((float)(p * c - q * s));
      v[2 * i + 1] = round_bf16((float)(p * s + q * c));
    }
  }
}

template <int DIM>
__global__ void __launch_bounds__(256) kv4_append_kernel(const RowsArgs a) {
  const long r = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (r >= a.n) return;
  const int lane = threadIdx.x & 63;
  const long seq = a.seq[r], row = a.row[r];
  if (row < 0) return;
  const uint16_t* x = a.x + r * a.x_rstride;
  const uint4 raw = *(const uint4*)(x + 8 * lane);
  const uint4 raw2 = DIM == 576 ? *(const uint4*)(x + 512 + 8 * (lane & 7)) : make_uint4(0, 0, 0, 0);
  const int p = kv4_page(a.map, seq, row);
  const long pos = row * a.ratio;
  if (p < 0 || a.refs[p] > 1 || (a.rd > 0 && pos >= a.n_pos)) {
    if (lane == 0) atomicOr(a.err, seq < 0 || seq >= a.map.slots ? kKv4Ignored : kKv4Dropped);
    return;
  }
  uint8_t* dst = a.pool + kv4_offset(a.map, p, row, kv4_row_bytes(DIM));
  float v[8];
  uint8_t scale;
  kv4_load(raw, 8 * lane, DIM, a, pos, v);
  const uint32_t codes = kv4_encode(v, &scale);
  ((uint32_t*)dst)[lane] = codes;
  if ((lane & 1) == 0) dst[256 + (lane >> 1)] = scale;
  if (DIM == 576) {
    kv4_load(raw2, 512 + 8 * (lane & 7), DIM, a, pos, v);
    const uint32_t tail = kv4_encode(v, &scale);
    if (lane < 8) {
      ((uint32_t*)dst)[72 + lane] = tail;
      if ((lane & 1) == 0) dst[320 + (lane >> 1)] = scale;
    } else if (lane < 11) {
      ((uint32_t*)dst)[73 + lane] = 0;
    }
  }
}

template <int DIM>
__global__ void __launch_bounds__(256) kv4_read_kernel(const RowsArgs a) {
  const long r = blockIdx.x * 4L + (threadIdx.x >> 6);
  if (r >= a.n) return;
  const int lane = threadIdx.x & 63;
  const long row = a.row[r];
  const int p = kv4_page(a.map, a.seq[r], row);
  uint16_t* out = a.out + r * DIM;
  uint4 v = make_uint4(0, 0, 0, 0), tail = v;
  if (p >= 0) {
    const uint8_t* src = a.pool + kv4_offset(a.map, p, row, kv4_row_bytes(DIM));
    v = kv4_bf16(((const uint32_t*)src)[lane], src[256 + (lane >> 1)]);
    if (DIM == 576) tail = kv4_bf16(((const uint32_t*)src)[72 + (lane & 7)], src[320 + ((lane & 7) >> 1)]);
  }
  *(uint4*)(out + 8 * lane) = v;
  if (DIM == 576 && lane < 8) *(uint4*)(out + 512 + 8 * lane) = tail;
}

void rows_args(RowsArgs& a, const dsv41_kv4& c, const long* seq, const long* row, long n) {
  a = RowsArgs{};
  a.seq = seq;
  a.row = row;
  a.n = n;
  a.pool = (uint8_t*)c.pool;
  a.map = kv4_map(c);
  a.refs = c.refs;
  a.err = c.err;
}

}  // namespace

extern "C" {

int dsv41_kv4_append(const dsv41_kv4* c, const void* x, long x_rstride, const long* seq, const long* row, long n,
                     int ratio, const float* cos_t, const float* sin_t, long n_pos, int rd, void* stream) {
  if (!kv4_ok(c) || n < 0 || n >= (1L << 32)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq || !row || !x || ((uintptr_t)x & 15) || x_rstride < c->dim || x_rstride % 8 || ratio < 1 || rd < 0 ||
      rd > c->dim || (rd & 1) || (rd > 0 && (!cos_t || !sin_t)))
    return (int)hipErrorInvalidValue;
  RowsArgs a;
  rows_args(a, *c, seq, row, n);
  a.x = (const uint16_t*)x;
  a.x_rstride = x_rstride;
  a.ratio = ratio;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.n_pos = n_pos;
  a.rd = rd;
  const unsigned grid = (unsigned)((n + 3) / 4);
  if (c->dim == 512)
    kv4_append_kernel<512><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    kv4_append_kernel<576><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

int dsv41_kv4_read(const dsv41_kv4* c, const long* seq, const long* row, long n, void* out, void* stream) {
  if (!kv4_ok(c) || n < 0 || n >= (1L << 32)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq || !row || !out || ((uintptr_t)out & 15)) return (int)hipErrorInvalidValue;
  RowsArgs a;
  rows_args(a, *c, seq, row, n);
  a.out = (uint16_t*)out;
  const unsigned grid = (unsigned)((n + 3) / 4);
  if (c->dim == 512)
    kv4_read_kernel<512><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    kv4_read_kernel<576><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
