// Rows of the paged 4-bit cache: written (rope, 4-bit grid, packed into the row's page) and read back as bf16.
//
// A wave has two rows: lane l holds values 8 l .. 8 l + 7 of each (one 16-byte load), so a group of 16 is a lane pair, the
// codes of a lane are one dword and a row's codes one 256-byte store; the last 64 values of rows of 576, which the rotation
// is of, take eight lanes a row, both rows' at once.  Page and address are scalar.
//
// Bound by latency for a step's rows (24 rows of 576: append 3.4 us, read 2.4) and by the way from sequence to page to row
// and the encoding for many: 16002 rows of 576 append 10.4 us, 24 MB at 2.3 TB/s, read 6.6, 3.6 TB/s (a large copy: 5.2).
// One row a wave, with exact quotients and the rotation in every lane: 23.3 and 7.6 us; with this encoding 15.2 and 8.0.
#include "kv4_core.h"

namespace {

constexpr int kRows = 2;  // rows a wave

struct RowsArgs {
  const uint16_t* x;
  long x_rstride;
  const long* seq;
  const long* row;
  long n;
  int ratio, by_pos;
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
// reciprocal (off by 2^-22 of themselves) rounded to bf16: one that is a border comes out as the border, which has 3 bits (the
// scale's 5).  Any other is at least 1/254 of a border away from it: the value, and the border times the divisor (of 7 bits,
// so even at 8), are two integers of 8 bits that differ; bf16 moves it by 2^-8 of the border at most.  The conversions round
// to even and saturate: the scale at 448, the codes at 6.  A group with an infinity or a NaN reads back as NaN (scale 0x7f).
DSV41_DEV uint32_t kv4_encode(const float* v, uint8_t* scale) {
  uint32_t top = 0;  // the largest magnitude's bits: a NaN's are above an infinity's
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
  const float a = group_max(__uint_as_float(min(top, 0x7f800000u)), 2);
  const float t = (float)(__bf16)fminf(fmaxf(a, 6.0f * 0.001953125f) * (1.0f / 6.0f), 448.0f);
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
  }
  const int from = dim - a.rd;
  if (e + 8 <= from) return;
  const float* const ct = a.cos_t + pos * (a.rd / 2);
  const float* const st = a.sin_t + pos * (a.rd / 2);
  float co[4], si[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int j = max(e + 2 * i - from, 0) >> 1;
    co[i] = ct[j];
    si[i] = st[j];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double c = co[i], s = si[i], p = v[2 * i], q = v[2 * i + 1];
    const float y = (float)(p * c - q * s), z = (float)(p * s + q * c);
    uint32_t w2;
    asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(w2) : "v"(y), "v"(z));
    const uint32_t y2 = e + 2 * i < from ? w[i] : w2;
    v[2 * i] = __uint_as_float(y2 << 16);
    v[2 * i + 1] = __uint_as_float(y2 & 0xffff0000u);
  }
}

template <int DIM>
__global__ void __launch_bounds__(256) kv4_append_kernel(const RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const long r0 = (blockIdx.x * 4L + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kRows;
  const uint16_t* const x = a.x + r0 * a.x_rstride;
  const int n = (int)min((long)kRows, a.n - r0);
  if (n <= 0) return;
  uint4 raw[kRows], tail;
  long pos[kRows];
  uint8_t* dst[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) raw[u] = *(const uint4*)(x + min(u, n - 1) * a.x_rstride + 8 * lane);
  if (DIM == 576) tail = *(const uint4*)(x + min((lane >> 3) % kRows, n - 1) * a.x_rstride + 512 + 8 * (lane & 7));
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const long seq = a.seq[r0 + min(u, n - 1)];
    long row = a.row[r0 + min(u, n - 1)];
    if (a.by_pos) {
      const uint32_t next = (uint32_t)row + 1, ratio = (uint32_t)a.ratio;
      row = row >= 0 && row < (1L << 31) && next % ratio == 0 ? (long)(next / ratio) - 1 : -1;
    }
    const int p = kv4_page(a.map, seq, row);
    pos[u] = row * a.ratio;
    dst[u] = nullptr;
    if (u >= n || row < 0) continue;
    if (p < 0 || a.refs[p] > 1 || (a.rd > 0 && pos[u] >= a.n_pos)) {
      if (lane == 0) atomicOr(a.err, seq < 0 || seq >= a.map.slots ? kKv4Ignored : kKv4Dropped);
    } else {
      dst[u] = a.pool + kv4_offset(a.map, p, row, kv4_row_bytes(DIM));
    }
  }
  float v[8];
  uint8_t scale;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    if (!dst[u]) continue;
    kv4_load(raw[u], 8 * lane, DIM, a, pos[u], v);
    ((uint32_t*)dst[u])[lane] = kv4_encode(v, &scale);
    if ((lane & 1) == 0) dst[u][256 + (lane >> 1)] = scale;
  }
  if (DIM == 576) {  // the last columns of all the rows at once, eight lanes each
    long at = pos[0];
    uint8_t* to = dst[0];
#pragma unroll
    for (int u = 1; u < kRows; ++u) {
      at = (lane >> 3) == u ? pos[u] : at;
      to = (lane >> 3) == u ? dst[u] : to;
    }
    if (lane >= 8 * kRows || !to) return;
    const int l = lane & 7;
    kv4_load(tail, 512 + 8 * l, DIM, a, at, v);
    ((uint32_t*)to)[72 + l] = kv4_encode(v, &scale);
    if ((l & 1) == 0) to[320 + (l >> 1)] = scale;
    if (l < 3) ((uint32_t*)to)[81 + l] = 0;
  }
}

template <int DIM>
__global__ void __launch_bounds__(256) kv4_read_kernel(const RowsArgs a) {
  const int lane = threadIdx.x & 63;
  const long r0 = (blockIdx.x * 4L + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * kRows;
  const int n = (int)min((long)kRows, a.n - r0);
  if (n <= 0) return;
  const uint8_t* src[kRows];
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    const long row = a.row[r0 + min(u, n - 1)];
    const int p = kv4_page(a.map, a.seq[r0 + min(u, n - 1)], row);
    src[u] = p >= 0 ? a.pool + kv4_offset(a.map, p, row, kv4_row_bytes(DIM)) : nullptr;
  }
  uint32_t code[kRows], sc[kRows], ct = 0, st = 0;
#pragma unroll
  for (int u = 0; u < kRows; ++u) {
    code[u] = src[u] ? ((const uint32_t*)src[u])[lane] : 0;
    sc[u] = src[u] ? src[u][256 + (lane >> 1)] : 0;
  }
  const int l = lane & 7;
  if (DIM == 576) {
    const uint8_t* from = src[0];
#pragma unroll
    for (int u = 1; u < kRows; ++u) from = (lane >> 3) == u ? src[u] : from;
    if (from) {
      ct = ((const uint32_t*)from)[72 + l];
      st = from[320 + (l >> 1)];
    }
  }
  uint16_t* const out = a.out + r0 * DIM;
#pragma unroll
  for (int u = 0; u < kRows; ++u)
    if (u < n) *(uint4*)(out + u * DIM + 8 * lane) = kv4_bf16(code[u], sc[u]);
  if (DIM == 576 && (lane >> 3) < n) *(uint4*)(out + (lane >> 3) * DIM + 512 + 8 * l) = kv4_bf16(ct, st);
}

long rows_blocks(long n) { return n / (4 * kRows) + (n % (4 * kRows) != 0); }

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
                     int ratio, int by_pos, const float* cos_t, const float* sin_t, long n_pos, int rd, void* stream) {
  if (!kv4_ok(c) || n < 0 || !kv4_grid_ok(rows_blocks(n))) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq || !row || !x || ((uintptr_t)x & 15) || x_rstride < c->dim || x_rstride % 8 || ratio < 1 || rd < 0 ||
      rd > c->dim || (rd & 1) || (rd > 0 && (!cos_t || !sin_t)))
    return (int)hipErrorInvalidValue;
  RowsArgs a;
  rows_args(a, *c, seq, row, n);
  a.x = (const uint16_t*)x;
  a.x_rstride = x_rstride;
  a.ratio = ratio;
  a.by_pos = by_pos;
  a.cos_t = cos_t;
  a.sin_t = sin_t;
  a.n_pos = n_pos;
  a.rd = rd;
  const unsigned grid = (unsigned)rows_blocks(n);
  if (c->dim == 512)
    kv4_append_kernel<512><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    kv4_append_kernel<576><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

int dsv41_kv4_read(const dsv41_kv4* c, const long* seq, const long* row, long n, void* out, void* stream) {
  if (!kv4_ok(c) || n < 0 || !kv4_grid_ok(rows_blocks(n))) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq || !row || !out || ((uintptr_t)out & 15)) return (int)hipErrorInvalidValue;
  RowsArgs a;
  rows_args(a, *c, seq, row, n);
  a.out = (uint16_t*)out;
  const unsigned grid = (unsigned)rows_blocks(n);
  if (c->dim == 512)
    kv4_read_kernel<512><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  else
    kv4_read_kernel<576><<<grid, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
