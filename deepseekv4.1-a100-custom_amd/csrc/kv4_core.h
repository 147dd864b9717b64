// The paged 4-bit cache of compressed rows: its row format and the way from a sequence's row to its bytes.
//
// A row of 512 (or 576: 512 and 64 more) values on the compressed rows' grid -- E2M1 times an e4m3 scale per 16 -- as
// the grid's own bits: 256 bytes of codes, two a byte with the lower value in the lower four bits, 32 scales; at 576
// then 32 bytes of codes and 4 scales of the last 64 values and 12 bytes of zeros, so that rows stay 16-byte aligned.
// Codes and scales of a row stand together: a gathered row is 288 (336) contiguous bytes, three 128-byte lines.
// Every value is exact in bf16 and in fp16 (6 significand bits, 2^-10 .. 2688).
#pragma once
#include "common.h"

struct Kv4Table {
  const int* table;  // [slots, cols]: the page of rows j << shift .. of a sequence, -1 none
  int slots, cols, pages;
  int shift;         // page = 1 << shift rows
};

namespace {

typedef _Float16 h16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 h16x8_t __attribute__((ext_vector_type(8)));

constexpr int kv4_row_bytes(int dim) { return dim == 512 ? 288 : 336; }

// Bits of the cache's error word.
constexpr int kKv4NoPages = 1;   // reserve found too few free pages
constexpr int kKv4Ignored = 2;   // an entry was left out: an index out of range, or one named twice
constexpr int kKv4Dropped = 4;   // an appended row had no page of its own, or no rope angle

// The page of row `row` of sequence `seq`, -1 where there is none.
DSV41_DEV int kv4_page(const Kv4Table& m, long seq, long row) {
  if (seq < 0 || seq >= m.slots || row < 0 || (row >> m.shift) >= m.cols) return -1;
  const int p = m.table[seq * m.cols + (row >> m.shift)];
  return (unsigned)p < (unsigned)m.pages ? p : -1;
}

// Byte offset of a row in the pool (past 32 bits in a large one).
DSV41_DEV long kv4_offset(const Kv4Table& m, int p, long row, int row_bytes) {
  return (((long)p << m.shift) + (row & ((1L << m.shift) - 1))) * row_bytes;
}

// The e4m3 scales of bytes 0, 1 (or, HI, 2, 3) of w.
template <bool HI>
DSV41_DEV h16x2_t kv4_scales(uint32_t w) {
  return __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI);
}

// Eight codes of one group and its scale: the values in fp16, exact.
DSV41_DEV uint4 kv4_values(uint32_t codes, _Float16 scale) {
  const h16x2_t s{scale, scale};
  return make_uint4(__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 0) * s),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 1) * s),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 2) * s),
                    __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.0f, 3) * s));
}

// Eight codes and their scale as bf16 (the values' fp32 bits end above bf16's last one).
DSV41_DEV uint4 kv4_bf16(uint32_t codes, uint32_t scale) {
  const uint4 h = kv4_values(codes, kv4_scales<false>(scale)[0]);
  const uint32_t w[4] = {h.x, h.y, h.z, h.w};
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const h16x2_t p = __builtin_bit_cast(h16x2_t, w[i]);
    o[i] = (__float_as_uint((float)p[0]) >> 16) | (__float_as_uint((float)p[1]) & 0xffff0000u);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// log2 of a page's rows, -1 where it is no power of two from 16 to 256.
inline int kv4_shift(int page) {
  for (int s = 4; s <= 8; ++s)
    if (page == 1 << s) return s;
  return -1;
}

inline bool kv4_ok(const dsv41_kv4* c) {
  return c && c->pool && ((uintptr_t)c->pool & 15) == 0 && c->table && c->refs && c->err && c->slots > 0 && c->cols > 0 &&
         (long)c->slots * c->cols <= (1L << 31) - (1L << 20) && c->pages > 0 && kv4_shift(c->page) >= 0 &&
         (long)c->pages * c->page < (1L << 31) && (c->dim == 512 || c->dim == 576);
}

// Whether a launch of so many workgroups of 256 stays under 2^32 lanes, the runtime's bound.
inline bool kv4_grid_ok(long blocks) { return blocks < 1L << 24; }

inline Kv4Table kv4_map(const dsv41_kv4& c) { return Kv4Table{c.table, c.slots, c.cols, c.pages, kv4_shift(c.page)}; }

}  // namespace
