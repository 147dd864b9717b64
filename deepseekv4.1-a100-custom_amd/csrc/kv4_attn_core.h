// Shared pieces of the attention kernels over the paged 4-bit cache: arguments, operand types, the layout of the values in
// LDS and what becomes of a finished output.
#pragma once
#include "kv4_core.h"

struct Kv4AttnArgs {
  const uint16_t* q;  // [R, H, DQK]
  long q_rstride;
  int R, H;
  const uint16_t* win;  // window rows: slot stride, rows a slot
  long win_sstride;
  int win_rows, win_slots;
  const int* widx;      // [R, wt] rows of win, or null: the ring by positions
  int wt;
  const uint8_t* pool;
  Kv4Table map;
  const int* idx;       // [R, t]
  int t;
  int rows_per_slot;    // query row r belongs to batch row r / rows_per_slot
  const long* seq;      // per batch row: its sequence (null: itself)
  const long* pos;      // ring: per row
  const long* pmax;
  const long* plim;
  float scale;          // softmax scale times log2(e)
  const float* sink;
  const float* cos_t;
  const float* sin_t;
  long n_pos;           // rows of the tables
  int rd;
  uint16_t* out;        // [R, H, 512]
  int wtiles, tiles, chunk, nsplit, groups;
  float* part;          // splits: [R, H, nsplit, 512] (16-byte aligned), then [R, H, nsplit, 2] reference and sum
};

namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

__device__ __align__(16) uint8_t g_kv4_none[1152];  // what a key that is not there reads

DSV41_DEV f32x4_t mfma_f16_16x16x32(uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8_t, a), __builtin_bit_cast(h16x8_t, b), c, 0, 0, 0);
}

typedef __bf16 b16x2_t __attribute__((ext_vector_type(2)));
DSV41_DEV uint32_t pack_bf16(float a, float b) { return __builtin_bit_cast(uint32_t, b16x2_t{(__bf16)a, (__bf16)b}); }
DSV41_DEV uint32_t pack_f16(float a, float b) { return __builtin_bit_cast(uint32_t, h16x2_t{(_Float16)a, (_Float16)b}); }

// LDS transpose read: within 16 lanes, lane i receives element i % 4 of the 8 bytes of lanes i/4, i/4+4, i/4+8, i/4+12.
DSV41_DEV uint2 lds_read_tr(uint32_t addr) {
  typedef __attribute__((ext_vector_type(4))) short s4;
  const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)addr);
  return __builtin_bit_cast(uint2, v);
}

// The values in LDS: row `key` of 1024 bytes, its 16-byte unit u at u ^ swizzle(key), so that neither the writes (16 keys,
// one unit each) nor the transpose reads (eight keys at a time, four and the four eight on, 32 bytes each) meet in a bank.
DSV41_DEV uint32_t v_swizzle(int key) { return ((key & 3) << 1) | (key & 8) | ((key >> 2) & 1); }

// Output of one (row, head, 4 columns from c on): the inverse rotation, one rounding.
DSV41_DEV uint2 finish4(const Kv4AttnArgs& a, long pos, int c, float4 o) {
  if (a.rd > 0 && c >= 512 - a.rd) {
    if (pos < 0 || pos >= a.n_pos) return make_uint2(0x7fc07fc0u, 0x7fc07fc0u);  // (no angle: NaN)
    const long j = pos * (a.rd / 2) + ((c - (512 - a.rd)) >> 1);
    const float c0 = a.cos_t[j], s0 = a.sin_t[j], c1 = a.cos_t[j + 1], s1 = a.sin_t[j + 1];
    o = make_float4(o.x * c0 + o.y * s0, o.y * c0 - o.x * s0, o.z * c1 + o.w * s1, o.w * c1 - o.z * s1);
  }
  return make_uint2(pack_bf16(o.x, o.y), pack_bf16(o.z, o.w));
}

}  // namespace

// Many query rows: the cache's rows in bf16, [b, slots' rows, dim], and one list of window and cache rows [R, wt + t].
void kv4_unpack_launch(const Kv4AttnArgs& a, int dim, int b, void* rows, int* list, hipStream_t st);
