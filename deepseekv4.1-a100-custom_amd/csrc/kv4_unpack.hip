// Many queries over one cache: its rows decoded once, to bf16 (exact), and the queries' two index lists made one.
//
// A chunk of a prompt selects each row of the cache many times (2048 queries of 2048 rows out of 16896: 248 times), so
// decoding at every use costs more than the bf16 copy: one pass over the mapped pages and one over the lists, in one launch,
// four rows a wave and eight entries a lane in flight.  2048 queries and 16896 rows of 576: 15.9 us, 61 MB at 3.8 TB/s.
#include "kv4_attn_core.h"

namespace {

struct UnpackArgs {
  const uint8_t* pool;
  Kv4Table map;
  const long* seq;
  int b, s;
  uint16_t* rows;    // [b, cols * page, DIM]
  const int* widx;   // [b * s, wt] rows of the window
  int wt, win_rows;
  const int* idx;    // [b * s, t]
  int t;
  int* list;         // [b * s, wt + t]: window rows, then win_rows + cache rows; -1: none
  int page_blocks;   // blocks of the first kind: four pages' rows each wave in turn
};

template <int DIM>
__global__ void __launch_bounds__(256) kv4_unpack_kernel(const UnpackArgs a) {
  constexpr int RB = kv4_row_bytes(DIM);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < a.page_blocks) {
    const int e = blockIdx.x / a.map.cols, j = blockIdx.x % a.map.cols;
    const long seq = a.seq ? a.seq[e] : e;
    const int p = kv4_page(a.map, seq, (long)j << a.map.shift);
    if (p < 0) return;
    const int page = 1 << a.map.shift;
    const uint8_t* src = a.pool + (long)p * page * RB;
    uint16_t* dst = a.rows + ((long)e * a.map.cols + j) * page * DIM;
    for (int r0 = wave; r0 < page; r0 += 16) {  // four rows a wave in flight
      uint32_t c[4], ct[4], f[4], ft[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint8_t* row = src + (long)(r0 + 4 * i) * RB;
        c[i] = ((const uint32_t*)row)[lane];
        f[i] = row[256 + (lane >> 1)];
        ct[i] = DIM == 576 ? ((const uint32_t*)row)[72 + (lane & 7)] : 0;
        ft[i] = DIM == 576 ? row[320 + ((lane & 7) >> 1)] : 0;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint16_t* row = dst + (long)(r0 + 4 * i) * DIM;
        *(uint4*)(row + 8 * lane) = kv4_bf16(c[i], f[i]);
        if (DIM == 576 && lane < 8) *(uint4*)(row + 512 + 8 * lane) = kv4_bf16(ct[i], ft[i]);
      }
    }
    return;
  }
  const long r = (long)blockIdx.x - a.page_blocks;
  const int e = (int)(r / a.s), n = a.wt + a.t;
  const long seq = a.seq ? a.seq[e] : e;
  int* const out = a.list + r * n;
  for (int i = threadIdx.x; i < a.wt; i += 256) {
    const int w = a.widx[r * a.wt + i];
    out[i] = w < a.win_rows ? w : -1;
  }
  const int* const in = a.idx + r * a.t;
  for (int i0 = threadIdx.x; i0 < a.t; i0 += 8 * 256) {  // eight entries a lane in flight
    int c[8], p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = in[min(i0 + 256 * j, a.t - 1)];
#pragma unroll
    for (int j = 0; j < 8; ++j) p[j] = kv4_page(a.map, seq, c[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (i0 + 256 * j < a.t) out[a.wt + i0 + 256 * j] = p[j] >= 0 ? a.win_rows + c[j] : -1;
  }
}

}  // namespace

void kv4_unpack_launch(const Kv4AttnArgs& a, int dim, int b, void* rows, int* list, hipStream_t st) {
  UnpackArgs u{a.pool, a.map, a.seq, b, a.rows_per_slot, (uint16_t*)rows, a.widx, a.wt, a.win_rows, a.idx, a.t, list,
               b * a.map.cols};
  const unsigned grid = (unsigned)(u.page_blocks + (long)b * a.rows_per_slot);
  if (dim == 512)
    kv4_unpack_kernel<512><<<grid, 256, 0, st>>>(u);
  else
    kv4_unpack_kernel<576><<<grid, 256, 0, st>>>(u);
}
