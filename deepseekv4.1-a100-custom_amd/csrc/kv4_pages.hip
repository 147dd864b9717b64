// The pages of a 4-bit cache: sequences forked, rows made writable, sequences cut short, the pool compacted, pages
// copied between pools.  Everything is kept on the device (a table of pages a sequence, a count of the table's entries
// that name a page), so the calls are stream-ordered and may be captured.
//
// Free pages are handed out lowest first, in the order of the arguments, from prefix sums: no result depends on the
// order in which workgroups run.  The counts are changed by integer atomics, whose order does not show.
//
// Release, fork and small calls are launches and little else (3 to 5 us).  A plan is one workgroup of 1024 lanes over the
// counts: reserve reads them from the front until it has found enough (8.2 us, of 63 sequences as of 4), compact all
// of them twice, 16 a lane (13.6 k pages 7.0 us; 8 a lane, one at a time, 14.1).  Moves and copies run at the memory's rate:
// compact 2400 pages of 21.5 kB, 104 MB, in 17.5 us, copy 6001 of them, 258 MB, in 46.7 us.
#include "kv4_core.h"

namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPer = 8;              // counts a thread looks at in one round of reserve
constexpr int kPlanPages = 16;       // and of compact
constexpr int kMostEntries = 4096;   // sequences of one reserve call
constexpr int kFewEntries = kPlanThreads / 256;  // of one that is one launch

struct PagesArgs {
  int* table;
  int slots, cols;
  int* refs;
  int pages, shift;
  int* err;
  uint8_t* pool;
  long page_bytes;
  const long* seq;    // (fork: the destinations)
  const long* src;
  const long* begin;  // (fork, release: rows kept)
  const long* end;
  int n;
  int* ws;
  int* live;
};

// Columns of a table that `rows` rows take.
DSV41_DEV int columns(long rows, int shift, int cols) {
  const long c = rows <= 0 ? 0 : ((rows - 1) >> shift) + 1;
  return c < cols ? (int)c : cols;
}

DSV41_DEV void copy_bytes(uint8_t* dst, const uint8_t* src, long bytes, int i = threadIdx.x) {  // by 256 lanes, 16 bytes each
  const uint4* s = (const uint4*)src;
  uint4* d = (uint4*)dst;
  const int n = (int)(bytes >> 4);
  constexpr int nt = 256;
  for (; i + 3 * nt < n; i += 4 * nt) {
    const uint4 a = s[i], b = s[i + nt], c = s[i + 2 * nt], e = s[i + 3 * nt];
    d[i] = a;
    d[i + nt] = b;
    d[i + 2 * nt] = c;
    d[i + 3 * nt] = e;
  }
  for (; i < n; i += nt) d[i] = s[i];
}

// ---- release: the pages behind the first `rows` rows of a sequence are named no more
__global__ void __launch_bounds__(256) release_kernel(const PagesArgs a) {
  const long s = a.seq[blockIdx.x];
  if (s < 0 || s >= a.slots) {
    if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.err, kKv4Ignored);
    return;
  }
  const int j = blockIdx.y * 256 + threadIdx.x;
  if (j >= a.cols || j < columns(a.begin ? a.begin[blockIdx.x] : 0, a.shift, a.cols)) return;
  const int p = atomicExch(a.table + s * a.cols + j, -1);  // (a sequence named twice gives a page up once)
  if ((unsigned)p < (unsigned)a.pages) atomicSub(a.refs + p, 1);
}

// ---- fork: sequence dst names the pages of src's first `rows` rows instead of its own
// A destination that is also a source, or that an earlier pair has, would be read and written at once: left out.
__global__ void __launch_bounds__(256) fork_kernel(const PagesArgs a) {
  const int i = blockIdx.x;
  const long s = a.src[i], d = a.seq[i];
  bool bad = s < 0 || s >= a.slots || d < 0 || d >= a.slots;
  for (int k = threadIdx.x; k < a.n; k += 256) bad |= a.src[k] == d || (k < i && a.seq[k] == d);
  if (__syncthreads_or(bad)) {
    if (threadIdx.x == 0 && blockIdx.y == 0) atomicOr(a.err, kKv4Ignored);
    return;
  }
  const int j = blockIdx.y * 256 + threadIdx.x;
  if (j >= a.cols) return;
  int* at = a.table + d * a.cols + j;
  const int old = *at;
  int p = j < columns(a.begin ? a.begin[i] : (1L << 62), a.shift, a.cols) ? a.table[s * a.cols + j] : -1;
  if ((unsigned)p >= (unsigned)a.pages) p = -1;
  if ((unsigned)old < (unsigned)a.pages) atomicSub(a.refs + old, 1);
  if (p >= 0) atomicAdd(a.refs + p, 1);
  *at = p;
}

// ---- reserve
// Workspace (int32): owner [slots], entry [pages], column [pages], page [pages], copy from [n], copy to [n].
DSV41_DEV int* ws_entry(const PagesArgs& a) { return a.ws + a.slots; }
DSV41_DEV int* ws_from(const PagesArgs& a) { return a.ws + a.slots + 3L * a.pages; }

// What the first of entry i's new pages held before `begin` goes with it.
DSV41_DEV void carry(const PagesArgs& a, int i, int lane) {
  const int from = ws_from(a)[i];
  if (from < 0) return;
  const long rows = a.begin[i] & ((1L << a.shift) - 1);
  copy_bytes(a.pool + ws_from(a)[a.n + i] * a.page_bytes, a.pool + from * a.page_bytes, rows * (a.page_bytes >> a.shift), lane);
}

// One workgroup: which columns of which entry need a page of their own (none there, or one that other entries name too),
// counted in the order of the arguments; the lowest free pages in as many; then the table and the counts; with up to four
// entries the copies too, 256 lanes each (a launch less: forking a prompt for four samples 25.9 -> 22.8 us).
__global__ void __launch_bounds__(kPlanThreads) reserve_plan_kernel(const PagesArgs a) {
  __shared__ int offs[kMostEntries + 1];
  __shared__ int tmp[kPlanThreads / 64];
  const int t = threadIdx.x;
  int* const owner = a.ws;
  int* const entry = ws_entry(a);
  int* const column = entry + a.pages;
  int* const page = column + a.pages;
  int* const from = ws_from(a);
  int* const to = from + a.n;
  for (int i = t; i < a.n; i += kPlanThreads) {
    from[i] = -1;
    const long s = a.seq[i];
    if (s >= 0 && s < a.slots) __hip_atomic_store(owner + s, a.n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  for (int i = t; i < a.n; i += kPlanThreads) {
    const long s = a.seq[i];
    if (s >= 0 && s < a.slots) atomicMin(owner + s, i);
  }
  __syncthreads();
  // columns of each entry, summed
  int total = 0;
  for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
    const int i = i0 + t;
    int c = 0;
    if (i < a.n) {
      const long s = a.seq[i], b = a.begin[i], e = a.end[i];
      const bool ok = s >= 0 && s < a.slots && b >= 0 && e <= ((long)a.cols << a.shift) &&
                      __hip_atomic_load(owner + s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == i;
      if (!ok)
        atomicOr(a.err, kKv4Ignored);
      else if (b < e)
        c = (int)(((e - 1) >> a.shift) - (b >> a.shift)) + 1;
    }
    int sum;
    const int before = block_scan_dpp<kPlanThreads>(c, tmp, &sum);
    if (i < a.n) offs[i] = total + before;
    total += sum;
  }
  if (t == 0) offs[a.n] = total;
  __syncthreads();
  // the needs, in order
  int needs = 0;
  for (int f0 = 0; f0 < total; f0 += kPlanThreads) {
    const int f = f0 + t;
    int i = 0, j = 0;
    bool need = false;
    if (f < total) {
      int hi = a.n;  // the last entry whose columns begin at f or before
      while (hi - i > 1) {
        const int mid = (i + hi) >> 1;
        if (offs[mid] <= f)
          i = mid;
        else
          hi = mid;
      }
      j = (int)(a.begin[i] >> a.shift) + f - offs[i];
      const int p = a.table[a.seq[i] * a.cols + j];
      need = (unsigned)p >= (unsigned)a.pages || a.refs[p] > 1;
    }
    int sum;
    const int r = needs + block_scan_dpp<kPlanThreads>(need, tmp, &sum);
    if (need && r < a.pages) {
      entry[r] = i;
      column[r] = j;
    }
    needs += sum;
  }
  // the lowest free pages
  int found = 0;
  for (int p0 = 0; p0 < a.pages && found < needs; p0 += kPlanThreads * kPer) {
    const int p = p0 + t * kPer;
    unsigned free = 0;
#pragma unroll
    for (int u = 0; u < kPer; ++u) free |= (p + u < a.pages && a.refs[p + u] <= 0) ? 1u << u : 0u;
    int sum;
    int r = found + block_scan_dpp<kPlanThreads>(__popc(free), tmp, &sum);
#pragma unroll
    for (int u = 0; u < kPer; ++u)
      if (free >> u & 1) {
        if (r < needs) page[r] = p + u;
        ++r;
      }
    found += sum;
  }
  if (t == 0 && found < needs) atomicOr(a.err, kKv4NoPages);
  __syncthreads();
  for (int r = t; r < (found < needs ? found : needs); r += kPlanThreads) {
    const int i = entry[r], j = column[r], p = page[r];
    int* at = a.table + a.seq[i] * a.cols + j;
    const int old = *at;
    *at = p;
    a.refs[p] = 1;
    if ((unsigned)old < (unsigned)a.pages) {
      atomicSub(a.refs + old, 1);
      if (j == (int)(a.begin[i] >> a.shift)) {
        to[i] = p;
        from[i] = old;
      }
    }
  }
  if (a.n > kFewEntries) return;
  __syncthreads();
  if (t >> 8 < a.n) carry(a, t >> 8, t & 255);
}

__global__ void __launch_bounds__(256) reserve_copy_kernel(const PagesArgs a) { carry(a, blockIdx.x, threadIdx.x); }

// ---- compact
// Workspace (int32): live, moves, from [pages], to [pages], where [pages] (the move of a page).
// One workgroup: L live pages; the live ones of L and above go, in order, to the free ones below L.  Sources and
// destinations do not meet, so the moves need no order.
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PagesArgs a) {
  __shared__ int2 tmp[2][kPlanThreads / 64];
  const int t = threadIdx.x;
  int* const from = a.ws + 2;
  int* const to = from + a.pages;
  int* const where = to + a.pages;
  // which of the kPlanPages pages of a round from p on are live, a bit each (refs is read 16 bytes at a time where it may)
  const bool wide = ((uintptr_t)a.refs & 15) == 0;
  auto bits = [&](int p) {
    unsigned m = 0;
    if (wide && p + kPlanPages <= a.pages) {
#pragma unroll
      for (int u = 0; u < kPlanPages; u += 4) {
        const int4 r = *(const int4*)(a.refs + p + u);
        m |= ((r.x > 0 ? 1u : 0u) | (r.y > 0 ? 2u : 0u) | (r.z > 0 ? 4u : 0u) | (r.w > 0 ? 8u : 0u)) << u;
      }
    } else {
      for (int u = 0; u < kPlanPages; ++u) m |= p + u < a.pages && a.refs[p + u] > 0 ? 1u << u : 0u;
    }
    return m;
  };
  const int step = kPlanThreads * kPlanPages;
  const unsigned first = bits(t * kPlanPages);
  int count = __popc(first);
  for (int p0 = step; p0 < a.pages; p0 += step) count += __popc(bits(p0 + t * kPlanPages));
  int2 total;
  block_scan2_dpp<kPlanThreads>(count, 0, tmp[0], &total);
  const int live = total.x;
  int2 base = make_int2(0, 0);
  for (int p0 = 0; p0 < a.pages; p0 += step) {
    const int p = p0 + t * kPlanPages;
    const unsigned l = p0 == 0 ? first : bits(p);
    const int n = min(max(live - p, 0), kPlanPages);  // pages of p .. that stay in front
    const unsigned front = n == 32 ? ~0u : (1u << n) - 1, held = a.pages - p >= kPlanPages ? ~0u : p < a.pages ? (1u << (a.pages - p)) - 1 : 0u;
    unsigned src = l & ~front, dst = ~l & front & held;
    const int which = (p0 / step + 1) & 1;
    const int2 r = block_scan2_dpp<kPlanThreads>(__popc(src), __popc(dst), tmp[which], &total);
    for (int i = base.x + r.x; src; src &= src - 1, ++i) {
      const int s = p + __ffs(src) - 1;
      from[i] = s;
      where[s] = i;
    }
    for (int i = base.y + r.y; dst; dst &= dst - 1) to[i++] = p + __ffs(dst) - 1;
    base.x += total.x;
    base.y += total.y;
  }
  if (t == 0) {
    a.ws[0] = live;
    a.ws[1] = base.x;
    *a.live = live;
  }
}

__global__ void __launch_bounds__(256) compact_move_kernel(const PagesArgs a) {
  const int live = a.ws[0], moves = a.ws[1];
  const int* const from = a.ws + 2;
  const int* const to = from + a.pages;
  const int* const where = to + a.pages;
  const int entries = a.slots * a.cols;
  for (long i = blockIdx.x * 256 + threadIdx.x; i < entries; i += gridDim.x * 256L) {
    const int p = a.table[i];
    if (p >= live && p < a.pages) {
      const int k = where[p];  // (what the workspace held where the page's count says that it is free: no move then)
      const bool moved = (unsigned)k < (unsigned)moves && from[k] == p;
      a.table[i] = moved ? to[k] : -1;
      if (!moved) atomicOr(a.err, kKv4Ignored);
    }
  }
  for (int r = blockIdx.x; r < moves; r += gridDim.x) {
    const int s = from[r], d = to[r];
    copy_bytes(a.pool + d * a.page_bytes, a.pool + s * a.page_bytes, a.page_bytes);
    if (threadIdx.x == 0) {
      a.refs[d] = a.refs[s];
      a.refs[s] = 0;
    }
  }
}

// ---- copies between pools
struct CopyArgs {
  const uint8_t* src;
  uint8_t* dst;
  int src_pages, dst_pages, n;
  long page_bytes;
  const long* from;
  const long* to;
  int* err;
  int* last;  // [dst_pages] or null
};

// The last pair that names a page as its destination, of many pairs.
__global__ void __launch_bounds__(256) copy_clear_kernel(const CopyArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < a.dst_pages) a.last[i] = -1;
}

__global__ void __launch_bounds__(256) copy_last_kernel(const CopyArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.n) return;
  const long d = a.to[i], s = a.from[i];
  if (d >= 0 && d < a.dst_pages && s >= 0 && s < a.src_pages) atomicMax(a.last + d, i);
}

// A workgroup has P pairs: it looks through those behind its own once.
template <int P>
__global__ void __launch_bounds__(256) copy_kernel(const CopyArgs a) {
  __shared__ int s_later;
  const int i0 = blockIdx.x * P, t = threadIdx.x;
  long s[P], d[P];
  int mine = 0, later = 0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    s[p] = i0 + p < a.n ? a.from[i0 + p] : -1;
    d[p] = i0 + p < a.n ? a.to[i0 + p] : -1;
    if (s[p] == -1 || d[p] == -1) continue;
    if (s[p] >= 0 && s[p] < a.src_pages && d[p] >= 0 && d[p] < a.dst_pages)
      mine |= 1 << p;
    else if (t == 0)
      atomicOr(a.err, kKv4Ignored);
  }
  if (mine == 0) return;
  if (t == 0) s_later = 0;
  if (a.last) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (mine >> p & 1) later |= a.last[d[p]] != i0 + p ? 1 << p : 0;
  } else {
    for (int k = i0 + 1 + t; k < a.n; k += 256) {
      const long to = a.to[k];
      int hit = 0;
#pragma unroll
      for (int p = 0; p < P; ++p) hit |= to == d[p] && k > i0 + p ? 1 << p : 0;
      if (hit && a.from[k] >= 0 && a.from[k] < a.src_pages) later |= hit;
    }
  }
  __syncthreads();
  if (later & mine) atomicOr(&s_later, later);
  __syncthreads();
  later = s_later & mine;
  if (later && t == 0) atomicOr(a.err, kKv4Ignored);
#pragma unroll
  for (int p = 0; p < P; ++p)
    if ((mine & ~later) >> p & 1) copy_bytes(a.dst + d[p] * a.page_bytes, a.src + s[p] * a.page_bytes, a.page_bytes);
}

// Pairs up to which every workgroup looks through those behind its own: a pair each up to kLone, beyond that four (in a
// graph, a pair and four: 129 pairs 4.6 and 6.3 us, 2048 15.8 and 18.0, 4001 31.2 and 32.5, 6001 52.3 and 49.9, 14000 of 5 kB
// 67.4 and 38.0; claims by two launches before the copy 7.7, 21.4, 34.5, 48.7, but 61 for 51 call by call).
constexpr int kLone = 4096, kFewCopies = 16384;

PagesArgs pages_args(const dsv41_kv4& c) {
  PagesArgs a{};
  a.table = c.table;
  a.slots = c.slots;
  a.cols = c.cols;
  a.refs = c.refs;
  a.pages = c.pages;
  a.shift = kv4_shift(c.page);
  a.err = c.err;
  a.pool = (uint8_t*)c.pool;
  a.page_bytes = (long)kv4_row_bytes(c.dim) * c.page;
  return a;
}

// A grid of a workgroup per entry and 256 columns.
bool grid_ok(const dsv41_kv4* c, int n) { return kv4_ok(c) && c->cols <= 256 * 65535 && n >= 0 && kv4_grid_ok(n); }

}  // namespace

extern "C" {

int dsv41_kv4_fork(const dsv41_kv4* c, const long* src, const long* dst, const long* rows, int n, void* stream) {
  if (!grid_ok(c, n)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!src || !dst) return (int)hipErrorInvalidValue;
  PagesArgs a = pages_args(*c);
  a.src = src;
  a.seq = dst;
  a.begin = rows;
  a.n = n;
  fork_kernel<<<dim3(n, (c->cols + 255) / 256), 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

int dsv41_kv4_release(const dsv41_kv4* c, const long* seq, const long* rows, int n, void* stream) {
  if (!grid_ok(c, n)) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq) return (int)hipErrorInvalidValue;
  PagesArgs a = pages_args(*c);
  a.seq = seq;
  a.begin = rows;
  a.n = n;
  release_kernel<<<dim3(n, (c->cols + 255) / 256), 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

long dsv41_kv4_reserve_workspace_bytes(const dsv41_kv4* c, int n) {
  return 4 * ((long)c->slots + 3L * c->pages + 2L * n);
}

int dsv41_kv4_reserve(const dsv41_kv4* c, const long* seq, const long* begin, const long* end, int n, void* ws,
                      long ws_bytes, void* stream) {
  if (!kv4_ok(c) || n < 0 || n > kMostEntries) return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!seq || !begin || !end || !ws || ((uintptr_t)ws & 3) || ws_bytes < dsv41_kv4_reserve_workspace_bytes(c, n))
    return (int)hipErrorInvalidValue;
  PagesArgs a = pages_args(*c);
  a.seq = seq;
  a.begin = begin;
  a.end = end;
  a.n = n;
  a.ws = (int*)ws;
  reserve_plan_kernel<<<1, kPlanThreads, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  if (n > kFewEntries) {
    reserve_copy_kernel<<<n, 256, 0, (hipStream_t)stream>>>(a);
    DSV41_CHECK_LAUNCH();
  }
  return 0;
}

long dsv41_kv4_compact_workspace_bytes(const dsv41_kv4* c) { return 4 * (2 + 3L * c->pages); }

int dsv41_kv4_compact(const dsv41_kv4* c, int* live, void* ws, long ws_bytes, void* stream) {
  if (!kv4_ok(c) || !live || !ws || ((uintptr_t)ws & 3) || ws_bytes < dsv41_kv4_compact_workspace_bytes(c))
    return (int)hipErrorInvalidValue;
  PagesArgs a = pages_args(*c);
  a.ws = (int*)ws;
  a.live = live;
  compact_plan_kernel<<<1, kPlanThreads, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  compact_move_kernel<<<c->pages < 2048 ? c->pages : 2048, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

long dsv41_kv4_copy_workspace_bytes(const dsv41_kv4* c, int n) { return n > kFewCopies ? 4L * c->pages : 0; }

int dsv41_kv4_copy(const dsv41_kv4* c, const dsv41_kv4* other, const long* src, const long* dst, int n, void* ws,
                   long ws_bytes, void* stream) {
  if (!kv4_ok(c) || !kv4_ok(other) || c->dim != other->dim || c->page != other->page || n < 0 || !kv4_grid_ok(n))
    return (int)hipErrorInvalidValue;
  if (n == 0) return 0;
  if (!src || !dst || (n > kFewCopies && (!ws || ((uintptr_t)ws & 3) || ws_bytes < dsv41_kv4_copy_workspace_bytes(c, n))))
    return (int)hipErrorInvalidValue;
  const long pb = (long)kv4_row_bytes(c->dim) * c->page;
  const char *s0 = (const char*)other->pool, *d0 = (const char*)c->pool;
  if (s0 < d0 + c->pages * pb && d0 < s0 + other->pages * pb) return (int)hipErrorInvalidValue;  // (one memory)
  CopyArgs a{(const uint8_t*)other->pool, (uint8_t*)c->pool, other->pages, c->pages, n, pb, src, dst, c->err,
             n > kFewCopies ? (int*)ws : nullptr};
  if (a.last) {
    copy_clear_kernel<<<(c->pages + 255) / 256, 256, 0, (hipStream_t)stream>>>(a);
    DSV41_CHECK_LAUNCH();
    copy_last_kernel<<<(n + 255) / 256, 256, 0, (hipStream_t)stream>>>(a);
    DSV41_CHECK_LAUNCH();
  }
  if (a.last || n <= kLone)
    copy_kernel<1><<<n, 256, 0, (hipStream_t)stream>>>(a);
  else
    copy_kernel<4><<<(n + 3) / 4, 256, 0, (hipStream_t)stream>>>(a);
  DSV41_CHECK_LAUNCH();
  return 0;
}

}  // extern "C"
