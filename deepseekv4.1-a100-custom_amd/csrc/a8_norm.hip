// norm_quant8: the residual's addition, the root-mean-square norm and the block quantisation in one pass,
//   h = bf16(x + r);  y = h / sqrt(mean(h^2) + eps) * w;  codes and scales of y (a8_core.h).
// y is rounded once, to 8 bits (norm_quant rounds to bf16 in between, as the reference does); the norm is that of the bf16
// stream, whose readers see what was normed.  Without w: the quantisation alone.  The reciprocal of the root is two floats,
// so that y = (h w) (hi + lo), h w exact, is rounded to fp32 once: codes at a border of two fall to the side of the sum.
// (The sum over the lanes and the root in 64 bits as well: 8192 rows of 5120 53 -> 57 us.)
//
// Bound: HBM, 2 bytes a value in (4 with r) and 1 + 1/32 out (3 + 1/32 with h).  A lane holds 8 adjacent values (16-byte
// loads, all of a row's in flight at once), so a row is read once and a block is 4 lanes; its codes leave as 8 bytes a
// lane after one exchange with the neighbour.
#include "a8_core.h"
#include "rowop.h"

namespace {

struct NormArgs {
  const uint16_t *x, *r, *w;
  float eps;
  uint16_t* h;
  uint8_t *a8, *s8;
  long rows, first;  // all of them; the launch's first
  int D;
};

// One row by nt lanes (t: this lane's number); red: the workgroup's exchange, null where a row is one wave's.
template <int IT, bool BLOCK>
DSV41_DEV void norm_row(const NormArgs& a, long row, bool live, int t, int nt, float* red) {
  const int nc = a.D / 8;
  const long base = row * a.D;
  uint4 xq[IT], rq[IT], wq[IT];
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = min(t + i * nt, nc - 1);  // (lanes past the row load its last chunk and store nothing)
    xq[i] = ((const uint4*)(a.x + base))[c];
    if (a.r) rq[i] = ((const uint4*)(a.r + base))[c];
    if (a.w) wq[i] = ((const uint4*)a.w)[c];
  }
  float v[IT][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const bool in = live && t + i * nt < nc;
    a8_unpack8(xq[i], v[i]);
    if (a.r) {
      float r[8];
      a8_unpack8(rq[i], r);
#pragma unroll
      for (int k = 0; k < 8; ++k) r[k] += v[i][k];
      const uint4 hq = a8_pack8(r);
      if (in) ((uint4*)(a.h + base))[t + i * nt] = hq;
      a8_unpack8(hq, v[i]);
    }
    if (in) {
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = __builtin_fmaf(v[i][k], v[i][k], ss);
    }
  }
  if (a.w) {
    ss = wave_sum(ss);
    if constexpr (BLOCK) {
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
      __syncthreads();
      ss = 0.0f;
      for (int k = 0; k < nt / 64; ++k) ss += red[k];
    }
    const float mean = __fdiv_rn(ss, (float)a.D) + a.eps;
    float hi = __fdiv_rn(1.0f, __fsqrt_rn(mean));
    // 1 - mean hi^2, its products exact: half of it is what hi is off by, relative
    const float root = mean * hi, off = __builtin_fmaf(-root, hi, 1.0f) - __builtin_fmaf(mean, hi, -root) * hi;
    // (2^8 from w to the reciprocal: h w of finite numbers stays finite, and y is 0 where the sum of squares is infinite)
    hi *= 256.0f;
    const float lo = hi > 0.0f && hi < 3.0e38f ? 0.5f * hi * off : 0.0f;
#pragma unroll
    for (int i = 0; i < IT; ++i) {
      float w[8];
      a8_unpack8(wq[i], w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float p = v[i][k] * (w[k] * 0.00390625f);
        v[i][k] = __builtin_fmaf(p, hi, p * lo);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int c = t + i * nt;
    int s;
    const uint2 q = a8_quant8(v[i], t & 1, &s);
    if (live && c < nc) {
      *(uint2*)(a.a8 + base + 8 * c) = q;
      if ((c & 3) == 0) {
        const int b = c >> 2;
        uint8_t* sp = a.s8 + ((long)(b >> 2) * a.rows + row) * 4 + (b & 3);
        *sp = (uint8_t)s;
        if (b == nc / 4 - 1)
          for (int k = (b & 3) + 1; k < 4; ++k) *++sp = 127;
      }
    }
  }
}

// A row a workgroup (its threads: the row's chunks, rounded up to whole waves, at most 1024).
template <int IT>
__global__ void __launch_bounds__(1024) norm_quant8_block_kernel(const NormArgs a) {
  __shared__ float red[16];
  norm_row<IT, true>(a, a.first + blockIdx.x, true, threadIdx.x, blockDim.x, red);
}

// A row a wave, four to a workgroup.
template <int IT>
__global__ void __launch_bounds__(256) norm_quant8_wave_kernel(const NormArgs a) {
  const long row = a.first + (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  norm_row<IT, false>(a, min(row, a.rows - 1), row < a.rows, threadIdx.x & 63, 64, nullptr);
}

}  // namespace

extern "C" int dsv41_norm_quant8(const void* x, const void* residual, const void* w, float eps, void* h, void* a8,
                                 void* s8, long n_rows, int D, void* stream) {
  if (n_rows <= 0) return 0;
  if (D <= 0 || D % 32 != 0 || D > 16384 || n_rows > 0x7fffffffl || (residual && !h)) return (int)hipErrorInvalidValue;
  if (!x || !a8 || !s8) return (int)hipErrorInvalidValue;
  if (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)w | (uintptr_t)h | (uintptr_t)a8) & 15)
    return (int)hipErrorInvalidValue;
  NormArgs a{(const uint16_t*)x, (const uint16_t*)residual, (const uint16_t*)w, eps, (uint16_t*)h,
             (uint8_t*)a8, (uint8_t*)s8, n_rows, 0, D};
  const hipStream_t st = (hipStream_t)stream;
  // (a launch has fewer than 2^32 threads: 64 a row, or up to 1024)
  const long most = D <= 2048 ? 1l << 25 : 1l << 21;
  for (; a.first < n_rows; a.first += most) {
    const long rows = min(n_rows - a.first, most);
    if (D <= 2048) {
      const dim3 g((unsigned)((rows + 3) / 4));
      if (D <= 512) norm_quant8_wave_kernel<1><<<g, 256, 0, st>>>(a);
      else if (D <= 1024) norm_quant8_wave_kernel<2><<<g, 256, 0, st>>>(a);
      else if (D <= 1536) norm_quant8_wave_kernel<3><<<g, 256, 0, st>>>(a);
      else norm_quant8_wave_kernel<4><<<g, 256, 0, st>>>(a);
    } else {
      const int nc = D / 8, nt = nc <= 1024 ? (nc + 63) / 64 * 64 : (nc / 2 + 63) / 64 * 64;
      if (nc <= 1024) norm_quant8_block_kernel<1><<<(unsigned)rows, nt, 0, st>>>(a);
      else norm_quant8_block_kernel<2><<<(unsigned)rows, nt, 0, st>>>(a);
    }
  }
  DSV41_CHECK_LAUNCH();
  return 0;
}
