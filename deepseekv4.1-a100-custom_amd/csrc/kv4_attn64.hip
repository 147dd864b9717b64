// Sparse attention of many query rows over two tables of bf16 rows (the window's, and a cache's rows decoded once).
//
// One workgroup of eight waves, two a SIMD: one query row, 64 heads, a run of 32-key tiles.  A tile's rows are gathered
// into LDS by direct loads two tiles ahead, four rows a wave (a row is 64 lanes of 16 bytes).  Waves 0-3 have heads 0-31,
// waves 4-7 heads 32-63, and share nothing but the rows.  S^T = K Q^T by 16x16x32 MFMAs: a wave scores 16 heads by 16
// keys, Q in registers; O^T += V^T P^T: a wave has its group's heads by 128 of the 512 value columns.
//
// Three tiles are in work at once: step 1 of iteration u has the scores of tile u and the product of tile u - 2 (values
// read into registers an iteration ahead), step 2 the probabilities of tile u - 1 (a reference that only a score more than
// 2^8 above it moves, noted through LDS), the gathers, and the masked scores of tile u.  One group's step 1 stands beside
// the other's step 2, a barrier after each: a wave alone issues a vector instruction in 8 cycles, so the matrix units and
// everything else only run at once in two waves.
#include "kv4_attn_core.h"

namespace {

typedef __attribute__((ext_vector_type(2))) float f32x2_t;

constexpr int kTile = 32;
constexpr int kThreads = 512;
constexpr int kVAt = 0;                 // rows' first 512 columns [4][32 keys] 1024 bytes
constexpr int kTAt = 4 * 32768;         // their last 64 [4][32 keys] 128 bytes
constexpr int kPAt = kTAt + 4 * 4096;   // probabilities [2][64 heads][32 keys]
constexpr int kRAt = kPAt + 2 * 4096;   // row pointers [8 pairs of tiles][64 keys]
constexpr int kIAt = kRAt + 8 * 512;    // indices [8][64]
constexpr int kMAt = kIAt + 8 * 256;    // maxima [2][64 heads][2 key blocks], where a wave notes one
constexpr int kFAt = kMAt + 2 * 512;    // whether it does [2][8 waves]
constexpr int kKAt = kFAt + 2 * 32;     // which keys there are [8 pairs] 64 bits
constexpr int kLds = kKAt + 64;

#define LDS(T, at) (*(__attribute__((address_space(3))) T*)(at))

// The 16-byte unit u of a key's row stands at u ^ swizzle(key): 16 keys' reads of one unit have 16 places, and so have the
// eight keys (four, and four eight on) whose 32 bytes a transpose read takes at a time.
DSV41_DEV uint32_t swizzle(int key) { return ((key & 3) << 1) | (key & 8) | ((key >> 2) & 1); }

template <int DQK>
__global__ void __launch_bounds__(kThreads, 2) kv4_attn64_kernel(const Kv4AttnArgs a) {
  constexpr int NK = DQK / 32;
  constexpr bool TAIL = DQK == 576;
  constexpr int kLoads = TAIL ? 5 : 4;  // of a wave and tile
  __shared__ __align__(1024) uint8_t lds[kLds];

  const int b = blockIdx.x;
  const int sp = b % a.nsplit, rh = b / a.nsplit;
  const int hg = rh % a.groups, r = rh / a.groups;
  const int h0 = hg * 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  // this wave's group of heads, its keys and head block (2 group + own) in the scores, its eight blocks of 16
  // columns (every fourth) in the product
  const int group = wave >> 2, kb = wave & 1, own = (wave >> 1) & 1, hb = 2 * group + own, cols = wave & 3;
  const int slot = r / a.rows_per_slot;
  const int t0 = sp * a.chunk, t1 = min(t0 + a.chunk, a.tiles), T = t1 - t0;

  const uint32_t base = lds_addr_of(lds);
  const int key = kb * 16 + l16;

  // ---- rows' pointers: wave w has the pairs of tiles w, w + 8, ..
  const int* const list = a.idx + (long)r * a.t + t0 * kTile;
  const int n = min(a.t - t0 * kTile, T * kTile);
  const uint8_t* const win = (const uint8_t*)(a.win + (long)slot * a.win_sstride);
  const uint8_t* const cache = a.pool + (long)slot * a.n2 * (2 * DQK);
  auto resolve = [&](int pp, int i) {
    const bool ok = pp * 64 + lane < n && i >= 0 && i < a.win_rows + a.n2;
    const uint8_t* p = i < a.win_rows ? win + (long)i * (2 * DQK) : cache + (long)(i - a.win_rows) * (2 * DQK);
    LDS(uint64_t, base + kRAt + wave * 512 + lane * 8) = (uint64_t)(ok ? p : g_kv4_none);
    LDS(uint64_t, base + kKAt + wave * 8) = __ballot(ok);  // (64 lanes, one value)
  };
  auto entry = [&](int pp) { return list + max(min(pp * 64 + lane, n - 1), 0); };
  resolve(wave, n > 0 ? *entry(wave) : -1);

  u32x4 q[NK];
  {
    const int h = h0 + 16 * hb + l16;
    const uint16_t* src = a.q + r * a.q_rstride + (long)(h < a.H ? h : a.H - 1) * DQK + 8 * g;
#pragma unroll
    for (int k = 0; k < NK; ++k) q[k] = *(const u32x4*)(src + 32 * k);
  }
  // the pipeline starts on nothing: no probabilities, zeros for values, no maxima
  for (int i = threadIdx.x * 16; i < 2 * 4096; i += kThreads * 16) LDS(u32x4, base + kPAt + i) = u32x4{0, 0, 0, 0};
  if (threadIdx.x < 16) LDS(int, base + kFAt + threadIdx.x * 4) = 0;
  if (threadIdx.x < 256) LDS(float, base + kMAt + threadIdx.x * 4) = -__builtin_inff();
  for (int i = threadIdx.x * 16; i < 32768; i += kThreads * 16) LDS(u32x4, base + kVAt + 3 * 32768 + i) = u32x4{0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < NK; ++k) asm volatile("" : "+v"(q[k]));  // (from here on the loads in flight are those counted here)
  lds_barrier();

  // ---- gathers: four rows a wave; lane i of a row's load has unit i ^ swizzle(key), of the tails' unit i % 8 of key i / 8
  const uint32_t rows_at = base + kRAt + wave * 32;  // pointers of keys 4 wave .. of the first tile of a pair
  auto gather = [&](int u) {
    const uint32_t at = rows_at + ((u >> 1) & 7) * 512 + (u & 1) * 256;
    const uint32_t dst = base + kVAt + (u & 3) * 32768 + wave * 4096;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t p = LDS(uint64_t, at + j * 8);
      lds_dma16_at((const uint8_t*)p + (((uint32_t)lane ^ swizzle(4 * wave + j)) << 4), dst + j * 1024);
    }
    if (TAIL) {
      const int k4 = (lane >> 3) & 3, kk = 4 * wave + k4;
      const uint64_t p = LDS(uint64_t, at + k4 * 8);
      if (lane < 32)
        lds_dma16_at((const uint8_t*)p + 1024 + (((lane & 7) ^ ((kk >> 1) & 7)) << 4), base + kTAt + (u & 3) * 4096 + wave * 512);
    }
  };
  gather(0);
  gather(1);
  if (group) gather(2);  // (the second group gathers three tiles ahead: it comes to it half an iteration later)

  f32x4_t o[2][8];  // head blocks, column blocks
  float m[2], l = 0.0f;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = -__builtin_inff();
#pragma unroll
    for (int c = 0; c < 8; ++c) o[i][c] = f32x4_t{0, 0, 0, 0};
  }
  f32x4_t sv;   // scores of the tile before
  u32x4 vf[8];  // values of the tile before that
#pragma unroll
  for (int i = 0; i < 4; ++i) sv[i] = -__builtin_inff();
#pragma unroll
  for (int c = 0; c < 8; ++c) vf[c] = u32x4{0, 0, 0, 0};

  // addresses: of unit 4 k + g the bits of k % 4 meet the swizzle's, those of k / 4 are an immediate; the values' alike
  uint32_t k_get[4], v_get[2][2];
  const int kr = g * 8 + (l16 >> 2);
#pragma unroll
  for (int i = 0; i < 4; ++i) k_get[i] = base + kVAt + key * 1024 + (((uint32_t)(4 * i + g) ^ swizzle(key)) << 4);
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int e = 0; e < 2; ++e)
      v_get[i][e] = base + kVAt + (kr + 4 * e) * 1024 +
                    (((uint32_t)(8 * i + 2 * cols + ((l16 & 3) >> 1)) ^ swizzle(kr + 4 * e)) << 4) + (l16 & 1) * 8;
  const uint32_t t_get = base + kTAt + key * 128 + ((g ^ ((key >> 1) & 7)) << 4);  // (unit 4 + g: bit 2 the other way)
  // (probabilities: a head's four units likewise, by the head)
  const uint32_t p_get = base + kPAt + (32 * group + l16) * 64 + ((g ^ (l16 >> 2)) << 4);
  const uint32_t p_put = base + kPAt + (16 * hb + l16) * 64 + (((kb * 2 + (g >> 1)) ^ (l16 >> 2)) << 4) + (g & 1) * 8;
  const uint32_t m_get = base + kMAt + (32 * group + l16) * 8, m_put = base + kMAt + (16 * hb + l16) * 8 + kb * 4;
  const uint32_t f_get = base + kFAt + group * 16, f_put = base + kFAt + wave * 4;

  if (group)
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
  else
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");
  lds_barrier();  // (tile 0 is there)
  if (group) lds_barrier();

#pragma unroll 1
  for (int u = 0; u < T + 2; ++u) {
    const uint32_t odd = u & 1, even = odd ^ 1;
    // ---- step 1: scores of tile u, the product of tile u - 2
    f32x4_t s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};
    const uint32_t buf = (u & 3) * 32768, old = ((u + 3) & 3) * 32768;
    u32x4 pb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) pb[i] = LDS(u32x4, p_get + odd * 4096 + i * 1024);
#pragma unroll
    for (int k = 0; k < NK; ++k) {
      const uint4 x = __builtin_bit_cast(uint4, k < 16 ? LDS(u32x4, k_get[k & 3] + buf + (k >> 2) * 256)
                                                       : LDS(u32x4, (k == 16 ? t_get : t_get ^ 64) + (u & 3) * 4096));
      const uint4 qa = __builtin_bit_cast(uint4, q[k]);
      if (k & 1)
        s1 = mfma_bf16_16x16x32(x, qa, s1);
      else
        s0 = mfma_bf16_16x16x32(x, qa, s0);
      if (k < 16) {
        const int i = k & 1, c = k >> 1;
        o[i][c] = mfma_bf16_16x16x32(__builtin_bit_cast(uint4, vf[c]), __builtin_bit_cast(uint4, pb[i]), o[i][c]);
        if (i == 1) {  // (this column block is done: its values of tile u - 1)
          const uint2 lo = lds_read_tr(v_get[c & 1][0] + old + (c >> 1) * 256), hi = lds_read_tr(v_get[c & 1][1] + old + (c >> 1) * 256);
          vf[c] = u32x4{lo.x, lo.y, hi.x, hi.y};
        }
      }
    }
    if (group) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");  // (tile u + 1 is there)
    lds_barrier();

    // ---- step 2: probabilities of tile u - 1
    const u32x4 fl = LDS(u32x4, f_get + even * 32);
    const uint32_t tile_keys = LDS(uint32_t, base + kKAt + ((u >> 1) & 7) * 8 + (u & 1) * 4);
    if ((u & 1) == 0) {  // the pairs of tiles behind those on their way
      const int pd = (u >> 1) + 7, pr = (u >> 1) + 5;
      if ((pd & 7) == wave && pd > 7 && n > 0) lds_dma4_at(entry(pd), base + kIAt + wave * 256);
      if ((pr & 7) == wave && pr > 7) resolve(pr, LDS(int, base + kIAt + wave * 256 + lane * 4));
    }
    gather(u + 2 + group);
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(fl[0] | fl[1] | fl[2] | fl[3]) != 0, 0)) {
      // (alike in the group's waves: all have the same maxima)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const f32x2_t w = LDS(f32x2_t, m_get + even * 512 + i * 128);
        const float t = fmaxf(fl[2 * i] ? w[0] : -__builtin_inff(), fl[2 * i + 1] ? w[1] : -__builtin_inff());
        const float up = t > m[i] + 8.0f ? t : m[i];
        const float f = up != m[i] ? __builtin_amdgcn_exp2f(m[i] - up) : 1.0f;
        m[i] = up;
        if (i == own) l *= f;
#pragma unroll
        for (int c = 0; c < 8; ++c) o[i][c] *= f;
      }
    }
    const float mine = own ? m[1] : m[0], ref = mine == -__builtin_inff() ? 0.0f : mine;
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __builtin_amdgcn_exp2f(sv[i] - ref);
    l += (p[0] + p[1]) + (p[2] + p[3]);
    LDS(uint64_t, p_put + even * 4096) = (uint64_t)pack_bf16(p[2], p[3]) << 32 | pack_bf16(p[0], p[1]);
    // masked scores of tile u
    const uint32_t there = u < T ? tile_keys >> (16 * kb + 4 * g) : 0u;
#pragma unroll
    for (int i = 0; i < 4; ++i) sv[i] = there >> i & 1 ? (s0[i] + s1[i]) * a.scale : -__builtin_inff();
    float top = fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3]));
    const bool moves = __any(top > mine + 8.0f);
    if (__builtin_expect(moves, 0)) {
      top = row_max4(top);
      LDS(float, m_put + odd * 512) = top;  // (four lanes, one value)
    }
    LDS(int, f_put + odd * 32) = moves;
    if (!group) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLoads) : "memory");  // (tile u + 1 is there)
    lds_barrier();
  }
  if (!group) lds_barrier();

  // ---- sums of the waves' keys, output
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (no load to LDS outlives the workgroup)
  LDS(float, m_put) = row_sum4(l);
  lds_barrier();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f32x2_t w = LDS(f32x2_t, m_get + i * 128);
    const float sum = w[0] + w[1];
    const int h = h0 + 16 * (2 * group + i) + l16;
    if (h >= a.H) continue;
    const int col = 16 * cols + 4 * g;
    if (a.nsplit > 1) {
      const long at = ((long)r * a.H + h) * a.nsplit + sp;
      if (cols == 0 && g == 0) *(float2*)(a.part + 2 * at) = make_float2(m[i], sum);
      float* dst = a.part + 2L * a.R * a.H * a.nsplit + at * 512 + col;
#pragma unroll
      for (int c = 0; c < 8; ++c) *(float4*)(dst + 64 * c) = make_float4(o[i][c][0], o[i][c][1], o[i][c][2], o[i][c][3]);
    } else {
      const float den = sum + exp2f(a.sink[h] * kLog2e - m[i]);
      const float inv = m[i] == -__builtin_inff() ? 0.0f : 1.0f / den;  // (no key: zeros)
      uint16_t* dst = a.out + ((long)r * a.H + h) * 512 + col;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        *(uint2*)(dst + 64 * c) = make_uint2(pack_bf16(o[i][c][0] * inv, o[i][c][1] * inv), pack_bf16(o[i][c][2] * inv, o[i][c][3] * inv));
    }
  }
}

}  // namespace

void kv4_attn64_launch(const Kv4AttnArgs& a, int dqk, hipStream_t st) {
  const unsigned grid = (unsigned)((long)a.R * a.groups * a.nsplit);
  if (dqk == 512)
    kv4_attn64_kernel<512><<<grid, kThreads, 0, st>>>(a);
  else
    kv4_attn64_kernel<576><<<grid, kThreads, 0, st>>>(a);
}
