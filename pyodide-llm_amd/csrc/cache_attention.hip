// cache_attention.hip — attention over the cache held in 8 bits (cache.hpp): softmax_j(q . k_j / sqrt(hs)) v_j of a token
// at position p over the positions before its block of 32 by their 8-bit values, and over its own block's up to p by their
// float32 rows.
//
// A wave takes 32 rows (tokens x query heads of one kv head) of one block of positions and goes over the cache's blocks
// once, with a running maximum and sum. The rows are the columns of every product, so that a row's statistics live in its
// lane (and the lane 32 past it):
//   S^T = K Q^T on i8 MFMA: a query in three signed base-256 digits, x = round(q * 8355000 / max|q|) = 65536 d0 + 256 d1 +
//     d2: float32's precision (2^-23 of the row's largest), the keys' bytes as they lie, the int32 sums exact;
//   O^T = V^T P^T on f16 MFMA: the values' bytes are exact in f16, a probability goes in two halves (22 bits).
// Maxima are rounded up to whole powers of two, so that every rescaling is exact; the products' scale (2^mw - 14) follows
// the largest probability times its block's value scale, so that halves neither overflow nor lose bits where the blocks'
// scales differ.
#include "cache.hpp"

namespace ple {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr float LOG2E = 1.44269504088896341f;
constexpr float NONE = -1e30f;  // no maximum yet (finite: its differences stay numbers)

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// a query's 16 values as three words of digits each four: round(x * m) = 65536 d0 + 256 d1 + d2
__device__ __forceinline__ void digits(const float4 x, float m, int32_t &d0, int32_t &d1, int32_t &d2) {
  const float in[4] = {x.x, x.y, x.z, x.w};
  uint32_t w0 = 0, w1 = 0, w2 = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int32_t n = (int32_t)__builtin_rintf(in[j] * m);
    const int32_t low = (int32_t)(int8_t)n, rest = (n - low) >> 8, mid = (int32_t)(int8_t)rest, high = (rest - mid) >> 8;
    w0 |= (uint32_t)(high & 255) << (8 * j);
    w1 |= (uint32_t)(mid & 255) << (8 * j);
    w2 |= (uint32_t)(low & 255) << (8 * j);
  }
  d0 = (int32_t)w0;
  d1 = (int32_t)w1;
  d2 = (int32_t)w2;
}

// four value bytes (value + 128) as two pairs of halves: 0x6400 | byte is 1024 + byte
__device__ __forceinline__ void widen(uint32_t w, f16x2 &a, f16x2 &b) {
  const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
  b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
}

// w in two halves, hi + lo = w to 22 bits, of two values at once. (The halves pass through a register that the compiler
// does not see into: it would otherwise form the one for the product and the one that is taken off w by different
// instructions, the product e * factor rounded once or twice, and leave an f16 step between them.)
__device__ __forceinline__ void split(float w0, float w1, f16x2 &hi, f16x2 &lo) {
  const f16x2 h = {(_Float16)w0, (_Float16)w1};
  uint32_t bits = __builtin_bit_cast(uint32_t, h);
  asm volatile("" : "+v"(bits));
  hi = __builtin_bit_cast(f16x2, bits);
  lo = f16x2{(_Float16)(w0 - (float)hi[0]), (_Float16)(w1 - (float)hi[1])};
}

// a row's running statistics: scores are in powers of two
struct Running {
  float m, l;  // sum of 2^(score - m), this lane's half of the positions
  float mw;    // the products' reference: O holds sum of 2^(score - mw + 14) value
};

template <int HS>
__global__ __launch_bounds__(256) void attend_kernel(const CacheAttn a, int tokens_log2) {
  constexpr int STEPS = (HS + 31) / 32, TILES = (HS + 31) / 32;
  const CacheView &c = a.rows.c;
  const int lane = threadIdx.x % 64, col = lane % 32, half = lane / 32, head = blockIdx.y;
  const int pos = a.rows.dpos ? *a.rows.dpos : a.rows.pos, end = pos + a.rows.count;
  const int group = a.nh / c.nkv, first_token = ((pos >> tokens_log2) + blockIdx.x * 4 + threadIdx.x / 64) << tokens_log2;
  if (first_token >= end) return;
  const int last_token = min(end, first_token + (1 << tokens_log2)) - 1;
  const int own = first_token / CACHE_BLOCK;  // the tile's tokens lie in one block
  const int token = first_token + col / group;
  const bool row = col / group < (1 << tokens_log2) && token >= pos && token < end;
  const int qhead = head * group + col % group;
  const float *q = a.q + (int64_t)(row ? token - pos : 0) * a.q_stride + qhead * HS;

  // the query's digits: lane (row, half) holds channels 32 s + 16 half .. + 15 of step s
  i32x4 q0[STEPS], q1[STEPS], q2[STEPS];
  float largest = 0.0f;
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * s + 16 * half + 4 * j;
      if (!row || d >= HS) continue;
      const float4 x = *reinterpret_cast<const float4 *>(q + d);
      largest = wmax(largest, wmax(wmax(__builtin_fabsf(x.x), __builtin_fabsf(x.y)),
                                   wmax(__builtin_fabsf(x.z), __builtin_fabsf(x.w))));
    }
  largest = wmax(largest, other_half(largest));
  // (below 2^-100 a query is taken as zero; one that is not finite makes its row's scores not a number)
  const bool finite = largest < __builtin_inff(), some = finite && largest > 0x1p-100f;
  const float to_digits = some ? 8355000.0f / largest : 0.0f;
  const float unit = LOG2E / __builtin_sqrtf((float)HS);
  const float from_digits = finite ? largest / 8355000.0f * unit : __builtin_nanf("");
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int d = 32 * s + 16 * half + 4 * j;
      float4 x = make_float4(0, 0, 0, 0);
      if (row && d < HS && some) x = *reinterpret_cast<const float4 *>(q + d);
      int32_t d0, d1, d2;
      digits(x, to_digits, d0, d1, d2);
      q0[s][j] = d0;
      q1[s][j] = d1;
      q2[s][j] = d2;
    }

  Running run = {NONE, 0.0f, NONE};
  f32x16 o[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) o[t] = (f32x16)(0.0f);
  // the statistics after a tile whose largest score is `top`, of values up to 2^bits: the factor of a probability in the
  // products
  auto advance = [&](float top, float bits) {
    const float up = __builtin_ceilf(top), m = __builtin_fmaxf(run.m, up), mw = __builtin_fmaxf(run.mw, up + bits);
    run.l *= __builtin_amdgcn_exp2f(run.m - m);
    const float gamma = __builtin_amdgcn_exp2f(run.mw - mw);
    if (__any(gamma != 1.0f)) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t] *= gamma;
    }
    run.m = m;
    run.mw = mw;
    return __builtin_amdgcn_exp2f(__builtin_fminf(m - mw + 14.0f, 126.0f));
  };

  const int64_t at = (int64_t)head * c.blocks;
  const int8_t *kp = c.keys + at * (CACHE_BLOCK * HS) + half * (CACHE_BLOCK * 16) + col * 16;
  const uint8_t *vp = c.values + at * (CACHE_BLOCK * HS) + col * CACHE_BLOCK + half * 16;
  for (int b = 0; b < own; ++b) {
    i32x16 s0 = (i32x16)(0), s1 = (i32x16)(0), s2 = (i32x16)(0);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      i32x4 k = (i32x4)(0);
      if (HS % 32 == 0 || 32 * s + 16 * half < HS)
        k = *reinterpret_cast<const i32x4 *>(kp + (int64_t)b * (CACHE_BLOCK * HS) + s * (CACHE_BLOCK * 32));
      s0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, q0[s], s0, 0, 0, 0);
      s1 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, q1[s], s1, 0, 0, 0);
      s2 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k, q2[s], s2, 0, 0, 0);
    }
    const float ks = c.scales[(at + b) * 2], vs = c.scales[(at + b) * 2 + 1];
    const float each = from_digits * ks;
    float p[16], top = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      p[r] = __builtin_fmaf((float)s0[r], 65536.0f, __builtin_fmaf((float)s1[r], 256.0f, (float)s2[r])) * each;
      top = __builtin_fmaxf(top, p[r]);
    }
    top = __builtin_fmaxf(top, other_half(top));
    const float bits = vs > 0.0f ? (float)((int)(__float_as_uint(vs) >> 23) - 126) : -200.0f;
    const float factor = advance(top, bits) * vs;
    f16x8 hi[2], lo[2];
#pragma unroll
    for (int r = 0; r < 16; r += 2) {
      const float e0 = __builtin_amdgcn_exp2f(p[r] - run.m), e1 = __builtin_amdgcn_exp2f(p[r + 1] - run.m);
      run.l += e0;
      run.l += e1;
      f16x2 h, l;
      split(e0 * factor, e1 * factor, h, l);
      hi[r / 8][r % 8] = h[0];
      hi[r / 8][r % 8 + 1] = h[1];
      lo[r / 8][r % 8] = l[0];
      lo[r / 8][r % 8 + 1] = l[1];
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (HS % 32 == 0 || 32 * t + col < HS)
        w = *reinterpret_cast<const uint4 *>(vp + (int64_t)b * (CACHE_BLOCK * HS) + t * (32 * CACHE_BLOCK));
      f16x2 h[8];
      widen(w.x, h[0], h[1]);
      widen(w.y, h[2], h[3]);
      widen(w.z, h[4], h[5]);
      widen(w.w, h[6], h[7]);
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const f16x8 v = {h[4 * s][0], h[4 * s][1], h[4 * s + 1][0], h[4 * s + 1][1],
                         h[4 * s + 2][0], h[4 * s + 2][1], h[4 * s + 3][0], h[4 * s + 3][1]};
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, hi[s], o[t], 0, 0, 0);
        o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, lo[s], o[t], 0, 0, 0);
      }
    }
  }

  // the tile's own block by its float32 rows, up to the tile's last token, on float32 MFMA
  {
    const int p0 = own * CACHE_BLOCK;
    auto source = [&](const float *x, const float *recent, int p) {
      if (p >= pos) return x + (int64_t)(p - pos) * a.rows.x_stride + head * HS;
      return recent + ((int64_t)(a.rows.displaced ? CACHE_RECENT + p % CACHE_BLOCK : p % CACHE_RECENT) * c.nkv + head) * HS;
    };
    const bool key = p0 + col <= last_token;
    const float *k = source(a.rows.k, c.recent_keys, key ? p0 + col : last_token) + half * (HS / 2);
    const float *qh = q + half * (HS / 2);
    f32x16 s = (f32x16)(0.0f);
#pragma unroll 2
    for (int i = 0; i < HS / 2; i += 4) {
      const float4 x = *reinterpret_cast<const float4 *>(k + i), y = *reinterpret_cast<const float4 *>(qh + i);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, y.x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, y.y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, y.z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, y.w, s, 0, 0, 0);
    }
    float p[16], top = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = p0 + 8 * (r / 4) + 4 * half + r % 4;
      p[r] = j <= token ? s[r] * unit : -__builtin_inff();
      top = __builtin_fmaxf(top, p[r]);
    }
    top = __builtin_fmaxf(top, other_half(top));
    const float factor = advance(top, 1.0f);
    float bad = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = p0 + 8 * (r / 4) + 4 * half + r % 4;
      const bool there = j <= last_token;
      const float *v = source(a.rows.v, c.recent_values, there ? j : last_token);
      const float e = j <= token ? __builtin_amdgcn_exp2f(p[r] - run.m) : 0.0f;
      run.l += e;
      const float w = e * factor;
      bool strange = false;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        float x = 0.0f;
        if (there && (HS % 32 == 0 || 32 * t + col < HS)) x = v[32 * t + col];
        const bool fine = __builtin_fabsf(x) < __builtin_inff();
        strange |= !fine;
        o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(fine ? x : 0.0f, w, o[t], 0, 0, 0);
      }
      // a value that is not finite is left out of the product (which would carry it to rows that do not see it) and makes
      // the rows that see it not a number
      const uint64_t any = __ballot(strange);
      const int j0 = p0 + 8 * (r / 4) + r % 4;
      if (((uint32_t)any && j0 <= token) || ((uint32_t)(any >> 32) && j0 + 4 <= token)) bad = __builtin_nanf("");
    }
    run.l += bad;
  }

  const float sum = run.l + other_half(run.l);
  const float scale = __builtin_amdgcn_exp2f(run.mw - run.m - 14.0f) / sum;
  if (!row) return;
  float *out = a.out + (int64_t)(token - pos) * a.out_stride + qhead * HS;
#pragma unroll
  for (int t = 0; t < TILES; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * t + 8 * (r / 4) + 4 * half;
      if (HS % 32 == 0 || d < HS)
        *reinterpret_cast<float4 *>(out + d) =
            make_float4(o[t][r] * scale, o[t][r + 1] * scale, o[t][r + 2] * scale, o[t][r + 3] * scale);
    }
}

}  // namespace

int64_t cache_attention_workspace(const CacheView &, int32_t, int32_t) { return 0; }

hipError_t launch_cache_attention(const CacheAttn &args, hipStream_t s) {
  CacheAttn a = args;
  a.rows.displaced = cache_displaces(a.rows.pos, a.rows.count);
  // tokens a tile: the largest power of two whose rows (token, query head) are at most 32, so that tiles that start at its
  // multiples never straddle two blocks
  const int group = a.nh / a.rows.c.nkv;
  int log2 = 0;
  while (log2 < 5 && (2 << log2) * group <= 32) ++log2;
  const int tiles = ((a.rows.pos + a.rows.count - 1) >> log2) - (a.rows.pos >> log2) + 1;
  const dim3 grid((tiles + 3) / 4, a.rows.c.nkv);
  switch (a.rows.c.hs) {
    case 16: hipLaunchKernelGGL(attend_kernel<16>, grid, dim3(256), 0, s, a, log2); break;
    case 32: hipLaunchKernelGGL(attend_kernel<32>, grid, dim3(256), 0, s, a, log2); break;
    case 48: hipLaunchKernelGGL(attend_kernel<48>, grid, dim3(256), 0, s, a, log2); break;
    case 64: hipLaunchKernelGGL(attend_kernel<64>, grid, dim3(256), 0, s, a, log2); break;
    case 96: hipLaunchKernelGGL(attend_kernel<96>, grid, dim3(256), 0, s, a, log2); break;
    case 128: hipLaunchKernelGGL(attend_kernel<128>, grid, dim3(256), 0, s, a, log2); break;
    case 256: hipLaunchKernelGGL(attend_kernel<256>, grid, dim3(256), 0, s, a, log2); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ple
