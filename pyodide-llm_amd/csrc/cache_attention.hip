// cache_attention.hip — attention over the cache held in 8 bits (cache.hpp): softmax_j(q . k_j / sqrt(hs)) v_j of a token
// at position p over the positions before its block of 32 by their 8-bit values, and over its own block's up to p by their
// float32 rows.
//
// A wave takes 32 rows (tokens x query heads of one kv head) of one block of positions and goes over the cache's blocks
// once, with a running maximum and sum. The rows are the columns of every product, so that a row's statistics live in its
// lane (and the lane 32 past it):
//   S^T = K Q^T on i8 MFMA: a query in three signed base-256 digits, x = round(q * 4160000 / max|q|) = 65536 d0 + 256 d1 +
//     d2: float32's precision (2^-23 of the row's largest), the keys' bytes as they lie, the int32 sums exact;
//   O^T = V^T P^T on f16 MFMA: the values' bytes are exact in f16, a probability goes in two halves (22 bits).
// Maxima are rounded up to whole powers of two, so that every rescaling is exact; the products' scale (2^mw - 14) follows
// the largest probability times its block's value scale, so that halves neither overflow nor lose bits where the blocks'
// scales differ.
//
// What bounds it: 32 rows by 32 positions of 128 channels take 28 MFMAs (890 cycles) and about 290 VALU instructions (1200),
// and a launch takes about as long as the two one after the other (two waves a SIMD, each with its own in turn): 2048 tokens of
// 32 / 8 heads of 128 from the start take 88 to 92 us, 1001 of 28 / 4 at 20,003 580 to 590 (500 TFLOP/s of the attention's 4 hs
// a score). One token over 131,077 positions, 268 MB, takes 54 us (4.9 TB/s; a plain streaming read of as much 44); over 4077
// 9.6, which is latency: a chain of loads, products and two barriers for the token's own block, a second launch that joins the
// parts.
#include <algorithm>

#include "cache.hpp"

namespace ple {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float LOG2E = 1.44269504088896341f;
constexpr float DIGITS = 4160000.0f;  // a query's largest value in digits (below 2^22 - 0x8080)
constexpr float NONE = -1e30f;  // no maximum yet (finite: its differences stay numbers)

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// 2^n of a whole n <= 0, what one reference is to another: a denormal too, which the exponential's instruction gives as 0
// (values below 2^-106 in 8 bits beside an own block would vanish)
__device__ __forceinline__ float power(float n) {
  return __builtin_amdgcn_ldexpf(1.0f, (int)__builtin_fmaxf(n, -200.0f));
}

// four of a query's values as three words of digits: round(x m) = 65536 d0 + 256 d1 + d2, below 2^22. Added to 1.5 * 2^23
// + 0x8080, the sum's low three bytes are d0 + 64, d1 + 128 and d2 + 128; they are gathered by value and taken back.
// (16 instructions; with conversions, shifts and masks 72)
__device__ __forceinline__ void digits(const float4 x, float m, int32_t &d0, int32_t &d1, int32_t &d2) {
  constexpr float BIAS = 12582912.0f + 32896.0f;
  const uint32_t a = __float_as_uint(__builtin_fmaf(x.x, m, BIAS)), b = __float_as_uint(__builtin_fmaf(x.y, m, BIAS)),
                 c = __float_as_uint(__builtin_fmaf(x.z, m, BIAS)), d = __float_as_uint(__builtin_fmaf(x.w, m, BIAS));
  const uint32_t low = __builtin_amdgcn_perm(b, a, 0x05010400u), high = __builtin_amdgcn_perm(d, c, 0x05010400u);
  d2 = (int32_t)(__builtin_amdgcn_perm(high, low, 0x05040100u) ^ 0x80808080u);
  d1 = (int32_t)(__builtin_amdgcn_perm(high, low, 0x07060302u) ^ 0x80808080u);
  const uint32_t top = __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0602u), __builtin_amdgcn_perm(b, a, 0x0c0c0602u),
                                             0x05040100u);
  d0 = (int32_t)(((top | 0x80808080u) - 0x40404040u) ^ 0x80808080u);  // (no byte borrows from the next)
}

// four value bytes (value + 128) as two pairs of halves: 0x6400 | byte is 1024 + byte
__device__ __forceinline__ void widen(uint32_t w, f16x2 &a, f16x2 &b) {
  const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - bias;
  b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - bias;
}

// w in two halves, hi + lo = w to 22 bits, of two values at once. (What is left of w is taken from the very register that
// goes to the product: formed from w anew, by an instruction that rounds the exponential's product once or twice, the half
// taken off could be an f16 step from the one kept.)
__device__ __forceinline__ void split(float w0, float w1, f16x2 &hi, f16x2 &lo) {
  const f16x2 h = {(_Float16)w0, (_Float16)w1};
  uint32_t bits = __builtin_bit_cast(uint32_t, h);
  float r0, r1;
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r0) : "v"(bits), "v"(w0));
  asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r1) : "v"(bits), "v"(w1));
  asm volatile("" : "+v"(bits));
  hi = __builtin_bit_cast(f16x2, bits);
  lo = f16x2{(_Float16)r0, (_Float16)r1};
}

// a row's running statistics: scores are in powers of two
struct Running {
  float m, l;  // sum of 2^(score - m), this lane's half of the positions
  float mw;    // the products' reference: O holds sum of 2^(score - mw + 14) value
};

// A wave's 32 rows: the tokens and query heads of its lanes' columns, the queries' digits, the running statistics and the
// output's columns
template <int HS>
struct Tile {
  static constexpr int STEPS = (HS + 31) / 32, TILES = (HS + 31) / 32;
  int lane, col, half, head, pos, group, first_token, last_token, own, token, qhead;
  bool row;
  const float *q;
  float unit, from_digits;
  i32x4 q0[STEPS], q1[STEPS], q2[STEPS];
  Running run;
  f32x16 o[TILES];

  // the rows of tile `index` (of 2^tokens_log2 tokens, from the multiple that holds pos on)
  __device__ __forceinline__ void place(const CacheAttn &a, int index, int tokens_log2) {
    lane = threadIdx.x % 64;
    col = lane % 32;
    half = lane / 32;
    pos = a.rows.dpos ? *a.rows.dpos : a.rows.pos;
    const int end = pos + a.rows.count;
    group = a.nh / a.rows.c.nkv;
    first_token = ((pos >> tokens_log2) + index) << tokens_log2;
    last_token = min(end, first_token + (1 << tokens_log2)) - 1;
    own = first_token / CACHE_BLOCK;  // the tile's tokens lie in one block
    const int mine = (int)(((float)col + 0.5f) * __builtin_amdgcn_rcpf((float)group));  // col / group
    token = first_token + mine;
    row = mine < (1 << tokens_log2) && token >= pos && token < end;
    qhead = head * group + col - mine * group;
    q = a.q + (int64_t)(row ? token - pos : 0) * a.q_stride + qhead * HS;
    unit = LOG2E / __builtin_sqrtf((float)HS);
    run = {NONE, 0.0f, NONE};
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = (f32x16)(0.0f);
  }

  // the queries' digits: lane (row, half) holds channels 32 s + 16 half .. + 15 of step s. (Every load first, none behind a
  // branch: one after the other they took 6 us. The first block's bytes are asked for right behind them.)
  __device__ __forceinline__ void read_queries(const CacheView &c, int first) {
    float4 x[STEPS][4];
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) x[s][j] = make_float4(0, 0, 0, 0);
    if (row) {  // (a column without a row asks for nothing: a wave's 1 KiB load takes 16 cycles of the CU's one port)
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int d = 32 * s + 16 * half;
        if (HS % 32 && d >= HS) continue;
        const float4 *from = reinterpret_cast<const float4 *>(q + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[s][j] = from[j];
      }
    }
    start(c, first);
    float largest = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        largest = wmax(largest, wmax(wmax(__builtin_fabsf(x[s][j].x), __builtin_fabsf(x[s][j].y)),
                                     wmax(__builtin_fabsf(x[s][j].z), __builtin_fabsf(x[s][j].w))));
      }
    largest = wmax(largest, other_half(largest));
    // (below 2^-100 a query is taken as zero; one that is not finite makes its row's scores not a number)
    const bool finite = largest < __builtin_inff();
    const float to_digits = finite && largest > 0x1p-100f ? DIGITS / largest : 0.0f;
    from_digits = finite ? largest / DIGITS * unit : __builtin_nanf("");
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        int32_t d0, d1, d2;
        digits(x[s][j], to_digits, d0, d1, d2);
        q0[s][j] = d0;
        q1[s][j] = d1;
        q2[s][j] = d2;
      }
  }

  // the statistics after positions whose largest score is `top`, of values up to 2^bits
  __device__ __forceinline__ void advance(float top, float bits) {
    const float up = __builtin_ceilf(top), m = __builtin_fmaxf(run.m, up), mw = __builtin_fmaxf(run.mw, up + bits);
    run.l *= __builtin_amdgcn_exp2f(run.m - m);
    const float gamma = power(run.mw - mw);
    if (__any(gamma != 1.0f)) {
#pragma unroll
      for (int t = 0; t < TILES; ++t) o[t] *= gamma;
    }
    run.m = m;
    run.mw = mw;
  }

  // the bytes and scales of a block
  i32x4 k[STEPS], v[TILES];
  const int8_t *kp;
  const uint8_t *vp;
  const float2 *sp;
  __device__ __forceinline__ void load_keys(int b) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      k[s] = (i32x4)(0);
      if (HS % 32 == 0 || 32 * s + 16 * half < HS)
        k[s] = *reinterpret_cast<const i32x4 *>(kp + (int64_t)b * (CACHE_BLOCK * HS) + s * (CACHE_BLOCK * 32));
    }
  }
  __device__ __forceinline__ void load_values(int b) {
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      v[t] = (i32x4)(0);
      if (HS % 32 == 0 || 32 * t + col < HS)
        v[t] = *reinterpret_cast<const i32x4 *>(vp + (int64_t)b * (CACHE_BLOCK * HS) + t * (32 * CACHE_BLOCK));
    }
  }
  // asks for the first block
  __device__ __forceinline__ void start(const CacheView &c, int first) {
    const int64_t at = (int64_t)head * c.blocks;
    kp = c.keys + at * (CACHE_BLOCK * HS) + half * (CACHE_BLOCK * 16) + col * 16;
    vp = c.values + at * (CACHE_BLOCK * HS) + col * CACHE_BLOCK + half * 16;
    sp = reinterpret_cast<const float2 *>(c.scales) + at;
    load_keys(first);
    load_values(first);
  }

  // blocks first, first + step, .. below to, by their 8-bit values, once start(first) has run: each one's bytes are asked for
  // once the products have taken those of the block before it
  __device__ __forceinline__ void blocks(int first, int to, int step) {
    i32x16 magic = (i32x16)(0x4B400000);  // (kept in registers where they suffice: made anew, it took 23 instructions a block)
    if (HS <= 128) asm volatile("" : "+v"(magic));
    for (int b = first; b < to; b += step) {
      const int next = b + step < to ? b + step : b;  // (the last one again, unused: a branch around the reads cost 10%)
      const float2 scale = sp[b];
      // 256 (K d0) + K d1 in one accumulator, K d2 in another that starts at 1.5 * 2^23's bits and is read as a float
      constexpr float MAGIC = 12582912.0f;
      i32x16 s0 = (i32x16)(0), s2 = magic;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) s0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[s], q0[s], s0, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) s2 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[s], q2[s], s2, 0, 0, 0);
      s0 <<= 8;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) s0 = __builtin_amdgcn_mfma_i32_32x32x32_i8(k[s], q1[s], s0, 0, 0, 0);
      const float ks = scale.x, vs = scale.y;
      load_keys(next);
      // a score (in powers of two): each (p - MAGIC)
      const float each = from_digits * ks;
      float p[16], top = -__builtin_inff();
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = __builtin_fmaf((float)s0[r], 256.0f, __int_as_float(s2[r]));
        top = __builtin_fmaxf(top, p[r]);
      }
      top = __builtin_fmaxf(top, other_half(top));
      advance((top - MAGIC) * each, vs > 0.0f ? (float)((int)(__float_as_uint(vs) >> 23) - 126) : -200.0f);
      // a probability comes with its block's value scale, 2^(score + log2 vs + 14 - mw), and goes to l with that taken back.
      // Where the block's values lie 2^100 below the reference (or are zero) they are left out, and l takes 2^(score - m)
      const float log_vs = __builtin_amdgcn_logf(vs), below = run.m - run.mw;
      const bool tiny = log_vs + below < -100.0f;
      const float scaled = tiny ? -below : log_vs, c = __builtin_fmaf(-MAGIC, each, scaled + 14.0f - run.mw);
      f16x8 hi[2], lo[2];
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float w0 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], each, c)),
                    w1 = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r + 1], each, c));
        sum += w0;
        sum += w1;
        f16x2 h, l;
        split(w0, w1, h, l);
        hi[r / 8][r % 8] = h[0];
        hi[r / 8][r % 8 + 1] = h[1];
        lo[r / 8][r % 8] = l[0];
        lo[r / 8][r % 8 + 1] = l[1];
      }
      run.l = __builtin_fmaf(sum, __builtin_amdgcn_exp2f(-14.0f - scaled - below), run.l);
      if (__any(tiny)) {
        const f16x8 zero = (f16x8)((_Float16)0.0f);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          hi[s] = tiny ? zero : hi[s];
          lo[s] = tiny ? zero : lo[s];
        }
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        f16x2 h[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) widen((uint32_t)v[t][j], h[2 * j], h[2 * j + 1]);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const f16x8 x = {h[4 * s][0], h[4 * s][1], h[4 * s + 1][0], h[4 * s + 1][1],
                           h[4 * s + 2][0], h[4 * s + 2][1], h[4 * s + 3][0], h[4 * s + 3][1]};
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, hi[s], o[t], 0, 0, 0);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, lo[s], o[t], 0, 0, 0);
        }
      }
      load_values(next);
    }
  }

  // The tile's own block by its float32 rows, up to the tile's last token, on float32 MFMA. PARTS waves share it (wave
  // `part`): each takes its share of the channels of the products of keys and queries, whose parts are added through
  // `shared` (PARTS x 64 x 16 floats; a barrier between own_scores and own_values), and of the output's; the sums of
  // probabilities count with part 0
  template <int PARTS>
  static constexpr int mine() {
    return PARTS > 1 ? (TILES + PARTS - 1) / PARTS : 1;
  }
  // the row of position p (this kv head's), for one that is not past the tile's last token
  __device__ __forceinline__ const float *source(const CacheAttn &a, const float *x, const float *recent, int p) const {
    const int kept = a.rows.displaced ? CACHE_RECENT + p % CACHE_BLOCK : p % CACHE_RECENT;
    const int64_t at = p >= pos ? (int64_t)(p - pos) * a.rows.x_stride : (int64_t)(kept * a.rows.c.nkv) * HS;
    return (p >= pos ? x : recent) + at + head * HS;
  }
  __device__ __forceinline__ void value_rows(const CacheAttn &a, const float *(&from)[16]) const {
#pragma unroll
    for (int r = 0; r < 16; ++r)
      from[r] = source(a, a.rows.v, a.rows.c.recent_values,
                       min(own * CACHE_BLOCK + 8 * (r / 4) + 4 * half + r % 4, last_token));
  }
  __device__ __forceinline__ void values(int t, const float *const (&from)[16], float (&to)[16]) const {
    const int d = HS % 32 == 0 || 32 * t + col < HS ? 32 * t + col : 0;
#pragma unroll
    for (int r = 0; r < 16; ++r) to[r] = from[r][d];
  }
  template <int PARTS>
  __device__ __forceinline__ void own_scores(const CacheAttn &a, int part, float *shared, float (&x)[mine<PARTS>()][16],
                                             f32x16 &s) const {
    // every load first: the keys and queries, and a shared block's values, which come while its scores are made
    constexpr int QUADS = (HS / 8 + PARTS - 1) / PARTS;
    const int key = min(own * CACHE_BLOCK + col, last_token);
    const float *k = source(a, a.rows.k, a.rows.c.recent_keys, key) + half * (HS / 2);
    const float *qh = q + half * (HS / 2);
    s = (f32x16)(0.0f);
    auto scores = [&](const float4 &kk, const float4 &y) {
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.x, y.x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.y, y.y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.z, y.z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_32x32x2f32(kk.w, y.w, s, 0, 0, 0);
    };
    if (PARTS > 1) {
      float4 kk[QUADS], y[QUADS];
#pragma unroll
      for (int n = 0; n < QUADS; ++n) {
        const int i = 4 * min(n * PARTS + part, HS / 8 - 1);
        kk[n] = *reinterpret_cast<const float4 *>(k + i);
        y[n] = *reinterpret_cast<const float4 *>(qh + i);
      }
      const float *from[16];
      value_rows(a, from);
#pragma unroll
      for (int i = 0; i < mine<PARTS>(); ++i) values(min(i * PARTS + part, TILES - 1), from, x[i]);
#pragma unroll
      for (int n = 0; n < QUADS; ++n)
        if (HS / 8 % PARTS == 0 || n * PARTS + part < HS / 8) scores(kk[n], y[n]);  // (the same in the whole wave)
#pragma unroll
      for (int r = 0; r < 16; ++r) shared[(part * 16 + r) * 64 + lane] = s[r];
    } else {
#pragma unroll 4
      for (int i = 0; i < HS / 2; i += 4)
        scores(*reinterpret_cast<const float4 *>(k + i), *reinterpret_cast<const float4 *>(qh + i));
    }
  }
  template <int PARTS>
  __device__ __forceinline__ void own_values(const CacheAttn &a, int part, const float *shared,
                                             float (&x)[mine<PARTS>()][16], f32x16 &s) {
    const int p0 = own * CACHE_BLOCK;
    if (PARTS > 1) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[r] = shared[r * 64 + lane];
#pragma unroll
        for (int w = 1; w < PARTS; ++w) s[r] += shared[(w * 16 + r) * 64 + lane];
      }
    }
    float p[16], top = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = p0 + 8 * (r / 4) + 4 * half + r % 4;
      // (an infinite score, of a key that is not finite: not a number, whichever its sign)
      p[r] = j <= token ? __builtin_fmaf(s[r], 0.0f, s[r] * unit) : -__builtin_inff();
      top = __builtin_fmaxf(top, p[r]);
    }
    top = __builtin_fmaxf(top, other_half(top));
    // (the reference lies 2^20 above the largest score: a probability comes as 2^-6 at most, and 32 of them times values of up to
    // the type's largest stay below 2^128. Their real size is not known yet where a wave reads them a part at a time)
    advance(top, 20.0f);
    const float factor = __builtin_amdgcn_exp2f(__builtin_fminf(run.m - run.mw + 14.0f, 126.0f));
    float sum = 0.0f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float e = __builtin_amdgcn_exp2f(p[r] - run.m);  // (0 behind the token)
      sum += e;
      p[r] = e * factor;
    }
    // a value that is not finite is left out of the product (which would carry it to rows that do not see it) and makes the
    // rows that see it not a number
    uint32_t strange = 0;  // bit r: this lane's value of its position r is not finite
    const float *from[16];
    if (PARTS == 1) value_rows(a, from);
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      if (PARTS > 1 && t % PARTS != part) continue;  // (the same in the whole wave)
      float(&v)[16] = x[PARTS > 1 ? t / PARTS : 0];
      if (PARTS == 1) values(t, from, v);
#pragma unroll
      for (int c = 0; c < 16; c += 4) {
        // (the same in the whole wave; where a wave reads its values only now, the branches would part its loads: 97 -> 108 us)
        if (PARTS > 1 && p0 + 2 * c > last_token) break;
#pragma unroll
        for (int r = c; r < c + 4; ++r) {
          const int j = p0 + 8 * (r / 4) + 4 * half + r % 4;
          if (j > last_token || (HS % 32 && 32 * t + col >= HS)) v[r] = 0.0f;
          const bool fine = __builtin_fabsf(v[r]) < __builtin_inff();
          strange |= fine ? 0u : 1u << r;
          o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(fine ? v[r] : 0.0f, p[r], o[t], 0, 0, 0);
        }
      }
    }
    float bad = 0.0f;
    if (__any(strange != 0)) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const uint64_t any = __ballot(strange >> r & 1);
        const int j0 = p0 + 8 * (r / 4) + r % 4;
        if (((uint32_t)any && j0 <= token) || ((uint32_t)(any >> 32) && j0 + 4 <= token)) bad = __builtin_nanf("");
      }
    }
    run.l = (PARTS > 1 && part ? 0.0f : run.l + sum) + bad;
  }
};

// Many tiles: one a wave. A workgroup of eight waves (four where a head's 256 values take twice the registers) takes half as
// many tiles in a row and as many as far from the end as these are from the start (`halves` such rows a kv head), so that
// every workgroup, and every SIMD, has as many blocks to go over as the others: a tile's blocks grow with its position. With
// parts > 1 a workgroup takes one part in `parts` of its tiles' blocks (the last the own block too) and leaves statistics and
// outputs in the workspace, as attend_part_kernel does.
// Workgroups that the eight XCDs take in turn are of different kv heads, so that an XCD's L2 holds few heads' blocks.
constexpr int OWN_BLOCKS = 8;
template <int HS>
constexpr int half_waves() { return HS <= 128 ? 4 : 2; }
template <int HS>
__global__ __launch_bounds__(128 * half_waves<HS>(), HS <= 128 ? 2 : 1) void attend_kernel(
    const CacheAttn a, int tokens_log2, int rows, int tiles, int halves, int parts) {
  constexpr int HALF = half_waves<HS>();
  Tile<HS> tile;
  const int wave = threadIdx.x / 64, nkv = a.rows.c.nkv;
  const int pair = blockIdx.x / nkv / parts, part = blockIdx.x / nkv % parts;
  const int half = wave < HALF ? pair : halves - 1 - pair, index = half * HALF + wave % HALF;
  if ((wave >= HALF && half == pair) || index >= tiles) return;  // (the middle row once; the last one's missing tiles)
  tile.head = blockIdx.x % nkv;
  tile.place(a, index, tokens_log2);
  // (the own block takes as long as eight earlier ones: 512 tokens 38 us with equal parts of these, 31 with it counted)
  const int units = tile.own + OWN_BLOCKS, from = min(tile.own, (int)((int64_t)units * part / parts)),
            to = part + 1 < parts ? min(tile.own, (int)((int64_t)units * (part + 1) / parts)) : tile.own;
  if (from < to) {
    tile.read_queries(a.rows.c, from);
    tile.blocks(from, to, 1);
  }
  if (part == parts - 1) {
    float x[Tile<HS>::template mine<1>()][16];
    f32x16 scores;
    tile.template own_scores<1>(a, 0, nullptr, x, scores);
    tile.template own_values<1>(a, 0, nullptr, x, scores);
  }
  const Running &run = tile.run;
  const float sum = run.l + other_half(run.l);
  if (tile.col >= rows || (parts == 1 && !tile.row)) return;
  float scale = 1.0f, *out;
  if (parts == 1) {
    scale = __builtin_amdgcn_exp2f(run.mw - run.m - 14.0f) / sum;
    out = a.out + (int64_t)(tile.token - tile.pos) * a.out_stride + tile.qhead * HS;
  } else {
    const int64_t at = (((int64_t)index * nkv + tile.head) * parts + part) * rows + tile.col;
    out = a.workspace + at * HS;
    if (tile.half == 0)
      reinterpret_cast<float4 *>(a.workspace + (int64_t)tiles * nkv * parts * rows * HS)[at] =
          make_float4(run.m, sum, run.mw, 0.0f);
  }
#pragma unroll
  for (int t = 0; t < Tile<HS>::TILES; ++t)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * t + 8 * (r / 4) + 4 * tile.half;
      const f32x16 &o = tile.o[t];
      if (HS % 32 == 0 || d < HS)
        *reinterpret_cast<float4 *>(out + d) =
            make_float4(o[r] * scale, o[r + 1] * scale, o[r + 2] * scale, o[r + 3] * scale);
    }
}

// The few parts of many rows together: four values of a (tile row, kv head, tile) a thread
template <int HS>
__global__ __launch_bounds__(256) void attend_join_rows_kernel(const CacheAttn a, int tokens_log2, int rows, int tiles,
                                                               int parts) {
  constexpr int QUADS = HS / 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, at = i / QUADS;  // (tile, kv head, row)
  const int nkv = a.rows.c.nkv, quad = (int)(i % QUADS), r = (int)(at % rows), group = a.nh / nkv;
  if (at >= (int64_t)tiles * nkv * rows) return;
  const int64_t unit = at / rows;
  const int tile = (int)(unit / nkv), head = (int)(unit % nkv), pos = a.rows.pos, mine = r / group;
  const int token = (((pos >> tokens_log2) + tile) << tokens_log2) + mine;
  if (token < pos || token >= pos + a.rows.count) return;
  const float4 *o = reinterpret_cast<const float4 *>(a.workspace) + (unit * parts * rows + r) * QUADS + quad;
  const float4 *stats = reinterpret_cast<const float4 *>(a.workspace + (int64_t)tiles * nkv * parts * rows * HS) +
                        unit * parts * rows + r;
  float m = NONE, l = 0.0f, mw = NONE;
  float4 y = make_float4(0, 0, 0, 0);
  for (int p = 0; p < parts; ++p) {
    const float4 x = o[(int64_t)p * rows * QUADS], s = stats[(int64_t)p * rows];
    const float top = __builtin_fmaxf(m, s.x), high = __builtin_fmaxf(mw, s.z);
    l = l * __builtin_amdgcn_exp2f(m - top) + s.y * __builtin_amdgcn_exp2f(s.x - top);
    const float f = power(mw - high), g = power(s.z - high);
    y = make_float4(y.x * f + x.x * g, y.y * f + x.y * g, y.z * f + x.z * g, y.w * f + x.w * g);
    m = top;
    mw = high;
  }
  const float scale = __builtin_amdgcn_exp2f(mw - m - 14.0f) / l;
  float *out = a.out + (int64_t)(token - pos) * a.out_stride + (head * group + r - mine * group) * HS + 4 * quad;
  *reinterpret_cast<float4 *>(out) = make_float4(y.x * scale, y.y * scale, y.z * scale, y.w * scale);
}

// The parts a tile's `own` earlier blocks are split into: a block for each of a part's four waves at least, and as many that
// the launch is one workgroup a CU (`most`, most_parts; 257 workgroups take 3 us more than 256), or two where that leaves
// waves more than eight blocks and the registers allow it. (By the tile alone, not by the launch, which may not know its
// position: the same sums either way.) 8 kv heads of 128, a token behind 16k, 32k, 64k, 128k positions: one a CU 13.9, 18.3,
// 34.6, 60.9 us, two 14.2, 18.7, 34.1, 57.7; of 256 values behind 32k, 64k: 35.7, 60.2, two 41.0, 66.5.
constexpr int PARTS_MOST = 255;  // (attend_join_kernel takes one more, the own block's)
template <int HS>
__host__ __device__ inline int parts_of(int own, int most) {
  if (HS <= 128 && own > 8 * 4 * most) most = most < PARTS_MOST / 2 ? 2 * most + 1 : PARTS_MOST;
  const int parts = (own + 3) / 4;
  return parts < 1 ? 1 : parts < most ? parts : most;
}

// Few tiles: the blocks of a tile in parts, one a workgroup, whose four waves take them in turn, and one part more for the
// tile's own block (the first, which takes the longest). 37 tokens of 32 / 8 heads at 1500 take 14.2 us (unsplit, a wave a
// tile, 86); one token over 32,001 of 28 / 4 13.5. A part's statistics (m, l, mw) and outputs go to the
// workspace: outputs [tile][kv head][part][rows][HS], then statistics [tile][kv head][part][rows] of 4 floats.
template <int HS>
__global__ __launch_bounds__(256, HS <= 128 ? 2 : 1) void attend_part_kernel(const CacheAttn a, int tokens_log2, int rows, int most) {
  extern __shared__ float4 lds[];
  constexpr int STRIDE = HS + 4;  // (rows of a wave's outputs 4 banks apart)
  float *const shared = reinterpret_cast<float *>(lds);
  __shared__ float stats[4][32][3];
  const int wave = threadIdx.x / 64, part = blockIdx.x;
  Tile<HS> tile;
  tile.head = blockIdx.z;
  tile.place(a, blockIdx.y, tokens_log2);
  const int splits = parts_of<HS>(tile.own, most);
  if (part > splits) return;  // (the whole workgroup)
  if (part == 0) {
    float x[Tile<HS>::template mine<4>()][16];
    f32x16 scores;
    tile.template own_scores<4>(a, wave, shared, x, scores);
    __syncthreads();
    tile.template own_values<4>(a, wave, shared, x, scores);
    __syncthreads();  // (shared holds the outputs next)
  } else {
    const int from = (int)((int64_t)tile.own * (part - 1) / splits), to = (int)((int64_t)tile.own * part / splits);
    if (from + wave < to) {
      tile.read_queries(a.rows.c, from + wave);
      tile.blocks(from + wave, to, 4);
    }
  }
  // the four waves' outputs and statistics through LDS, put on one reference by the threads that add them
  const Running &run = tile.run;
  const float sum = run.l + other_half(run.l);
  if (tile.half == 0) {
    stats[wave][tile.col][0] = run.m;
    stats[wave][tile.col][1] = sum;
    stats[wave][tile.col][2] = run.mw;
  }
  if (tile.col < rows) {
#pragma unroll
    for (int t = 0; t < Tile<HS>::TILES; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * t + 8 * (r / 4) + 4 * tile.half;
        const f32x16 &o = tile.o[t];
        if (HS % 32 == 0 || d < HS)
          *reinterpret_cast<float4 *>(shared + (wave * rows + tile.col) * STRIDE + d) =
              make_float4(o[r], o[r + 1], o[r + 2], o[r + 3]);
      }
  }
  __syncthreads();
  const int64_t at = ((int64_t)blockIdx.y * gridDim.z + blockIdx.z) * gridDim.x + part;
  float4 *const out = reinterpret_cast<float4 *>(a.workspace) + at * rows * (HS / 4);
  for (int i = threadIdx.x; i < rows * (HS / 4); i += 256) {
    const int row = i / (HS / 4);
    const float *x = shared + row * STRIDE + i % (HS / 4) * 4;
    float mw = NONE;
#pragma unroll
    for (int w = 0; w < 4; ++w) mw = __builtin_fmaxf(mw, stats[w][row][2]);
    float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 z = *reinterpret_cast<const float4 *>(x + w * rows * STRIDE);
      const float f = power(stats[w][row][2] - mw);
      y.x = __builtin_fmaf(z.x, f, y.x);
      y.y = __builtin_fmaf(z.y, f, y.y);
      y.z = __builtin_fmaf(z.z, f, y.z);
      y.w = __builtin_fmaf(z.w, f, y.w);
    }
    out[i] = y;
  }
  float m = NONE, l = 0.0f, mw = NONE;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    m = __builtin_fmaxf(m, stats[w][tile.col][0]);
    mw = __builtin_fmaxf(mw, stats[w][tile.col][2]);
  }
#pragma unroll
  for (int w = 0; w < 4; ++w) l += stats[w][tile.col][1] * __builtin_amdgcn_exp2f(stats[w][tile.col][0] - m);
  if (threadIdx.x < rows)  // (wave 0: lane = column)
    (reinterpret_cast<float4 *>(a.workspace) + (int64_t)gridDim.x * gridDim.y * gridDim.z * rows * (HS / 4))[
        at * rows + tile.col] = make_float4(m, l, mw, 0.0f);
}

// One token over a short cache (short_cache): a workgroup of eight waves a kv head, four for the token's own block and four
// for the earlier ones, whose outputs are put together through LDS: one launch in place of the parts and their join. By the
// cache's size, not the token's position, which a launch may not know. At the end of a cache of 256, 512, 1024 positions, one
// launch against the parts: 6 kv heads of 48 7.4, 9.0, 11.9 us against 8.8; 8 of 64 7.2, 8.5, 11.2 against 8.6; 8 of 128 9.1,
// 10.9, 14.5 against 9.1.
constexpr bool short_cache(int blocks, int hs) { return blocks <= 16 && blocks * hs <= 1024; }
template <int HS>
__global__ __launch_bounds__(512, HS <= 128 ? 2 : 1) void attend_short_kernel(const CacheAttn a, int rows) {
  extern __shared__ float4 lds[];
  constexpr int STRIDE = HS + 4;
  float *const shared = reinterpret_cast<float *>(lds), *const outputs = shared + 4 * 16 * 64;
  __shared__ float stats[8][32][3];
  const int wave = threadIdx.x / 64;
  Tile<HS> tile;
  tile.head = blockIdx.x;
  tile.place(a, 0, 0);
  float x[Tile<HS>::template mine<4>()][16];
  f32x16 scores;
  if (wave < 4) {
    tile.template own_scores<4>(a, wave, shared, x, scores);
  } else if (wave - 4 < tile.own) {
    tile.read_queries(a.rows.c, wave - 4);
    tile.blocks(wave - 4, tile.own, 4);
  }
  __syncthreads();
  if (wave < 4) tile.template own_values<4>(a, wave, shared, x, scores);
  const Running &run = tile.run;
  const float sum = run.l + other_half(run.l);
  if (tile.half == 0) {
    stats[wave][tile.col][0] = run.m;
    stats[wave][tile.col][1] = sum;
    stats[wave][tile.col][2] = run.mw;
  }
  if (tile.col < rows) {
#pragma unroll
    for (int t = 0; t < Tile<HS>::TILES; ++t)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const int d = 32 * t + 8 * (r / 4) + 4 * tile.half;
        const f32x16 &o = tile.o[t];
        if (HS % 32 == 0 || d < HS)
          *reinterpret_cast<float4 *>(outputs + (wave * rows + tile.col) * STRIDE + d) =
              make_float4(o[r], o[r + 1], o[r + 2], o[r + 3]);
      }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (HS / 4); i += 512) {
    const int row = i / (HS / 4);
    const float *from = outputs + row * STRIDE + i % (HS / 4) * 4;
    float m = NONE, mw = NONE, l = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      m = __builtin_fmaxf(m, stats[w][row][0]);
      mw = __builtin_fmaxf(mw, stats[w][row][2]);
    }
    float4 y = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const float4 z = *reinterpret_cast<const float4 *>(from + w * rows * STRIDE);
      const float f = power(stats[w][row][2] - mw);
      l += stats[w][row][1] * __builtin_amdgcn_exp2f(stats[w][row][0] - m);
      y.x = __builtin_fmaf(z.x, f, y.x);
      y.y = __builtin_fmaf(z.y, f, y.y);
      y.z = __builtin_fmaf(z.z, f, y.z);
      y.w = __builtin_fmaf(z.w, f, y.w);
    }
    const float scale = __builtin_amdgcn_exp2f(mw - m - 14.0f) / l;
    float *out = a.out + ((int)blockIdx.x * rows + row) * HS + i % (HS / 4) * 4;
    *reinterpret_cast<float4 *>(out) = make_float4(y.x * scale, y.y * scale, y.z * scale, y.w * scale);
  }
}

// A row's parts together: one (tile row, kv head, tile) a workgroup
template <int HS>
__global__ __launch_bounds__(256) void attend_join_kernel(const CacheAttn a, int tokens_log2, int rows, int most, int stride) {
  constexpr int QUADS = HS / 4, GROUPS = 256 / QUADS;
  constexpr int AHEAD = 8;  // parts a thread reads before it knows their weights
  __shared__ float4 sums[GROUPS * QUADS];
  __shared__ float scales[4][256];
  const int tid = threadIdx.x, lane = tid % 64, r = blockIdx.x, head = blockIdx.y, tile = blockIdx.z;
  const int pos = a.rows.dpos ? *a.rows.dpos : a.rows.pos, group = a.nh / a.rows.c.nkv;
  const int mine = (int)(((float)r + 0.5f) * __builtin_amdgcn_rcpf((float)group));  // r / group
  const int token = (((pos >> tokens_log2) + tile) << tokens_log2) + mine;
  if (token < pos || token >= pos + a.rows.count) return;  // (the whole workgroup)
  const int parts = parts_of<HS>(token / CACHE_BLOCK, most) + 1;
  const int64_t at = ((int64_t)tile * gridDim.y + head) * stride;
  const float4 *o = reinterpret_cast<const float4 *>(a.workspace) + (at * rows + r) * QUADS + tid % QUADS;
  const float4 *stats = reinterpret_cast<const float4 *>(a.workspace) + (int64_t)stride * gridDim.y * gridDim.z * rows * QUADS +
                        at * rows + r;
  float4 stat[4], x[AHEAD];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    stat[j] = make_float4(NONE, 0.0f, NONE, 0.0f);
    if (lane + 64 * j < parts) stat[j] = stats[(int64_t)(lane + 64 * j) * rows];
  }
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    x[i] = o[(int64_t)min(tid / QUADS + i * GROUPS, parts - 1) * rows * QUADS];
  // (every wave for itself: no barrier before the sums)
  float m = NONE, mw = NONE, l = 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    m = __builtin_fmaxf(m, stat[j].x);
    mw = __builtin_fmaxf(mw, stat[j].z);
  }
  m = wave_top(m);
  mw = wave_top(mw);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    l += stat[j].y * __builtin_amdgcn_exp2f(stat[j].x - m);
    scales[tid / 64][lane + 64 * j] = power(stat[j].z - mw);
  }
  l = wave_sum(l);
  wave_sync_lds();
  if (tid < GROUPS * QUADS) {
    float4 y = make_float4(0, 0, 0, 0);
    auto add = [&](const float4 &v, int p) {
      const float f = scales[tid / 64][p];
      y.x = __builtin_fmaf(v.x, f, y.x);
      y.y = __builtin_fmaf(v.y, f, y.y);
      y.z = __builtin_fmaf(v.z, f, y.z);
      y.w = __builtin_fmaf(v.w, f, y.w);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      if (tid / QUADS + i * GROUPS < parts) add(x[i], tid / QUADS + i * GROUPS);
    for (int p = tid / QUADS + AHEAD * GROUPS; p < parts; p += GROUPS) add(o[(int64_t)p * rows * QUADS], p);
    sums[tid] = y;
  }
  __syncthreads();
  if (tid >= QUADS) return;
  float4 y = sums[tid];
#pragma unroll
  for (int g = 1; g < GROUPS; ++g) {
    const float4 z = sums[g * QUADS + tid];
    y.x += z.x;
    y.y += z.y;
    y.z += z.z;
    y.w += z.w;
  }
  const float scale = __builtin_amdgcn_exp2f(mw - m - 14.0f) / l;
  float *out = a.out + (int64_t)(token - pos) * a.out_stride + (head * group + r - mine * group) * HS + 4 * tid;
  *reinterpret_cast<float4 *>(out) = make_float4(y.x * scale, y.y * scale, y.z * scale, y.w * scale);
}

// How a call is laid out: the tokens a tile takes (2^log2: the largest power of two whose rows, token and query head, are at
// most 32, and no larger than the call needs; tiles start at its multiples, so that none straddles two blocks); with many tiles
// (at least FEW waves of them) one a wave, their blocks in `parts`; with few, and for a single token, whose position the launch
// may not know, each tile's blocks in at most `most` parts
struct Layout {
  int log2, rows, tiles, most, parts;
};
constexpr int FEW = 192;
int tokens_log2(int group, int count) {
  int log2 = 0;
  while (log2 < 5 && (2 << log2) * group <= 32 && 1 << log2 < count) ++log2;
  return log2;
}
// (each tile's own block is a part more)
int most_parts(int64_t waves) { return (int)std::min<int64_t>(PARTS_MOST, std::max<int64_t>(1, 256 / waves - 1)); }
// parts that fill the card's SIMDs with two waves (one where a head's 256 values take twice the registers), of two blocks at
// least
int tile_parts(int64_t waves, int hs, int blocks) {
  return (int)std::max<int64_t>(1, std::min<int64_t>({16, (hs <= 128 ? 2048 : 1024) / waves, blocks / 2}));
}
Layout layout_of(const CacheAttn &a) {
  Layout l;
  const int group = a.nh / a.rows.c.nkv, last = a.rows.pos + a.rows.count - 1;
  l.log2 = tokens_log2(group, a.rows.count);
  l.rows = group << l.log2;
  l.tiles = (last >> l.log2) - (a.rows.pos >> l.log2) + 1;
  const int64_t waves = (int64_t)l.tiles * a.rows.c.nkv;
  l.most = waves < FEW || a.rows.count == 1 ? most_parts(waves) : 0;
  l.parts = tile_parts(waves, a.rows.c.hs, last / CACHE_BLOCK);
  return l;
}

template <int HS>
hipError_t launch(const CacheAttn &a, hipStream_t s) {
  const Layout l = layout_of(a);
  const int last = (a.rows.pos + a.rows.count - 1) / CACHE_BLOCK;
  if constexpr (HS <= 128) {
    const size_t bytes = (4 * 16 * 64 + 8 * l.rows * (HS + 4)) * sizeof(float);
    if (a.rows.count == 1 && short_cache(a.rows.c.blocks, HS) && bytes <= 65536 - 4096) {  // (and `stats`)
      hipLaunchKernelGGL(attend_short_kernel<HS>, dim3(a.rows.c.nkv), dim3(512), bytes, s, a, l.rows);
      return hipGetLastError();
    }
  }
  if (!l.most) {
    const int halves = (l.tiles + half_waves<HS>() - 1) / half_waves<HS>();
    hipLaunchKernelGGL(attend_kernel<HS>, dim3((halves + 1) / 2 * a.rows.c.nkv * l.parts), dim3(128 * half_waves<HS>()), 0, s,
                       a, l.log2, l.rows, l.tiles, halves, l.parts);
    if (l.parts > 1) {
      const int64_t threads = (int64_t)l.tiles * a.rows.c.nkv * l.rows * (HS / 4);
      hipLaunchKernelGGL(attend_join_rows_kernel<HS>, dim3((uint32_t)((threads + 255) / 256)), dim3(256), 0, s, a, l.log2,
                         l.rows, l.tiles, l.parts);
    }
    return hipGetLastError();
  }
  const size_t bytes = std::max<size_t>(4 * l.rows * (HS + 4), 4 * 16 * 64) * sizeof(float);
  if (bytes + sizeof(float[4][32][3]) > 65536) {  // (and `stats`)
    const hipError_t err = hipFuncSetAttribute(reinterpret_cast<const void *>(attend_part_kernel<HS>),
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (err != hipSuccess) return err;
  }
  const int stride = parts_of<HS>(last, l.most) + 1;
  hipLaunchKernelGGL(attend_part_kernel<HS>, dim3(stride, l.tiles, a.rows.c.nkv), dim3(256), bytes, s, a, l.log2, l.rows,
                     l.most);
  hipLaunchKernelGGL(attend_join_kernel<HS>, dim3(l.rows, a.rows.c.nkv, l.tiles), dim3(256), 0, s, a, l.log2, l.rows,
                     l.most, stride);
  return hipGetLastError();
}

}  // namespace

// (the most over the positions: count tokens make one tile more where they start inside one)
int64_t cache_attention_workspace(const CacheView &c, int32_t nh, int32_t count) {
  const int log2 = tokens_log2(nh / c.nkv, count);
  const int64_t rows = nh / c.nkv << log2, fewest = ((int64_t)count + (1 << log2) - 1) >> log2;
  int64_t most = 0;
  for (int64_t tiles = fewest; tiles <= fewest + (count > 1); ++tiles) {
    const int64_t waves = tiles * c.nkv;
    int64_t parts;
    if (waves < FEW || count == 1) {
      parts = (c.hs <= 128 ? parts_of<16> : parts_of<256>)(c.blocks, most_parts(waves)) + 1;
    } else {
      parts = tile_parts(waves, c.hs, c.blocks);
      if (parts == 1) parts = 0;  // (nothing to join)
    }
    most = std::max(most, waves * parts * rows * (c.hs + 4) * (int64_t)sizeof(float));
  }
  return most;
}

hipError_t launch_cache_attention(const CacheAttn &args, hipStream_t s) {
  CacheAttn a = args;
  a.rows.displaced = cache_displaces(a.rows.pos, a.rows.count);
  switch (a.rows.c.hs) {
    case 16: return launch<16>(a, s);
    case 32: return launch<32>(a, s);
    case 48: return launch<48>(a, s);
    case 64: return launch<64>(a, s);
    case 96: return launch<96>(a, s);
    case 128: return launch<128>(a, s);
    case 256: return launch<256>(a, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace ple
