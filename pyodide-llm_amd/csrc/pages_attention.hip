// pages_attention.hip — attention of one new token a row over the cache in pages: softmax_j(q . k_j / sqrt(hs)) v_j over the
// first lengths[i] positions of its sequence.
//
// A workgroup takes the query heads of one kv head (up to 8 of them over a float16 cache, 16 over a float32 one) of one row
// over one part of its positions; its waves take the part's blocks of 32 positions in turn, each with a running maximum and
// sum, and join at the end; the parts of a longer row are joined by a second launch. The heads are the columns of every
// product, so that a head's statistics live in its lanes:
//   S^T = K Q^T: a lane's 16 bytes of a key row as they lie; the channels in the order that these loads give;
//   O^T = V^T P^T: the probabilities go from the first product's output registers to the second's input. A lane reads a
//     few neighbouring channels of its positions' value rows; channel i of each is one product's.
// A float16 cache's products are float16's, with float32's bits: queries and probabilities go in two halves, x = hi + lo / 2048,
// each rounded to nearest (2^-23 of x is left at most), in columns 0-7 and 8-15 of one product. A float32 cache's are float32's.
// Outputs are divided by the probabilities' sum at the end alone: what they add up to before has float32's range too.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 32;   // positions a wave takes at a time
constexpr int WAVES = 4;
constexpr int UNIT = BLOCK * WAVES, LEAST = 2;  // positions of a piece: a multiple of UNIT, at least LEAST of them
constexpr int PLANNED = 256;  // rows a launch's workgroups look through
constexpr float LOG2E = 1.44269504088896341f;
constexpr float INF = __builtin_inff();
constexpr float PIECE_UP = 64.0f;  // what float16 halves of probabilities are raised by: up to 2^15
constexpr float LOW = 2048.0f;     // the second half's scale
constexpr float WHOLE = 0x1p24f;   // from here on float32 has not every whole number
constexpr float LOWEST = -3.402823466e38f;

template <bool HALF>
struct Kind {
  typedef _Float16 type;
  static constexpr int heads = 8;
  // how far (log2) a score may lie above the reference (and its rounding) before that moves
  static constexpr float ahead = 8.0f;
};
template <>
struct Kind<false> {
  typedef float type;
  static constexpr int heads = 16;
  static constexpr float ahead = 0.0f;  // (values may be large: no probability is above 1, but for a score's rounding)
};

// lane ^ 8 within 16: the other half of a column's products
__device__ __forceinline__ float other_half(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, true));  // row_ror:8
}
// over a column's lanes (l, l ^ 16, l ^ 32)
template <class F>
__device__ __forceinline__ float column(float x, F f) {
  x = f(x, __shfl_xor(x, 16));
  return f(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float column_sum(float x) {
  return column(x, [](float a, float b) { return a + b; });
}
__device__ __forceinline__ float column_max(float x) {
  return column(x, [](float a, float b) { return __builtin_fmaxf(a, b); });
}

template <int BYTES>
struct Bits {
  typedef uint16_t type;
};
template <>
struct Bits<4> {
  typedef uint32_t type;
};

// channels a lane reads at once of a value row whose `rest` channels are left
template <bool HALF>
__host__ __device__ constexpr int width(int rest) {
  return HALF && rest >= 128 ? 8 : rest >= 64 ? 4 : rest >= 32 ? 2 : 1;
}

// a lane's values of 32 positions: channels BASE + W c.. of its eight positions, and those past BASE + 16 W
template <int HS, bool HALF, int BASE = 0>
struct Values {
  typedef typename Kind<HALF>::type T;
  static constexpr int W = width<HALF>(HS - BASE), AT = BASE / 16;
  typedef T piece __attribute__((ext_vector_type(W)));
  piece x[8];
  Values<HS, HALF, BASE + 16 * W> rest;

  __device__ __forceinline__ void read(const T *v, int c, int j) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      x[e] = *reinterpret_cast<const piece *>(v + ((e & 4) * 4 + 4 * j + (e & 3)) * HS + BASE + W * c);
    rest.read(v, c, j);
  }
  // zeros at the positions from `left` on (what lies behind the row's end may be anything): by masks, since selects of these
  // vectors became a branch under whose exec mask the compiler reused a value's registers (wrong outputs at heads of 128)
  __device__ __forceinline__ void cut(int left, int j) {
    typedef typename Bits<sizeof(T)>::type bits __attribute__((ext_vector_type(W)));
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int32_t keep = ((e & 4) * 4 + 4 * j + (e & 3) - left) >> 31;  // all ones before it
      x[e] = __builtin_bit_cast(piece, __builtin_bit_cast(bits, x[e]) & (bits)((typename Bits<sizeof(T)>::type)keep));
    }
    rest.cut(left, j);
  }
  // tiles of 16 channels: channel i of each lane's
  __device__ __forceinline__ void add(f32x4 *o, const f16x8 &ph, const f32x4 (&p)[2]) const {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (HALF) {
        f16x8 a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = x[e][i];
        o[AT + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, ph, o[AT + i], 0, 0, 0);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          o[AT + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e][i], p[e >> 2][e & 3], o[AT + i], 0, 0, 0);
      }
    }
    rest.add(o, ph, p);
  }
};
template <int HS, bool HALF>
struct Values<HS, HALF, HS> {
  typedef typename Kind<HALF>::type T;
  __device__ __forceinline__ void read(const T *, int, int) {}
  __device__ __forceinline__ void cut(int, int) {}
  __device__ __forceinline__ void add(f32x4 *, const f16x8 &, const f32x4 (&)[2]) const {}
};

// a wave's queries, accumulators and statistics
template <int HS, bool HALF>
struct Wave {
  typedef typename Kind<HALF>::type T;
  typedef T chunk __attribute__((ext_vector_type(16 / sizeof(T))));  // 16 bytes
  static constexpr int KEYS = HALF ? (HS + 31) / 32 : HS / 16;       // of them a lane takes of a key row
  static constexpr int TILES = HS / 16;
  float4 raw[HALF ? 2 * KEYS : KEYS];
  f16x8 q[HALF ? KEYS : 1];
  chunk k[2][KEYS];
  Values<HS, HALF> v;
  float up, up_low;  // what a product is multiplied by: a score in log2
  // the scores' reference, and how far above it one may lie (-INF: there is no reference yet; LOWEST: none is taken as it is)
  float reference = 0.0f, bar = -INF, sum = 0.0f;
  f32x4 o[TILES];
  int c, j;  // the lane's column and quarter

  __device__ __forceinline__ static bool within(int d) { return HS % 32 == 0 || !HALF || d < HS; }

  __device__ __forceinline__ void read_queries(const float *from, int heads) {
    const int h = min(HALF ? c & 7 : c, heads - 1);  // (columns past the heads: the last one's, to no end)
#pragma unroll
    for (int s = 0; s < KEYS; ++s) {
      const int d = HALF ? 32 * s + 8 * j : 16 * s + 4 * j;
      const float *at = from + h * HS + (within(d) ? d : 0);
      if constexpr (HALF) {
        raw[2 * s] = *reinterpret_cast<const float4 *>(at);
        raw[2 * s + 1] = *reinterpret_cast<const float4 *>(at + 4);
      } else {
        raw[s] = *reinterpret_cast<const float4 *>(at);
      }
    }
  }
  __device__ __forceinline__ void read_keys(const T *from) {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s = 0; s < KEYS; ++s) {
        const int d = HALF ? 32 * s + 8 * j : 16 * s + 4 * j;
        k[t][s] = *reinterpret_cast<const chunk *>(from + (16 * t + c) * HS + (within(d) ? d : 0));
      }
  }
  __device__ __forceinline__ void read_values(const T *from) { v.read(from, c, j); }

  // the queries as the products take them
  __device__ __forceinline__ void begin() {
    const float scale = LOG2E / __builtin_sqrtf((float)HS);
    if constexpr (HALF) {
      float most = 0.0f;
#pragma unroll
      for (int s = 0; s < KEYS; ++s) {
        if (!within(32 * s + 8 * j)) raw[2 * s] = raw[2 * s + 1] = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float4 x = raw[2 * s + i];
          most = __builtin_fmaxf(most, __builtin_fmaxf(__builtin_fmaxf(__builtin_fabsf(x.x), __builtin_fabsf(x.y)),
                                                       __builtin_fmaxf(__builtin_fabsf(x.z), __builtin_fabsf(x.w))));
        }
      }
      most = column_max(most);
      const int e = __builtin_amdgcn_frexp_expf(most);  // |q| < 2^e; (of 0 and of what is not finite 0)
#pragma unroll
      for (int s = 0; s < KEYS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float4 x = raw[2 * s + i / 4];
          const float y = __builtin_amdgcn_ldexpf(i % 4 == 0 ? x.x : i % 4 == 1 ? x.y : i % 4 == 2 ? x.z : x.w, 15 - e);
          const _Float16 hi = (_Float16)y;
          q[s][i] = c < 8 ? hi : (_Float16)((y - (float)hi) * LOW);
        }
      up = __builtin_amdgcn_ldexpf(scale, e - 15);
      up_low = __builtin_amdgcn_ldexpf(scale, e - 26);
    } else {
      up = scale;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = f32x4{0, 0, 0, 0};
  }

  // position 16 t + 4 j + r of column c in s[t][r]
  __device__ __forceinline__ void products(f32x4 (&s)[2]) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) s[t] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < KEYS; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if constexpr (HALF) {
          f16x8 x = k[t][i];
          if constexpr (HS % 32 != 0) {  // (the last load's upper half is past the row)
            typedef uint32_t words __attribute__((ext_vector_type(4)));
            if (i == KEYS - 1) x = __builtin_bit_cast(f16x8, __builtin_bit_cast(words, x) & (words)((uint32_t)((j - 2) >> 31)));
          }
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[i], s[t], 0, 0, 0);
        } else {
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i].x, raw[i].x, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i].y, raw[i].y, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i].z, raw[i].z, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][i].w, raw[i].w, s[t], 0, 0, 0);
        }
      }
  }

  // the products' scores (log2) over `from`, and the largest of the lane's: one rounding at their own size, not at the scores'
  __device__ __forceinline__ float scores(const f32x4 (&s)[2], f32x4 (&x)[2], int left, float from) const {
    float most = -INF;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float y;
        if constexpr (HALF) {
          const float other = other_half(s[t][r]);
          y = __builtin_fmaf(c < 8 ? other : s[t][r], up_low, __builtin_fmaf(c < 8 ? s[t][r] : other, up, -from));
        } else {
          y = __builtin_fmaf(s[t][r], up, -from);
        }
        if (16 * t + 4 * j + r >= left) y = -INF;
        x[t][r] = y;
        most = __builtin_fmaxf(most, y);
      }
    return most;
  }

  // the probabilities of the products' scores, as the second product takes them; `left` of the positions are the row's
  __device__ __forceinline__ void probabilities(const f32x4 (&s)[2], int left, f16x8 &ph, f32x4 (&p)[2]) {
    const float most = scores(s, p, left, reference);
    if (__any(most > bar)) {
      // the reference is the largest score as float32 has it, and what is held follows that: a score that is met again, and lies
      // above its float32, moves nothing
      const bool held = bar > -INF;
      const float top = column_max(__any(held) ? scores(s, p, left, 0.0f) : most);
      const float next = held ? __builtin_fmaxf(reference, top) : top > -INF ? top : 0.0f;
      if (__any(held && next != reference)) {
        const float less = held ? __builtin_amdgcn_exp2f(reference - next) : 1.0f;
        sum *= less;
#pragma unroll
        for (int t = 0; t < TILES; ++t) o[t] *= less;
      }
      reference = next;
      // From 2^24 on float32's numbers are two apart, and what a rounding leaves of a score is no exponent any more (from 2^28 on it
      // made infinities, or zeros everywhere): there the scores are float32's too, block by block
      const bool whole = __builtin_fabsf(next) >= WHOLE;
      if (top > -INF) bar = whole ? LOWEST : __builtin_fmaf(__builtin_fabsf(next), 0x1p-24f, Kind<HALF>::ahead);
      const f32x4 rounded[2] = {p[0], p[1]};
      scores(s, p, left, next);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) p[t][r] = whole ? rounded[t][r] - next : p[t][r];
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = __builtin_amdgcn_exp2f(p[t][r]);
        sum += x;
        if constexpr (HALF) {
          x *= PIECE_UP;
          const _Float16 hi = (_Float16)x;
          ph[4 * t + r] = c < 8 ? hi : (_Float16)((x - (float)hi) * LOW);
        }
        p[t][r] = x;
      }
  }
};

// channel of element r of quarter j's output in tile n (Values' order)
template <int HS, bool HALF>
__device__ __forceinline__ constexpr int channel(int n, int row) {
  int base = 0;
  while (n >= base / 16 + width<HALF>(HS - base)) base += 16 * width<HALF>(HS - base);
  return base + width<HALF>(HS - base) * row + n - base / 16;
}

// Which positions of which row a workgroup takes. Up to PLANNED rows a launch, every workgroup works that out from all lengths:
// the rows' positions, in units of UNIT, over the pieces that the launch is made for, are a piece's; a row longer than one has
// several, one after another, so that all are about equal whatever the rows' lengths are. Of more rows each has the same
// number of pieces (which lie behind its end if it is short).
struct Piece {
  int row, seq, len;    // len 0: no attention (zeros)
  bool wrong;           // a row that cannot be (NaN)
  int chunk;            // positions a piece
  int first, part;      // the row's first piece, and which of the row's this is
};

__device__ __forceinline__ bool impossible(const PagesAttn &a, int seq, int len) {
  return len > 0 && seq >= 0 && (seq >= a.c.n_seqs || len > a.longest || len > a.c.slots * a.c.page);
}

// `find`: the row, or the piece whose row is looked for (past the last: row -1)
template <bool ROW>
__device__ __forceinline__ Piece piece_of(const PagesAttn &a, int find, int lane) {
  Piece p;
  if (a.parts) {
    p.row = ROW ? find : find / a.parts;
    p.part = ROW ? 0 : find % a.parts;
    p.first = p.row * a.parts;
    p.chunk = a.chunk;
    p.len = a.lengths[p.row];
    p.seq = a.seqs ? a.seqs[p.row] : p.row;
    p.wrong = impossible(a, p.seq, p.len);
    if (p.seq < 0 || p.len < 0 || p.wrong) p.len = 0;
    return p;
  }
  int len, seq, units;
  bool wrong;
  auto read = [&](int row) {
    const int at = min(row, a.rows - 1);
    len = a.lengths[at];
    seq = a.seqs ? a.seqs[at] : at;
    wrong = impossible(a, seq, len);
    if (seq < 0 || len < 0 || wrong || row >= a.rows) len = 0;
    units = (len + UNIT - 1) / UNIT;
  };
  read(lane);
  uint32_t total = (uint32_t)__builtin_amdgcn_readlane((int)wave_up_to(units), 63);
  for (int base = 64; base < a.rows; base += 64) {
    read(base + lane);
    total += (uint32_t)__builtin_amdgcn_readlane((int)wave_up_to(units), 63);
  }
  // units a piece (the total may be 2^31)
  const uint32_t row_most = (a.longest + UNIT - 1) / UNIT;
  const int each = max(LEAST, (int)min((total + a.pieces - 1) / a.pieces, row_most));
  p.chunk = each * UNIT;
  p.row = -1;
  for (int base = 0, before = 0; base < a.rows; base += 64) {
    if (a.rows > 64) read(base + lane);
    const int mine = base + lane < a.rows ? max(1, (units + each - 1) / each) : 0;
    const int upto = before + (int)wave_up_to(mine);
    const uint64_t here = __ballot(ROW ? base + lane == find : upto > find && upto - mine <= find);
    if (here) {
      const int l = __builtin_ctzll(here);
      p.row = base + l;
      p.first = __builtin_amdgcn_readlane(upto - mine, l);
      p.part = ROW ? 0 : find - p.first;
      p.len = __builtin_amdgcn_readlane(len, l);
      p.seq = __builtin_amdgcn_readlane(seq, l);
      p.wrong = __builtin_amdgcn_readlane(wrong ? 1 : 0, l);
      break;
    }
    before = __builtin_amdgcn_readlane(upto, 63);
  }
  return p;
}

// a piece's results: references and sums [piece][head], then outputs [piece][head][HS]
__device__ __forceinline__ float2 *statistics(const PagesAttn &a, int64_t piece, int h) {
  return reinterpret_cast<float2 *>(a.workspace) + piece * a.nh + h;
}
template <int HS>
__device__ __forceinline__ float *outputs(const PagesAttn &a, int64_t piece, int h) {
  return a.workspace + ((a.most * a.nh * 2 + 3) & ~3) + (piece * a.nh + h) * HS;
}

// waves a SIMD that the registers are kept for: a block's keys and values, the queries and the outputs
constexpr int occupancy(int hs, bool half) {
  return half ? (hs <= 64 ? 4 : hs <= 128 ? 3 : 1) : (hs <= 48 ? 4 : hs <= 64 ? 3 : hs <= 128 ? 2 : 1);
}

template <int HS, bool HALF>
__global__ __launch_bounds__(64 * WAVES, occupancy(HS, HALF)) void attend_kernel(const PagesAttn a) {
  typedef typename Kind<HALF>::type T;
  constexpr int HEADS = Kind<HALF>::heads;
  __shared__ float tops[WAVES][HEADS], sums[WAVES][HEADS];
  __shared__ float outs[WAVES][HEADS][HS + 4];  // (a column's lanes four banks apart)
  const PagesView &c = a.c;
  const int group = a.nh / c.nkv, tiles = (group + HEADS - 1) / HEADS;
  const int g = blockIdx.y / tiles, first = g * group + blockIdx.y % tiles * HEADS;
  const int heads = min(HEADS, (g + 1) * group - first);
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const Piece piece = piece_of<false>(a, blockIdx.x, lane);
  const int row = piece.row, len = piece.len;
  if (row < 0) return;
  float *out = a.out + (int64_t)row * a.out_stride + (int64_t)first * HS;
  if (len == 0) {
    if (piece.part == 0)
      for (int i = tid; i < heads * HS; i += 64 * WAVES) out[i] = piece.wrong ? __builtin_nanf("") : 0.0f;
    return;
  }
  const int64_t begin = (int64_t)piece.part * piece.chunk;
  if (begin >= len) return;
  const int p0 = (int)begin + BLOCK * wave;  // the wave's first block
  const int p1 = (int)min((int64_t)len, begin + piece.chunk);
  // the pages of the wave's next 64 blocks, a lane each
  const int32_t *table = c.tables + (int64_t)piece.seq * c.slots;
  const int shift = __builtin_ctz(c.page);
  bool lost = false;
  auto pages = [&](int p) {
    const int64_t mine = min(p + (int64_t)lane * (BLOCK * WAVES), (int64_t)p1 - 1);  // (past the last: the last position's)
    const int32_t page = table[mine >> shift];
    const bool none = (uint32_t)page >= (uint32_t)c.n_pages;
    lost = lost || __any(none);
    return none ? 0 : page;
  };
  Wave<HS, HALF> w;
  w.c = lane & 15;
  w.j = lane >> 4;
  w.read_queries(a.q + (int64_t)row * a.q_stride + (int64_t)first * HS, heads);
  int32_t held = pages(p0);
  const int64_t layer = (int64_t)a.layer * c.n_pages;
  auto place = [&](int p, int turn) {
    if (turn % 64 == 0 && turn) held = pages(p);
    const int64_t page = __builtin_amdgcn_readlane(held, turn % 64);
    return (((layer + page) * c.nkv + g) * c.page + (p & (c.page - 1))) * HS;
  };
  const T *keys = reinterpret_cast<const T *>(c.keys), *values = reinterpret_cast<const T *>(c.values);
  int64_t at = 0;
  if (p0 < p1) {
    at = place(p0, 0);
    w.read_keys(keys + at);
    w.read_values(values + at);
  }
  w.begin();
  for (int p = p0, turn = 0; p < p1; p += BLOCK * WAVES, ++turn) {
    f32x4 s[2], prob[2];
    f16x8 ph;
    w.products(s);
    __builtin_amdgcn_sched_barrier(0);
    const bool more = p + BLOCK * WAVES < p1;
    if (more) {
      at = place(p + BLOCK * WAVES, turn + 1);
      w.read_keys(keys + at);
    }
    __builtin_amdgcn_sched_barrier(0);
    w.probabilities(s, p1 - p, ph, prob);
    if (p1 - p < BLOCK) w.v.cut(p1 - p, w.j);
    w.v.add(w.o, ph, prob);
    __builtin_amdgcn_sched_barrier(0);
    if (more) w.read_values(values + at);
  }
  if (lost) w.sum = __builtin_nanf("");
  w.sum = column_sum(w.sum);
  if (w.j == 0 && w.c < HEADS) {
    tops[wave][w.c] = w.bar > -INF ? w.reference : -INF;
    sums[wave][w.c] = w.sum;
  }
#pragma unroll
  for (int t = 0; t < HS / 16; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = w.o[t][r];
      if (HALF) {
        x *= w.c < 8 ? 1.0f / PIECE_UP : 1.0f / (PIECE_UP * LOW);
        x += other_half(x);
      }
      if (w.c < HEADS) outs[wave][w.c][channel<HS, HALF>(t, 4 * w.j + r)] = x;
    }
  __syncthreads();
  const bool whole = len <= piece.chunk;
  for (int i = tid; i < heads * HS; i += 64 * WAVES) {
    const int h = i / HS, d = i % HS;
    float top = tops[0][h];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) top = __builtin_fmaxf(top, tops[k][h]);
    const float from = top > -INF ? top : 0.0f;
    float sum = 0.0f, o = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const float f = __builtin_amdgcn_exp2f(tops[k][h] - from);
      sum += sums[k][h] * f;
      o += outs[k][h][d] * f;
    }
    if (whole) {
      out[i] = o / sum;
    } else {
      outputs<HS>(a, blockIdx.x, first + h)[d] = o;
      if (d == 0) *statistics(a, blockIdx.x, first + h) = make_float2(top, sum);
    }
  }
}

// the pieces of a (row, head) with more than one: a thread takes four channels of every EACH-th
template <int HS>
__global__ __launch_bounds__(256) void join_kernel(const PagesAttn a) {
  constexpr int QUADS = HS / 4, EACH = 256 / QUADS;
  __shared__ float tops[4];
  __shared__ float sums[EACH];
  __shared__ float4 outs[EACH][QUADS];
  const int row = blockIdx.y, h = blockIdx.x, tid = threadIdx.x;
  const Piece piece = piece_of<true>(a, row, tid & 63);
  if (piece.len <= piece.chunk) return;
  const int parts = (int)(((int64_t)piece.len + piece.chunk - 1) / piece.chunk);
  const float2 *stats = statistics(a, piece.first, h);
  const float4 *from = reinterpret_cast<const float4 *>(outputs<HS>(a, piece.first, h));
  float top = -INF;
  for (int p = tid; p < parts; p += 256) top = __builtin_fmaxf(top, stats[(int64_t)p * a.nh].x);
  top = wave_all(top, [](float x, float y) { return __builtin_fmaxf(x, y); });
  if ((tid & 63) == 0) tops[tid >> 6] = top;
  __syncthreads();
  top = __builtin_fmaxf(__builtin_fmaxf(tops[0], tops[1]), __builtin_fmaxf(tops[2], tops[3]));
  if (!(top > -INF)) top = 0.0f;
  const int part = tid / QUADS, d = tid % QUADS;
  float sum = 0.0f;
  float4 o = make_float4(0, 0, 0, 0);
  if (part < EACH) {
    for (int p = part; p < parts; p += EACH) {
      const float2 own = stats[(int64_t)p * a.nh];
      const float f = __builtin_amdgcn_exp2f(own.x - top);
      const float4 x = from[(int64_t)p * a.nh * QUADS + d];
      sum += own.y * f;
      o.x += x.x * f, o.y += x.y * f, o.z += x.z * f, o.w += x.w * f;
    }
    if (d == 0) sums[part] = sum;
    outs[part][d] = o;
  }
  __syncthreads();
  if (tid < HS) {
    float y = 0.0f;
    sum = 0.0f;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      y += reinterpret_cast<const float *>(outs[e])[tid];
      sum += sums[e];
    }
    a.out[(int64_t)row * a.out_stride + (int64_t)h * HS + tid] = y / sum;
  }
}

// workgroups that the heads of a row's piece take
int tiles_of(const PagesView &c, int32_t nh) {
  const int group = nh / c.nkv, most = c.half ? Kind<true>::heads : Kind<false>::heads;
  return c.nkv * ((group + most - 1) / most);
}

template <int HS>
void launch(const PagesAttn &a, hipStream_t s) {
  const dim3 grid(a.most, tiles_of(a.c, a.nh));
  if (a.c.half) hipLaunchKernelGGL((attend_kernel<HS, true>), grid, dim3(64 * WAVES), 0, s, a);
  else hipLaunchKernelGGL((attend_kernel<HS, false>), grid, dim3(64 * WAVES), 0, s, a);
  if (a.most > a.rows) hipLaunchKernelGGL(join_kernel<HS>, dim3(a.nh, a.rows), dim3(256), 0, s, a);
}

// how a launch of `rows` rows of at most `longest` positions is cut
void cut(PagesAttn &a) {
  const int tiles = tiles_of(a.c, a.nh);
  a.parts = a.pieces = 0;
  // every row one piece where cutting it and joining its pieces takes longer: a block of a wave after another 1.3 us, the join
  // about 4 (one row of 512 positions 12.3 us against 9.7 and the join); where the rows fill the CUs by themselves up to twice
  // as many (96 rows of up to 900 positions of 8 heads 44 us against 49 and 5)
  if (a.longest <= 5 * UNIT || (a.longest <= 8 * UNIT && (int64_t)a.rows * tiles >= 256)) {
    a.parts = 1;
    a.chunk = std::max(a.longest, 1);
    a.most = a.rows;
  } else if (a.rows <= PLANNED) {
    const int places = 256 * occupancy(a.c.hs, a.c.half) / tiles;
    a.pieces = std::max(1, places - std::min(a.rows, places) / 2);
    a.most = std::min<int64_t>(a.pieces + a.rows, (int64_t)a.rows * ((a.longest + LEAST * UNIT - 1) / (LEAST * UNIT)));
  } else {  // (by the longest: one row of 131,072 positions among 511 of 200 takes 1042 us, among 255, planned, 174)
    a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(16384 / ((int64_t)a.rows * tiles), (a.longest + 2047) / 2048));
    a.chunk = ((a.longest + a.parts - 1) / a.parts + UNIT - 1) / UNIT * UNIT;
    a.most = (int64_t)a.rows * a.parts;
  }
}

}  // namespace

// for any launch of at most as many rows of at most as many positions: a program's largest step sizes it once
int64_t pages_attention_workspace(const PagesView &c, int32_t nh, int32_t rows, int32_t longest) {
  if (longest <= 5 * UNIT) return 0;
  const int tiles = tiles_of(c, nh);
  const int64_t planned = std::min(rows, PLANNED), two = (longest + LEAST * UNIT - 1) / (LEAST * UNIT);
  int64_t most = std::min(256 * occupancy(c.hs, c.half) / tiles + 1 + planned, planned * two);
  if (rows > PLANNED && longest > 2048) most = std::max<int64_t>(most, std::min<int64_t>(16384 / tiles, (int64_t)rows * ((longest + 2047) / 2048)));
  return 4 * (((most * nh * 2 + 3) & ~3) + most * nh * c.hs);
}

hipError_t launch_pages_attention(const PagesAttn &args, hipStream_t s) {
  PagesAttn a = args;
  cut(a);
  switch (a.c.hs) {
    case 16: launch<16>(a, s); break;
    case 32: launch<32>(a, s); break;
    case 48: launch<48>(a, s); break;
    case 64: launch<64>(a, s); break;
    case 96: launch<96>(a, s); break;
    case 128: launch<128>(a, s); break;
    case 256: launch<256>(a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ple
