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
// each rounded to nearest (2^-24 of x is left), in columns 0-7 and 8-15 of one product. A float32 cache's are float32's.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BLOCK = 32;   // positions a wave takes at a time
constexpr int WAVES = 4;
constexpr float LOG2E = 1.44269504088896341f;
constexpr float INF = __builtin_inff();
constexpr float AHEAD = 8.0f;     // how far (log2) a score may lie above the reference before that moves
constexpr float PIECE_UP = 64.0f;  // probabilities go up to 2^AHEAD, their float16 halves to 2^14
constexpr float LOW = 2048.0f;     // the second half's scale

template <bool HALF>
struct Kind {
  typedef _Float16 type;
  static constexpr int heads = 8, widest = 8;
};
template <>
struct Kind<false> {
  typedef float type;
  static constexpr int heads = 16, widest = 4;
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

// a wave's accumulators and statistics
template <int HS, bool HALF>
struct Wave {
  typedef typename Kind<HALF>::type T;
  static constexpr int KEYS = HALF ? (HS + 31) / 32 : HS / 16;  // loads of a key row
  static constexpr int TILES = HS / 16;
  f16x8 qh[HALF ? KEYS : 1];
  float4 qf[HALF ? 1 : KEYS];
  float up;        // what a product is multiplied by: a score in log2
  float top = -INF, reference = 0.0f, sum = 0.0f;
  f32x4 o[TILES];
  int lane, c, j;  // the lane, its column and its quarter

  // the row's queries of the tile's heads as products take them
  __device__ __forceinline__ void queries(const float *q, int heads, float scale) {
    const int h = HALF ? c & 7 : c;
    const bool mine = h < heads;
    if constexpr (HALF) {
      float x[KEYS][8], most = 0.0f;
#pragma unroll
      for (int s = 0; s < KEYS; ++s) {
        const int d = 32 * s + 8 * j;
        const bool in = mine && (HS % 32 == 0 || d < HS);
        const float4 a = in ? *reinterpret_cast<const float4 *>(q + h * HS + d) : make_float4(0, 0, 0, 0),
                     b = in ? *reinterpret_cast<const float4 *>(q + h * HS + d + 4) : make_float4(0, 0, 0, 0);
        x[s][0] = a.x, x[s][1] = a.y, x[s][2] = a.z, x[s][3] = a.w;
        x[s][4] = b.x, x[s][5] = b.y, x[s][6] = b.z, x[s][7] = b.w;
#pragma unroll
        for (int i = 0; i < 8; ++i) most = __builtin_fmaxf(most, __builtin_fabsf(x[s][i]));
      }
      most = column_max(most);
      const int e = __builtin_amdgcn_frexp_expf(most);  // |q| < 2^e; (of 0 and of what is not finite 0)
#pragma unroll
      for (int s = 0; s < KEYS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __builtin_amdgcn_ldexpf(x[s][i], 15 - e);
          const _Float16 hi = (_Float16)y;
          const _Float16 lo = (_Float16)((y - (float)hi) * LOW);
          qh[s][i] = c < 8 ? hi : lo;
        }
      up = __builtin_amdgcn_ldexpf(scale * LOG2E, e - 15);
      if (c >= 8) up = up / LOW;
    } else {
#pragma unroll
      for (int s = 0; s < KEYS; ++s)
        qf[s] = mine ? *reinterpret_cast<const float4 *>(q + h * HS + 16 * s + 4 * j) : make_float4(0, 0, 0, 0);
      up = scale * LOG2E;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = f32x4{0, 0, 0, 0};
  }

  // the scores of 32 positions whose key rows begin at k: position 16 t + 4 j + r of column c in s[t][r]
  __device__ __forceinline__ void scores(const T *k, f32x4 (&s)[2]) const {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{0, 0, 0, 0};
      const T *row = k + (16 * t + c) * HS;
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        if constexpr (HALF) {
          const int d = 32 * i + 8 * j;
          f16x8 x = {};
          if (HS % 32 == 0 || d < HS) x = *reinterpret_cast<const f16x8 *>(row + d);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, qh[i], s[t], 0, 0, 0);
        } else {
          const float4 x = *reinterpret_cast<const float4 *>(row + 16 * i + 4 * j);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, qf[i].x, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, qf[i].y, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, qf[i].z, s[t], 0, 0, 0);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, qf[i].w, s[t], 0, 0, 0);
        }
      }
    }
  }

  // channels BASE.. of the values: tiles of 16 from tile AT on
  template <int BASE, int AT>
  __device__ __forceinline__ void values(const T *v, int left, const f16x8 &ph, const f32x4 (&p)[2]) {
    constexpr int REST = HS - BASE;
    if constexpr (REST > 0) {
      constexpr int W = HALF && REST >= 128 ? 8 : REST >= 64 ? 4 : REST >= 32 ? 2 : 1;  // channels a lane
      typedef T piece __attribute__((ext_vector_type(W)));
      piece x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int t = (e & 4) * 4 + 4 * j + (e & 3);
        x[e] = *reinterpret_cast<const piece *>(v + t * HS + BASE + W * c);
        if (t >= left) x[e] = piece(0);  // (what lies behind the row's end may be anything)
      }
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
      values<BASE + 16 * W, AT + W>(v, left, ph, p);
    }
  }

  // 32 positions, `left` of them (or more) before the row's end
  __device__ __forceinline__ void block(const T *k, const T *v, int left) {
    f32x4 s[2];
    scores(k, s);
    float most = -INF;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float x = s[t][r] * up;
        if (HALF) x = x + other_half(x);
        if (16 * t + 4 * j + r >= left) x = -INF;
        s[t][r] = x;
        most = __builtin_fmaxf(most, x);
      }
    if (__any(most > top + AHEAD)) {
      const float next = __builtin_fmaxf(top, column_max(most));
      const float other = next > -INF ? next : 0.0f, less = __builtin_amdgcn_exp2f(top - other);
      top = next;
      reference = other;
      sum *= less;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        // a product's output has the column's statistics in its own lane
        o[t] *= less;
      }
    }
    f16x8 ph = {};
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float p = __builtin_amdgcn_exp2f(s[t][r] - reference);
        sum += p;
        if constexpr (HALF) {
          p *= PIECE_UP;
          const _Float16 hi = (_Float16)p, lo = (_Float16)((p - (float)hi) * LOW);
          ph[4 * t + r] = c < 8 ? hi : lo;
        }
        s[t][r] = p;
      }
    values<0, 0>(v, left, ph, s);
  }
};

// channel of element r of quarter j's output in tile n (Wave::values' order)
template <int HS, bool HALF>
__device__ __forceinline__ constexpr int channel(int n, int row) {
  int base = 0, at = 0;
  while (true) {
    const int rest = HS - base, w = HALF && rest >= 128 ? 8 : rest >= 64 ? 4 : rest >= 32 ? 2 : 1;
    if (n < at + w) return base + w * row + n - at;
    base += 16 * w;
    at += w;
  }
}

template <int HS, bool HALF>
__global__ __launch_bounds__(64 * WAVES) void attend_kernel(const PagesAttn a) {
  typedef typename Kind<HALF>::type T;
  constexpr int HEADS = Kind<HALF>::heads;
  __shared__ float tops[WAVES][HEADS], sums[WAVES][HEADS];
  __shared__ float outs[WAVES][HEADS][HS];
  const PagesView &c = a.c;
  const int group = a.nh / c.nkv, tiles = (group + HEADS - 1) / HEADS;
  const int part = blockIdx.x, g = blockIdx.y / tiles, first = g * group + blockIdx.y % tiles * HEADS, row = blockIdx.z;
  const int heads = min(HEADS, (g + 1) * group - first);
  const int tid = threadIdx.x, wave = tid >> 6;
  int len = a.lengths[row];
  const int32_t seq = a.seqs ? a.seqs[row] : row;
  if (seq < 0 || len < 0) len = 0;
  const bool wrong = len > 0 && (seq >= c.n_seqs || len > a.longest || len > c.slots * c.page);
  float *out = a.out + (int64_t)row * a.out_stride + (int64_t)first * HS;
  if (len == 0 || wrong) {
    if (part == 0)
      for (int i = tid; i < heads * HS; i += 64 * WAVES) out[i] = wrong ? __builtin_nanf("") : 0.0f;
    return;
  }
  const int p0 = part * a.chunk, p1 = min(len, p0 + a.chunk);
  if (p0 >= len) return;
  Wave<HS, HALF> w;
  w.lane = tid & 63;
  w.c = w.lane & 15;
  w.j = w.lane >> 4;
  w.queries(a.q + (int64_t)row * a.q_stride + (int64_t)first * HS, heads, 1.0f / __builtin_sqrtf((float)HS));
  const int32_t *table = c.tables + (int64_t)seq * c.slots;
  bool lost = false;
  for (int p = p0 + BLOCK * wave; p < p1; p += BLOCK * WAVES) {
    int32_t page = table[p / c.page];
    if ((uint32_t)page >= (uint32_t)c.n_pages) page = 0, lost = true;
    const int64_t at = ((((int64_t)a.layer * c.n_pages + page) * c.nkv + g) * c.page + p % c.page) * HS;
    w.block(reinterpret_cast<const T *>(c.keys) + at, reinterpret_cast<const T *>(c.values) + at, p1 - p);
  }
  if (lost) w.sum = __builtin_nanf("");
  w.sum = column_sum(w.sum);
  if (w.j == 0 && w.c < HEADS) {
    tops[wave][w.c] = w.top;
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
  const bool whole = len <= a.chunk;
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
      float *to = a.workspace + (((int64_t)row * a.nh + first + h) * a.parts + part) * (HS + 2);
      to[2 + d] = o;
      if (d == 0) to[0] = top, to[1] = sum;
    }
  }
}

// the parts of a (row, head) whose positions are more than one part's
template <int HS>
__global__ __launch_bounds__(HS) void join_kernel(const PagesAttn a) {
  const int row = blockIdx.y, h = blockIdx.x, d = threadIdx.x;
  const int len = a.lengths[row];
  const int32_t seq = a.seqs ? a.seqs[row] : row;
  if (seq < 0 || seq >= a.c.n_seqs || len <= a.chunk || len > a.longest || len > a.c.slots * a.c.page) return;
  const int parts = (len + a.chunk - 1) / a.chunk;
  const float *from = a.workspace + ((int64_t)row * a.nh + h) * a.parts * (HS + 2);
  float top = -INF;
  for (int p = 0; p < parts; ++p) top = __builtin_fmaxf(top, from[p * (HS + 2)]);
  if (!(top > -INF)) top = 0.0f;
  float sum = 0.0f, o = 0.0f;
  for (int p = 0; p < parts; ++p) {
    const float f = __builtin_amdgcn_exp2f(from[p * (HS + 2)] - top);
    sum += from[p * (HS + 2) + 1] * f;
    o += from[p * (HS + 2) + 2 + d] * f;
  }
  a.out[(int64_t)row * a.out_stride + (int64_t)h * HS + d] = o / sum;
}

// positions a part takes, a multiple of the waves' blocks
int32_t chunk_of(const PagesView &c, int32_t nh, int32_t rows, int32_t longest) { return 512; }

template <int HS>
void launch(const PagesAttn &a, hipStream_t s) {
  const int group = a.nh / a.c.nkv, most = a.c.half ? 8 : 16;
  const dim3 grid(a.parts, a.c.nkv * ((group + most - 1) / most), a.rows);
  if (a.c.half) hipLaunchKernelGGL((attend_kernel<HS, true>), grid, dim3(64 * WAVES), 0, s, a);
  else hipLaunchKernelGGL((attend_kernel<HS, false>), grid, dim3(64 * WAVES), 0, s, a);
  if (a.parts > 1) hipLaunchKernelGGL(join_kernel<HS>, dim3(a.nh, a.rows), dim3(HS), 0, s, a);
}

}  // namespace

int64_t pages_attention_workspace(const PagesView &c, int32_t nh, int32_t rows, int32_t longest) {
  const int64_t chunk = chunk_of(c, nh, rows, longest), parts = (longest + chunk - 1) / chunk;
  return parts > 1 ? 4 * (int64_t)rows * nh * parts * (c.hs + 2) : 0;
}

hipError_t launch_pages_attention(const PagesAttn &args, hipStream_t s) {
  PagesAttn a = args;
  a.chunk = chunk_of(a.c, a.nh, a.rows, a.longest);
  a.parts = std::max(1, (a.longest + a.chunk - 1) / a.chunk);
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
