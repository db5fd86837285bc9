// four.hip — products with 4-bit matrices (include/pyodide_llm_hip.h hk_matmul_four): w in -8..7 with a scale a row and group
// of columns, against activations quantized per group of 32.
//
// y[t][r] = sum_g ws[r][g] xs[t][g] S_g, S_g = the sum of w (xq - bias) over the 32 columns of group g, exact in int32; the
// float32 sums over the groups run in no order of the reference's, which has no 4-bit kernels.
//
// 128 columns of a row are four chunks of 16 bytes, and chunk j has eight columns of each of the four groups: what a lane of
// the matrix core's products takes of each (16 rows by 32 columns an instruction, columns by quarters of the wave), so that a
// lane's one load feeds four products. The four bits go to the upper half of a byte (three instructions for eight values):
// sixteen times the value, taken off the result.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));

template <bool HALF>
struct Scale {
  typedef float type;
};
template <>
struct Scale<true> {
  typedef _Float16 type;
};

constexpr int WAVES = 4;
constexpr float SIXTEENTH = 0.0625f;

__device__ __forceinline__ uint32_t low_bits(uint32_t w) { return (w << 4) & 0xF0F0F0F0u; }
__device__ __forceinline__ uint32_t high_bits(uint32_t w) { return w & 0xF0F0F0F0u; }

__device__ __forceinline__ float dpp_xor2(float v) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), 0x4E, 0xF, 0xF, true));
}
__device__ __forceinline__ int32_t dpp_xor2(int32_t v) { return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true); }

// s[i], i = 0..3, added over the four lanes of a quad: lane j has s[j]'s sum (nine instructions)
template <class T>
__device__ __forceinline__ T quad_sums(const T (&s)[4], int j) {
  const bool odd = j & 1, high = j & 2;
  const T a = (odd ? s[1] : s[0]) + dpp_xor1(odd ? s[0] : s[1]), b = (odd ? s[3] : s[2]) + dpp_xor1(odd ? s[2] : s[3]);
  return (high ? b : a) + dpp_xor2(high ? a : b);
}

// ---- one token ----

// LANES lanes a row (16, 64 or all waves'), which take its chunks LANES apart, STEPS of them at most; they take four rows at a
// time and go on the launch's rows further. A lane's activations stay in its registers from row to row. No load is conditional,
// which would wait for each: what lies past the columns is taken as zero. Bound by the weights' bytes where there are many
// (128,256 rows of 4096 columns, 271 MB in 48.4 us, 5.6 TB/s), by latency where not (4096 rows, 10.5 MB, 4.0 us; 5.5 with
// conditional loads).
template <int LANES, int STEPS, bool HALF>
__global__ __launch_bounds__(64 * WAVES) void gemv_kernel(const FourArgs a) {
  constexpr int ROWS = WAVES * 64 / LANES * 4;  // a workgroup takes at a time
  constexpr bool WIDE = LANES > 64;
  __shared__ float parts[WIDE ? 2 : 1][4][WAVES];
  const int nc = (a.k + 127) / 128, l = threadIdx.x % LANES, j = threadIdx.x & 3;
  const int shift = a.group == 32 ? 0 : a.group == 64 ? 1 : 2;
  uint32_t x[STEPS][8];
  float xs[STEPS];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int q = l + LANES * s, first = 32 * q - 28 * j;  // (the chunk's first column: 128 of 128s, 4 j)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int column = first + 16 * e;
      x[s][e] = *reinterpret_cast<const uint32_t *>(a.xq + min(column, a.k - 4));
      if (column >= a.k) x[s][e] = a.bias ? 0x40404040u : 0;
    }
    xs[s] = a.xs[min(q, a.k / 32 - 1)];
    if (q >= a.k / 32) xs[s] = 0.0f;
  }
  int turn = 0;
  for (int64_t base = (int64_t)blockIdx.x * ROWS; base < a.rows; base += (int64_t)gridDim.x * ROWS, turn ^= 1) {
    const int64_t row0 = base + threadIdx.x / LANES * 4;
    uint4 w[4][STEPS];
    float ws[4][STEPS];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = min(row0 + r, (int64_t)a.rows - 1);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const int q = min(l + LANES * s, nc * 4 - 1);  // (past the row's end: its last chunk, against zeros)
        w[r][s] = reinterpret_cast<const uint4 *>(a.w)[row * nc * 4 + q];
        const int64_t at = row * (nc * 4 >> shift) + (q >> shift);
        ws[r][s] = HALF ? (float)reinterpret_cast<const _Float16 *>(a.ws)[at] : reinterpret_cast<const float *>(a.ws)[at];
      }
    }
    if (base == (int64_t)blockIdx.x * ROWS && a.bias) {  // (here, so that the first rows are asked for before)
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) x[s][e] = centre4(x[s][e]);
    }
    float acc[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      acc[r] = 0.0f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t in[4] = {w[r][s].x, w[r][s].y, w[r][s].z, w[r][s].w};
        int32_t sums[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) sums[g] = dot4(low_bits(in[g]), x[s][2 * g], dot4(high_bits(in[g]), x[s][2 * g + 1], 0));
        acc[r] = __builtin_fmaf((float)quad_sums(sums, j), ws[r][s] * xs[s], acc[r]);
      }
    }
    float y = quad_sums(acc, j);  // row j's, over the lane's quad
    y += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x124, 0xF, 0xF, true));  // row_ror:4
    y += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x128, 0xF, 0xF, true));  // row_ror:8
    if (LANES >= 64) {
      y += __shfl_xor(y, 16);
      y += __shfl_xor(y, 32);
    }
    if (WIDE) {  // (the next turn's go to the other half: one barrier)
      if ((threadIdx.x & 63) < 4) parts[turn][j][threadIdx.x >> 6] = y;
      __syncthreads();
      y = 0.0f;
#pragma unroll
      for (int k = 0; k < WAVES; ++k) y += parts[turn][j][k];
    }
    if (l < 4 && row0 + j < a.rows) a.y[row0 + j] = y * SIXTEENTH;
  }
}

// ---- more tokens ----

constexpr int GEMM_WAVES = 8, GEMM_THREADS = 64 * GEMM_WAVES;

// the activations of 16 TILES tokens for PLACES times 128 columns, in the order in which a product takes them, and their scales
template <int TILES, int PLACES>
struct Tokens {
  uint4 x[TILES][PLACES][2][64];
  float xs[TILES][PLACES][64];
};

// a thread's part in bringing them there: 16 columns of a token, and a group's scale, a load; all loads before the stores
template <int TILES, int PLACES>
struct Carrier {
  static constexpr int LOADS = TILES * PLACES * 128 / GEMM_THREADS, SCALES = LOADS / 2;
  uint4 v[LOADS];
  float f[SCALES];
  // (token, 16 columns of 64, which 64, then tiles and places)
  __device__ __forceinline__ static int token() { return threadIdx.x & 15; }
  __device__ __forceinline__ static int part() { return threadIdx.x >> 4 & 3; }
  __device__ __forceinline__ static int half() { return threadIdx.x >> 6 & 1; }
  __device__ __forceinline__ static int load(int i) { return (threadIdx.x >> 7) + 4 * i; }
  __device__ __forceinline__ static int scale(int i) { return (threadIdx.x >> 6) + 8 * i; }

  __device__ __forceinline__ void read(const FourArgs &a, int t0, int c0) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int column = (c0 + load(i) / TILES) * 128 + half() * 64 + part() * 16, t = t0 + load(i) % TILES * 16 + token();
      v[i] = *reinterpret_cast<const uint4 *>(a.xq + (int64_t)min(t, a.m - 1) * a.k + min(column, a.k - 16));
    }
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int group = (c0 + scale(i) / TILES) * 4 + part(), t = t0 + scale(i) % TILES * 16 + token();
      f[i] = a.xs[(int64_t)min(t, a.m - 1) * (a.k / 32) + min(group, a.k / 32 - 1)];
    }
  }
  __device__ __forceinline__ void write(const FourArgs &a, int c0, Tokens<TILES, PLACES> &to) const {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int q = load(i) / TILES;
      const uint32_t keep = (c0 + q) * 128 + half() * 64 + part() * 16 < a.k ? ~0u : 0u;
      uint4 y = v[i];
      if (a.bias) y.x = centre4(y.x), y.y = centre4(y.y), y.z = centre4(y.z), y.w = centre4(y.w);
      uint32_t *at = reinterpret_cast<uint32_t *>(&to.x[load(i) % TILES][q][half()][token()]) + part();
      at[0] = y.x & keep, at[64] = y.y & keep, at[128] = y.z & keep, at[192] = y.w & keep;
    }
#pragma unroll
    for (int i = 0; i < SCALES; ++i) {
      const int q = scale(i) / TILES;
      to.xs[scale(i) % TILES][q][part() * 16 + token()] = (c0 + q) * 4 + part() < a.k / 32 ? f[i] : 0.0f;
    }
  }
};

// what a product of 16 tokens and 128 columns takes of them, of one lane
struct Operand {
  uint4 lo, hi;
  float f;
};
template <int TILES, int PLACES>
__device__ __forceinline__ Operand operand(const Tokens<TILES, PLACES> &tokens, int tile, int place) {
  const int lane = threadIdx.x & 63;
  Operand x;
  x.lo = tokens.x[tile][place][0][lane];
  x.hi = tokens.x[tile][place][1][lane];
  x.f = tokens.xs[tile][place][lane];
  return x;
}

// a lane's weights of 128 columns, and the scale of its quarter's group, of a row
template <int GROUP, bool HALF>
struct Weights {
  typedef typename Scale<HALF>::type scale;
  static constexpr int EACH = 128 / GROUP;  // scales of a row's 128 columns
  uint4 in;
  scale sc;

  __device__ __forceinline__ void read(const FourArgs &a, int64_t row, int place, int nc) {
    const int j = (threadIdx.x & 63) >> 4;
    in = reinterpret_cast<const uint4 *>(a.w)[(row * nc + place) * 4 + j];
    sc = reinterpret_cast<const scale *>(a.ws)[(row * nc + place) * EACH + j * EACH / 4];
  }
  // D = X W^T, 16 tokens by 16 rows, a group a product; and so the scales: one product of single columns has xs ws of the four
  // groups, each in the place of its sum, and leaves a conversion and an fma a sum (16 tokens by 4096 rows of 4096 columns 7.7 ->
  // 7.2 us, 32 by 14336 19 -> 17, against scaling by the tokens' and the rows' one after the other)
  __device__ __forceinline__ void multiply(const Operand &x, float4 &acc) const {
    const uint32_t bits[4] = {in.x, in.y, in.z, in.w};
    const long av[4] = {(long)((uint64_t)x.lo.y << 32 | x.lo.x), (long)((uint64_t)x.lo.w << 32 | x.lo.z),
                        (long)((uint64_t)x.hi.y << 32 | x.hi.x), (long)((uint64_t)x.hi.w << 32 | x.hi.z)};
    const f32x16 f = __builtin_amdgcn_mfma_f32_16x16x1f32(x.f, (float)sc, f32x16{}, 0, 0, 0);
    i32x4 s[4];
#pragma unroll
    for (int g = 0; g < 4; ++g)
      s[g] = __builtin_amdgcn_mfma_i32_16x16x32_i8(av[g], (long)((uint64_t)high_bits(bits[g]) << 32 | low_bits(bits[g])),
                                                   i32x4{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      acc.x = __builtin_fmaf((float)s[g][0], f[4 * g], acc.x);
      acc.y = __builtin_fmaf((float)s[g][1], f[4 * g + 1], acc.y);
      acc.z = __builtin_fmaf((float)s[g][2], f[4 * g + 2], acc.z);
      acc.w = __builtin_fmaf((float)s[g][3], f[4 * g + 3], acc.w);
    }
  }
};

// the waves' sums of 16 tokens and 16 RT rows, [row tile][wave][lane], added up and stored
template <int RT>
__device__ __forceinline__ void finish(const FourArgs &a, const float4 *sums, int t0, int64_t row0) {
  for (int e = threadIdx.x; e < RT * 256; e += GEMM_THREADS) {
    const int col = e & 15, r = e >> 4 & 3, quarter = e >> 6 & 3, rt = e >> 8;
    const float *from = reinterpret_cast<const float *>(sums + rt * GEMM_THREADS + quarter * 16 + col) + r;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < GEMM_WAVES; ++k) y += from[k * 256];
    const int t = t0 + quarter * 4 + r;
    const int64_t row = row0 + rt * 16 + col;
    if (t < a.m && row < a.rows) a.y[(int64_t)t * a.rows + row] = y * SIXTEENTH;
  }
}

// Up to 16 TILES tokens of up to 1024 DEEP columns: they stay in LDS, and the workgroup goes from 16 rows to 16 rows, its waves
// sharing their columns. A wave's loads for its next rows go out as its present weights are used, into their registers. One
// workgroup a CU, whose waves all wait for the tokens before the first product. 16 tokens by 2304 rows of 768 columns take 3.7 us;
// 32 by 14336 of 4096 18, by 4096 12.
template <int TILES, int DEEP, int GROUP, bool HALF>
__global__ __launch_bounds__(GEMM_THREADS, 2) void rows_kernel(const FourArgs a) {
  __shared__ Tokens<TILES, GEMM_WAVES * DEEP> tokens;
  __shared__ float4 sums[2][GEMM_THREADS];
  const int nc = (a.k + 127) / 128, first = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * DEEP, mine = threadIdx.x & 15;
  const int64_t step = (int64_t)gridDim.x * 16;
  Weights<GROUP, HALF> w[DEEP];
  auto row = [&](int64_t row0) { return min(row0 + mine, (int64_t)a.rows - 1); };
  {
    Carrier<TILES, GEMM_WAVES * DEEP> carrier;
    carrier.read(a, 0, 0);  // (before the weights, for which it would wait otherwise)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) w[d].read(a, row((int64_t)blockIdx.x * 16), min(first + d, nc - 1), nc);
    __builtin_amdgcn_sched_barrier(0);
    carrier.write(a, 0, tokens);
  }
  __syncthreads();
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * 16; row0 < a.rows; row0 += step) {
    const int64_t next = row(row0 + step);
    float4 acc[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[t] = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {  // (places past the columns: zeros)
      const Weights<GROUP, HALF> now = w[d];
#pragma unroll
      for (int t = 0; t < TILES; ++t) now.multiply(operand(tokens, t, first + d), acc[t]);
      w[d].read(a, next, min(first + d, nc - 1), nc);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
      sums[turn][threadIdx.x] = acc[t];
      __syncthreads();  // (the next go to the other half)
      finish<1>(a, sums[turn], 16 * t, row0);
      turn ^= 1;
    }
  }
}

// Up to 16 tokens of 1025 to 4096 columns: as rows_kernel, with the tokens in registers (a wave's columns stay the same) and the
// weights on their way there through LDS. A wave's load takes 64 DEEP bytes of a row, whole cache lines, from 16 / DEEP rows; the
// products' order, 64 bytes of each of 16, is LDS's: chunk k of row r lies at place k ^ r of the row's, so that neither side meets
// a bank twice. 128,256 rows of 4096 columns, 271 MB, take 59 us (64 with loads of 64 bytes of 16 rows), 14336 12.0, of which
// about 6 pass until the first rows are done, 4096 7.5. Rows two turns ahead: the same.
template <int DEEP, int GROUP, bool HALF>
__global__ __launch_bounds__(GEMM_THREADS, 2) void lines_kernel(const FourArgs a) {
  constexpr int EACH = Weights<GROUP, HALF>::EACH;
  typedef typename Scale<HALF>::type scales __attribute__((ext_vector_type(EACH)));
  constexpr int CHUNKS = 4 * DEEP, ROWS = 64 / CHUNKS;  // of a row a load, and rows a load
  __shared__ Tokens<1, GEMM_WAVES * DEEP> tokens;
  __shared__ float4 sums[2][GEMM_THREADS];
  __shared__ u32x4 chunks[GEMM_WAVES][16 * CHUNKS];
  __shared__ scales factors[GEMM_WAVES][DEEP][16];
  const int nc = (a.k + 127) / 128, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = wave * DEEP;
  const int lane = threadIdx.x & 63, c = lane & 15, j = lane >> 4, d_mine = min(j, DEEP - 1);
  const int64_t step = (int64_t)gridDim.x * 16;
  u32x4 in[DEEP];
  scales sc;
  auto read = [&](int64_t row0) {
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const int r = ROWS * i + lane / CHUNKS, k = lane % CHUNKS ^ r % CHUNKS;
      const int64_t row = min(row0 + r, (int64_t)a.rows - 1);
      in[i] = reinterpret_cast<const u32x4 *>(a.w)[row * nc * 4 + min(first * 4 + k, nc * 4 - 1)];
    }
    sc = reinterpret_cast<const scales *>(a.ws)[min(row0 + c, (int64_t)a.rows - 1) * nc + min(first + d_mine, nc - 1)];
  };
  {
    Carrier<1, GEMM_WAVES * DEEP> carrier;
    carrier.read(a, 0, 0);  // (before the weights, for which it would wait otherwise)
    __builtin_amdgcn_sched_barrier(0);
    read((int64_t)blockIdx.x * 16);
    __builtin_amdgcn_sched_barrier(0);
    carrier.write(a, 0, tokens);
  }
  __syncthreads();
  Operand x[DEEP];
#pragma unroll
  for (int d = 0; d < DEEP; ++d) x[d] = operand(tokens, 0, first + d);
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * 16; row0 < a.rows; row0 += step, turn ^= 1) {
#pragma unroll
    for (int i = 0; i < DEEP; ++i) chunks[wave][64 * i + lane] = in[i];
    factors[wave][d_mine][c] = sc;
    wave_sync_lds();  // (a wave's own part)
    read(row0 + step);
    __builtin_amdgcn_sched_barrier(0);
    float4 acc = make_float4(0, 0, 0, 0);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {  // (places past the columns: zeros)
      Weights<GROUP, HALF> w;
      w.in = __builtin_bit_cast(uint4, chunks[wave][c * CHUNKS + ((4 * d + j) ^ c % CHUNKS)]);
      w.sc = reinterpret_cast<const typename Scale<HALF>::type *>(&factors[wave][d][c])[j * EACH / 4];
      w.multiply(x[d], acc);
    }
    wave_sync_lds();
    sums[turn][threadIdx.x] = acc;
    __syncthreads();  // (the next go to the other half)
    finish<1>(a, sums[turn], 0, row0);
  }
}

// Any number of tokens and columns: 16 RT rows by 16 TILES tokens a workgroup, the activations a stage at a time, the next
// stage's on their way meanwhile.
template <int RT, int TILES, int GROUP, bool HALF>
__global__ __launch_bounds__(GEMM_THREADS, TILES == 1 && (HALF || GROUP > 32) ? 4 : 2) void stages_kernel(const FourArgs a) {
  constexpr int DEEP = 4 / TILES, STAGE = GEMM_WAVES * DEEP;
  __shared__ Tokens<TILES, STAGE> tokens;
  const int nc = (a.k + 127) / 128, t0 = blockIdx.y * (16 * TILES), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row0 = (int64_t)blockIdx.x * (16 * RT);
  float4 acc[RT][TILES];
#pragma unroll
  for (int r = 0; r < RT; ++r)
#pragma unroll
    for (int t = 0; t < TILES; ++t) acc[r][t] = make_float4(0, 0, 0, 0);
  Carrier<TILES, STAGE> carrier;
  carrier.read(a, t0, 0);
  int64_t row[RT];
#pragma unroll
  for (int r = 0; r < RT; ++r) row[r] = min(row0 + 16 * r + (threadIdx.x & 15), (int64_t)a.rows - 1);
  for (int c0 = 0; c0 < nc; c0 += STAGE) {
    Weights<GROUP, HALF> w[RT][DEEP];
#pragma unroll
    for (int d = 0; d < DEEP; ++d)
#pragma unroll
      for (int r = 0; r < RT; ++r) w[r][d].read(a, row[r], min(c0 + wave * DEEP + d, nc - 1), nc);
    __builtin_amdgcn_sched_barrier(0);
    if (c0) __syncthreads();  // (the last stage's have been read)
    carrier.write(a, c0, tokens);
    __syncthreads();
    if (c0 + STAGE < nc) carrier.read(a, t0, c0 + STAGE);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      if (c0 + wave * DEEP + d >= nc) break;
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const Operand x = operand(tokens, t, wave * DEEP + d);
#pragma unroll
        for (int r = 0; r < RT; ++r) w[r][d].multiply(x, acc[r][t]);
      }
    }
  }
  float4 *sums = reinterpret_cast<float4 *>(tokens.x);
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; ++r) sums[r * GEMM_THREADS + threadIdx.x] = acc[r][t];
    __syncthreads();
    finish<RT>(a, sums, t0 + 16 * t, row0);
  }
}

template <int LANES, int STEPS, bool HALF>
void launch_gemv(const FourArgs &a, hipStream_t s) {
  constexpr int ROWS = WAVES * 64 / LANES * 4;
  const int blocks = std::min((a.rows + ROWS - 1) / ROWS, 1024);
  hipLaunchKernelGGL((gemv_kernel<LANES, STEPS, HALF>), dim3(blocks), dim3(64 * WAVES), 0, s, a);
}

template <int TILES, int DEEP, bool HALF>
void launch_rows(const FourArgs &a, hipStream_t s) {
  // as many turns for every workgroup as for the most
  const int blocks = (a.rows + 15) / 16, turns = (blocks + 255) / 256, grid = (blocks + turns - 1) / turns;
  if (a.group == 32) hipLaunchKernelGGL((rows_kernel<TILES, DEEP, 32, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((rows_kernel<TILES, DEEP, 64, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else hipLaunchKernelGGL((rows_kernel<TILES, DEEP, 128, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
}

template <int DEEP, bool HALF>
void launch_lines(const FourArgs &a, hipStream_t s) {
  const int blocks = (a.rows + 15) / 16, turns = (blocks + 255) / 256, grid = (blocks + turns - 1) / turns;
  if (a.group == 32) hipLaunchKernelGGL((lines_kernel<DEEP, 32, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((lines_kernel<DEEP, 64, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else hipLaunchKernelGGL((lines_kernel<DEEP, 128, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
}

template <int RT, int TILES, bool HALF>
void launch_stages(const FourArgs &a, hipStream_t s) {
  const dim3 grid((a.rows + 16 * RT - 1) / (16 * RT), (a.m + 16 * TILES - 1) / (16 * TILES)), block(GEMM_THREADS);
  if (a.group == 32) hipLaunchKernelGGL((stages_kernel<RT, TILES, 32, HALF>), grid, block, 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((stages_kernel<RT, TILES, 64, HALF>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((stages_kernel<RT, TILES, 128, HALF>), grid, block, 0, s, a);
}

template <int TILES, bool HALF>
void launch_gemm(const FourArgs &a, hipStream_t s) {
  // rows a workgroup: the fewest whose workgroups are not more than the CUs, since each brings the activations to LDS for itself
  // (64 tokens by 14336 rows: 62 us at 16, 45 at 32, 29 at 64; by 4096 rows 19, 23, 30; 2048 tokens by 4096 rows 408 at 16, 217
  // at 64); with one tile of tokens two of rows take more registers than two workgroups a CU leave (4096 rows of 14336 columns:
  // 21 us, 35). Past 64 rows a workgroup there is no larger shape: 128 tokens by 8192 rows, 256 workgroups, take 31 us, by 9000
  // rows, 282 of them, 58.
  if constexpr (TILES == 1) {
    launch_stages<1, 1, HALF>(a, s);
  } else {
    const int64_t rows = (int64_t)a.rows * ((a.m + 16 * TILES - 1) / (16 * TILES));  // times the tiles of tokens
    if (rows > 8192) launch_stages<4, TILES, HALF>(a, s);
    else if (rows > 4096) launch_stages<2, TILES, HALF>(a, s);
    else launch_stages<1, TILES, HALF>(a, s);
  }
}

template <bool HALF>
void launch(const FourArgs &a, hipStream_t s) {
  const int chunks = (a.k + 127) / 128 * 4;
  if (a.m == 1 && chunks <= 1024) {
    if (chunks <= 16) launch_gemv<16, 1, HALF>(a, s);
    else if (chunks <= 32) launch_gemv<16, 2, HALF>(a, s);
    else if (chunks <= 64) launch_gemv<64, 1, HALF>(a, s);
    else if (chunks <= 128) launch_gemv<64, 2, HALF>(a, s);
    else if (chunks <= 256) launch_gemv<64, 4, HALF>(a, s);
    else if (chunks <= 512) launch_gemv<256, 2, HALF>(a, s);
    else launch_gemv<256, 4, HALF>(a, s);
  } else if (a.m <= 16 && chunks <= 128) {
    if (chunks <= 32) launch_rows<1, 1, HALF>(a, s);
    else if (chunks <= 64) launch_lines<2, HALF>(a, s);
    else launch_lines<4, HALF>(a, s);
  } else if (a.m <= 32 && chunks <= 128) {
    if (chunks <= 32) launch_rows<2, 1, HALF>(a, s);
    else if (chunks <= 64) launch_rows<2, 2, HALF>(a, s);
    else launch_rows<2, 4, HALF>(a, s);
  } else if (a.m <= 16) {
    launch_gemm<1, HALF>(a, s);
  } else if (a.m <= 32) {
    launch_gemm<2, HALF>(a, s);
  } else {
    launch_gemm<4, HALF>(a, s);
  }
}

}  // namespace

hipError_t launch_matmul_four(const FourArgs &a, hipStream_t s) {
  if (a.half) launch<true>(a, s);
  else launch<false>(a, s);
  return hipGetLastError();
}

}  // namespace ple
