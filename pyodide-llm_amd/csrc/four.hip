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

// ---- one token or two ----

// LANES lanes a row (16, 64 or all waves'), which take its chunks LANES apart, STEPS of them at most; they take four rows at a
// time and go on the launch's rows further. A lane's activations stay in its registers from row to row. Bound by the weights'
// bytes.
template <int LANES, int STEPS, int M, bool HALF>
__global__ __launch_bounds__(64 * WAVES) void gemv_kernel(const FourArgs a) {
  constexpr int ROWS = WAVES * 64 / LANES * 4;  // a workgroup takes at a time
  constexpr bool WIDE = LANES > 64;
  __shared__ float parts[WIDE ? 2 : 1][M][4][WAVES];
  const int nc = (a.k + 127) / 128, l = threadIdx.x % LANES, j = threadIdx.x & 3;
  const int shift = a.group == 32 ? 0 : a.group == 64 ? 1 : 2;
  uint32_t x[M][STEPS][8];
  float xs[M][STEPS];
#pragma unroll
  for (int t = 0; t < M; ++t)
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int q = l + LANES * s, first = 32 * q - 28 * j;  // (the chunk's first column: 128 of 128s, 4 j)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int column = first + 16 * e;
        uint32_t v = 0;
        if (column < a.k) {
          v = *reinterpret_cast<const uint32_t *>(a.xq + (int64_t)t * a.k + column);
          if (a.bias) v = centre4(v);
        }
        x[t][s][e] = v;
      }
      xs[t][s] = q < a.k / 32 ? a.xs[(int64_t)t * (a.k / 32) + q] : 0.0f;
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
#pragma unroll
    for (int t = 0; t < M; ++t) {
      float acc[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        acc[r] = 0.0f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const uint32_t in[4] = {w[r][s].x, w[r][s].y, w[r][s].z, w[r][s].w};
          int32_t sums[4];
#pragma unroll
          for (int g = 0; g < 4; ++g)
            sums[g] = dot4(low_bits(in[g]), x[t][s][2 * g], dot4(high_bits(in[g]), x[t][s][2 * g + 1], 0));
          acc[r] = __builtin_fmaf((float)quad_sums(sums, j), ws[r][s] * xs[t][s], acc[r]);
        }
      }
      float y = quad_sums(acc, j);  // row j's, over the lane's quad
      y += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x124, 0xF, 0xF, true));  // row_ror:4
      y += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(y), 0x128, 0xF, 0xF, true));  // row_ror:8
      if (LANES >= 64) {
        y += __shfl_xor(y, 16);
        y += __shfl_xor(y, 32);
      }
      if (WIDE) {
        if ((threadIdx.x & 63) < 4) parts[turn][t][j][threadIdx.x >> 6] = y;
      } else if (l < 4 && row0 + j < a.rows) {
        a.y[(int64_t)t * a.rows + row0 + j] = y * SIXTEENTH;
      }
    }
    if (WIDE) {  // (the next turn's go to the other half: one barrier)
      __syncthreads();
      if (threadIdx.x < 4 * M) {
        const int t = threadIdx.x >> 2;
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) y += parts[turn][t][j][k];
        if (row0 + j < a.rows) a.y[(int64_t)t * a.rows + row0 + j] = y * SIXTEENTH;
      }
    }
  }
}

// ---- more tokens ----

constexpr int GEMM_WAVES = 8, GEMM_THREADS = 64 * GEMM_WAVES;

// the activations of 16 TILES tokens for PLACES times 128 columns, in the order in which a product takes them, and their scales
template <int TILES, int PLACES>
struct Tokens {
  uint4 x[TILES][PLACES][2][64];
  float4 xs[TILES][PLACES][4][4];
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
      reinterpret_cast<float *>(to.xs[scale(i) % TILES][q][part()])[token()] = (c0 + q) * 4 + part() < a.k / 32 ? f[i] : 0.0f;
    }
  }
};

// a wave's weights of 16 RT rows: DEEP times 128 columns of them, GEMM_WAVES apart, and their scales
template <int RT, int DEEP, int GROUP, bool HALF>
struct Weights {
  static constexpr int EACH = 128 / GROUP;
  typedef typename Scale<HALF>::type scales __attribute__((ext_vector_type(EACH)));
  uint4 in[RT][DEEP];
  scales sc[RT][DEEP];

  __device__ __forceinline__ void read(const FourArgs &a, int64_t row0, int place, int nc) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const int64_t row = min(row0 + 16 * r + (lane & 15), (int64_t)a.rows - 1);
      const uint4 *w = reinterpret_cast<const uint4 *>(a.w) + row * nc * 4 + (lane >> 4);
      const scales *ws = reinterpret_cast<const scales *>(a.ws) + row * nc;
#pragma unroll
      for (int d = 0; d < DEEP; ++d) {
        const int q = min(place + GEMM_WAVES * d, nc - 1);
        in[r][d] = w[q * 4];
        sc[r][d] = ws[q];
      }
    }
  }

  // their products with the tokens at places GEMM_WAVES d + wave of `left`
  template <int TILES, int PLACES>
  __device__ __forceinline__ void multiply(const Tokens<TILES, PLACES> &tokens, int left, float4 (&acc)[RT][TILES]) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int q = GEMM_WAVES * d + wave;
      if (q >= left) break;
      long b[RT][4];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const uint32_t bits[4] = {in[r][d].x, in[r][d].y, in[r][d].z, in[r][d].w};
#pragma unroll
        for (int g = 0; g < 4; ++g) b[r][g] = (long)((uint64_t)high_bits(bits[g]) << 32 | low_bits(bits[g]));
      }
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const uint4 lo = tokens.x[t][q][0][lane], hi = tokens.x[t][q][1][lane];
        const long av[4] = {(long)((uint64_t)lo.y << 32 | lo.x), (long)((uint64_t)lo.w << 32 | lo.z),
                            (long)((uint64_t)hi.y << 32 | hi.x), (long)((uint64_t)hi.w << 32 | hi.z)};
#pragma unroll
        for (int g = 0; g < 4; g += 4 / EACH)
#pragma unroll
          for (int r = 0; r < RT; ++r) {
            float4 y;  // of the groups that share a scale
#pragma unroll
            for (int i = 0; i < 4 / EACH; ++i) {
              const i32x4 s = __builtin_amdgcn_mfma_i32_16x16x32_i8(av[g + i], b[r][g + i], i32x4{0, 0, 0, 0}, 0, 0, 0);
              const float4 fs = tokens.xs[t][q][g + i][lane >> 4];
              if (i == 0) {
                y = make_float4((float)s[0] * fs.x, (float)s[1] * fs.y, (float)s[2] * fs.z, (float)s[3] * fs.w);
              } else {
                y.x = __builtin_fmaf((float)s[0], fs.x, y.x);
                y.y = __builtin_fmaf((float)s[1], fs.y, y.y);
                y.z = __builtin_fmaf((float)s[2], fs.z, y.z);
                y.w = __builtin_fmaf((float)s[3], fs.w, y.w);
              }
            }
            const float scale = (float)sc[r][d][g * EACH / 4];
            acc[r][t].x = __builtin_fmaf(y.x, scale, acc[r][t].x);
            acc[r][t].y = __builtin_fmaf(y.y, scale, acc[r][t].y);
            acc[r][t].z = __builtin_fmaf(y.z, scale, acc[r][t].z);
            acc[r][t].w = __builtin_fmaf(y.w, scale, acc[r][t].w);
          }
      }
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

// D = X W^T, 16 tokens by 16 rows a product: a lane has one row's sums for four tokens, so that the row's scales are its own and
// the tokens' come from LDS four at a time. The waves of a workgroup take the 128s of columns in turn.

// Up to 16 tokens of up to 4096 columns: they stay in LDS, and the workgroup goes from row to row, the next rows' weights on
// their way meanwhile.
constexpr int RESIDENT = 32;  // 128s of columns
template <int GROUP, bool HALF>
__global__ __launch_bounds__(GEMM_THREADS, 4) void rows_kernel(const FourArgs a) {
  constexpr int DEEP = RESIDENT / GEMM_WAVES;
  __shared__ Tokens<1, RESIDENT> tokens;
  __shared__ float4 sums[GEMM_THREADS];  // (half of a CU's LDS in all)
  const int nc = (a.k + 127) / 128, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t step = (int64_t)gridDim.x * 16;
  Weights<1, DEEP, GROUP, HALF> w;
  w.read(a, (int64_t)blockIdx.x * 16, wave, nc);
  Carrier<1, RESIDENT> carrier;
  carrier.read(a, 0, 0);
  carrier.write(a, 0, tokens);
  __syncthreads();
  for (int64_t row0 = (int64_t)blockIdx.x * 16; row0 < a.rows; row0 += step) {
    Weights<1, DEEP, GROUP, HALF> next;
    if (row0 + step < a.rows) next.read(a, row0 + step, wave, nc);
    __builtin_amdgcn_sched_barrier(0);
    float4 acc[1][1] = {{make_float4(0, 0, 0, 0)}};
    w.multiply(tokens, nc, acc);
    sums[threadIdx.x] = acc[0][0];
    __syncthreads();
    finish<1>(a, sums, 0, row0);
    __syncthreads();
    w = next;
  }
}

// Any number of tokens and columns: 16 RT rows by 16 TILES tokens a workgroup, the activations a stage at a time, the next
// stage's on their way meanwhile.
template <int RT, int TILES, int GROUP, bool HALF>
__global__ __launch_bounds__(GEMM_THREADS, RT * TILES <= 2 ? 4 : 2) void stages_kernel(const FourArgs a) {
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
  for (int c0 = 0; c0 < nc; c0 += STAGE) {
    Weights<RT, DEEP, GROUP, HALF> w;
    w.read(a, row0, c0 + wave, nc);
    __builtin_amdgcn_sched_barrier(0);
    if (c0) __syncthreads();  // (the last stage's have been read)
    carrier.write(a, c0, tokens);
    __syncthreads();
    if (c0 + STAGE < nc) carrier.read(a, t0, c0 + STAGE);
    __builtin_amdgcn_sched_barrier(0);
    w.multiply(tokens, nc - c0, acc);
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

template <int LANES, int STEPS, int M, bool HALF>
void launch_gemv(const FourArgs &a, hipStream_t s) {
  constexpr int ROWS = WAVES * 64 / LANES * 4;
  const int blocks = std::min((a.rows + ROWS - 1) / ROWS, 1024);
  hipLaunchKernelGGL((gemv_kernel<LANES, STEPS, M, HALF>), dim3(blocks), dim3(64 * WAVES), 0, s, a);
}

template <bool HALF>
void launch_rows(const FourArgs &a, hipStream_t s) {
  // one workgroup a CU, two where each has many turns (14336 rows 15.8 us against 17.6, 128,256 rows 83 against 73); as many
  // turns for all as for the most
  const int blocks = (a.rows + 15) / 16, most = blocks > 2048 ? 512 : 256;
  const int turns = (blocks + most - 1) / most, grid = (blocks + turns - 1) / turns;
  if (a.group == 32) hipLaunchKernelGGL((rows_kernel<32, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((rows_kernel<64, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
  else hipLaunchKernelGGL((rows_kernel<128, HALF>), dim3(grid), dim3(GEMM_THREADS), 0, s, a);
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
  // rows a workgroup: as many as leave about one workgroup a CU, since each brings the activations to LDS for itself (64 tokens by
  // 14336 rows: 62 us at 16, 45 at 32, 33 at 64; by 4096 rows 21, 23, 31); with one tile of tokens two of rows take more
  // registers than two workgroups a CU leave (4096 rows of 14336 columns: 21 us, 35)
  if constexpr (TILES == 1) {
    launch_stages<1, 1, HALF>(a, s);
  } else {
    if (a.rows >= 12800) launch_stages<4, TILES, HALF>(a, s);
    else if (a.rows >= 6400) launch_stages<2, TILES, HALF>(a, s);
    else launch_stages<1, TILES, HALF>(a, s);
  }
}

template <bool HALF>
void launch(const FourArgs &a, hipStream_t s) {
  const int chunks = (a.k + 127) / 128 * 4;
  // two tokens go this way only over many short rows, whose 128s of columns are fewer than the other kernel's waves (32000 rows
  // of 768 columns: 8.8 us against 15.8; 2304 of 768: 6.1, 5.3; 4096 of 4096: 7.3, 6.9; 4096 of 14336: 17.8, 13.8)
  if (a.m == 2 && chunks <= 32 && a.rows > 8192) {
    if (chunks <= 16) launch_gemv<16, 1, 2, HALF>(a, s);
    else launch_gemv<16, 2, 2, HALF>(a, s);
  } else if (a.m == 1 && chunks <= 1024) {
    if (chunks <= 16) launch_gemv<16, 1, 1, HALF>(a, s);
    else if (chunks <= 32) launch_gemv<16, 2, 1, HALF>(a, s);
    else if (chunks <= 64) launch_gemv<64, 1, 1, HALF>(a, s);
    else if (chunks <= 128) launch_gemv<64, 2, 1, HALF>(a, s);
    else if (chunks <= 256) launch_gemv<64, 4, 1, HALF>(a, s);
    else if (chunks <= 512) launch_gemv<256, 2, 1, HALF>(a, s);
    else launch_gemv<256, 4, 1, HALF>(a, s);
  } else if (a.m <= 16 && chunks <= 4 * RESIDENT) {
    launch_rows<HALF>(a, s);
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
