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

// 16 rows by TILES times 16 tokens a workgroup, whose waves take the 128s of columns in turn. The activations go through LDS,
// a stage at a time, in the order in which a product takes them. D = X W^T: a lane has one row's sums for four tokens, so that
// the row's scales are its own and the tokens' come from LDS four at a time.
template <int TILES, int GROUP, bool HALF>
__global__ __launch_bounds__(64 * WAVES) void gemm_kernel(const FourArgs a) {
  constexpr int DEEP = TILES == 4 ? 1 : 4 / TILES, STAGE = WAVES * DEEP;  // 128s of columns a wave and a stage take
  constexpr int EACH = 128 / GROUP;                                       // scales a row has for them
  __shared__ uint4 x[TILES][STAGE][2][64];
  __shared__ float4 xs[TILES][STAGE][4][4];
  const int nc = (a.k + 127) / 128, t0 = blockIdx.y * (16 * TILES);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, j = lane >> 4;
  const int64_t row = (int64_t)blockIdx.x * 16 + c, held = min(row, (int64_t)a.rows - 1);
  const uint4 *w = reinterpret_cast<const uint4 *>(a.w) + held * nc * 4 + j;
  const int64_t scales = held * nc * EACH;
  float4 acc[TILES];
#pragma unroll
  for (int t = 0; t < TILES; ++t) acc[t] = make_float4(0, 0, 0, 0);
  uint4 in[DEEP];
  float ws[DEEP][EACH];
  auto read = [&](int c0) {
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int q = min(c0 + WAVES * d + wave, nc - 1);
      in[d] = w[q * 4];
#pragma unroll
      for (int i = 0; i < EACH; ++i) {
        const int64_t at = scales + q * EACH + i;
        ws[d][i] = HALF ? (float)reinterpret_cast<const _Float16 *>(a.ws)[at] : reinterpret_cast<const float *>(a.ws)[at];
      }
    }
  };
  read(0);
  for (int c0 = 0; c0 < nc; c0 += STAGE) {
    __syncthreads();
    for (int e = threadIdx.x; e < TILES * STAGE * 128; e += 64 * WAVES) {
      const int token = e & 15, part = e >> 4 & 3, half = e >> 6 & 1, q = (e >> 7) % STAGE, tile = (e >> 7) / STAGE;
      const int column = (c0 + q) * 128 + half * 64 + part * 16, t = t0 + tile * 16 + token;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (t < a.m && column < a.k) {
        v = *reinterpret_cast<const uint4 *>(a.xq + (int64_t)t * a.k + column);
        if (a.bias) v.x = centre4(v.x), v.y = centre4(v.y), v.z = centre4(v.z), v.w = centre4(v.w);
      }
      uint32_t *to = reinterpret_cast<uint32_t *>(&x[tile][q][half][token]) + part;
      to[0] = v.x, to[64] = v.y, to[128] = v.z, to[192] = v.w;
    }
    for (int e = threadIdx.x; e < TILES * STAGE * 64; e += 64 * WAVES) {
      const int token = e & 15, g = e >> 4 & 3, q = (e >> 6) % STAGE, tile = (e >> 6) / STAGE;
      const int group = (c0 + q) * 4 + g, t = t0 + tile * 16 + token;
      reinterpret_cast<float *>(xs[tile][q][g])[token] =
          t < a.m && group < a.k / 32 ? a.xs[(int64_t)t * (a.k / 32) + group] : 0.0f;
    }
    __syncthreads();
    uint4 now[DEEP];
    float sc[DEEP][EACH];
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      now[d] = in[d];
#pragma unroll
      for (int i = 0; i < EACH; ++i) sc[d][i] = ws[d][i];
    }
    if (c0 + STAGE < nc) read(c0 + STAGE);
#pragma unroll
    for (int d = 0; d < DEEP; ++d) {
      const int q = WAVES * d + wave;
      const uint32_t n[4] = {now[d].x, now[d].y, now[d].z, now[d].w};
      long b[4];
#pragma unroll
      for (int g = 0; g < 4; ++g) b[g] = (long)((uint64_t)high_bits(n[g]) << 32 | low_bits(n[g]));
#pragma unroll
      for (int t = 0; t < TILES; ++t) {
        const uint4 lo = x[t][q][0][lane], hi = x[t][q][1][lane];
        const long av[4] = {(long)((uint64_t)lo.y << 32 | lo.x), (long)((uint64_t)lo.w << 32 | lo.z),
                            (long)((uint64_t)hi.y << 32 | hi.x), (long)((uint64_t)hi.w << 32 | hi.z)};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const i32x4 s = __builtin_amdgcn_mfma_i32_16x16x32_i8(av[g], b[g], i32x4{0, 0, 0, 0}, 0, 0, 0);
          const float4 f = xs[t][q][g][j];
          const float r = sc[d][g * EACH / 4];
          acc[t].x = __builtin_fmaf((float)s[0], r * f.x, acc[t].x);
          acc[t].y = __builtin_fmaf((float)s[1], r * f.y, acc[t].y);
          acc[t].z = __builtin_fmaf((float)s[2], r * f.z, acc[t].z);
          acc[t].w = __builtin_fmaf((float)s[3], r * f.w, acc[t].w);
        }
      }
    }
  }
  __syncthreads();
  float4 *sums = reinterpret_cast<float4 *>(x);  // [tile][wave][lane]
#pragma unroll
  for (int t = 0; t < TILES; ++t) sums[(t * WAVES + wave) * 64 + lane] = acc[t];
  __syncthreads();
  for (int e = threadIdx.x; e < TILES * 256; e += 64 * WAVES) {
    const int col = e & 15, r = e >> 4 & 3, quarter = e >> 6 & 3, tile = e >> 8;
    const float *from = reinterpret_cast<const float *>(sums + tile * WAVES * 64 + quarter * 16 + col) + r;
    float y = 0.0f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) y += from[k * 256];
    const int t = t0 + tile * 16 + quarter * 4 + r;
    const int64_t out = (int64_t)blockIdx.x * 16 + col;
    if (t < a.m && out < a.rows) a.y[(int64_t)t * a.rows + out] = y * SIXTEENTH;
  }
}

template <int LANES, int STEPS, bool HALF>
void launch_gemv(const FourArgs &a, hipStream_t s) {
  constexpr int ROWS = WAVES * 64 / LANES * 4;
  const int blocks = std::min((a.rows + ROWS - 1) / ROWS, 1024);
  if (a.m == 1) hipLaunchKernelGGL((gemv_kernel<LANES, STEPS, 1, HALF>), dim3(blocks), dim3(64 * WAVES), 0, s, a);
  else hipLaunchKernelGGL((gemv_kernel<LANES, STEPS, 2, HALF>), dim3(blocks), dim3(64 * WAVES), 0, s, a);
}

template <int TILES, bool HALF>
void launch_gemm(const FourArgs &a, hipStream_t s) {
  const dim3 grid((a.rows + 15) / 16, (a.m + 16 * TILES - 1) / (16 * TILES)), block(64 * WAVES);
  if (a.group == 32) hipLaunchKernelGGL((gemm_kernel<TILES, 32, HALF>), grid, block, 0, s, a);
  else if (a.group == 64) hipLaunchKernelGGL((gemm_kernel<TILES, 64, HALF>), grid, block, 0, s, a);
  else hipLaunchKernelGGL((gemm_kernel<TILES, 128, HALF>), grid, block, 0, s, a);
}

template <bool HALF>
void launch(const FourArgs &a, hipStream_t s) {
  const int chunks = (a.k + 127) / 128 * 4;
  if (a.m <= 2 && chunks <= 1024) {
    if (chunks <= 16) launch_gemv<16, 1, HALF>(a, s);
    else if (chunks <= 32) launch_gemv<16, 2, HALF>(a, s);
    else if (chunks <= 64) launch_gemv<64, 1, HALF>(a, s);
    else if (chunks <= 128) launch_gemv<64, 2, HALF>(a, s);
    else if (chunks <= 256) launch_gemv<64, 4, HALF>(a, s);
    else if (chunks <= 512) launch_gemv<256, 2, HALF>(a, s);
    else launch_gemv<256, 4, HALF>(a, s);
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
