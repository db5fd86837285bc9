// four.hip — products with 4-bit matrices (include/pyodide_llm_hip.h hk_matmul_four): w in -8..7 with a scale a row and group
// of columns, against activations quantized per group of 32.
//
// y[t][r] = sum_g ws[r][g] xs[t][g] S_g, S_g = the sum of w (xq - bias) over the 32 columns of group g, exact in int32; the
// float32 sums over the groups run in no order of the reference's, which has no 4-bit kernels.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

constexpr int TOKENS = 4;  // a workgroup's tokens
constexpr int WAVES = 4;

// s[g], g = 0..3, added over the four lanes of a quad: the lane j has group j's sum
__device__ __forceinline__ int32_t quad_sums(const int32_t (&s)[4], int j) {
  const bool odd = j & 1, high = j & 2;
  const int32_t a = (odd ? s[1] : s[0]) + dpp_xor1(odd ? s[0] : s[1]), b = (odd ? s[3] : s[2]) + dpp_xor1(odd ? s[2] : s[3]);
  return (high ? b : a) + __builtin_amdgcn_mov_dpp(high ? a : b, 0x4E, 0xF, 0xF, true);  // lane ^ 2
}

constexpr int STAGE = 64;  // of 128 columns, whose activations lie in LDS at a time

// A wave a row. A lane takes 16 bytes at a time: eight columns of each of four groups (chunk j of the 128 columns c); the four
// lanes' sums of a group come together in one of them.
template <int GROUP, bool HALF>
__global__ __launch_bounds__(64 * WAVES) void four_kernel(const FourArgs a) {
  // the tokens' values in the rows' order: a lane's low columns, then its high ones; and the groups' scales
  __shared__ uint4 x[TOKENS][STAGE * 4][2];
  __shared__ float xs[TOKENS][STAGE * 4];
  const int nc = (a.k + 127) / 128, t0 = blockIdx.y * TOKENS, m = min(TOKENS, a.m - t0);
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6);
  const uint4 *w = reinterpret_cast<const uint4 *>(a.w) + row * nc * 4;
  float acc[TOKENS] = {};
  for (int c0 = 0; c0 < nc; c0 += STAGE) {
    const int n = min(STAGE, nc - c0);
    __syncthreads();
    for (int e = threadIdx.x; e < m * n * 32; e += 64 * WAVES) {
      const int t = e / (n * 32), d = e % (n * 32), c = d / 32, g = d / 8 % 4, h = d / 4 % 2, j = d % 4;
      const int column = c0 * 128 + 4 * d;
      uint32_t v = 0;
      if (column < a.k) {
        v = *reinterpret_cast<const uint32_t *>(a.xq + (int64_t)(t0 + t) * a.k + column);
        if (a.bias) v = centre4(v);
      }
      reinterpret_cast<uint32_t *>(&x[t][c * 4 + j][h])[g] = v;
    }
    for (int e = threadIdx.x; e < m * n * 4; e += 64 * WAVES) {
      const int t = e / (n * 4), g = e % (n * 4);
      xs[t][g] = c0 * 4 + g < a.k / 32 ? a.xs[(int64_t)(t0 + t) * (a.k / 32) + c0 * 4 + g] : 0.0f;
    }
    __syncthreads();
    if (row >= a.rows) continue;
    for (int q = lane; q < n * 4; q += 64) {
      const uint4 v = w[c0 * 4 + q];
      const int64_t at = (row * nc + c0) * (128 / GROUP) + q / (GROUP / 32);
      const float s = HALF ? (float)reinterpret_cast<const _Float16 *>(a.ws)[at] : reinterpret_cast<const float *>(a.ws)[at];
      const uint32_t in[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int t = 0; t < TOKENS; ++t) {
        if (t >= m) break;
        const uint4 lo = x[t][q][0], hi = x[t][q][1];
        const uint32_t xl[4] = {lo.x, lo.y, lo.z, lo.w}, xh[4] = {hi.x, hi.y, hi.z, hi.w};
        int32_t sums[4];
#pragma unroll
        for (int g = 0; g < 4; ++g)  // (four bits in the upper half of a byte: sixteen times the value)
          sums[g] = dot4((in[g] << 4) & 0xF0F0F0F0u, xl[g], dot4(in[g] & 0xF0F0F0F0u, xh[g], 0));
        acc[t] += (float)quad_sums(sums, q & 3) * (s * xs[t][q]);
      }
    }
  }
  if (row >= a.rows) return;
#pragma unroll
  for (int t = 0; t < TOKENS; ++t) {
    if (t >= m) break;
    const float y = wave_sum(acc[t]) * 0.0625f;
    if (lane == 0) a.y[(int64_t)(t0 + t) * a.rows + row] = y;
  }
}

template <int GROUP, bool HALF>
void launch(const FourArgs &a, hipStream_t s) {
  hipLaunchKernelGGL((four_kernel<GROUP, HALF>), dim3((a.rows + WAVES - 1) / WAVES, (a.m + TOKENS - 1) / TOKENS), dim3(64 * WAVES), 0, s,
                     a);
}

}  // namespace

hipError_t launch_matmul_four(const FourArgs &a, hipStream_t s) {
  switch (a.group * 2 + (a.half ? 1 : 0)) {
    case 64: launch<32, false>(a, s); break;
    case 65: launch<32, true>(a, s); break;
    case 128: launch<64, false>(a, s); break;
    case 129: launch<64, true>(a, s); break;
    case 256: launch<128, false>(a, s); break;
    case 257: launch<128, true>(a, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ple
