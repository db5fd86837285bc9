// logprobs.hip — log probabilities of given tokens, the entropy and the largest alternatives of rows of logits.
#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

// One row a workgroup of 256 threads. With m the row's largest logit: Z = sum exp(x - m), logp = x_t - m - log Z, the entropy
// log Z - sum exp(x - m) (x - m) / Z. A row whose largest logit is not finite has no probabilities: NaN everywhere, no
// alternatives (-1). A logit of minus infinity has probability 0: no alternative, nothing of the entropy.
__global__ __launch_bounds__(256) void logprobs_kernel(const LogprobArgs a) {
  const float *x = a.logits + (int64_t)blockIdx.x * a.stride;
  const int tid = threadIdx.x;
  __shared__ float sf[256];
  __shared__ double sd[256];
  __shared__ int si[256];
  float m = -__builtin_inff();
  for (int i = tid; i < a.n; i += 256) m = wmax(m, x[i]);
  sf[tid] = m;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (tid < o) sf[tid] = wmax(sf[tid], sf[tid + o]);
    __syncthreads();
  }
  m = sf[0];
  double z = 0, h = 0;
  for (int i = tid; i < a.n; i += 256) {
    const float d = x[i] - m, e = __expf(d);
    z += e;
    if (e > 0.0f) h += (double)(e * d);
  }
  sd[tid] = z;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (tid < o) sd[tid] += sd[tid + o];
    __syncthreads();
  }
  z = sd[0];
  __syncthreads();
  sd[tid] = h;
  __syncthreads();
  for (int o = 128; o; o >>= 1) {
    if (tid < o) sd[tid] += sd[tid + o];
    __syncthreads();
  }
  h = sd[0];
  const bool fine = __builtin_fabsf(m) < __builtin_inff();
  const float nan = __builtin_nanf("");
  const double logz = log(z);
  if (tid == 0 && a.entropy) a.entropy[blockIdx.x] = fine ? (float)(logz - h / z) : nan;
  for (int g = tid; g < a.n_given; g += 256) {
    const int t = a.given[(int64_t)blockIdx.x * a.n_given + g];
    a.logp[(int64_t)blockIdx.x * a.n_given + g] = fine && t >= 0 && t < a.n ? (float)((double)x[t] - m - logz) : nan;
  }
  // the alternatives one at a time: the largest logit behind the one before it, the lowest index among equals
  float last = __builtin_inff();
  int at = -1;
  for (int k = 0; k < a.top; ++k) {
    float best = -__builtin_inff();
    int bi = 0x7fffffff;
    for (int i = tid; i < a.n; i += 256) {
      const float v = x[i];
      if (v < last || (v == last && i > at))
        if (v > best) {
          best = v;
          bi = i;
        }
    }
    __syncthreads();
    sf[tid] = best;
    si[tid] = bi;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
      if (tid < o && (sf[tid + o] > sf[tid] || (sf[tid + o] == sf[tid] && si[tid + o] < si[tid]))) {
        sf[tid] = sf[tid + o];
        si[tid] = si[tid + o];
      }
      __syncthreads();
    }
    last = sf[0];
    at = si[0];
    if (tid == 0) {
      const bool one = fine && last > -__builtin_inff();
      a.ids[(int64_t)blockIdx.x * a.top + k] = one ? at : -1;
      a.logps[(int64_t)blockIdx.x * a.top + k] = one ? (float)((double)last - m - logz) : fine ? last : nan;
    }
  }
}

}  // namespace

int64_t logprobs_workspace(int32_t, int32_t, int32_t) { return 0; }

hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s) {
  hipLaunchKernelGGL(logprobs_kernel, dim3(a.m), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ple
