// logprobs.hip — log probabilities of given tokens, the entropy and the largest alternatives of rows of logits.
//
// With m a row's largest logit and Z = sum exp(x - m): logp_t = x_t - m - log Z, the entropy log Z - H / Z with H = sum
// exp(x - m) (x - m). One pass over the logits: every thread keeps its m, Z and H (rescaled when m grows), and the largest
// are picked out on the way by a threshold that only ever grows. Bound by reading the logits once; a few rows are split
// over many workgroups, whose parts a second launch joins.
#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

constexpr float LOG2E = 1.44269504088896341f;
constexpr float LOWEST = -3.402823466e38f;
constexpr int THREADS = 256, QUADS = 4, BATCH = 4 * QUADS;  // logits a thread takes at once
constexpr int LIST = 1024;  // candidates a workgroup holds: a batch adds at most 16 x 32 behind its threshold

// What a workgroup's part of a row comes to. A logit's key orders logits by value, the lower index first among equals; 0:
// none (a logit of minus infinity has no key).
struct Part {
  float m, z, h;
  int32_t unused;
};

__device__ __forceinline__ uint64_t key_of(float x, uint32_t i) {
  const uint32_t u = __float_as_uint(x + 0.0f);  // (-0 is 0)
  const uint32_t ordered = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x > -__builtin_inff() ? (uint64_t)ordered << 32 | (0xffffffffu - i) : 0;
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

// m, Z, H of two parts together (z 0: an empty part, whatever its m)
template <class T>
__device__ __forceinline__ void join(T &m, T &z, T &h, T m2, T z2, T h2) {
  const T top = m2 > m || m2 != m2 ? m2 : m;  // (a NaN stays)
  // (a part's m may lie 2^128 below: its factor is 0, its difference kept finite)
  const T d1 = m - top < (T)-1e30 ? (T)-1e30 : m - top, d2 = m2 - top < (T)-1e30 ? (T)-1e30 : m2 - top;
  const T f1 = (T)__builtin_amdgcn_exp2f((float)(d1 * (T)LOG2E)), f2 = (T)__builtin_amdgcn_exp2f((float)(d2 * (T)LOG2E));
  h = (h + z * d1) * f1 + (h2 + z2 * d2) * f2;
  z = z * f1 + z2 * f2;
  m = top;
}

struct Shared {
  uint64_t list[LIST];
  uint64_t tops[THREADS];
  uint64_t threshold;
  int count;
  Part parts[THREADS / 64];
};

// the k-th largest of the workgroup's threads' keys (k <= THREADS): no fewer than k keys of the workgroup reach it. By
// counting, for each key, those before it (equal ones, which are 0, by thread).
__device__ __forceinline__ uint64_t kth_of_threads(Shared &s, uint64_t key, int k) {
  const int tid = threadIdx.x;
  __syncthreads();
  s.tops[tid] = key;
  __syncthreads();
  int before = 0;
  for (int i = 0; i < THREADS; i += 2) {
    const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&s.tops[i]);
    before += (o.x > key || (o.x == key && i < tid)) + (o.y > key || (o.y == key && i + 1 < tid));
  }
  if (before == k - 1) s.threshold = key;
  __syncthreads();
  return s.threshold;
}

// the k largest keys of the list, in order, to its front; the list then holds at most k
__device__ __forceinline__ void tighten(Shared &s, int k) {
  const int tid = threadIdx.x, n = s.count;
  uint64_t mine[LIST / THREADS];
  int place[LIST / THREADS];
#pragma unroll
  for (int j = 0; j < LIST / THREADS; ++j) {
    const int i = tid + THREADS * j;
    mine[j] = i < n ? s.list[i] : 0;
    place[j] = 0;
  }
  if (tid + 1 == THREADS && n % 2) s.list[n] = 0;  // (n < LIST)
  __syncthreads();
  for (int i = 0; i < n; i += 2) {
    const ulonglong2 o = *reinterpret_cast<const ulonglong2 *>(&s.list[i]);
#pragma unroll
    for (int j = 0; j < LIST / THREADS; ++j) place[j] += (o.x > mine[j]) + (o.y > mine[j]);
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < LIST / THREADS; ++j)
    if (mine[j] && place[j] < k) s.list[place[j]] = mine[j];
  if (tid == 0) s.count = min(n, k);
  __syncthreads();
}

// up to BATCH keys a thread into the list, those that reach the threshold (which grows where they are too many)
template <int N>
__device__ __forceinline__ void take(Shared &s, const uint64_t (&key)[N], uint64_t &threshold, int k) {
  const int tid = threadIdx.x;
  int n = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) n += key[j] >= threshold;
  if (!__syncthreads_or(n)) return;
  const int held = s.count;
  int at = n ? atomicAdd(&s.count, n) : 0;
  __syncthreads();
  if (s.count >= LIST) {  // (the same in the whole workgroup)
    __syncthreads();
    if (tid == 0) s.count = held;
    uint64_t top = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) top = key[j] > top ? key[j] : top;
    const uint64_t t = kth_of_threads(s, top, k);  // at most k threads' keys reach it: N k in all
    threshold = t > threshold ? t : threshold;
    if (held + N * k >= LIST) {
      tighten(s, k);
      if (s.count == k && s.list[k - 1] > threshold) threshold = s.list[k - 1];
    }
    n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += key[j] >= threshold;
    __syncthreads();
    at = n ? atomicAdd(&s.count, n) : 0;
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (key[j] >= threshold) s.list[at++] = key[j];
}

// the row's results from its joined part and its sorted alternatives
__device__ __forceinline__ void finish(const LogprobArgs &a, int64_t row, double m, double z, double h, const uint64_t *list,
                                       int held) {
  const float *x = a.logits + row * a.stride;
  const bool fine = z > 0.0 && m > (double)-__builtin_inff() && m < (double)__builtin_inff();
  const double nan = __builtin_nan(""), logz = log(z);
  if (threadIdx.x == 0 && a.entropy) a.entropy[row] = (float)(fine ? logz - h / z : nan);
  for (int g = threadIdx.x; g < a.n_given; g += THREADS) {
    const int t = a.given[row * a.n_given + g];
    a.logp[row * a.n_given + g] = (float)(fine && t >= 0 && t < a.n ? (double)x[t] - m - logz : nan);
  }
  for (int i = threadIdx.x; i < a.top; i += THREADS) {
    const bool one = fine && i < held;
    a.ids[row * a.top + i] = one ? (int32_t)(0xffffffffu - (uint32_t)list[i]) : -1;
    a.logps[row * a.top + i] =
        (float)(one ? (double)value_of(list[i]) - m - logz : fine ? (double)-__builtin_inff() : nan);
  }
}

// Workgroup (part, row): `quads` aligned quads of the row's logits from part * quads on. ALONE: the row's only part.
template <bool ALONE, bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(const LogprobArgs a, int quads) {
  __shared__ Shared s;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.y;
  const float *x = a.logits + row * a.stride;
  const int ahead = (int)(reinterpret_cast<uintptr_t>(x) % 16 / 4);  // floats between an aligned address and the row
  const float *base = x - ahead;
  const int all = (int)(((int64_t)ahead + a.n + 3) / 4), from = blockIdx.x * quads, to = min(all, from + quads);
  if (TOP && tid == 0) s.count = 0;
  float m = LOWEST, z = 0.0f, h = 0.0f;
  uint64_t threshold = 0;
  float bar = -__builtin_inff();
  for (int q0 = from; q0 < to; q0 += THREADS * QUADS) {
    float v[BATCH];
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
      const int q = q0 + THREADS * j + tid;
      const int64_t e = (int64_t)q * 4 - ahead;  // the quad's first logit
      float4 w = make_float4(-__builtin_inff(), -__builtin_inff(), -__builtin_inff(), -__builtin_inff());
      if (q < to) {
        if (e >= 0 && e + 4 <= a.n) {
          w = *reinterpret_cast<const float4 *>(base + (int64_t)q * 4);
        } else {
          if (e >= 0 && e < a.n) w.x = x[e];
          if (e + 1 >= 0 && e + 1 < a.n) w.y = x[e + 1];
          if (e + 2 >= 0 && e + 2 < a.n) w.z = x[e + 2];
          if (e + 3 >= 0 && e + 3 < a.n) w.w = x[e + 3];
        }
      }
      v[4 * j] = w.x;
      v[4 * j + 1] = w.y;
      v[4 * j + 2] = w.z;
      v[4 * j + 3] = w.w;
    }
    float most = v[0];
#pragma unroll
    for (int j = 1; j < BATCH; ++j) most = wmax(most, v[j]);
    const float top = wmax(m, most), d = __builtin_fmaxf(m - top, -1e30f), f = __builtin_amdgcn_exp2f(d * LOG2E);
    h = (h + z * d) * f;
    z = z * f;
    m = top;
    float zs = 0.0f, hs = 0.0f;
#pragma unroll
    for (int j = 0; j < BATCH; ++j) {
      const float t = __builtin_fmaxf(v[j] - m, -150.0f), e = __builtin_amdgcn_exp2f(t * LOG2E);
      zs += e;
      hs = __builtin_fmaf(e, t, hs);
    }
    z += zs;
    h += hs;
    if (TOP) {
      if (q0 == from || __syncthreads_or(most >= bar)) {
        uint64_t key[BATCH], best = 0;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          key[j] = key_of(v[j], (uint32_t)((q0 + THREADS * (j / 4) + tid) * 4 - ahead + j % 4));
          best = key[j] > best ? key[j] : best;
        }
        if (q0 == from) {  // the first threshold: the k-th of the threads' largest
          const uint64_t t = kth_of_threads(s, best, a.top);
          threshold = t > 1 ? t : 1;
        }
        take(s, key, threshold, a.top);
        bar = value_of(threshold);
      }
    }
  }
  // the workgroup's part: across the lanes, then the waves
#pragma unroll
  for (int o = 32; o; o >>= 1) join(m, z, h, __shfl_xor(m, o), __shfl_xor(z, o), __shfl_xor(h, o));
  if (tid % 64 == 0) s.parts[tid / 64] = Part{m, z, h, 0};
  __syncthreads();
  if (TOP) tighten(s, a.top);
  double dm = s.parts[0].m, dz = s.parts[0].z, dh = s.parts[0].h;
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w)
    join(dm, dz, dh, (double)s.parts[w].m, (double)s.parts[w].z, (double)s.parts[w].h);
  if (ALONE) {
    finish(a, row, dm, dz, dh, s.list, TOP ? s.count : 0);
    return;
  }
  const int64_t part = row * gridDim.x + blockIdx.x;
  if (tid == 0) reinterpret_cast<Part *>(a.workspace)[part] = Part{(float)dm, (float)dz, (float)dh, 0};
  if (TOP && tid < a.top)
    reinterpret_cast<uint64_t *>(a.workspace + sizeof(Part) * gridDim.x * gridDim.y)[part * a.top + tid] =
        tid < s.count ? s.list[tid] : 0;
}

// the parts of a row (blockIdx.x) together
template <bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_join_kernel(const LogprobArgs a, int parts) {
  __shared__ Shared s;
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x;
  const Part *p = reinterpret_cast<const Part *>(a.workspace) + row * parts;
  if (TOP && tid == 0) s.count = 0;
  float m = LOWEST, z = 0.0f, h = 0.0f;
  for (int i = tid; i < parts; i += THREADS) join(m, z, h, p[i].m, p[i].z, p[i].h);
#pragma unroll
  for (int o = 32; o; o >>= 1) join(m, z, h, __shfl_xor(m, o), __shfl_xor(z, o), __shfl_xor(h, o));
  if (tid % 64 == 0) s.parts[tid / 64] = Part{m, z, h, 0};
  __syncthreads();
  if (TOP) {
    const uint64_t *keys = reinterpret_cast<const uint64_t *>(a.workspace + sizeof(Part) * parts * (int64_t)gridDim.x) +
                           row * parts * a.top;
    uint64_t threshold = 1;
    for (int at = 0; at < parts * a.top; at += THREADS * BATCH) {
      uint64_t key[BATCH], best = 0;
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const int i = at + THREADS * j + tid;
        key[j] = i < parts * a.top ? keys[i] : 0;
        best = key[j] > best ? key[j] : best;
      }
      if (at == 0) {
        const uint64_t t = kth_of_threads(s, best, a.top);
        threshold = t > 1 ? t : 1;
      }
      take(s, key, threshold, a.top);
    }
    __syncthreads();
    tighten(s, a.top);
  }
  double dm = s.parts[0].m, dz = s.parts[0].z, dh = s.parts[0].h;
#pragma unroll
  for (int w = 1; w < THREADS / 64; ++w)
    join(dm, dz, dh, (double)s.parts[w].m, (double)s.parts[w].z, (double)s.parts[w].h);
  finish(a, row, dm, dz, dh, s.list, TOP ? s.count : 0);
}

// a row's parts: enough workgroups for the card, each with at least a thousand logits
int parts_of(int32_t m, int32_t n) {
  const int64_t most = ((int64_t)n + 1023) / 1024, wanted = (1024 + (int64_t)m - 1) / m;
  return (int)(wanted < most ? wanted : most);
}

}  // namespace

int64_t logprobs_workspace(int32_t m, int32_t n, int32_t top) {
  const int64_t parts = parts_of(m, n);
  return parts == 1 ? 0 : parts * m * ((int64_t)sizeof(Part) + 8 * top);
}

hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s) {
  const int parts = parts_of(a.m, a.n);
  // (three floats more than n where a row starts behind an aligned address)
  const int quads = (int)((((int64_t)a.n + 6) / 4 + parts - 1) / parts);
  for (int32_t row = 0; row < a.m; row += 65535) {
    LogprobArgs b = a;
    b.m = a.m - row < 65535 ? a.m - row : 65535;
    if (a.logp) b.logp = a.logp + (int64_t)row * a.n_given;
    if (a.given) b.given = a.given + (int64_t)row * a.n_given;
    if (a.entropy) b.entropy = a.entropy + row;
    if (a.ids) b.ids = a.ids + (int64_t)row * a.top;
    if (a.logps) b.logps = a.logps + (int64_t)row * a.top;
    b.logits = a.logits + row * a.stride;
    const dim3 grid(parts, b.m);
    if (parts == 1) {
      if (a.top) hipLaunchKernelGGL((logprobs_kernel<true, true>), grid, dim3(THREADS), 0, s, b, quads);
      else hipLaunchKernelGGL((logprobs_kernel<true, false>), grid, dim3(THREADS), 0, s, b, quads);
    } else if (a.top) {
      hipLaunchKernelGGL((logprobs_kernel<false, true>), grid, dim3(THREADS), 0, s, b, quads);
      hipLaunchKernelGGL(logprobs_join_kernel<true>, dim3(b.m), dim3(THREADS), 0, s, b, parts);
    } else {
      hipLaunchKernelGGL((logprobs_kernel<false, false>), grid, dim3(THREADS), 0, s, b, quads);
      hipLaunchKernelGGL(logprobs_join_kernel<false>, dim3(b.m), dim3(THREADS), 0, s, b, parts);
    }
  }
  return hipGetLastError();
}

}  // namespace ple
