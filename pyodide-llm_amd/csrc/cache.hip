// cache.hip — rows into and out of the cache held in 8 bits (cache.hpp): append, read and rewind.
#include "cache.hpp"

namespace ple {

namespace {

// the float32 row (this kv head's hs values) of position p, which lies in the call's first block or after it: an earlier
// one from the recent rows, the call's own from k / v
__device__ __forceinline__ const float *row_of(const CacheRows &a, const float *x, const float *recent, int p, int pos,
                                               int head) {
  if (p >= pos) return x + (int64_t)(p - pos) * a.x_stride + head * a.c.hs;
  const int row = a.displaced ? CACHE_RECENT + p % CACHE_BLOCK : p % CACHE_RECENT;
  return recent + ((int64_t)row * a.c.nkv + head) * a.c.hs;
}

// q = x / s rounded to the nearest integer, ties to even, exactly: the float32 quotient is off by half a step of its own
// at most, so its nearest integer n is the answer or next to it, and x - n s is exact in one fma (n s has 31 bits and
// lies within s of x), so that comparing twice it with s decides
__device__ __forceinline__ int nearest_quotient(float x, float s) {
  if (!(s > 0.0f) || !(s < __builtin_inff())) return 0;  // (a scale that is not finite stands for what is not a number)
  float n = __builtin_rintf(x / s);
  const float over = __builtin_fmaf(-n, s, x), twice = over + over;
  const bool odd = ((int)n & 1) != 0;
  if (twice > s || (twice == s && odd)) n += 1.0f;
  else if (-twice > s || (-twice == s && odd)) n -= 1.0f;
  return max(-127, min(127, (int)n));  // (past it only where the scale is a denormal of few bits)
}

// One (block, kv head, keys or values) a workgroup: the block's rows read once, kept in registers; a complete block's
// largest magnitude gives its scale, its bytes go through LDS into the cache's order; the call's rows among the latest
// 128 positions are copied. Bound by memory: each float32 value is read once, each byte written once.
template <int HS>
__global__ __launch_bounds__(256) void append_kernel(const CacheRows a) {
  constexpr int QUADS = CACHE_BLOCK * HS / 4, EACH = (QUADS + 255) / 256;
  const int pos = a.dpos ? *a.dpos : a.pos, end = pos + a.count;
  const int block = pos / CACHE_BLOCK + blockIdx.x, head = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
  const int p0 = block * CACHE_BLOCK;
  const float *x = which ? a.v : a.k;
  float *recent = which ? a.c.recent_values : a.c.recent_keys;
  const bool whole = p0 + CACHE_BLOCK <= end;
  float4 v[EACH];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int f = tid + 256 * i, t = f / (HS / 4), d = f % (HS / 4) * 4, p = p0 + t;
    v[i] = make_float4(0, 0, 0, 0);
    if (QUADS % 256 && f >= QUADS) continue;
    if (p < end && (whole || p >= pos))
      v[i] = *reinterpret_cast<const float4 *>(row_of(a, x, recent, p, pos, head) + d);
    top = wmax(top, wmax(wmax(__builtin_fabsf(v[i].x), __builtin_fabsf(v[i].y)),
                         wmax(__builtin_fabsf(v[i].z), __builtin_fabsf(v[i].w))));
  }
  __shared__ float tops[4];
  __shared__ alignas(16) uint8_t bytes[CACHE_BLOCK * HS];
  if (whole) {  // (the same in the whole workgroup)
#pragma unroll
    for (int o = 32; o; o >>= 1) top = wmax(top, __shfl_xor(top, o));
    if (tid % 64 == 0) tops[tid / 64] = top;
    __syncthreads();
    const float s = wmax(wmax(tops[0], tops[1]), wmax(tops[2], tops[3])) * (1.0f / 127.0f);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int f = tid + 256 * i, t = f / (HS / 4), d = f % (HS / 4) * 4;
      if (QUADS % 256 && f >= QUADS) continue;
      const float in[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
      uint32_t packed = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = nearest_quotient(in[j], s);
        if (which) bytes[(d + j) * CACHE_BLOCK + value_byte(t)] = (uint8_t)(q + 128);
        else packed |= (uint32_t)(uint8_t)(int8_t)q << (8 * j);
      }
      if (!which) *reinterpret_cast<uint32_t *>(bytes + (d / 16 * CACHE_BLOCK + t) * 16 + d % 16) = packed;
    }
    __syncthreads();
    const int64_t at = (int64_t)head * a.c.blocks + block;
    uint8_t *out = (which ? a.c.values : reinterpret_cast<uint8_t *>(a.c.keys)) + at * (CACHE_BLOCK * HS);
    for (int i = tid; i < CACHE_BLOCK * HS / 16; i += 256)
      reinterpret_cast<uint4 *>(out)[i] = reinterpret_cast<const uint4 *>(bytes)[i];
    if (tid == 0) a.c.scales[at * 2 + which] = s;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int f = tid + 256 * i, t = f / (HS / 4), d = f % (HS / 4) * 4, p = p0 + t;
    if (QUADS % 256 && f >= QUADS) continue;
    if (p >= pos && p < end && p >= end - CACHE_RECENT)
      *reinterpret_cast<float4 *>(recent + ((int64_t)(p % CACHE_RECENT) * a.c.nkv + head) * HS + d) = v[i];
  }
}

// the recent rows of positions first..pos-1 into the places that a longer call's rows cannot displace
__global__ __launch_bounds__(256) void set_apart_kernel(const CacheView c, int first, int pos) {
  const int width = c.nkv * c.hs, p = first + blockIdx.x;
  for (int i = threadIdx.x; i < width; i += 256) {
    const int64_t from = (int64_t)(p % CACHE_RECENT) * width + i, to = (int64_t)(CACHE_RECENT + p - first) * width + i;
    c.recent_keys[to] = c.recent_keys[from];
    c.recent_values[to] = c.recent_values[from];
  }
}

// positions from.. as float32 rows: by their 8-bit values, those of block `recent_block` from the recent rows; into
// k / v [count][n_kv * hs], or (k null) into the recent rows
__global__ __launch_bounds__(256) void read_kernel(const CacheView c, float *k, float *v, int from, int recent_block) {
  const int p = from + blockIdx.x, width = c.nkv * c.hs, block = p / CACHE_BLOCK, t = p % CACHE_BLOCK;
  const int64_t recent = (int64_t)(p % CACHE_RECENT) * width;
  for (int i = threadIdx.x; i < width; i += 256) {
    const int head = i / c.hs, d = i % c.hs;
    float kv, vv;
    if (block != recent_block) {
      const int64_t at = (int64_t)head * c.blocks + block, base = at * CACHE_BLOCK * c.hs;
      kv = (float)c.keys[base + (d / 16 * CACHE_BLOCK + t) * 16 + d % 16] * c.scales[at * 2];
      vv = (float)((int)c.values[base + (int64_t)d * CACHE_BLOCK + value_byte(t)] - 128) * c.scales[at * 2 + 1];
    } else {
      kv = c.recent_keys[recent + i];
      vv = c.recent_values[recent + i];
    }
    if (k) {
      k[(int64_t)blockIdx.x * width + i] = kv;
      v[(int64_t)blockIdx.x * width + i] = vv;
    } else {
      c.recent_keys[recent + i] = kv;
      c.recent_values[recent + i] = vv;
    }
  }
}

template <int HS>
void launch_append(const CacheRows &a, int blocks, hipStream_t s) {
  hipLaunchKernelGGL(append_kernel<HS>, dim3(blocks, a.c.nkv, 2), dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_cache_append(const CacheRows &rows, hipStream_t s) {
  CacheRows a = rows;
  const int first = a.pos / CACHE_BLOCK * CACHE_BLOCK;
  a.displaced = cache_displaces(a.pos, a.count);
  if (a.displaced && a.pos > first)
    hipLaunchKernelGGL(set_apart_kernel, dim3(a.pos - first), dim3(256), 0, s, a.c, first, a.pos);
  const int blocks = (a.pos + a.count - 1) / CACHE_BLOCK - a.pos / CACHE_BLOCK + 1;
  switch (a.c.hs) {
    case 16: launch_append<16>(a, blocks, s); break;
    case 32: launch_append<32>(a, blocks, s); break;
    case 48: launch_append<48>(a, blocks, s); break;
    case 64: launch_append<64>(a, blocks, s); break;
    case 96: launch_append<96>(a, blocks, s); break;
    case 128: launch_append<128>(a, blocks, s); break;
    case 256: launch_append<256>(a, blocks, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_cache_read(const CacheView &c, float *keys, float *values, int32_t from, int32_t count, int32_t recent,
                             hipStream_t s) {
  hipLaunchKernelGGL(read_kernel, dim3(count), dim3(256), 0, s, c, keys, values, from, recent);
  return hipGetLastError();
}

}  // namespace ple
