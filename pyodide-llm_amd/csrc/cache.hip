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

// x / s rounded to the nearest integer, ties to even, exactly: x times 1 / s is off by 2^-22 of itself at most, so its nearest
// integer n is the answer or next to it, and x - n s is exact in one fma (n s has 31 bits and lies within s of x), so that
// comparing twice it with s decides. A scale that is next to nothing is taken up by 2^64 first, and x with it. (A
// division for every value: 15.3 us for 2048 tokens of 8 heads of 128 in and out again; so 14.2.)
struct Quotient {
  float s, inverse, up;
  bool none;
  __device__ __forceinline__ explicit Quotient(float scale) {
    none = !(scale > 0.0f) || !(scale < __builtin_inff());  // (a scale that is not finite stands for what is not a number)
    up = scale < 0x1p-60f ? 0x1p64f : 1.0f;
    s = scale * up;
    inverse = 1.0f / s;
  }
  __device__ __forceinline__ int operator()(float x) const {
    x *= up;
    const float n = __builtin_rintf(x * inverse), over = __builtin_fmaf(-n, s, x), twice = over + over;
    int q = (int)n;
    const int odd = q & 1;
    q += (twice > s) + (odd & (twice == s)) - (-twice > s) - (odd & (-twice == s));
    return none ? 0 : max(-127, min(127, q));  // (past it only where the scale is a denormal of few bits)
  }
};

// where a block's bytes lie in LDS on their way into (and out of) the cache's order: a chunk of 16 channels of keys takes
// 512 + 16 bytes, a channel of values 32 + 4, so that the lanes of a row, four channels apart, meet few others' banks
__device__ __forceinline__ constexpr int key_at(int t, int d) { return d / 16 * 528 + t * 16 + d % 16; }
__device__ __forceinline__ constexpr int value_at(int byte, int d) { return d * 36 + byte; }
template <int HS>
constexpr int lds_bytes() { return HS * 36; }

// One (block, kv head, keys or values) a workgroup; a thread takes four positions of four channels, so that keys leave it as
// a word a position and values as a word a channel. The block's rows are read once and kept in registers; a complete
// block's largest magnitude gives its scale, its bytes go through LDS into the cache's order; the call's rows among the
// latest 128 positions are copied. Bound by memory: each float32 value is read once, each byte written once (2048 tokens of 8
// heads of 128: 7.4 us, 21 MB; out again by read_kernel 5.9). A token's call is latency, 3 us.
template <int HS>
__global__ __launch_bounds__(256) void append_kernel(const CacheRows a) {
  constexpr int UNITS = CACHE_BLOCK / 4 * (HS / 4), EACH = (UNITS + 255) / 256;
  const int pos = a.dpos ? *a.dpos : a.pos, end = pos + a.count;
  const int block = pos / CACHE_BLOCK + blockIdx.x, head = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
  const int p0 = block * CACHE_BLOCK;
  const float *x = which ? a.v : a.k;
  float *recent = which ? a.c.recent_values : a.c.recent_keys;
  const bool whole = p0 + CACHE_BLOCK <= end;
  float4 v[EACH][4];
  float top = 0.0f;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int u = tid + 256 * i, t = u / (HS / 4) * 4, d = u % (HS / 4) * 4;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + t + r;
      v[i][r] = make_float4(0, 0, 0, 0);
      if ((UNITS % 256 == 0 || u < UNITS) && p < end && (whole || p >= pos))
        v[i][r] = *reinterpret_cast<const float4 *>(row_of(a, x, recent, p, pos, head) + d);
    }
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      top = wmax(top, wmax(wmax(__builtin_fabsf(v[i][r].x), __builtin_fabsf(v[i][r].y)),
                           wmax(__builtin_fabsf(v[i][r].z), __builtin_fabsf(v[i][r].w))));
  __shared__ float tops[4];
  __shared__ alignas(16) uint8_t bytes[lds_bytes<HS>()];
  if (whole) {  // (the same in the whole workgroup)
    top = wave_top(top);
    if (tid % 64 == 0) tops[tid / 64] = top;
    __syncthreads();
    const float s = wmax(wmax(tops[0], tops[1]), wmax(tops[2], tops[3])) * (1.0f / 127.0f);
    const Quotient quotient(s);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const int u = tid + 256 * i, t = u / (HS / 4) * 4, d = u % (HS / 4) * 4;
      if (UNITS % 256 && u >= UNITS) continue;
      uint32_t q[4][4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float in[4] = {v[i][r].x, v[i][r].y, v[i][r].z, v[i][r].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) q[r][j] = (uint32_t)(quotient(in[j]) + (which ? 128 : 0)) & 255u;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<uint32_t *>(bytes + (which ? value_at(value_byte(t), d + r) : key_at(t + r, d))) =
            which ? q[0][r] | q[1][r] << 8 | q[2][r] << 16 | q[3][r] << 24
                  : q[r][0] | q[r][1] << 8 | q[r][2] << 16 | q[r][3] << 24;
    }
    __syncthreads();
    const int64_t at = (int64_t)head * a.c.blocks + block;
    uint8_t *out = (which ? a.c.values : reinterpret_cast<uint8_t *>(a.c.keys)) + at * (CACHE_BLOCK * HS);
    for (int i = tid; i < CACHE_BLOCK * HS / 16; i += 256) {
      const uint32_t *from = reinterpret_cast<const uint32_t *>(
          bytes + (which ? value_at(i % 2 * 16, i / 2) : key_at(i % CACHE_BLOCK, i / CACHE_BLOCK * 16)));
      reinterpret_cast<uint4 *>(out)[i] = make_uint4(from[0], from[1], from[2], from[3]);
    }
    if (tid == 0) a.c.scales[at * 2 + which] = s;
  }
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int u = tid + 256 * i, t = u / (HS / 4) * 4, d = u % (HS / 4) * 4;
    if (UNITS % 256 && u >= UNITS) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int p = p0 + t + r;
      if (p >= pos && p < end && p >= end - CACHE_RECENT)
        *reinterpret_cast<float4 *>(recent + ((int64_t)(p % CACHE_RECENT) * a.c.nkv + head) * HS + d) = v[i][r];
    }
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

// One (block, kv head, keys or values) a workgroup: positions from..to - 1 of it as float32 rows, by their 8-bit values (read
// in the cache's order, turned through LDS), those of block `recent_block` from the recent rows; into k / v
// [to - from][n_kv * hs], or (null) into the recent rows
template <int HS>
__global__ __launch_bounds__(256) void read_kernel(const CacheView c, float *k, float *v, int from, int to,
                                                   int recent_block) {
  const int block = from / CACHE_BLOCK + blockIdx.x, head = blockIdx.y, which = blockIdx.z, tid = threadIdx.x;
  const int p0 = block * CACHE_BLOCK;
  float *recent = which ? c.recent_values : c.recent_keys, *out = which ? v : k;
  const bool eight = block != recent_block;
  __shared__ alignas(16) uint8_t bytes[lds_bytes<HS>()];
  float s = 0.0f;
  if (eight) {  // (the same in the whole workgroup)
    const int64_t at = (int64_t)head * c.blocks + block;
    const uint8_t *in = (which ? c.values : reinterpret_cast<const uint8_t *>(c.keys)) + at * (CACHE_BLOCK * HS);
    s = c.scales[at * 2 + which];
    for (int i = tid; i < CACHE_BLOCK * HS / 16; i += 256) {
      const uint4 w = reinterpret_cast<const uint4 *>(in)[i];
      uint32_t *to_lds = reinterpret_cast<uint32_t *>(
          bytes + (which ? value_at(i % 2 * 16, i / 2) : key_at(i % CACHE_BLOCK, i / CACHE_BLOCK * 16)));
      to_lds[0] = w.x;
      to_lds[1] = w.y;
      to_lds[2] = w.z;
      to_lds[3] = w.w;
    }
    __syncthreads();
  }
  for (int f = tid; f < CACHE_BLOCK * (HS / 4); f += 256) {
    const int t = f / (HS / 4), d = f % (HS / 4) * 4, p = p0 + t;
    if (p < from || p >= to) continue;
    float *kept = recent + ((int64_t)(p % CACHE_RECENT) * c.nkv + head) * HS + d;
    float4 y;
    if (!eight) {
      y = *reinterpret_cast<const float4 *>(kept);
    } else if (which) {
      const uint8_t *b = bytes + value_at(value_byte(t), d);
      y = make_float4((float)((int)b[0] - 128) * s, (float)((int)b[36] - 128) * s, (float)((int)b[72] - 128) * s,
                      (float)((int)b[108] - 128) * s);
    } else {
      const uint32_t w = *reinterpret_cast<const uint32_t *>(bytes + key_at(t, d));
      y = make_float4((float)(int8_t)w * s, (float)(int8_t)(w >> 8) * s, (float)(int8_t)(w >> 16) * s,
                      (float)(int8_t)(w >> 24) * s);
    }
    float *to_row = out ? out + ((int64_t)(p - from) * c.nkv + head) * HS + d : kept;
    *reinterpret_cast<float4 *>(to_row) = y;
  }
}

template <int HS>
void launch_append(const CacheRows &a, int blocks, hipStream_t s) {
  hipLaunchKernelGGL(append_kernel<HS>, dim3(blocks, a.c.nkv, 2), dim3(256), 0, s, a);
}
template <int HS>
void launch_read(const CacheView &c, float *k, float *v, int from, int to, int recent, hipStream_t s) {
  hipLaunchKernelGGL(read_kernel<HS>, dim3((to - 1) / CACHE_BLOCK - from / CACHE_BLOCK + 1, c.nkv, 2), dim3(256), 0, s, c, k,
                     v, from, to, recent);
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
  const int to = from + count;
  switch (c.hs) {
    case 16: launch_read<16>(c, keys, values, from, to, recent, s); break;
    case 32: launch_read<32>(c, keys, values, from, to, recent, s); break;
    case 48: launch_read<48>(c, keys, values, from, to, recent, s); break;
    case 64: launch_read<64>(c, keys, values, from, to, recent, s); break;
    case 96: launch_read<96>(c, keys, values, from, to, recent, s); break;
    case 128: launch_read<128>(c, keys, values, from, to, recent, s); break;
    case 256: launch_read<256>(c, keys, values, from, to, recent, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace ple
