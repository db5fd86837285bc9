// logprobs.hip — log probabilities of given tokens, the entropy and the largest alternatives of rows of logits.
//
// With m a row's largest logit and Z = sum exp(x - m): logp_t = x_t - m - log Z, the entropy log Z - H / Z with H = sum
// exp(x - m) (x - m). One pass over the logits: every thread keeps its m, Z and H (rescaled when m grows), and the largest
// are picked out on the way by a threshold that only ever grows. A few rows are split over many workgroups, whose parts a
// second launch joins.
//
// 512 rows of 128256 with 5 alternatives take 56 us, 4.7 TB/s (a plain streaming read 41): the VALU issues in 0.6 of the
// cycles, an exponential, a maximum and four other operations a logit and the candidates' ballots. One row takes 10.5, a chain of
// latencies: the read, the bar, the join's reads and its ordering.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

constexpr float LOG2E = 1.44269504088896341f, LN2 = 0.693147180559945309f;
constexpr float LOWEST = -3.402823466e38f;
constexpr int THREADS = 256, WAVES = THREADS / 64, QUADS = 4, BATCH = 4 * QUADS;  // logits a thread takes at once
constexpr int HELD = 256;  // candidates a wave holds

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

// m, Z, H (in nats) of two parts together (z 0: an empty part, whatever its m)
template <class T>
__device__ __forceinline__ void join(T &m, T &z, T &h, T m2, T z2, T h2) {
  const T top = m2 > m || m2 != m2 ? m2 : m;  // (a NaN stays)
  // (a part's m may lie 2^128 below, or be minus infinity: its factor is 0, its difference kept finite)
  const T d1 = m - top > (T)-1e30 ? m - top : (T)-1e30, d2 = m2 - top > (T)-1e30 ? m2 - top : (T)-1e30;
  const T f1 = (T)__builtin_amdgcn_exp2f((float)(d1 * (T)LOG2E)), f2 = (T)__builtin_amdgcn_exp2f((float)(d2 * (T)LOG2E));
  h = (h + z * d1) * f1 + (h2 + z2 * d2) * f2;
  z = z * f1 + z2 * f2;
  m = top;
}

// the candidates a part passes on: what is left of them behind its bar, as a rule
__host__ __device__ constexpr int slots_of(int top) { return top ? 3 * top + 4 : 0; }

struct Shared {
  uint64_t held[WAVES][HELD];  // the waves' candidates
  uint64_t list[WAVES * HELD + 8];
  uint64_t best[WAVES];
  uint32_t bars[WAVES][2];
  int count;
  Part parts[WAVES];
};

__device__ __forceinline__ uint32_t ordered_of(float x) { return (uint32_t)(key_of(x, 0) >> 32); }

// a value that at least k (at most 64) of the wave's lanes reach, the largest of 16 leading bits (in ordered_of's bits; 0
// where fewer lanes hold one): two bits at a time, by counting lanes
__device__ __forceinline__ uint32_t reached_by(uint32_t mine, int k) {
  uint32_t t = 0;
#pragma unroll
  for (int bit = 30; bit >= 16; bit -= 2) {
    const uint32_t one = t | 1u << bit, two = t | 2u << bit, three = t | 3u << bit;
    const int a = __popcll(__ballot(mine >= one)), b = __popcll(__ballot(mine >= two)), c = __popcll(__ballot(mine >= three));
    t = c >= k ? three : b >= k ? two : a >= k ? one : t;
  }
  return t;
}

// the parts of the wave's lanes as one (z 0: an empty part, whatever its m)
__device__ __forceinline__ void join_lanes(float &m, float &z, float &h) {
  const float top = wave_top(m), d = z > 0.0f ? __builtin_fmaxf(m - top, -1e30f) : 0.0f;
  const float f = __builtin_amdgcn_exp2f(d * LOG2E);
  h = wave_sum(__builtin_fmaf(d, z, h) * f);
  z = wave_sum(z * f);
  m = top;
}

// a bar that at least k of the workgroup's threads reach: one that k of some wave's lanes reach (`alone`), or each wave's
// share of k
__device__ __forceinline__ void raise_bars(Shared &s, uint32_t alone, uint32_t mine, int k) {
  const uint32_t share = reached_by(mine, (k + WAVES - 1) / WAVES);
  if (threadIdx.x % 64 == 0) {
    s.bars[threadIdx.x / 64][0] = alone;
    s.bars[threadIdx.x / 64][1] = share;
  }
}
__device__ __forceinline__ uint32_t highest_bar(const Shared &s) {
  uint32_t alone = s.bars[0][0], share = s.bars[0][1];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) {
    alone = s.bars[w][0] > alone ? s.bars[w][0] : alone;
    share = s.bars[w][1] < share ? s.bars[w][1] : share;
  }
  return share > alone ? share : alone;
}

// the lanes of a mask before this one
__device__ __forceinline__ int before_me(uint64_t lanes) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(lanes >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)lanes, 0));
}

__device__ __forceinline__ uint64_t wave_most(uint64_t x) {
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    const uint64_t y = __shfl_xor(x, o);
    x = y > x ? y : x;
  }
  return x;
}

// the k largest of a wave's n candidates to the front, in order, one at a time (where they pass HELD: rows of ties)
__device__ __forceinline__ int wave_tighten(uint64_t *held, int n, int k) {
  const int lane = threadIdx.x % 64;
  uint64_t mine[HELD / 64];
#pragma unroll
  for (int j = 0; j < HELD / 64; ++j) mine[j] = lane + 64 * j < n ? held[lane + 64 * j] : 0;
  wave_sync_lds();
  const int kept = min(n, k);
#pragma unroll 1
  for (int i = 0; i < kept; ++i) {
    uint64_t top = 0;
#pragma unroll
    for (int j = 0; j < HELD / 64; ++j) top = mine[j] > top ? mine[j] : top;
    top = wave_most(top);
    if (lane == 0) held[i] = top;
#pragma unroll
    for (int j = 0; j < HELD / 64; ++j) mine[j] = mine[j] == top ? 0 : mine[j];
  }
  wave_sync_lds();
  return kept;
}

// the k largest of the list's n keys to its front, in order: each key's place is the number of keys before it. (The list
// holds zeros for eight places from n on.)
__device__ __forceinline__ void sort_list(Shared &s, int n, int k) {
  const int tid = threadIdx.x;
  constexpr int EACH = WAVES * HELD / THREADS;
  uint64_t mine[EACH];
  int place[EACH];
#pragma unroll
  for (int j = 0; j < EACH; ++j) mine[j] = place[j] = 0;
  if (n <= THREADS) {
    if (tid < n) {
      mine[0] = s.list[tid];
#pragma unroll 1
      for (int i = 0; i < n; i += 8) {
        uint64_t o[8];  // (eight reads in flight)
#pragma unroll
        for (int u = 0; u < 8; ++u) o[u] = s.list[i + u];
#pragma unroll
        for (int u = 0; u < 8; ++u) place[0] += o[u] > mine[0];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < EACH; ++j) mine[j] = tid + THREADS * j < n ? s.list[tid + THREADS * j] : 0;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
      const uint64_t o = s.list[i];
#pragma unroll
      for (int j = 0; j < EACH; ++j) place[j] += o > mine[j];
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EACH; ++j)
    if (mine[j] && place[j] < k) s.list[place[j]] = mine[j];
  if (tid == 0) s.count = min(n, k);
  __syncthreads();
}

// the row's results from its joined part and its sorted alternatives
__device__ __forceinline__ void finish(const LogprobArgs &a, int64_t row, double m, double z, double h, const uint64_t *list,
                                       int held) {
  const float *x = a.logits + row * a.stride;
  const bool fine = z > 0.0 && m > (double)-__builtin_inff() && m < (double)__builtin_inff();
  // (Z is 1 at least, the largest logit's own term, and the entropy not negative: where a peaked row's sums round below, a
  // caller's log(1 - p) or square root would be no number)
  const double nan = __builtin_nan(""), logz = z > 1.0 ? (double)logf((float)z) : 0.0, entropy = logz - h / z;
  if (threadIdx.x == 0 && a.entropy) a.entropy[row] = (float)(!fine ? nan : entropy > 0.0 ? entropy : 0.0);
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
// Every wave picks its own candidates for the largest: a logit that reaches a bar which at least `top` of the wave's lanes
// have reached so far. The bar is found again once eight lanes have reached it; at the end the highest of the waves' bars leaves a
// few dozen candidates to sort.
template <bool ALONE, bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_kernel(const LogprobArgs a, int quads) {
  __shared__ Shared s;
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int64_t row = blockIdx.y;
  const float *x = a.logits + row * a.stride;
  const int ahead = (int)(reinterpret_cast<uintptr_t>(x) % 16 / 4);  // floats between an aligned address and the row
  const float *base = x - ahead;
  const int all = (int)(((int64_t)ahead + a.n + 3) / 4), from = blockIdx.x * quads, to = blockIdx.x + 1 == gridDim.x ? all : min(all, from + quads);
  // the thread's largest logit m, and against a reference of m: Z = sum 2^t, H = sum 2^t t, t = x log2(e) - up, up the next
  // whole number above m log2(e): a multiply-add an exponential's argument, every rescaling exact. (Logits past 2^20, where
  // that loses t, are taken against m itself: t = (x - m) log2(e).)
  float m = -__builtin_inff(), up = 0.0f, z = 0.0f, h = 0.0f;
  bool plain = false;  // (the same in the whole wave)
  auto to_plain = [&] {  // Z and H against m itself
    const float g = plain ? 0.0f : z > 0.0f ? __builtin_fmaf(-m, LOG2E, up) : 0.0f;
    h = __builtin_fmaf(g, z, h);
    const float f = __builtin_amdgcn_exp2f(g);
    z *= f;
    h *= f;
  };
  float bar = LOWEST;
  int reached_since = 0;  // lanes that have reached the bar since it was found
  uint64_t least = 0;  // a key that candidates are above, once ties have filled the wave's list
  int held = 0;
  const int inside = min(to, (int)(((int64_t)ahead + a.n) / 4));  // quads from here on are not whole, or another part's
  float4 next[QUADS];  // a batch is read while the one before it is worked on
  auto read = [&](int q0) {
    // (the same in the whole workgroup: a batch that lies inside the row and the part)
    if (q0 * 4 >= ahead && q0 + THREADS * QUADS <= inside) {
      const float4 *from = reinterpret_cast<const float4 *>(base) + q0 + tid;
#pragma unroll
      for (int j = 0; j < QUADS; ++j) next[j] = from[THREADS * j];
      return;
    }
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
      next[j] = w;
    }
  };
  read(from);
  for (int q0 = from; q0 < to; q0 += THREADS * QUADS) {
    float v[BATCH];
#pragma unroll
    for (int j = 0; j < QUADS; ++j) {
      v[4 * j] = next[j].x;
      v[4 * j + 1] = next[j].y;
      v[4 * j + 2] = next[j].z;
      v[4 * j + 3] = next[j].w;
    }
    if (q0 + THREADS * QUADS < to) read(q0 + THREADS * QUADS);
    float most = v[0];
#pragma unroll
    for (int j = 1; j < BATCH; ++j) most = wmax(most, v[j]);
    const float top = wmax(m, most);
    if (!plain && __any(!(__builtin_fabsf(top) <= 0x1p20f) && top != -__builtin_inff())) {
      to_plain();
      plain = true;
      up = m > -__builtin_inff() ? m : 0.0f;
    }
    float zs = 0.0f, hs = 0.0f;
    m = top;
    if (!plain) {
      const float to_up = m > -__builtin_inff() ? __builtin_ceilf(m * LOG2E) : 0.0f;
      const float f = z > 0.0f ? __builtin_amdgcn_exp2f(up - to_up) : 0.0f;
      h = __builtin_fmaf(up - to_up, z, h) * f;
      z = z * f;
      up = to_up;
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const float t = __builtin_fmaxf(__builtin_fmaf(v[j], LOG2E, -up), -150.0f), e = __builtin_amdgcn_exp2f(t);
        zs += e;
        hs = __builtin_fmaf(e, t, hs);
      }
    } else {
      const float to_up = m > -__builtin_inff() ? m : 0.0f;
      const float d = z > 0.0f ? __builtin_fmaxf((up - to_up) * LOG2E, -1e30f) : 0.0f, f = __builtin_amdgcn_exp2f(d);
      h = __builtin_fmaf(d, z, h) * f;
      z = z * f;
      up = to_up;
#pragma unroll
      for (int j = 0; j < BATCH; ++j) {
        const float t = __builtin_fmaxf((v[j] - up) * LOG2E, -150.0f), e = __builtin_amdgcn_exp2f(t);
        zs += e;
        hs = __builtin_fmaf(e, t, hs);
      }
    }
    z += zs;
    h += hs;
    if (TOP) {
      const int lanes = __popcll(__ballot(most >= bar));
      if (lanes) {
        reached_since += lanes;
        if (q0 == from || reached_since >= 8) {
          reached_since = 0;
          const uint32_t reached = reached_by(ordered_of(m), a.top);
          if (reached) bar = __builtin_fmaxf(bar, value_of((uint64_t)reached << 32));
        }
        uint64_t takes[BATCH];
        int all = 0;
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
          takes[j] = __ballot(v[j] >= bar);
          all += __popcll(takes[j]);
        }
        const uint32_t first = (uint32_t)((q0 + tid) * 4 - ahead);  // the lane's first logit
        if (!least && held + all <= HELD) {
#pragma unroll
          for (int j = 0; j < BATCH; ++j) {
            if (!takes[j]) continue;
            if (v[j] >= bar)
              s.held[wave][held + before_me(takes[j])] = key_of(v[j], first + (uint32_t)(THREADS * (j / 4) * 4 + j % 4));
            held += __popcll(takes[j]);
          }
          continue;
        }
        // ties or an ascending row: a value a lane at a time, the list tightened where it is full
#pragma unroll 1
        for (int j = 0; j < BATCH; ++j) {
          const float x = v[0];
#pragma unroll
          for (int i = 1; i < BATCH; ++i) v[i - 1] = v[i];
          uint64_t takes = __ballot(x >= bar);
          if (!takes) continue;
          const uint64_t key = key_of(x, first + (uint32_t)(THREADS * (j / 4) * 4 + j % 4));
          bool mine = x >= bar && key > least;
          takes = __ballot(mine);
          if (held + __popcll(takes) > HELD) {
            held = wave_tighten(s.held[wave], held, a.top);
            if (held == a.top) {
              least = s.held[wave][held - 1];
              bar = __builtin_fmaxf(bar, value_of(least));
            }
            mine = x >= bar && key > least;
            takes = __ballot(mine);
          }
          if (mine)
            s.held[wave][held + before_me(takes)] = key;
          held += __popcll(takes);
        }
      }
    }
  }
  // the workgroup's part: across the lanes, then the waves (H by whole exponentials' arguments: in nats)
  to_plain();
  h *= LN2;
  if (TOP) raise_bars(s, bar > LOWEST ? ordered_of(bar) : 0, ordered_of(m), a.top);
  join_lanes(m, z, h);
  if (lane == 0) s.parts[wave] = Part{m, z, h, 0};
  if (TOP && tid == 0) s.count = 0;
  __syncthreads();
  if (TOP) {
    const uint32_t high = highest_bar(s);
    for (int i = lane; i < held; i += 64) {
      const uint64_t key = s.held[wave][i];
      if ((uint32_t)(key >> 32) >= high) s.list[atomicAdd(&s.count, 1)] = key;
    }
    __syncthreads();
    const int count = s.count;
    // (a part's candidates are sorted only where they are more than its slots)
    if (ALONE || count > slots_of(a.top)) {
      if (tid < 8) s.list[count + tid] = 0;
      __syncthreads();
      sort_list(s, count, a.top);
    }
  }
  double dm = s.parts[0].m, dz = s.parts[0].z, dh = s.parts[0].h;
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
    join(dm, dz, dh, (double)s.parts[w].m, (double)s.parts[w].z, (double)s.parts[w].h);
  if (ALONE) {
    finish(a, row, dm, dz, dh, s.list, TOP ? s.count : 0);
    return;
  }
  const int64_t part = row * gridDim.x + blockIdx.x;
  if (tid == 0) reinterpret_cast<Part *>(a.workspace)[part] = Part{(float)dm, (float)dz, (float)dh, 0};
  if (TOP && tid < slots_of(a.top))
    reinterpret_cast<uint64_t *>(a.workspace + sizeof(Part) * gridDim.x * gridDim.y)[part * slots_of(a.top) + tid] =
        tid < s.count ? s.list[tid] : 0;
}

// the parts of a row (blockIdx.x) together
template <bool TOP>
__global__ __launch_bounds__(THREADS) void logprobs_join_kernel(const LogprobArgs a, int parts) {
  __shared__ Shared s;
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int64_t row = blockIdx.x;
  const Part *p = reinterpret_cast<const Part *>(a.workspace) + row * parts;
  const uint64_t *keys = reinterpret_cast<const uint64_t *>(a.workspace + sizeof(Part) * parts * (int64_t)gridDim.x) +
                         row * parts * slots_of(a.top);
  const int n = TOP ? parts * slots_of(a.top) : 0;
  uint64_t mine[8], best = 0;  // (the first 2048 are read once)
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    mine[j] = tid + THREADS * j < n ? keys[tid + THREADS * j] : 0;
    best = mine[j] > best ? mine[j] : best;
  }
  for (int i = tid + THREADS * 8; i < n; i += THREADS) best = keys[i] > best ? keys[i] : best;
  float m = LOWEST, z = 0.0f, h = 0.0f;
  for (int i = tid; i < parts; i += THREADS) join(m, z, h, p[i].m, p[i].z, p[i].h);
  join_lanes(m, z, h);
  if (TOP) raise_bars(s, reached_by((uint32_t)(best >> 32), a.top), (uint32_t)(best >> 32), a.top);
  if (lane == 0) s.parts[wave] = Part{m, z, h, 0};
  if (tid == 0) s.count = 0;
  __syncthreads();
  if (TOP) {
    const uint32_t high = highest_bar(s);
    const uint64_t least = high ? (uint64_t)high << 32 : 1;
    auto take = [&](uint64_t key) {
      if (key < least) return;
      const int at = atomicAdd(&s.count, 1);
      if (at < WAVES * HELD) s.list[at] = key;
    };
#pragma unroll
    for (int j = 0; j < 8; ++j) take(mine[j]);
    for (int i = tid + THREADS * 8; i < n; i += THREADS) take(keys[i]);
    __syncthreads();
    const int count = s.count;
    if (tid < 8 && count <= WAVES * HELD) s.list[count + tid] = 0;
    __syncthreads();
    if (count <= WAVES * HELD) {
      sort_list(s, count, a.top);
    } else {  // ties by the thousand: the largest one at a time
      uint64_t last = ~0ull;
      for (int k = 0; k < a.top; ++k) {
        best = 0;
        for (int i = tid; i < n; i += THREADS) best = keys[i] < last && keys[i] > best ? keys[i] : best;
        best = wave_most(best);
        if (lane == 0) s.best[wave] = best;
        __syncthreads();
        last = s.best[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) last = s.best[w] > last ? s.best[w] : last;
        if (tid == 0) s.list[k] = last;
        __syncthreads();
      }
      if (tid == 0) s.count = a.top;
      __syncthreads();
    }
  }
  double dm = s.parts[0].m, dz = s.parts[0].z, dh = s.parts[0].h;
#pragma unroll
  for (int w = 1; w < WAVES; ++w)
    join(dm, dz, dh, (double)s.parts[w].m, (double)s.parts[w].z, (double)s.parts[w].h);
  finish(a, row, dm, dz, dh, s.list, TOP ? s.count : 0);
}

// A row's parts, of whole batches of a workgroup: enough workgroups to fill the card. Rows from 640 on are not split: of 20,011,
// 32,000, 50,257, 128,256 logits 639 rows take 23.0, 28.9, 37.9, 70.4 us in parts, 640 unsplit 16.8, 21.9, 30.3, 62.7. (Below,
// the better side goes by the length: 512 rows of 128,256 take 57 in two parts, 61 unsplit.)
int parts_of(int32_t m, int32_t n) {
  if (m >= 640) return 1;
  const int64_t batches = ((int64_t)n + THREADS * BATCH - 1) / (THREADS * BATCH);
  const int64_t each = std::max<int64_t>(1, batches * m / 1024);
  return (int)((batches + each - 1) / each);
}

}  // namespace

int64_t logprobs_workspace(int32_t m, int32_t n, int32_t top) {
  const int64_t parts = parts_of(m, n);
  return parts == 1 ? 0 : parts * m * ((int64_t)sizeof(Part) + 8 * slots_of(top));
}

hipError_t launch_logprobs(const LogprobArgs &a, hipStream_t s) {
  const int parts = parts_of(a.m, a.n);
  // (three floats more than n where a row starts behind an aligned address: the last part takes them)
  const int64_t batches = ((int64_t)a.n + THREADS * BATCH - 1) / (THREADS * BATCH);
  const int quads = (int)((batches + parts - 1) / parts) * THREADS * QUADS;
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
