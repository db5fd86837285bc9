// pages.hip — the cache in pages (include/pyodide_llm_hip.h hk_pages): sequences forked, given room, cut and compacted, and
// rows into their pages.
//
// The tables and counts are small (4 bytes a page of a sequence, 4 a page of the pool); what costs is the rows that are
// copied. So one workgroup decides which pages go where, in a defined order (lowest pages first, in the order of the lists),
// and leaves a list; a second launch, whose workgroups take the list's pieces in turn, copies.
#include <algorithm>

#include "common.hpp"
#include "kernels.hpp"

namespace ple {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int THREADS = 1024;  // of the workgroup that decides
constexpr int BATCH = 16;      // counts a thread reads at a time
constexpr int COPIERS = 2048, MOVERS = 4096;  // workgroups of a launch that copies rows, and of one that moves pages
constexpr int FORKERS = 1 << 16;  // of one that forks, at most (a launch has fewer than 2^32 threads, a table up to 2^25 slots)

__device__ __forceinline__ bool a_page(const PagesView &c, int32_t p) { return (uint32_t)p < (uint32_t)c.n_pages; }

__device__ __forceinline__ int64_t entry(const PagesView &c, int32_t seq, int32_t slot) { return (int64_t)seq * c.slots + slot; }

// whether the lists of a call are such that it may be made: every sequence within the tables and at most once, every number
// in 0..the positions of a table's row. Negative sequences are passed over. The same answer in every thread of the workgroup.
template <class Numbers>
__device__ bool lists_hold(const PagesView &c, const int32_t *seqs, int n, uint32_t *seen, Numbers numbers) {
  for (int i = threadIdx.x; i < PAGES_SEQS_MOST / 32; i += blockDim.x) seen[i] = 0;
  __syncthreads();
  int wrong = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t s = seqs[i];
    if (s < 0) continue;
    if (s >= c.n_seqs || !numbers(i)) {
      wrong = 1;
    } else {
      const uint32_t bit = 1u << (s & 31);
      if (atomicOr(&seen[s >> 5], bit) & bit) wrong = 1;
    }
  }
  return !__syncthreads_or(wrong);
}

__device__ __forceinline__ bool position(const PagesView &c, int32_t p) { return p >= 0 && p <= c.slots * c.page; }

// the sum of x over the workgroup's threads before this one, and over all of them
__device__ __forceinline__ uint32_t before(uint32_t x, uint32_t (&sums)[THREADS / 64], uint32_t &all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t upto = wave_up_to(x);
  __syncthreads();  // (the sums of the last time have been read)
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  const uint32_t waves = wave_up_to(lane < THREADS / 64 ? sums[lane] : 0);
  all = __builtin_amdgcn_readlane(waves, THREADS / 64 - 1);
  return upto - x + (wave ? __builtin_amdgcn_readlane(waves, __builtin_amdgcn_readfirstlane(wave) - 1) : 0);
}

// BATCH counts from page p on, those past the pool's end as `past`
__device__ __forceinline__ void counts(const PagesView &c, int32_t p, int32_t past, int32_t (&r)[BATCH]) {
  if (p + BATCH <= c.n_pages) {
#pragma unroll
    for (int i = 0; i < BATCH; i += 4) {
      const int4 x = *reinterpret_cast<const int4 *>(c.refs + p + i);
      r[i] = x.x, r[i + 1] = x.y, r[i + 2] = x.z, r[i + 3] = x.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) r[i] = p + i < c.n_pages ? c.refs[p + i] : past;
  }
}

// ---- fork ----

// A workgroup takes `cols` slots of every listed sequence, and goes on a launch further: what their rows shall hold is read before
// any of it is written, so that a sequence may be read and written by one call. Latency: the lists, the tables, the counts (16
// sequences 4.8 us).
__global__ __launch_bounds__(256) void fork_kernel(const PagesView c, const int32_t *to, const int32_t *from,
                                                   const int32_t *lengths, int n, int cols, int32_t *status) {
  extern __shared__ int32_t lds[];
  uint32_t *seen = reinterpret_cast<uint32_t *>(lds);
  int32_t *next = lds + PAGES_SEQS_MOST / 32;
  const bool good = lists_hold(c, to, n, seen, [&](int i) {
    return from[i] >= 0 && from[i] < c.n_seqs && position(c, lengths[i]);
  });
  if (blockIdx.x == 0 && threadIdx.x == 0 && status) *status = good ? 0 : -1;
  if (!good) return;
  for (int first = blockIdx.x * cols; first < c.slots; first += gridDim.x * cols) {
    for (int e = threadIdx.x; e < n * cols; e += 256) {
      const int i = e / cols, slot = first + e % cols;
      int32_t a = -1;
      if (to[i] >= 0 && slot < c.slots && slot * c.page < lengths[i]) a = c.tables[entry(c, from[i], slot)];
      next[e] = a_page(c, a) ? a : -1;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n * cols; e += 256) {  // (a thread's own entries of `next`)
      const int32_t s = to[e / cols], slot = first + e % cols, a = next[e];
      if (s < 0 || slot >= c.slots) continue;
      int32_t *at = &c.tables[entry(c, s, slot)];
      const int32_t b = *at;
      if (a == b) continue;
      if (a >= 0) atomicAdd(&c.refs[a], 1);
      if (a_page(c, b)) atomicSub(&c.refs[b], 1);
      *at = a;
    }
  }
}

// ---- free ----

__global__ __launch_bounds__(256) void free_kernel(const PagesView c, const int32_t *seqs, const int32_t *kept) {
  const int slot = blockIdx.x * 256 + threadIdx.x;
  const int32_t s = seqs[blockIdx.y];
  if (s < 0 || s >= c.n_seqs || slot >= c.slots) return;
  if (kept && slot * c.page < kept[blockIdx.y]) return;
  int32_t *at = &c.tables[entry(c, s, slot)];
  if (*at < 0) return;
  const int32_t p = atomicExch(at, -1);  // (a sequence listed twice gives its page back once)
  if (a_page(c, p)) atomicSub(&c.refs[p], 1);
}

// ---- reserve ----

// the workspace: the copies' number and the copies; then the free pages taken, and for each the list's entry, the slot, and the
// page there now
struct Copies {
  int32_t *n, *from, *to, *rows;
  __host__ __device__ explicit Copies(int32_t *w)
      : n(w), from(w + 4), to(from + PAGES_SEQS_MOST), rows(to + PAGES_SEQS_MOST) {}
  static constexpr int64_t INTS = 4 + 3 * PAGES_SEQS_MOST;
};
struct Taken {
  int32_t *pages, *which, *slot, *old;
  __host__ __device__ Taken(int32_t *w, int64_t n) : pages(w), which(w + n), slot(which + n), old(slot + n) {}
};
constexpr int HERE = 2048;  // pages whose lists stay in LDS

// One workgroup. The slots that the listed positions lie in, in order, make pairs (entry, slot); those without a page, or with
// one that other entries name, ask for one, and the k-th asks for the k-th free page. Nothing is written before all are found.
// Latency: the lists, the tables, the counts (7.1 us; 64 sequences with one position more and nothing to copy 5.4); the first
// counts are asked for before it is known how many are needed.
__global__ __launch_bounds__(THREADS) void reserve_kernel(const PagesView c, const int32_t *seqs, const int32_t *starts,
                                                          const int32_t *ends, int n, int32_t *status, int32_t *workspace) {
  __shared__ uint32_t seen[PAGES_SEQS_MOST / 32];
  __shared__ uint32_t sums[THREADS / 64];
  __shared__ int32_t pairs_before[PAGES_SEQS_MOST + 1], n_copies, here[4 * HERE];
  const Copies copies(workspace);
  const int tid = threadIdx.x;
  int32_t x[BATCH];
  counts(c, min(tid * BATCH, c.n_pages), 1, x);
  const bool good = lists_hold(c, seqs, n, seen, [&](int i) { return position(c, starts[i]) && position(c, ends[i]); });
  if (tid == 0) {
    *copies.n = 0;
    n_copies = 0;
    if (!good && status) *status = -1;
  }
  if (!good) return;
  uint32_t pairs = 0, all;
  for (int base = 0; base < n; base += THREADS) {
    const int i = base + tid;
    uint32_t mine = 0;
    if (i < n && seqs[i] >= 0 && ends[i] > starts[i]) mine = (ends[i] - 1) / c.page - starts[i] / c.page + 1;
    const uint32_t ahead = pairs + before(mine, sums, all);
    if (i < n) pairs_before[i] = ahead;
    pairs += all;
  }
  if (tid == 0) pairs_before[n] = pairs;
  __syncthreads();
  const bool few = pairs <= HERE;
  const Taken r(few ? here : workspace + Copies::INTS, few ? HERE : c.n_pages);
  uint32_t asked = 0;
  for (uint32_t base = 0; base < pairs; base += THREADS) {
    const int at = base + tid;
    int32_t slot = 0, old = -1;
    int asks = 0, lo = 0;
    if (at < (int)pairs) {
      int hi = n;  // the last entry whose pairs begin at `at` or before
      while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (pairs_before[mid] <= at) lo = mid;
        else hi = mid;
      }
      slot = starts[lo] / c.page + at - pairs_before[lo];
      old = c.tables[entry(c, seqs[lo], slot)];
      if (!a_page(c, old)) old = -1;
      asks = old < 0 || c.refs[old] > 1;
    }
    const uint32_t k = asked + before(asks, sums, all);
    if (asks && k < (uint32_t)c.n_pages) r.which[k] = lo, r.slot[k] = slot, r.old[k] = old;
    asked += all;
  }
  uint32_t found = 0;
  for (int64_t base = 0; base < c.n_pages && found < asked; base += THREADS * BATCH) {
    const int32_t p = (int32_t)min(base + tid * BATCH, (int64_t)c.n_pages);
    if (base) counts(c, p, 1, x);
    uint32_t mine = 0;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) mine += x[i] == 0;
    uint32_t k = found + before(mine, sums, all);
#pragma unroll
    for (int i = 0; i < BATCH; ++i)
      if (x[i] == 0) {
        if (k < asked) r.pages[k] = p + i;
        ++k;
      }
    found += all;
  }
  if (tid == 0 && status) *status = (int32_t)(asked - min(asked, found));
  if (found < asked) return;
  __threadfence_block();
  __syncthreads();
  for (uint32_t k = tid; k < asked; k += THREADS) {
    const int32_t page = r.pages[k], i = r.which[k], slot = r.slot[k], old = r.old[k];
    c.tables[entry(c, seqs[i], slot)] = page;
    c.refs[page] = 1;
    if (old < 0) continue;
    atomicSub(&c.refs[old], 1);
    const int rows = starts[i] - slot * c.page;  // of the first slot: those before the first position
    if (rows > 0) {
      const int at = atomicAdd(&n_copies, 1);
      copies.from[at] = old, copies.to[at] = page, copies.rows[at] = rows;
    }
  }
  __syncthreads();
  if (tid == 0) *copies.n = n_copies;
}

// The first rows of copied pages: a piece is a (copy, kv head) of one layer's keys or values. Through the caches: several
// sequences part from one page (16 times 40 rows of 8 heads of 128 in 32 layers, 84 MB written, 25 us; past them 29).
__global__ __launch_bounds__(256) void copy_rows_kernel(const PagesView c, int32_t *workspace) {
  const Copies list(workspace);
  const int copies = *list.n, row = c.hs * (c.half ? 2 : 4);
  uint8_t *pool = reinterpret_cast<uint8_t *>(blockIdx.y & 1 ? c.values : c.keys);
  const int64_t head = (int64_t)c.page * row, layer = (int64_t)(blockIdx.y >> 1) * c.n_pages;
  for (int64_t u = blockIdx.x; u < (int64_t)copies * c.nkv; u += gridDim.x) {
    const int i = (int)(u / c.nkv), g = (int)(u % c.nkv);
    const u32x4 *from = reinterpret_cast<const u32x4 *>(pool + ((layer + list.from[i]) * c.nkv + g) * head);
    u32x4 *to = reinterpret_cast<u32x4 *>(pool + ((layer + list.to[i]) * c.nkv + g) * head);
    const int n = list.rows[i] * row / 16;
    for (int e = threadIdx.x; e < n; e += 1024) {
      u32x4 x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (e + 256 * r < n) x[r] = from[e + 256 * r];
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (e + 256 * r < n) to[e + 256 * r] = x[r];
    }
  }
}

// ---- compact ----

// the workspace: the pages that move and the used pages; where they go, where they lie, and for a page its place among them
struct Moves {
  int32_t *head, *to, *from, *place;
  __host__ __device__ Moves(int32_t *w, int64_t n_pages) : head(w), to(w + 4), from(to + n_pages), place(from + n_pages) {}
  static int64_t ints(int64_t n_pages) { return 4 + 3 * n_pages; }
};

// One workgroup, twice over the counts: the used pages, then the free ones below their number and the used ones from it on (at
// most THREADS * BATCH = 2^14 of each at a time: both in one sum). Latency: 4.7 us up to as many pages, about 1 more for each as
// many after them.
__global__ __launch_bounds__(THREADS) void moves_kernel(const PagesView c, int32_t *used_out, int32_t *workspace) {
  __shared__ uint32_t sums[THREADS / 64];
  const Moves m(workspace, c.n_pages);
  const int tid = threadIdx.x;
  uint32_t count = 0, all;
  int32_t x[BATCH];
  for (int64_t base = 0; base < c.n_pages; base += THREADS * BATCH) {
    counts(c, (int32_t)min(base + tid * BATCH, (int64_t)c.n_pages), 0, x);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) count += x[i] > 0;
  }
  before(count, sums, all);
  const int used = (int)all;
  int holes = 0, moved = 0;
  for (int64_t base = 0; base < c.n_pages; base += THREADS * BATCH) {
    const int32_t p = (int32_t)min(base + tid * BATCH, (int64_t)c.n_pages);
    if (c.n_pages > THREADS * BATCH) counts(c, p, 0, x);
    uint32_t both = 0;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) both += p + i < used ? x[i] <= 0 : x[i] > 0 ? 1 << 16 : 0;
    const uint32_t ahead = before(both, sums, all);
    int h = holes + (int)(ahead & 0xFFFF), k = moved + (int)(ahead >> 16);
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (p + i < used && x[i] <= 0) m.to[h++] = p + i;
      if (p + i >= used && x[i] > 0) {
        m.place[p + i] = k;
        m.from[k++] = p + i;
      }
    }
    holes += (int)(all & 0xFFFF);
    moved += (int)(all >> 16);
  }
  if (tid == 0) {
    m.head[0] = moved;
    m.head[1] = used;
    if (used_out) *used_out = used;
  }
}

constexpr int PIECE = 256 * 4 * 16;  // bytes a workgroup copies at a time

// Pages to their places: a piece of one layer's keys or values a workgroup and turn. Bound by HBM, both ways: 470 MB in 97 us (4.9
// TB/s; read and written past the caches, which hold nothing of them: 104 through them). The last row of workgroups takes the
// tables and the counts.
__global__ __launch_bounds__(256) void move_kernel(const PagesView c, int32_t *workspace) {
  const Moves m(workspace, c.n_pages);
  const int moved = m.head[0], used = m.head[1];
  if (moved == 0) return;
  if (blockIdx.y == 2 * c.layers) {
    const int64_t entries = (int64_t)c.n_seqs * c.slots, step = (int64_t)gridDim.x * 256;
    for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < entries; e += step) {
      const int32_t p = c.tables[e];
      if (p < used || p >= c.n_pages) continue;
      const int32_t k = m.place[p];  // (of a page that no count says is used: anything)
      if ((uint32_t)k < (uint32_t)moved && m.from[k] == p) c.tables[e] = m.to[k];
    }
    for (int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x; k < moved; k += step) {
      c.refs[m.to[k]] = c.refs[m.from[k]];
      c.refs[m.from[k]] = 0;
    }
    return;
  }
  uint8_t *pool = reinterpret_cast<uint8_t *>(blockIdx.y & 1 ? c.values : c.keys);
  const int64_t bytes = (int64_t)c.nkv * c.page * c.hs * (c.half ? 2 : 4), layer = (int64_t)(blockIdx.y >> 1) * c.n_pages;
  const int64_t pieces = (bytes + PIECE - 1) / PIECE;
  int64_t u = blockIdx.x;
  if (u >= moved * pieces) return;
  int32_t source = m.from[u / pieces], target = m.to[u / pieces];
  while (true) {
    const int64_t at = u % pieces * PIECE + threadIdx.x * 16;
    const uint8_t *from = pool + (layer + source) * bytes;
    uint8_t *to = pool + (layer + target) * bytes;
    u32x4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * 4096 < bytes) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(from + at + i * 4096));
    u += gridDim.x;
    const bool more = u < moved * pieces;
    if (more) source = m.from[u / pieces], target = m.to[u / pieces];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i * 4096 < bytes) __builtin_nontemporal_store(x[i], reinterpret_cast<u32x4 *>(to + at + i * 4096));
    if (!more) return;
  }
}

// ---- append ----

// A thread takes four channels of a row's keys and values. A step's rows are latency (64 rows 3.0 us), a prompt's bound by HBM
// (2048 rows of 8 heads of 128 in float32, 34 MB, 7.3).
template <bool HALF>
__global__ __launch_bounds__(256) void append_kernel(const PagesRows a) {
  const PagesView &c = a.c;
  const int units = c.nkv * c.hs / 4;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < (int64_t)a.count * units; e += (int64_t)gridDim.x * 256) {
    const int i = (int)(e / units), d = (int)(e % units) * 4;
    const int32_t s = a.seqs ? a.seqs[i] : i, p = a.positions[i];
    if (s < 0 || s >= c.n_seqs || p < 0 || p >= c.slots * c.page) continue;
    const int32_t page = c.tables[entry(c, s, p / c.page)];
    if (!a_page(c, page)) continue;
    const int64_t at = ((((int64_t)a.layer * c.n_pages + page) * c.nkv + d / c.hs) * c.page + p % c.page) * c.hs + d % c.hs;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const float4 x = *reinterpret_cast<const float4 *>((which ? a.v : a.k) + (int64_t)i * a.stride + d);
      void *pool = which ? c.values : c.keys;
      if (HALF) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<f16x4 *>(reinterpret_cast<_Float16 *>(pool) + at) =
            f16x4{(_Float16)x.x, (_Float16)x.y, (_Float16)x.z, (_Float16)x.w};
      } else {
        *reinterpret_cast<float4 *>(reinterpret_cast<float *>(pool) + at) = x;
      }
    }
  }
}

}  // namespace

int64_t pages_workspace(const PagesView &c) {
  return 4 * std::max(Copies::INTS + 4 * (int64_t)c.n_pages, Moves::ints(c.n_pages));
}

hipError_t launch_pages_fork(const PagesView &c, const int32_t *to, const int32_t *from, const int32_t *lengths, int32_t n,
                             int32_t *status, hipStream_t s) {
  const int cols = std::max(1, std::min(16, 8192 / n));
  hipLaunchKernelGGL(fork_kernel, dim3(std::min((c.slots + cols - 1) / cols, FORKERS)), dim3(256), PAGES_SEQS_MOST / 8 + 4 * n * cols,
                     s, c, to, from, lengths, n, cols, status);
  return hipGetLastError();
}

hipError_t launch_pages_reserve(const PagesView &c, const int32_t *seqs, const int32_t *starts, const int32_t *ends, int32_t n,
                                int32_t *status, int32_t *workspace, hipStream_t s) {
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(THREADS), 0, s, c, seqs, starts, ends, n, status, workspace);
  const int64_t pieces = (int64_t)n * c.nkv;
  hipLaunchKernelGGL(copy_rows_kernel, dim3((uint32_t)std::min<int64_t>(pieces, std::max(1, COPIERS / (2 * c.layers))), 2 * c.layers),
                     dim3(256), 0, s, c, workspace);
  return hipGetLastError();
}

hipError_t launch_pages_free(const PagesView &c, const int32_t *seqs, const int32_t *kept, int32_t n, hipStream_t s) {
  hipLaunchKernelGGL(free_kernel, dim3((c.slots + 255) / 256, n), dim3(256), 0, s, c, seqs, kept);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesView &c, int32_t *used, int32_t *workspace, hipStream_t s) {
  hipLaunchKernelGGL(moves_kernel, dim3(1), dim3(THREADS), 0, s, c, used, workspace);
  hipLaunchKernelGGL(move_kernel, dim3(std::max(1, MOVERS / (2 * c.layers)), 2 * c.layers + 1), dim3(256), 0, s, c, workspace);
  return hipGetLastError();
}

hipError_t launch_pages_append(const PagesRows &a, hipStream_t s) {
  const int64_t units = (int64_t)a.count * (a.c.nkv * a.c.hs / 4);
  const dim3 grid((uint32_t)std::min<int64_t>((units + 255) / 256, 1 << 20));
  if (a.c.half) hipLaunchKernelGGL(append_kernel<true>, grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL(append_kernel<false>, grid, dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace ple
