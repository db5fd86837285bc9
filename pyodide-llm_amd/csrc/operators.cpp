// operators.cpp — the C ABI of the operators that stand beside the engine's own kernels (include/pyodide_llm_hip.h): the cache
// held in 8 bits with its attention, and the log probabilities. Arguments are checked here, before any launch; nothing
// allocates or waits.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/pyodide_llm_hip.h"
#include "cache.hpp"
#include "kernels.hpp"

using namespace ple;

namespace {

static_assert(HK_CACHE_BLOCK == CACHE_BLOCK && HK_CACHE_RECENT == CACHE_RECENT, "the cache's sizes");
static_assert(HK_LOGPROBS_TOP_MOST == LOGPROBS_TOP_MOST, "the alternatives a row");

bool aligned(const void *p, uintptr_t to = 16) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

int32_t launched(const char *what, hipError_t err) {
  return err == hipSuccess ? HE_OK : failed(HE_E_HIP, std::string(what) + ": " + hipGetErrorString(err));
}

bool cache_head_size(int32_t hs) {
  return hs == 16 || hs == 32 || hs == 48 || hs == 64 || hs == 96 || hs == 128 || hs == 256;
}

int32_t view_of(const char *what, const hk_cache *c, CacheView &v) {
  if (!c) return failed(HE_E_ARG, std::string(what) + ": cache is null");
  if (!cache_head_size(c->head_size))
    return failed(HE_E_ARG, std::string(what) + ": head_size is one of 16, 32, 48, 64, 96, 128, 256");
  if (c->n_kv_heads < 1 || c->n_kv_heads > 65535 || c->seq_len < 1 || c->seq_len > HK_CACHE_MOST)
    return failed(HE_E_ARG, std::string(what) + ": n_kv_heads is in 1..65535, seq_len in 1..HK_CACHE_MOST (16777216)");
  v = {reinterpret_cast<int8_t *>(c->keys), reinterpret_cast<uint8_t *>(c->values), reinterpret_cast<float *>(c->scales),
       reinterpret_cast<float *>(c->recent_keys), reinterpret_cast<float *>(c->recent_values), c->n_kv_heads,
       c->head_size, (c->seq_len + HK_CACHE_BLOCK - 1) / HK_CACHE_BLOCK};
  return HE_OK;
}

int32_t buffers_of(const char *what, const CacheView &v) {
  const void *ptrs[] = {v.keys, v.values, v.scales, v.recent_keys, v.recent_values};
  for (const void *p : ptrs)
    if (!p || !aligned(p)) return failed(HE_E_ARG, std::string(what) + ": a cache buffer is null or not 16-byte aligned");
  return HE_OK;
}

// the tokens' rows k / v of a call on the cache
int32_t rows_of(const char *what, const hk_cache *cache, const void *k, const void *v, int32_t kv_stride, int32_t count,
                int32_t pos, CacheRows &rows) {
  int32_t rc = view_of(what, cache, rows.c);
  if (!rc) rc = buffers_of(what, rows.c);
  if (rc) return rc;
  if (!k || !v || !aligned(k) || !aligned(v))
    return failed(HE_E_ARG, std::string(what) + ": k or v is null or not 16-byte aligned");
  if ((int64_t)rows.c.nkv * rows.c.hs > kv_stride || kv_stride % 4)
    return failed(HE_E_ARG, std::string(what) + ": kv_stride is a multiple of 4, at least n_kv_heads * head_size");
  if (count < 1 || pos < 0) return failed(HE_E_ARG, std::string(what) + ": count is at least 1, pos at least 0");
  if ((int64_t)pos + count > cache->seq_len)
    return failed(HE_E_STATE, std::string(what) + ": the positions run past the context (seq_len)");
  rows.k = reinterpret_cast<const float *>(k);
  rows.v = reinterpret_cast<const float *>(v);
  rows.x_stride = kv_stride;
  rows.count = count;
  rows.pos = pos;
  rows.dpos = nullptr;
  rows.displaced = 0;
  return HE_OK;
}

int32_t heads_of(const char *what, const CacheView &v, int32_t n_heads) {
  if (n_heads < 1 || n_heads % v.nkv || n_heads / v.nkv > HK_CACHE_GROUP_MOST)
    return failed(HE_E_ARG, std::string(what) + ": n_heads is a multiple of n_kv_heads, at most 32 times it");
  return HE_OK;
}

}  // namespace

extern "C" {

int32_t hk_cache_append(const hk_cache *cache, const void *k, const void *v, int32_t kv_stride, int32_t count,
                        int32_t pos, void *stream) {
  CacheRows rows;
  const int32_t rc = rows_of("hk_cache_append", cache, k, v, kv_stride, count, pos, rows);
  if (rc) return rc;
  return launched("hk_cache_append", launch_cache_append(rows, reinterpret_cast<hipStream_t>(stream)));
}

int32_t hk_cache_attention(void *out, const void *q, const void *k, const void *v, const hk_cache *cache,
                           int32_t n_heads, int32_t q_stride, int32_t kv_stride, int32_t out_stride, int32_t count,
                           int32_t pos, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *what = "hk_cache_attention";
  CacheAttn a;
  int32_t rc = rows_of(what, cache, k, v, kv_stride, count, pos, a.rows);
  if (!rc) rc = heads_of(what, a.rows.c, n_heads);
  if (rc) return rc;
  if (!out || !q || !aligned(out) || !aligned(q))
    return failed(HE_E_ARG, "hk_cache_attention: out or q is null or not 16-byte aligned");
  const int64_t width = (int64_t)n_heads * a.rows.c.hs;
  if (q_stride < width || out_stride < width || q_stride % 4 || out_stride % 4)
    return failed(HE_E_ARG, "hk_cache_attention: q_stride and out_stride are multiples of 4, at least n_heads * head_size");
  const int64_t need = cache_attention_workspace(a.rows.c, n_heads, count);
  if (need > 0 && (!workspace || !aligned(workspace) || workspace_bytes < need))
    return failed(HE_E_ARG, "hk_cache_attention: the workspace is null, not 16-byte aligned or smaller than hk_cache_workspace");
  a.q = reinterpret_cast<const float *>(q);
  a.out = reinterpret_cast<float *>(out);
  a.nh = n_heads;
  a.q_stride = q_stride;
  a.out_stride = out_stride;
  a.workspace = reinterpret_cast<float *>(workspace);
  return launched(what, launch_cache_attention(a, reinterpret_cast<hipStream_t>(stream)));
}

int64_t hk_cache_workspace(const hk_cache *cache, int32_t n_heads, int32_t count) {
  CacheView v;
  int32_t rc = view_of("hk_cache_workspace", cache, v);
  if (!rc) rc = heads_of("hk_cache_workspace", v, n_heads);
  if (!rc && (count < 1 || count > cache->seq_len))
    rc = failed(HE_E_ARG, "hk_cache_workspace: count is in 1..seq_len");
  return rc ? rc : cache_attention_workspace(v, n_heads, count);
}

int32_t hk_cache_read(void *keys, void *values, const hk_cache *cache, int32_t from, int32_t count, int32_t end,
                      void *stream) {
  CacheView v;
  int32_t rc = view_of("hk_cache_read", cache, v);
  if (!rc) rc = buffers_of("hk_cache_read", v);
  if (rc) return rc;
  if (!keys || !values || !aligned(keys) || !aligned(values))
    return failed(HE_E_ARG, "hk_cache_read: keys or values is null or not 16-byte aligned");
  if (from < 0 || count < 0 || (int64_t)from + count > end || end > cache->seq_len)
    return failed(HE_E_ARG, "hk_cache_read: positions out of range");
  if (count == 0) return HE_OK;
  return launched("hk_cache_read",
                  launch_cache_read(v, reinterpret_cast<float *>(keys), reinterpret_cast<float *>(values), from, count,
                                    end / HK_CACHE_BLOCK, reinterpret_cast<hipStream_t>(stream)));
}

int32_t hk_cache_rewind(const hk_cache *cache, int32_t pos, void *stream) {
  CacheView v;
  int32_t rc = view_of("hk_cache_rewind", cache, v);
  if (!rc) rc = buffers_of("hk_cache_rewind", v);
  if (rc) return rc;
  if (pos < 0 || pos >= cache->seq_len) return failed(HE_E_ARG, "hk_cache_rewind: pos is outside the context (seq_len)");
  if (pos % HK_CACHE_BLOCK == 0) return HE_OK;
  return launched("hk_cache_rewind",
                  launch_cache_read(v, nullptr, nullptr, pos / HK_CACHE_BLOCK * HK_CACHE_BLOCK, pos % HK_CACHE_BLOCK, -1,
                                    reinterpret_cast<hipStream_t>(stream)));
}

int64_t hk_logprobs_workspace(int32_t m, int32_t n, int32_t top) {
  if (m < 1 || m > 1 << 30 || n < 1 || n > 1 << 30 || top < 0 || top > HK_LOGPROBS_TOP_MOST)
    return failed(HE_E_ARG, "hk_logprobs: m and n are in 1..2^30, top in 0..HK_LOGPROBS_TOP_MOST (32)");
  return logprobs_workspace(m, n, top);
}

int32_t hk_logprobs(void *logp, void *entropy, void *ids, void *logps, const void *logits, int64_t stride,
                    const void *given, int32_t n_given, int32_t m, int32_t n, int32_t top, void *workspace,
                    int64_t workspace_bytes, void *stream) {
  const int64_t need = hk_logprobs_workspace(m, n, top);
  if (need < 0) return (int32_t)need;
  if (!logits || stride < n || !aligned(logits, 4))
    return failed(HE_E_ARG, "hk_logprobs: logits is null or not 4-byte aligned, or stride is less than n");
  if (n_given < 0 || (n_given > 0 && (!given || !logp)))
    return failed(HE_E_ARG, "hk_logprobs: given tokens need given and logp");
  if (top > 0 && (!ids || !logps)) return failed(HE_E_ARG, "hk_logprobs: alternatives need ids and logps");
  if (!n_given && !top && !entropy) return failed(HE_E_ARG, "hk_logprobs: nothing is asked for");
  if (need > 0 && (!workspace || !aligned(workspace) || workspace_bytes < need))
    return failed(HE_E_ARG, "hk_logprobs: the workspace is null, not 16-byte aligned or smaller than hk_logprobs_workspace");
  const LogprobArgs a = {reinterpret_cast<float *>(logp), reinterpret_cast<float *>(entropy),
                         reinterpret_cast<int32_t *>(ids), reinterpret_cast<float *>(logps),
                         reinterpret_cast<const float *>(logits), stride, reinterpret_cast<const int32_t *>(given),
                         n_given, m, n, top, reinterpret_cast<uint8_t *>(workspace)};
  return launched("hk_logprobs", launch_logprobs(a, reinterpret_cast<hipStream_t>(stream)));
}

}  // extern "C"
