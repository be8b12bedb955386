// The paged 8-bit K/V cache as the kernels see it, and the rules that its kernels share.
#pragma once

#include "common.cuh"
#include "../../include/so101_b200_text.h"

namespace so101 {

using KvPages = so101_kv_pages;

// Host side: whether the handle describes a cache that the kernels can run on.
inline bool kv_pages_ok(const KvPages* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->table || !c->lengths || !c->refs || !c->scratch)
    return false;
  const auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!a16(c->k) || !a16(c->v) || !a16(c->k_scale) || !a16(c->v_scale)) return false;
  if (c->n_layers < 1 || c->n_pages < 1 || c->n_kv < 1 || c->max_seqs < 1 || c->max_pages < 1) return false;
  if (c->n_kv > 1024 || c->n_pages > (1 << 20) || static_cast<long long>(c->max_pages) * c->page > (1LL << 30)) return false;
  if (c->page != 16 && c->page != 32 && c->page != 64) return false;
  return c->hd == 64 || c->hd == 128;
}

// The scratch ints: number of moves, arrivals, the plan's flag and departures (the last three zero between
// calls), then src[most], dst[most] (most = max(n_pages, max_seqs)), then remap[n_pages], per list entry running
// offsets or parents' lengths [max_seqs] and places [max_seqs], and per sequence whether its last reservation was
// refused [max_seqs].
__host__ __device__ inline long long kv_scratch_most(const KvPages& c) { return c.n_pages > c.max_seqs ? c.n_pages : c.max_seqs; }
__host__ __device__ inline long long kv_refused_at(const KvPages& c) {
  return 4 + 2 * kv_scratch_most(c) + c.n_pages + 2LL * c.max_seqs;
}

// Element offset of (layer, page id, kv head) in the code arrays (slot 0, dim 0) and in the scales.
// A long cache passes 32 bits.
__device__ __forceinline__ long long kv_scale_at(const KvPages& c, int layer, int id, int head) {
  return (static_cast<long long>(layer) * c.n_pages + id) * c.n_kv + head;
}
__device__ __forceinline__ long long kv_code_at(const KvPages& c, int layer, int id, int head) {
  return kv_scale_at(c, layer, id, head) * (c.page * c.hd);
}

// The pages and rows of list entry i: its sequence, its packed rows [row0, row0 + n). False (with
// the error recorded) where an index is out of range.
__device__ __forceinline__ bool kv_rows(const KvPages& c, const int* starts, const int* seqs, int i, long long rows,
                                        int& seq, int& row0, int& n, int* status) {
  seq = seqs ? __ldg(seqs + i) : i;
  row0 = starts ? __ldg(starts + i) : i;
  n = starts ? __ldg(starts + i + 1) - row0 : 1;
  if (seq < 0 || seq >= c.max_seqs || row0 < 0 || n < 0 || static_cast<long long>(row0) + n > rows) {
    record_error(status, SO101_ERR_PAGES);
    return false;
  }
  return true;
}

// A sequence's length, at most what its table row can name.
__device__ __forceinline__ int kv_length(const KvPages& c, int seq, int* status) {
  const int len = c.lengths[seq];
  if (len < 0 || len > c.max_pages * c.page) {
    record_error(status, SO101_ERR_PAGES);
    return 0;
  }
  return len;
}

}  // namespace so101
