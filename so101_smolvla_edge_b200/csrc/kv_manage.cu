// The pages of the 8-bit cache: taken (so101_kv_reserve), given back (so101_kv_free), shared and copied
// (so101_kv_fork, so101_kv_copy) and moved together (so101_kv_compact).
//
// All on the device, so that a serving loop neither waits for the GPU nor mirrors its tables. A plan
// kernel of one CTA orders what has to be ordered (free pages by number, list entries by place) with
// prefix sums: the same inputs give the same pages, and a call that cannot be met changes nothing.
// It leaves a list of page moves in the scratch ints, which a second launch over the whole GPU
// carries out: a page is n_layers x 2 runs of n_kv * page * hd bytes (20 KB for five heads of 64 and
// 64 slots), read and written once in 16-byte pieces, which the HBM copy rate bounds.
#include "kv_pages.cuh"

namespace so101 {

constexpr int kPlanThreads = 1024;

// Scratch ints: [0] number of moves, then src[most], dst[most] (most = max(n_pages, max_seqs)), then
// remap[n_pages] and the parents' lengths / running offsets [max_seqs].
struct Scratch {
  int* moves;
  int* src;
  int* dst;
  int* remap;
  int* aux;
};

__host__ __device__ inline long long scratch_most(const KvPages& c) { return c.n_pages > c.max_seqs ? c.n_pages : c.max_seqs; }

__device__ __forceinline__ Scratch scratch_of(const KvPages& c) {
  const long long most = scratch_most(c);
  Scratch s;
  s.moves = c.scratch;
  s.src = c.scratch + 4;
  s.dst = s.src + most;
  s.remap = s.dst + most;
  s.aux = s.remap + c.n_pages;
  return s;
}

// Exclusive prefix sum of one int per thread over the CTA, and the total.
__device__ __forceinline__ int block_scan(int x, int& total, int* warp_sums) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = x;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += y;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = warp_sums[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, w, d);
      if (lane >= d) w += y;
    }
    warp_sums[lane] = w;
  }
  __syncthreads();
  const int before = warp ? warp_sums[warp - 1] : 0;
  total = warp_sums[31];
  __syncthreads();
  return before + inc - x;
}

// The lowest `want` free pages, ascending, into list; false if there are fewer. Whole CTA.
__device__ __forceinline__ bool free_pages(const KvPages& c, int want, int* list, int* warp_sums) {
  int found = 0;
  for (int p0 = 0; p0 < c.n_pages && found < want; p0 += kPlanThreads) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const int free = p < c.n_pages && c.refs[p] <= 0 ? 1 : 0;
    int here;
    const int rank = found + block_scan(free, here, warp_sums);
    if (free && rank < want) list[rank] = p;
    found += here;
  }
  __syncthreads();
  return found >= want;
}

__device__ __forceinline__ int pages_for(const KvPages& c, int tokens) { return (tokens + c.page - 1) / c.page; }

struct ListArgs {
  KvPages c;
  const int* a;  // sequences (reserve), parents (fork), source pages (copy)
  const int* b;  // tokens (reserve), children (fork), destination pages (copy)
  int n;
  int* status;
};

__global__ void __launch_bounds__(kPlanThreads, 1) kv_reserve_kernel(const ListArgs g) {
  __shared__ int warp_sums[32];
  __shared__ int bad;
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = g.c;
  const Scratch s = scratch_of(c);
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  // pages that each entry needs, as running offsets
  int want = 0;
  for (int i0 = 0; i0 < g.n; i0 += kPlanThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    int need = 0;
    if (i < g.n) {
      const int seq = g.a[i], add = g.b[i];
      const int len = seq >= 0 && seq < c.max_seqs ? c.lengths[seq] : -1;
      if (len < 0 || add < 0 || static_cast<long long>(len) + add > static_cast<long long>(c.max_pages) * c.page)
        bad = 1;
      else
        need = min(pages_for(c, len + add) - pages_for(c, len), c.n_pages + 1);  // the sums stay in 32 bits
    }
    int here;
    const int off = block_scan(need, here, warp_sums);
    if (i < g.n) s.aux[i] = want + off;
    want = min(want + here, c.n_pages + 1);  // more than the pool has is refused below
    if (here > c.n_pages) bad = 1;
  }
  __syncthreads();
  const bool enough = !bad && want <= c.n_pages && free_pages(c, want, s.src, warp_sums);
  if (!enough) {
    if (threadIdx.x == 0) record_error(g.status, SO101_ERR_PAGES);
    return;
  }
  for (int i = threadIdx.x >> 5; i < g.n; i += kPlanThreads / 32) {  // a warp per entry
    const int lane = threadIdx.x & 31;
    const int seq = g.a[i], add = g.b[i], len = c.lengths[seq];
    const int have = pages_for(c, len), need = pages_for(c, len + add) - have;
    for (int j = lane; j < need; j += 32) {
      const int id = s.src[s.aux[i] + j];
      c.table[static_cast<long long>(seq) * c.max_pages + have + j] = id;
      c.refs[id] = 1;
    }
    __syncwarp();
    if (lane == 0) c.lengths[seq] = len + add;
  }
}

constexpr int kFreeThreads = 128;

// A warp per sequence; the exchange of its length makes a sequence named twice harmless.
__global__ void __launch_bounds__(kFreeThreads) kv_free_kernel(const ListArgs g) {
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = g.c;
  const int i = (blockIdx.x * kFreeThreads + threadIdx.x) >> 5, lane = threadIdx.x & 31;
  if (i >= g.n) return;
  const int seq = g.a[i];
  if (seq < 0 || seq >= c.max_seqs) {
    if (lane == 0) record_error(g.status, SO101_ERR_PAGES);
    return;
  }
  int len = lane == 0 ? atomicExch(c.lengths + seq, 0) : 0;
  len = __shfl_sync(0xffffffffu, len, 0);
  int* row = c.table + static_cast<long long>(seq) * c.max_pages;
  const int held = min(pages_for(c, max(len, 0)), c.max_pages);
  for (int j = lane; j < held; j += 32) {
    const int id = row[j];
    row[j] = -1;
    if (id < 0 || id >= c.n_pages) {
      record_error(g.status, SO101_ERR_PAGES);
    } else if (atomicSub(c.refs + id, 1) <= 0) {
      atomicAdd(c.refs + id, 1);
      record_error(g.status, SO101_ERR_PAGES);
    }
  }
}

__global__ void __launch_bounds__(kPlanThreads, 1) kv_fork_kernel(const ListArgs g) {
  __shared__ int warp_sums[32];
  __shared__ int bad;
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = g.c;
  const Scratch s = scratch_of(c);
  if (threadIdx.x == 0) {
    bad = 0;
    *s.moves = 0;
  }
  __syncthreads();
  // entry i: its parent's length into aux, its place among the copies kept beside it (remap)
  int copies = 0;
  for (int i0 = 0; i0 < g.n; i0 += kPlanThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    int part = 0, len = 0;
    if (i < g.n) {
      const int par = g.a[i], chi = g.b[i];
      if (par < 0 || par >= c.max_seqs || chi < 0 || chi >= c.max_seqs || c.lengths[chi] != 0 ||
          (len = c.lengths[par]) < 0 || len > c.max_pages * c.page) {
        bad = 1;
        len = 0;
      }
      part = len % c.page ? 1 : 0;
      s.aux[i] = len;
    }
    int here;
    const int off = block_scan(part, here, warp_sums);
    if (i < g.n) s.dst[i] = copies + off;
    copies += here;
  }
  __syncthreads();
  // the fresh pages, listed where the remap of a compaction would be
  const bool enough = !bad && copies <= c.n_pages && free_pages(c, copies, s.remap, warp_sums);
  if (!enough) {
    if (threadIdx.x == 0) record_error(g.status, SO101_ERR_PAGES);
    return;
  }
  for (int i = threadIdx.x >> 5; i < g.n; i += kPlanThreads / 32) {  // a warp per entry
    const int lane = threadIdx.x & 31;
    const int par = g.a[i], chi = g.b[i], len = s.aux[i], whole = len / c.page;
    const int* from = c.table + static_cast<long long>(par) * c.max_pages;
    int* to = c.table + static_cast<long long>(chi) * c.max_pages;
    for (int j = lane; j < c.max_pages; j += 32) {
      int id = -1;
      if (j < whole) {
        id = from[j];
        if (id >= 0 && id < c.n_pages) atomicAdd(c.refs + id, 1);
        else record_error(g.status, SO101_ERR_PAGES);
      } else if (j == whole && len % c.page) {
        const int k = s.dst[i];
        id = s.remap[k];
        s.src[k] = from[j];
        c.refs[id] = 1;
      }
      if (par != chi) to[j] = id;
    }
    __syncwarp();
    if (lane == 0) c.lengths[chi] = len;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < copies; k += kPlanThreads) s.dst[k] = s.remap[k];
  if (threadIdx.x == 0) *s.moves = copies;
}

// Live pages past the live count into the free ones below it, both ascending.
__global__ void __launch_bounds__(kPlanThreads, 1) kv_compact_kernel(const ListArgs g) {
  __shared__ int warp_sums[32];
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = g.c;
  const Scratch s = scratch_of(c);
  int live = 0;
  for (int p = threadIdx.x; p < c.n_pages; p += kPlanThreads) live += c.refs[p] > 0 ? 1 : 0;
  int total;
  block_scan(live, total, warp_sums);
  int high = 0, holes = 0;
  for (int p0 = 0; p0 < c.n_pages; p0 += kPlanThreads) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const bool in = p < c.n_pages;
    const bool used = in && c.refs[p] > 0;
    const int move = used && p >= total, hole = in && !used && p < total;
    int sum;  // both counts in one scan: at most 1024 of each per turn
    const int off = block_scan(move | hole << 16, sum, warp_sums);
    if (move) s.src[high + (off & 0xFFFF)] = p;
    if (hole) s.dst[holes + (off >> 16)] = p;
    if (in) s.remap[p] = p;
    high += sum & 0xFFFF;
    holes += sum >> 16;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < high; k += kPlanThreads) {
    const int from = s.src[k], to = s.dst[k];
    s.remap[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  if (threadIdx.x == 0) *s.moves = high;
}

constexpr int kMoveThreads = 256;
constexpr int kMovePieces = 4;  // 16-byte pieces that a thread holds at once

// The moves of the list, one unit at a time per CTA: unit u is (move, layer, keys or values, part);
// with `remap`, the table entries too. src / dst given: n pairs; null: the scratch list.
__global__ void __launch_bounds__(kMoveThreads) kv_move_kernel(const ListArgs g, const int remap) {
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = g.c;
  const Scratch s = scratch_of(c);
  const int* src = g.a ? g.a : s.src;
  const int* dst = g.a ? g.b : s.dst;
  const int moves = g.a ? g.n : *s.moves;
  const int pieces = c.n_kv * c.page * c.hd / 16;  // of a page, per layer, keys or values
  constexpr int kUnit = kMoveThreads * kMovePieces;
  const int parts = (pieces + kUnit - 1) / kUnit;
  const long long units = static_cast<long long>(moves) * c.n_layers * 2 * parts;
  for (long long u = blockIdx.x; u < units; u += gridDim.x) {
    const int part = static_cast<int>(u % parts);
    const long long w = u / parts;
    const int which = static_cast<int>(w & 1);
    const int layer = static_cast<int>((w >> 1) % c.n_layers);
    const int k = static_cast<int>((w >> 1) / c.n_layers);
    const int from = src[k], to = dst[k];
    if (from < 0 || from >= c.n_pages || to < 0 || to >= c.n_pages) {
      if (threadIdx.x == 0) record_error(g.status, SO101_ERR_PAGES);
      continue;
    }
    int8_t* codes = which ? c.v : c.k;
    const uint4* x = reinterpret_cast<const uint4*>(codes + kv_code_at(c, layer, from, 0));
    uint4* y = reinterpret_cast<uint4*>(codes + kv_code_at(c, layer, to, 0));
    uint4 t[kMovePieces];
#pragma unroll
    for (int i = 0; i < kMovePieces; ++i) {
      const int p = part * kUnit + i * kMoveThreads + static_cast<int>(threadIdx.x);
      if (p < pieces) t[i] = x[p];
    }
#pragma unroll
    for (int i = 0; i < kMovePieces; ++i) {
      const int p = part * kUnit + i * kMoveThreads + static_cast<int>(threadIdx.x);
      if (p < pieces) y[p] = t[i];
    }
    if (part == 0) {
      float* sc = which ? c.v_scale : c.k_scale;
      for (int h = threadIdx.x; h < c.n_kv; h += kMoveThreads)
        sc[kv_scale_at(c, layer, to, h)] = sc[kv_scale_at(c, layer, from, h)];
    }
  }
  if (remap) {
    const long long entries = static_cast<long long>(c.max_seqs) * c.max_pages;
    for (long long e = static_cast<long long>(blockIdx.x) * kMoveThreads + threadIdx.x; e < entries;
         e += static_cast<long long>(gridDim.x) * kMoveThreads) {
      const int id = c.table[e];
      if (id >= 0 && id < c.n_pages) c.table[e] = s.remap[id];
    }
  }
}

namespace {

int sm_count() {
  int dev = 0, n = 0;
  cudaGetDevice(&dev);
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) n = 148;
  return n;
}

ListArgs list_args(const KvPages* c, const int* a, const int* b, int n) {
  ListArgs g;
  g.c = *c;
  g.a = a;
  g.b = b;
  g.n = n;
  g.status = status_ptr();
  return g;
}

// The copies of at most `most` moves (an upper bound is enough: the list's own length rules).
int move_pages(const ListArgs& g, long long most, int remap, cudaStream_t stream) {
  const long long pieces = static_cast<long long>(g.c.n_kv) * g.c.page * g.c.hd / 16;
  const long long parts = (pieces + kMoveThreads * kMovePieces - 1) / (kMoveThreads * kMovePieces);
  const long long units = most * g.c.n_layers * 2 * parts;
  const long long full = static_cast<long long>(sm_count()) * 8;
  const dim3 grid(static_cast<unsigned>(units < full ? units : full));
  return launch_kernel(kv_move_kernel, grid, dim3(kMoveThreads), 0, stream, g, remap);
}

}  // namespace

}  // namespace so101

using namespace so101;

extern "C" int so101_kv_scratch(const so101_kv_pages* c, int64_t* ints) {
  if (!c || !ints || c->n_pages < 1 || c->max_seqs < 1) return SO101_ERR_ARG;
  *ints = 4 + 2 * scratch_most(*c) + c->n_pages + c->max_seqs;
  return SO101_OK;
}

extern "C" int so101_kv_reserve(const so101_kv_pages* c, const int* seqs, const int* tokens, int n,
                                cudaStream_t stream) {
  if (!kv_pages_ok(c) || n < 0 || n > c->max_seqs || (n > 0 && (!seqs || !tokens))) return SO101_ERR_ARG;
  if (n == 0) return SO101_OK;
  return launch_kernel(kv_reserve_kernel, dim3(1), dim3(kPlanThreads), 0, stream, list_args(c, seqs, tokens, n));
}

extern "C" int so101_kv_free(const so101_kv_pages* c, const int* seqs, int n, cudaStream_t stream) {
  if (!kv_pages_ok(c) || n < 0 || n > c->max_seqs || (n > 0 && !seqs)) return SO101_ERR_ARG;
  if (n == 0) return SO101_OK;
  const int per = kFreeThreads / 32;
  return launch_kernel(kv_free_kernel, dim3(static_cast<unsigned>((n + per - 1) / per)), dim3(kFreeThreads), 0, stream,
                       list_args(c, seqs, nullptr, n));
}

extern "C" int so101_kv_fork(const so101_kv_pages* c, const int* parents, const int* children, int n,
                             cudaStream_t stream) {
  if (!kv_pages_ok(c) || n < 0 || n > c->max_seqs || (n > 0 && (!parents || !children))) return SO101_ERR_ARG;
  if (n == 0) return SO101_OK;
  const int rc = launch_kernel(kv_fork_kernel, dim3(1), dim3(kPlanThreads), 0, stream,
                               list_args(c, parents, children, n));
  return rc ? rc : move_pages(list_args(c, nullptr, nullptr, 0), n, 0, stream);
}

extern "C" int so101_kv_copy(const so101_kv_pages* c, const int* src, const int* dst, int n, cudaStream_t stream) {
  if (!kv_pages_ok(c) || n < 0 || n > c->n_pages || (n > 0 && (!src || !dst))) return SO101_ERR_ARG;
  if (n == 0) return SO101_OK;
  return move_pages(list_args(c, src, dst, n), n, 0, stream);
}

extern "C" int so101_kv_compact(const so101_kv_pages* c, cudaStream_t stream) {
  if (!kv_pages_ok(c)) return SO101_ERR_ARG;
  const ListArgs g = list_args(c, nullptr, nullptr, 0);
  const int rc = launch_kernel(kv_compact_kernel, dim3(1), dim3(kPlanThreads), 0, stream, g);
  return rc ? rc : move_pages(g, c->n_pages, 1, stream);
}
