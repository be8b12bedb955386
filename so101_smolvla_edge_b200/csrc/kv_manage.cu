// The pages of the 8-bit cache: taken (so101_kv_reserve), given back (so101_kv_free), shared and copied
// (so101_kv_fork, so101_kv_copy) and moved together (so101_kv_compact).
//
// All on the device, so that a serving loop neither waits for the GPU nor mirrors its tables. One CTA
// orders what has to be ordered (free pages by number, list entries by place) with prefix sums: the
// same inputs give the same pages, and a call that cannot be met changes nothing. Fork and compact leave
// a list of page moves, which all CTAs of the same launch carry out. A page is n_layers x 2 runs of
// n_kv * page * hd bytes (20 KB for five heads of 64 and 64 slots); the runs go through shared
// memory in bulk copies, eight in flight per SM, bounded by the HBM copy rate: a compaction that moves 335 MB takes
// 113 us, 5.9 TB/s read and written (156 us with a launch of its own for the moves and 16-byte loads and stores).
#include <atomic>
#include <type_traits>

#include "kv_pages.cuh"

namespace so101 {

constexpr int kPlanThreads = 512;

struct Scratch {  // kv_pages.cuh: kv_refused_at

  int* moves;
  int* arrived;
  int* ready;
  int* left;
  int* src;
  int* dst;
  int* remap;
  int* aux;
  int* place;
  int* refused;
};

__device__ __forceinline__ Scratch scratch_of(const KvPages& c) {
  const long long most = kv_scratch_most(c);
  Scratch s;
  s.moves = c.scratch;
  s.arrived = c.scratch + 1;
  s.ready = c.scratch + 2;
  s.left = c.scratch + 3;
  s.src = c.scratch + 4;
  s.dst = s.src + most;
  s.remap = s.dst + most;
  s.aux = s.remap + c.n_pages;
  s.place = s.aux + c.max_seqs;
  s.refused = c.scratch + kv_refused_at(c);
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
  const int w = lane < kPlanThreads / 32 ? warp_sums[lane] : 0;
  const int before = static_cast<int>(__reduce_add_sync(0xffffffffu, lane < warp ? w : 0));
  total = static_cast<int>(__reduce_add_sync(0xffffffffu, w));
  __syncthreads();
  return before + inc - x;
}

// The count of the thread's page among the first kPlanThreads; asked for early, beside other look-ups.
__device__ __forceinline__ int first_ref(const KvPages& c) {
  return static_cast<int>(threadIdx.x) < c.n_pages ? c.refs[threadIdx.x] : 1;
}

// The lowest `want` free pages, ascending, into list; false if there are fewer. Whole CTA; first: first_ref.
__device__ __forceinline__ bool free_pages(const KvPages& c, int want, int* list, int* warp_sums, int first) {
  int found = 0;
  for (int p0 = 0; p0 < c.n_pages && found < want; p0 += kPlanThreads) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const int free = p < c.n_pages && (p0 ? c.refs[p] : first) <= 0 ? 1 : 0;
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
  const int first = first_ref(c);
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
      if (seq >= 0 && seq < c.max_seqs) s.place[seq] = i;
    }
    int here;
    const int off = block_scan(need, here, warp_sums);
    if (i < g.n) s.aux[i] = want + off;
    want = min(want + here, c.n_pages + 1);  // more than the pool has is refused below
    if (here > c.n_pages) bad = 1;
  }
  __syncthreads();
  // a sequence named twice: one of its entries finds the other's number (their lengths and pages would be worked out
  // apart and written over one another, past the end of the table row where both fit only alone)
  bool twice = false;
  for (int i = threadIdx.x; i < g.n; i += kPlanThreads)
    if (g.a[i] >= 0 && g.a[i] < c.max_seqs && s.place[g.a[i]] != i) twice = true;
  const bool enough = !bad && want <= c.n_pages && free_pages(c, want, s.src, warp_sums, first);
  if (__syncthreads_or(twice) || !enough) {
    if (threadIdx.x == 0) record_error(g.status, SO101_ERR_PAGES);
    // the lengths stay, so what is appended next would land on older tokens: kv_append leaves these sequences alone
    for (int i = threadIdx.x; i < g.n; i += kPlanThreads)
      if (g.a[i] >= 0 && g.a[i] < c.max_seqs) s.refused[g.a[i]] = 1;
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
    if (lane == 0) {
      c.lengths[seq] = len + add;
      s.refused[seq] = 0;
    }
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
  if (lane == 0) c.scratch[kv_refused_at(c) + seq] = 0;
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

// What a fork or a compaction moves, worked out from the cache as it stands, nothing changed: page src[k] to page
// dst[k]. For a fork also each entry's parent length and its place among the copies (-1: none).
struct MovePlan {
  int* src;
  int* dst;
  int* len;
  int* place;
};

// The number of copies; -1 where the call cannot be met. Whole CTA.
__device__ __forceinline__ int plan_fork(const ListArgs& g, const MovePlan& m, int* warp_sums) {
  __shared__ int bad;
  const KvPages& c = g.c;
  if (threadIdx.x == 0) bad = 0;
  __syncthreads();
  int copies = 0;
  const int first = first_ref(c);
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
      m.len[i] = len;
    }
    const int page = part ? c.table[static_cast<long long>(g.a[i]) * c.max_pages + len / c.page] : 0;
    int here;
    const int off = copies + block_scan(part, here, warp_sums);
    if (i < g.n) m.place[i] = part ? off : -1;
    if (part) m.src[off] = page;
    copies += here;
  }
  __syncthreads();
  return !bad && copies <= c.n_pages && free_pages(c, copies, m.dst, warp_sums, first) ? copies : -1;
}

// The bookkeeping of a planned fork, a warp per entry, by warps [first, first + warps) of the CTA.
__device__ __forceinline__ void apply_fork(const ListArgs& g, const MovePlan& m, int first, int warps) {
  const KvPages& c = g.c;
  const int lane = threadIdx.x & 31;
  for (int i = static_cast<int>(threadIdx.x >> 5) - first; i < g.n; i += warps) {
    const int par = g.a[i], chi = g.b[i], len = m.len[i], whole = len / c.page, place = m.place[i];
    const int* from = c.table + static_cast<long long>(par) * c.max_pages;
    int* to = c.table + static_cast<long long>(chi) * c.max_pages;
    for (int j = lane; j < c.max_pages; j += 32) {
      int id = -1;
      if (j < whole) {
        id = from[j];
        if (id >= 0 && id < c.n_pages) atomicAdd(c.refs + id, 1);
        else record_error(g.status, SO101_ERR_PAGES);
      } else if (j == whole && place >= 0) {
        id = m.dst[place];
        c.refs[id] = 1;
      }
      if (par != chi) to[j] = id;
    }
    __syncwarp();
    if (lane == 0) c.lengths[chi] = len;
  }
}

// Live pages past the live count into the free ones below it, both ascending: how many. Whole CTA.
__device__ __forceinline__ int plan_compact(const ListArgs& g, const MovePlan& m, int* warp_sums) {
  const KvPages& c = g.c;
  int live = 0;
  uint32_t seen = 0u;  // of the thread's first 32 pages, which are in use
#pragma unroll 4
  for (int i = 0; i * kPlanThreads < c.n_pages; ++i) {
    const int p = i * kPlanThreads + static_cast<int>(threadIdx.x);
    if (p < c.n_pages && c.refs[p] > 0) {
      ++live;
      if (i < 32) seen |= 1u << i;
    }
  }
  int total;
  block_scan(live, total, warp_sums);
  int high = 0, holes = 0;
  for (int p0 = 0, i = 0; p0 < c.n_pages; p0 += kPlanThreads, ++i) {
    const int p = p0 + static_cast<int>(threadIdx.x);
    const bool used = i < 32 ? seen >> i & 1u : p < c.n_pages && c.refs[p] > 0;
    const int move = used && p >= total, hole = p < c.n_pages && !used && p < total;
    int sum;  // both counts in one scan: at most 512 of each per turn
    const int off = block_scan(move | hole << 16, sum, warp_sums);
    if (move) m.src[high + (off & 0xFFFF)] = p;
    if (hole) m.dst[holes + (off >> 16)] = p;
    high += sum & 0xFFFF;
    holes += sum >> 16;
  }
  __syncthreads();
  return high;
}

// The counts of a planned compaction, and every page's new number into remap (-> the tables), by the threads
// from `first` on, which meet at named barrier 1.
__device__ __forceinline__ void apply_compact(const ListArgs& g, const MovePlan& m, int moves, int* remap, int first) {
  const KvPages& c = g.c;
  const int t = static_cast<int>(threadIdx.x) - first, step = kPlanThreads - first;
  for (int p = t; p < c.n_pages; p += step) remap[p] = p;
  asm volatile("bar.sync 1, %0;" ::"r"(step) : "memory");
  for (int k = t; k < moves; k += step) {
    const int from = m.src[k], to = m.dst[k];
    remap[from] = to;
    c.refs[to] = c.refs[from];
    c.refs[from] = 0;
  }
  asm volatile("bar.sync 1, %0;" ::"r"(step) : "memory");
}

enum { kMoveCopy, kMoveFork, kMoveCompact };
constexpr int kMoveStages = 8;
constexpr int kMoveChunk = 16384;  // bytes of a run that go at once, at most

constexpr int kMoveBatch = 512;  // units whose addresses the CTA works out together

constexpr int kSmallList = 4096;   // moves and fork entries that a plan in shared memory holds
constexpr int kSmallTable = 16384;  // table entries that one CTA rewrites

struct MoveSmem {
  uint8_t data[kMoveStages][kMoveChunk];
  int src[kSmallList], dst[kSmallList], len[kSmallList], place[kSmallList];
  const int8_t* from[kMoveBatch];
  int8_t* to[kMoveBatch];
  int bytes[kMoveBatch];  // 0: a page out of range
  uint64_t full[kMoveStages];
};

__device__ __forceinline__ void bulk_in(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void bulk_out(void* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;\n\tcp.async.bulk.commit_group;" ::"l"(dst),
               "r"(src), "r"(bytes)
               : "memory");
}

__device__ __forceinline__ int ld_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void st_release(int* p, int v) {
  asm volatile("st.release.gpu.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}

// Plan (fork, compact), then move. SMALL: every CTA works the plan out for itself, in shared memory, and starts to
// copy; the CTA that is last to have done so (an atomic count) then changes the bookkeeping, beside its copies, so
// that nobody waits. Larger lists and tables: the first CTA to arrive plans for all, in the scratch ints, the
// others wait (bounded) for its flag. (64 sequences freed and forked again, their part-filled pages 1.3 MB each:
// 17.5 us, 23.8 with the flag. The count is asked for by the threads that do not copy: 19.5 with the copies behind it
// and each look-up behind the one before.)
// Unit u of the moves is (move, layer, keys or values, chunk); CTA b
// takes units b, b + gridDim.x, ...: all its threads work out the addresses of a batch of them (a single
// thread that looks each page number up itself moves a unit in 2 us: 266 us for 335 MB), then
// thread 0 keeps kMoveStages / 2 loads ahead of the stores.
template <int MODE, bool SMALL>
__global__ void __launch_bounds__(kPlanThreads, 1) kv_move_kernel(const ListArgs g) {
  extern __shared__ __align__(128) uint8_t smem_raw[];
  MoveSmem& sm = *reinterpret_cast<MoveSmem*>(smem_raw);
  __shared__ int warp_sums[32];
  __shared__ int shared;
  const KvPages& c = g.c;
  const Scratch s = scratch_of(c);
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMoveStages; ++i) mbar_init(&sm.full[i], 1);
    fence_mbar_init();
  }
  grid_dep_launch();
  grid_dep_wait();
  int moves = g.n;
  bool settle = false;   // this CTA changes the bookkeeping
  bool planned = true;
  // whether the CTA, having planned, is the last to have done so (one thread of each asks)
  auto planned_last = [&]() {
    __threadfence();
    const bool last = atomicAdd(s.left, 1) == static_cast<int>(gridDim.x) - 1;
    if (last) *s.left = 0;
    __threadfence();
    return last;
  };
  MovePlan m = {s.src, s.dst, s.aux, s.place};
  if (SMALL) m = {sm.src, sm.dst, sm.len, sm.place};
  if (MODE != kMoveCopy && SMALL) {
    __syncthreads();
    moves = MODE == kMoveFork ? plan_fork(g, m, warp_sums) : plan_compact(g, m, warp_sums);
    __syncthreads();
    if (moves < 0) {
      if (threadIdx.x == 0 && planned_last()) record_error(g.status, SO101_ERR_PAGES);
      return;
    }
  } else if (MODE != kMoveCopy) {
    // the first CTA to arrive plans: it is running, so the others may wait for it
    if (threadIdx.x == 0) shared = atomicAdd(s.arrived, 1);
    __syncthreads();
    if (shared == 0) {
      moves = MODE == kMoveFork ? plan_fork(g, m, warp_sums) : plan_compact(g, m, warp_sums);
      if (moves >= 0) {
        if (MODE == kMoveFork) apply_fork(g, m, 0, kPlanThreads / 32);
        else apply_compact(g, m, moves, s.remap, 0);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        if (moves < 0) record_error(g.status, SO101_ERR_PAGES);
        *s.moves = max(moves, 0);
        __threadfence();
        st_release(s.ready, 1);
      }
    } else if (threadIdx.x == 0) {
      const uint64_t t0 = globaltimer();
      while (!ld_acquire(s.ready)) {
        if (globaltimer() - t0 > kWaitLimitNs) {
          record_error(g.status, SO101_ERR_TIMEOUT);
          break;
        }
        __nanosleep(50);
      }
    }
    __syncthreads();
    planned = ld_acquire(s.ready);
    moves = planned ? __ldcg(s.moves) : 0;
  }
  // a move's pages: from the caller's lists, the CTA's own, or the scratch ints that another SM wrote
  auto src_of = [&](int k) { return MODE == kMoveCopy ? g.a[k] : SMALL ? sm.src[k] : __ldcg(s.src + k); };
  auto dst_of = [&](int k) { return MODE == kMoveCopy ? g.b[k] : SMALL ? sm.dst[k] : __ldcg(s.dst + k); };
  const int run = c.n_kv * c.page * c.hd;  // bytes per move, layer, keys or values
  const int chunks = (run + kMoveChunk - 1) / kMoveChunk;
  const int chunk = ((run + chunks - 1) / chunks + 15) / 16 * 16;
  using Count = typename std::conditional<SMALL, unsigned, long long>::type;  // (the host sees to their size)
  const Count units = static_cast<Count>(moves) * c.n_layers * 2 * chunks;
  // the scales, and after a compaction the tables: by the warps that do not copy
  auto small_work = [&]() {
    const int t = static_cast<int>(threadIdx.x) - 32, step = kPlanThreads - 32;
    const Count scales = static_cast<Count>(moves) * c.n_layers * c.n_kv * 2;
    for (Count e = static_cast<Count>(blockIdx.x) * step + t; e < scales; e += static_cast<Count>(gridDim.x) * step) {
      const int which = static_cast<int>(e & 1);
      const int h = static_cast<int>((e >> 1) % c.n_kv);
      const Count w = (e >> 1) / c.n_kv;
      const int layer = static_cast<int>(w % c.n_layers), k = static_cast<int>(w / c.n_layers);
      const int from = src_of(k), to = dst_of(k);
      if (from < 0 || from >= c.n_pages || to < 0 || to >= c.n_pages) continue;
      float* sc = which ? c.v_scale : c.k_scale;
      sc[kv_scale_at(c, layer, to, h)] = sc[kv_scale_at(c, layer, from, h)];
    }
    if (MODE != kMoveCopy && SMALL) {
      if (t == 0) shared = planned_last();
      asm volatile("bar.sync 1, %0;" ::"r"(step) : "memory");
      settle = shared;
    }
    if (MODE == kMoveFork && SMALL && settle) apply_fork(g, m, 1, kPlanThreads / 32 - 1);
    if (MODE == kMoveCompact && (SMALL ? settle : planned)) {
      if (SMALL) apply_compact(g, m, moves, s.remap, 32);
      const long long entries = static_cast<long long>(c.max_seqs) * c.max_pages;
      const long long at = SMALL ? t : static_cast<long long>(blockIdx.x) * step + t;
      for (long long e = at; e < entries; e += SMALL ? step : static_cast<long long>(gridDim.x) * step) {
        const int id = c.table[e];
        if (id >= 0 && id < c.n_pages) c.table[e] = __ldcg(s.remap + id);
      }
    }
  };
  const Count mine = units > blockIdx.x ? (units - blockIdx.x + gridDim.x - 1) / gridDim.x : 0;
  constexpr int kAhead = kMoveStages / 2;
  bool ok = true;
  for (Count i0 = 0; i0 < mine || i0 == 0; i0 += kMoveBatch) {
    const int n = static_cast<int>(mine - i0 < kMoveBatch ? mine - i0 : kMoveBatch);
    __syncthreads();  // thread 0 is done with the batch before
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
      const Count u = blockIdx.x + (i0 + i) * gridDim.x, w = u / chunks;
      const int off = static_cast<int>(u % chunks) * chunk;
      const int layer = static_cast<int>((w >> 1) % c.n_layers), k = static_cast<int>((w >> 1) / c.n_layers);
      const int from = src_of(k), to = dst_of(k);
      const bool valid = from >= 0 && from < c.n_pages && to >= 0 && to < c.n_pages;
      if (!valid) record_error(g.status, SO101_ERR_PAGES);
      int8_t* codes = (w & 1) ? c.v : c.k;
      sm.from[i] = codes + (valid ? kv_code_at(c, layer, from, 0) + off : 0);
      sm.to[i] = codes + (valid ? kv_code_at(c, layer, to, 0) + off : 0);
      sm.bytes[i] = valid ? min(chunk, run - off) : 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      // stage and phase of unit i of the batch: its batch's predecessors are whole batches, so i serves
      static_assert(kMoveBatch % (2 * kMoveStages) == 0, "a batch ends on an even phase");
      for (int i = 0; i < n + kAhead && ok; ++i) {
        if (i < n) {  // load unit i; its stage's last store has read it
          asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(kMoveStages - kAhead - 1) : "memory");
          const int st = i % kMoveStages;
          const uint32_t bytes = static_cast<uint32_t>(sm.bytes[i]);
          mbar_arrive_expect_tx(&sm.full[st], bytes);
          if (bytes) bulk_in(smem_u32(sm.data[st]), sm.from[i], bytes, &sm.full[st]);
        }
        const int j = i - kAhead;
        if (j >= 0) {  // store unit j
          ok = mbar_wait(&sm.full[j % kMoveStages], static_cast<uint32_t>(j / kMoveStages) & 1u, g.status);
          if (ok && sm.bytes[j])
            bulk_out(sm.to[j], smem_u32(sm.data[j % kMoveStages]), static_cast<uint32_t>(sm.bytes[j]));
          else
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");  // the groups count units
          if (!ok)  // a wait ran out: the loads still in flight must land before this CTA's shared memory goes
            for (int k = j + 1; k <= i && k < n; ++k)
              mbar_wait(&sm.full[k % kMoveStages], static_cast<uint32_t>(k / kMoveStages) & 1u, g.status);
        }
      }
    } else if (threadIdx.x >= 32 && i0 == 0) {
      small_work();
    }
  }
  if (threadIdx.x == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  if (MODE != kMoveCopy && !SMALL) {
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(s.left, 1) == static_cast<int>(gridDim.x) - 1) {
      *s.arrived = 0;
      *s.left = 0;
      *s.ready = 0;
    }
  }
}

namespace {

ListArgs list_args(const KvPages* c, const int* a, const int* b, int n) {
  ListArgs g;
  g.c = *c;
  g.a = a;
  g.b = b;
  g.n = n;
  g.status = status_ptr();
  return g;
}

// At most `most` moves (an upper bound is enough: the list's own length rules), one CTA per SM.
template <int MODE, bool SMALL>
int launch_moves(const ListArgs& g, long long most, cudaStream_t stream) {
  static std::atomic<int> sms[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return SO101_ERR_DRIVER;
  int full = sms[dev].load();
  if (!full) {
    cudaError_t e = cudaFuncSetAttribute(kv_move_kernel<MODE, SMALL>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(sizeof(MoveSmem)));
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&full, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return launch_error(e);
    sms[dev].store(full);
  }
  const long long run = static_cast<long long>(g.c.n_kv) * g.c.page * g.c.hd;
  const long long units = most * g.c.n_layers * 2 * ((run + kMoveChunk - 1) / kMoveChunk);
  const dim3 grid(static_cast<unsigned>(units < full ? units : full));
  return launch_kernel(kv_move_kernel<MODE, SMALL>, grid, dim3(kPlanThreads), sizeof(MoveSmem), stream, g);
}

// Every CTA plans for itself where the lists and the tables are small enough.
template <int MODE>
int move_pages(const ListArgs& g, long long most, cudaStream_t stream) {
  const long long run = static_cast<long long>(g.c.n_kv) * g.c.page * g.c.hd;
  const long long units = 2LL * kSmallList * g.c.n_layers * ((run + kMoveChunk - 1) / kMoveChunk);  // at most
  const bool small = g.c.n_pages <= 2 * kSmallList && g.n <= kSmallList &&
                     static_cast<long long>(g.c.max_seqs) * g.c.max_pages <= kSmallTable && units < (1LL << 30) &&
                     2LL * kSmallList * g.c.n_layers * g.c.n_kv < (1LL << 30);
  return small ? launch_moves<MODE, true>(g, most, stream) : launch_moves<MODE, false>(g, most, stream);
}

}  // namespace

}  // namespace so101

using namespace so101;

extern "C" int so101_kv_scratch(const so101_kv_pages* c, int64_t* ints) {
  if (!c || !ints || c->n_pages < 1 || c->max_seqs < 1) return SO101_ERR_ARG;
  *ints = kv_refused_at(*c) + c->max_seqs;
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
  return move_pages<kMoveFork>(list_args(c, parents, children, n), n, stream);
}

extern "C" int so101_kv_copy(const so101_kv_pages* c, const int* src, const int* dst, int n, cudaStream_t stream) {
  if (!kv_pages_ok(c) || n < 0 || n > c->n_pages || (n > 0 && (!src || !dst))) return SO101_ERR_ARG;
  if (n == 0) return SO101_OK;
  return launch_moves<kMoveCopy, false>(list_args(c, src, dst, n), n, stream);
}

extern "C" int so101_kv_compact(const so101_kv_pages* c, cudaStream_t stream) {
  if (!kv_pages_ok(c)) return SO101_ERR_ARG;
  return move_pages<kMoveCompact>(list_args(c, nullptr, nullptr, 0), c->n_pages, stream);
}
