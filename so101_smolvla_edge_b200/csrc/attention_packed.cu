// Causal grouped-query attention over prompts packed end to end (so101_attention_packed), on tcgen05.
//
//   o_i = sum_{j <= i} 2^(f q_i . k_j - m_i) v_j / sum_{j <= i} 2^(f q_i . k_j - m_i),  f = scale * log2(e)
//
// The query heads of a kv head are stacked: row r of (sequence, kv head) is token r / group, head
// r % group of the group, so 128 MMA rows span few tokens (43 at three heads per kv head), little of
// a 128-key tile is masked at the diagonal, and one K / V tile serves every head that reads it.
// A work item is 256 such rows (two groups of 128) of one kv head. One CTA per SM walks its items, a
// sequence's last blocks (most keys) first, in six warp groups that split the registers unevenly:
//   0  warp 0: TMA, K_j and V_j (128 keys) into rings that run on across items
//      warps 1, 2: the MMAs of group 0 / 1, S_g = Q_g K_j^T -> TMEM, O_g += P_g V_j, P_g read from TMEM
//      warp 3: the list of items, ahead of the rest
//   1  the queries of the next item: loaded, rotated in fp32, rounded to bf16 into swizzled tiles (head_dim 128: loaded;
//      the softmax threads rotate)
//   2-5  the softmax, and O / l to the output rows: two threads per row (TMEM lane)
// While a group's softmax runs, the tensor pipe works for the other one. TMEM holds S (128 columns), P and O of
// both groups at head_dim 64; at 128, S and O only, and P takes the place of the S that it came from.
// Rotated queries are kept in two bf16 parts (value and remainder, two MMAs into one S): the error against 64 bits falls
// from 2.6e-3 to 1.9e-3 (1.6e-3 is the rounding of the result). At 128 the second part takes the place of a tile of K and V,
// which go through one ring of three then: one sequence of 8191 tokens 800 us, 636 with one part (tiles of 64 keys, two of
// each: 1058); 64 prompts of 113 to 305 150 us, 128 with one part.
// The row maximum is only raised when a tile exceeds it by more than 2^8 (as in the SigLIP kernel).
// Keys past the row's own token are masked by their index. Their values still meet P = 0 in the MMA, where an
// infinity or a NaN in a value the row must not see would make the row NaN, so a row whose result is
// not finite is computed again key by key over what it sees (never with finite values).
// Measured: one sequence of 8191 tokens, 32 heads on 8 of 128, 620-640 us (0.86-0.89 PFLOP/s; 724 us with a CTA per
// 128 rows and one softmax thread per row); with heads of 64, 430 us. The chain
// S -> maximum -> exponentials -> P V -> next S bounds it, with the issue slots half and the tensor pipe 41 to 55% busy.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kv_pages.cuh"
#include "tc_attn.cuh"

namespace so101 {

struct PackedArgs {
  const __nv_bfloat16* q;
  const __nv_bfloat16* k;
  const __nv_bfloat16* v;
  __nv_bfloat16* o;
  long long ldq, ldk, ldv, ldo;
  const int* starts;
  int n_seqs, rows, group, n_kv;
  int block;      // rows of an item: 256, or 128 where that leaves SMs without one (the second group idle)
  int group_inv;  // 65536 / group + 1: x / group = x * group_inv >> 16 for x < 512
  const float* cos;
  const float* sin;
  float scale_log2;
  int* status;
};

constexpr int kPkRows = 128;  // rows per group (MMA M)
constexpr float kPkStaleMax = 8.f;
// PARTS: bf16 parts of a query that are held (2: it is rotated here, always at head_dim 64).
template <int HD, int PARTS>
struct PkCfg {
  static constexpr int kHalves = HD / 64;             // 64-dim (128-byte) tiles of a row
  static constexpr int kKeys = 128;                   // keys per tile
  static constexpr int kQTile = kPkRows * 128;        // 16 KB: 128 rows x 64 dims
  static constexpr int kKTile = kKeys * 128;          // kKeys rows x 64 dims
  static constexpr int kStage = kHalves * kKTile;     // a K or V tile
  static constexpr int kQBufs = HD == 64 ? 2 : 1;     // items whose queries are held
  // K and V tiles: two of each, or, beside two parts of queries of 128 dims, three in one ring that they take in turn
  static constexpr bool kOneRing = HD == 128 && PARTS == 2;
  static constexpr int kSlots = kOneRing ? 3 : 4;
  static constexpr int kBars = kOneRing ? 3 : 2;      // barriers of a kind (K's and V's are the same in one ring)
  __device__ static constexpr int k_slot(int t) { return kOneRing ? 2 * t % 3 : t % 2; }
  __device__ static constexpr int k_use(int t) { return kOneRing ? 2 * t / 3 : t / 2; }
  __device__ static constexpr int v_slot(int t) { return kOneRing ? (2 * t + 1) % 3 : t % 2; }
  __device__ static constexpr int v_use(int t) { return kOneRing ? (2 * t + 1) / 3 : t / 2; }
  static constexpr int kQGroup = PARTS * kHalves * kQTile;  // a group's queries
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kQBufs * 2 * kQGroup;
  static constexpr int kOffV = kOneRing ? kOffK : kOffK + 2 * kStage;
  // [2][2 groups][2 halves][128] values between half rows: floats, or their halves where floats do not fit
  static constexpr int kOffSwap = kOffK + kSlots * kStage;
  static constexpr int kOffBar = kOffSwap + (kOneRing ? 2048 : 4096);
  static constexpr int kSmem = kOffBar + 768 + (kOneRing ? 0 : 1024);
  // TMEM columns of a group. head_dim 64: S (128), P (64) and O (64) side by side; 128: S and O (128 each), P in
  // the place of the S that it came from.
  static constexpr bool kAlias = HD == 128;
  static constexpr uint32_t kColS = 0, kColP = HD == 64 ? 128 : 0, kColO = HD == 64 ? 192 : 128, kGroupCols = 256;
  // Warps: four for loads, MMAs and the item list, then the queries', then 16 for the softmax. Registers per thread
  // of each kind: together no more than the threads start with (80 of 768 threads).
  // At head_dim 128 the softmax threads turn the queries that those four bring, between an item's last P and its O
  // (64 prompts of 113 to 305 tokens, 32 heads on 8, in one part: 135 us, 182 with the four turning them); at 64, with two
  // buffers, the four do (15 heads on 5: 54 us, 55; 64 prompts of 512 120 and 129).
  static constexpr bool kSoftTurns = HD == 128 && PARTS == 2;
  static constexpr int kQWarps = 4;
  static constexpr int kThreads = 32 * (4 + kQWarps + 16);
  static constexpr int kRegsLoad = HD == 64 ? 40 : 48, kRegsQuery = HD == 64 ? 72 : 40, kRegsSoft = HD == 64 ? 88 : 96;
  static constexpr int kItemReaders = 1 + 4 + kQWarps + 16;  // reads of each item: loads, MMAs 2 x 2 (S, P V), queries, softmax
};
static_assert(PkCfg<64, 2>::kSmem <= 232448 && PkCfg<128, 1>::kSmem <= 232448 && PkCfg<128, 2>::kSmem <= 232448,
              "227 KB of shared memory per CTA");

// One output row in plain fp32 over the keys it may see, by a whole warp: lane l holds dims
// l, l + 32, ... Only for rows that came out not finite. A warp takes up to 16 of them one after another while the CTA's
// others wait, for two seconds at most: those are reached at 750000 tokens (heads of 64; 430000 of 128), at 200000 and
// 130000 with 32 rows a warp and one key at a time.
template <int HD>
__device__ __forceinline__ void packed_row_alone(const PackedArgs& a, int start, int tok, int head, int kvh) {
  const int lane = threadIdx.x & 31;
  constexpr int N = HD / 32;
  float q[N], o[N];
  const __nv_bfloat16* qr = a.q + (start + tok) * a.ldq + head * HD;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 32 * i;
    q[i] = __bfloat162float(qr[d]);
    if (a.cos) {
      const long long p = static_cast<long long>(start + tok) * (HD / 2) + d % (HD / 2);
      const float other = __bfloat162float(qr[(d + HD / 2) % HD]);
      q[i] = d < HD / 2 ? q[i] * a.cos[p] - other * a.sin[p] : q[i] * a.cos[p] + other * a.sin[p];
    }
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  constexpr int kAt = 256 / HD;  // keys at a time, their loads in flight together
  for (int j0 = 0; j0 <= tok; j0 += kAt) {
    float s[kAt];
#pragma unroll
    for (int b = 0; b < kAt; ++b) {
      const __nv_bfloat16* kr = a.k + (start + min(j0 + b, tok)) * a.ldk + kvh * HD;
      s[b] = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s[b] = fmaf(q[i], __bfloat162float(kr[lane + 32 * i]), s[b]);
    }
    float mn = m;
#pragma unroll
    for (int b = 0; b < kAt; ++b) {
#pragma unroll
      for (int d = 16; d; d >>= 1) s[b] += __shfl_xor_sync(0xffffffffu, s[b], d);
      s[b] = j0 + b <= tok ? s[b] * a.scale_log2 : -INFINITY;
      mn = fmaxf(mn, s[b]);
    }
    const float base = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - base);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] *= alpha;
#pragma unroll
    for (int b = 0; b < kAt; ++b) {
      const __nv_bfloat16* vr = a.v + (start + min(j0 + b, tok)) * a.ldv + kvh * HD;
      const float p = exp2f(s[b] - base);
      l += p;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = __bfloat162float(vr[lane + 32 * i]);
        if (j0 + b <= tok) o[i] = fmaf(p, x, o[i]);
      }
    }
  }
  __nv_bfloat16* out = a.o + (start + tok) * a.ldo + head * HD;
#pragma unroll
  for (int i = 0; i < N; ++i) out[lane + 32 * i] = __float2bfloat16(l == 0.f ? 0.f : o[i] / l);
}

// Eight dims (x1) and their partners HD / 2 later (x2) of a query turned by the angles of cv / sv: each operation
// rounded to fp32, the results to bf16, and with PARTS == 2 what that loses, in bf16 too, in l1 / l2.
template <int PARTS>
__device__ __forceinline__ void packed_turn(uint4& x1, uint4& x2, uint4& l1, uint4& l2, const float* cv, const float* sv) {
  __nv_bfloat162* h1 = reinterpret_cast<__nv_bfloat162*>(&x1);
  __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&x2);
  __nv_bfloat162* r1 = reinterpret_cast<__nv_bfloat162*>(&l1);
  __nv_bfloat162* r2 = reinterpret_cast<__nv_bfloat162*>(&l2);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 v1 = __bfloat1622float2(h1[e]), v2 = __bfloat1622float2(h2[e]);
    const float y0 = __fsub_rn(__fmul_rn(v1.x, cv[2 * e]), __fmul_rn(v2.x, sv[2 * e]));
    const float y1 = __fsub_rn(__fmul_rn(v1.y, cv[2 * e + 1]), __fmul_rn(v2.y, sv[2 * e + 1]));
    const float y2 = __fadd_rn(__fmul_rn(v2.x, cv[2 * e]), __fmul_rn(v1.x, sv[2 * e]));
    const float y3 = __fadd_rn(__fmul_rn(v2.y, cv[2 * e + 1]), __fmul_rn(v1.y, sv[2 * e + 1]));
    h1[e] = __floats2bfloat162_rn(y0, y1);
    h2[e] = __floats2bfloat162_rn(y2, y3);
    if (PARTS == 2) {
      const float2 b1 = __bfloat1622float2(h1[e]), b2 = __bfloat1622float2(h2[e]);
      r1[e] = __floats2bfloat162_rn(y0 - b1.x, y1 - b1.y);
      r2[e] = __floats2bfloat162_rn(y2 - b2.x, y3 - b2.y);
    }
  }
}

// The largest of three (NaN only if all are).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// A work item: rows [row_first, row_first + rows) (of the stacked ones) of the sequence that begins at packed
// row `start`, kv head kvh. rows == 0: no more items. What every warp would divide for is worked out with it: row r of the
// item is token tok + (lead + r) / group, head (lead + r) % group, and row group g has tiles[g] key tiles (0: no rows).
struct __align__(16) PackedItem {
  int start, row_first, rows, kvh;
  int tok, lead, tiles[2];

  __device__ __forceinline__ int tiles_of(int g) const { return g ? tiles[1] : tiles[0]; }
  __device__ __forceinline__ int all_tiles() const { return max(tiles[0], tiles[1]); }
  __device__ __forceinline__ void divide(const PackedArgs& a, int keys) {
    tok = row_first / a.group;
    lead = row_first - tok * a.group;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int here = min(rows - g * kPkRows, kPkRows);
      tiles[g] = here <= 0 ? 0 : (tok + ((lead + g * kPkRows + here - 1) * a.group_inv >> 16)) / keys + 1;
    }
  }
};

// The items of one CTA, in order, worked out by one warp for all: item w is kv head w % n_kv of block
// w / n_kv, the blocks (256 rows) of all sequences counted in turn, each sequence's from its last, 32 sequences at a time.
// CTA b takes item b of the first gridDim.x, the b-th last of the second, and so on in turn: items get smaller along
// a sequence, and with the same place in every turn the first CTA would have 14% more than the average.
struct PackedWalk {
  int turn, s0, before;  // items taken; the window's first sequence and the blocks before it

  __device__ __forceinline__ PackedItem next(const PackedArgs& a, int keys) {
    const int lane = threadIdx.x & 31;
    const int g = static_cast<int>(gridDim.x), b = static_cast<int>(blockIdx.x);
    const int w = turn * g + (turn & 1 ? g - 1 - b : b);
    ++turn;
    const int block = w / a.n_kv;
    PackedItem it;
    it.kvh = w - block * a.n_kv;
    it.start = it.row_first = it.rows = it.tok = it.lead = it.tiles[0] = it.tiles[1] = 0;
    for (; s0 < a.n_seqs; s0 += 32) {
      const int s = s0 + lane;
      int at = 0, len = 0;
      if (s < a.n_seqs) {
        at = __ldg(a.starts + s);
        len = __ldg(a.starts + s + 1) - at;
        if (at < 0 || len < 0 || static_cast<long long>(at) + len > a.rows) {
          record_error(a.status, SO101_ERR_PAGES);
          len = 0;
        }
      }
      int inc = static_cast<int>((static_cast<long long>(len) * a.group + a.block - 1) / a.block);
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > block);
      if (hit) {
        const int x = __ffs(hit) - 1;
        it.start = __shfl_sync(0xffffffffu, at, x);
        const int n = __shfl_sync(0xffffffffu, len, x);
        it.row_first = (before + __shfl_sync(0xffffffffu, inc, x) - 1 - block) * a.block;
        it.rows = min(a.block, n * a.group - it.row_first);
        it.divide(a, keys);
        return it;
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    return it;
  }
};

constexpr int kPkItems = 8;           // items that the list in shared memory holds

template <int HD, int PARTS>
__global__ void __launch_bounds__(PkCfg<HD, PARTS>::kThreads, 1)
    attention_packed_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const PackedArgs a) {
  using Cfg = PkCfg<HD, PARTS>;
  constexpr int kBars = Cfg::kBars, kQBufs = Cfg::kQBufs, kKeys = Cfg::kKeys;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  if (Cfg::kOneRing && smem != smem_raw) {  // no bytes to spare (dynamic shared memory starts on 1024 bytes here)
    if (threadIdx.x == 0) record_error(a.status, SO101_ERR_LAUNCH);
    return;
  }
  PackedItem* items = reinterpret_cast<PackedItem*>(smem + Cfg::kOffBar);
  uint64_t* item_full = reinterpret_cast<uint64_t*>(items + kPkItems);  // [kPkItems]
  uint64_t* item_empty = item_full + kPkItems;                         // [kPkItems] read by every warp
  uint64_t* q_full = item_empty + kPkItems;  // [kQBufs][2] a group's queries of an item are ready
  uint64_t* q_raw = q_full + 2 * kQBufs;     // [kQBufs] an item's queries are there, to be turned
  uint64_t* q_empty = q_raw + kQBufs;        // [kQBufs] both groups' S MMAs have read them
  uint64_t* q_first = q_empty + kQBufs;      // [1] the first item's queries are written
  uint64_t* k_full = q_first + 1;            // [kBars]
  uint64_t* k_empty = k_full + kBars;        // [kBars]
  uint64_t* v_full = Cfg::kOneRing ? k_full : k_empty + kBars;  // [kBars]
  uint64_t* v_empty = Cfg::kOneRing ? k_empty : v_full + kBars;  // [kBars]
  uint64_t* s_full = v_empty + kBars;        // [2] per group: S written
  uint64_t* s_free = s_full + 2;             // [2] S read into registers (head_dim 64)
  uint64_t* p_full = s_free + 2;             // [2] P written, O rescaled
  // [2] P V added to O; everyone waits for each of them (a phase's parity only tells it from its neighbours)
  uint64_t* o_full = p_full + 2;
  uint64_t* o_free = o_full + 2;             // [2] an item's O read out
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  static_assert(kPkItems * sizeof(PackedItem) + (2 * kPkItems + 4 + 4 + 16 + 4 + 12) * 8 + 4 <= 768, "barrier region");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  PackedWalk walk;  // warp 3's
  PackedItem walked;
  if (warp == 0) {
    if (lane < kPkItems) {
      mbar_init(&item_full[lane], 1);
      mbar_init(&item_empty[lane], Cfg::kItemReaders);
    }
    if (lane < kQBufs) {
      mbar_init(&q_full[2 * lane], a.cos && Cfg::kSoftTurns ? 8 : Cfg::kQWarps);
      mbar_init(&q_full[2 * lane + 1], a.cos && Cfg::kSoftTurns ? 8 : Cfg::kQWarps);
      mbar_init(&q_raw[lane], Cfg::kQWarps);
      mbar_init(&q_empty[lane], 2);
    }
    if (lane == 0) mbar_init(q_first, 16);
    if (lane < kBars) {
      mbar_init(&k_full[lane], 1);
      mbar_init(&k_empty[lane], 2);
    }
    if (lane < kBars && !Cfg::kOneRing) {
      mbar_init(&v_full[lane], 1);
      mbar_init(&v_empty[lane], 2);
    }
    if (lane < 2) {
      mbar_init(&s_full[lane], 1);
      mbar_init(&s_free[lane], 8);
      mbar_init(&p_full[lane], 8);
      mbar_init(&o_full[lane], 1);
      mbar_init(&o_free[lane], 8);
    }
    fence_mbar_init();
  } else if (warp == 3) {  // the first item, beside the set-up
    grid_dep_wait();
    walk.turn = walk.s0 = walk.before = 0;
    walked = walk.next(a, kKeys);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  grid_dep_launch();
  grid_dep_wait();

  const bool parted = PARTS == 2 && a.cos != nullptr;  // a second part of the queries
  // waits whose outcome is the same for the whole warp; the n-th use (from 0) of a barrier
  auto wait = [&](uint64_t* b, int n) {
    return __all_sync(0xffffffffu, mbar_wait(b, static_cast<uint32_t>(n) & 1u, a.status));
  };
  // item i of this CTA; rows == 0 past the last, or where a wait ran out. Each reader takes an item once (a look
  // does not count).
  auto item_at = [&](int i, bool look = false) {
    PackedItem it = {};
    if (wait(&item_full[i % kPkItems], i / kPkItems)) {
      it = items[i % kPkItems];
    }
    __syncwarp();
    if (lane == 0 && !look) mbar_arrive(&item_empty[i % kPkItems]);
    return it;
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsLoad));
    if (warp == 3) {
      // ---- the list of items
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (i > 0) walked = walk.next(a, kKeys);
        if (i >= kPkItems) ok = wait(&item_empty[i % kPkItems], i / kPkItems - 1);
        if (ok && lane == 0) {
          items[i % kPkItems] = walked;
          mbar_arrive(&item_full[i % kPkItems]);
        }
        __syncwarp();
        if (walked.rows == 0) break;
      }
    } else if (warp == 0) {
      // ---- K and V tiles
      if (lane == 0) {
        tma_prefetch_desc(&tm_k);
        tma_prefetch_desc(&tm_v);
      }
      const uint64_t keep = policy_evict_normal();
      int t = 0;  // this CTA's key tiles so far (ring slot and phase)
      int k_loads = 0, v_loads = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const PackedItem it = item_at(i);
        if (it.rows == 0) break;
        const int n_tiles = it.all_tiles();
        for (int j = 0; j < n_tiles && ok; ++j, ++t) {
          const int ks = Cfg::k_slot(t), vs = Cfg::v_slot(t);
          if (Cfg::k_use(t) > 0) ok = wait(&k_empty[ks], Cfg::k_use(t) - 1);
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&k_full[ks], Cfg::kStage);
            for (int h = 0; h < Cfg::kHalves; ++h)
              tma_load_2d(smem + Cfg::kOffK + ks * Cfg::kStage + h * Cfg::kKTile, &tm_k, &k_full[ks],
                          it.kvh * HD + 64 * h, it.start + j * kKeys, keep);
          }
          if (!ok) break;
          k_loads = t + 1;
          if (Cfg::v_use(t) > 0) ok = wait(&v_empty[vs], Cfg::v_use(t) - 1);
          if (ok && elect_one()) {
            mbar_arrive_expect_tx(&v_full[vs], Cfg::kStage);
            for (int h = 0; h < Cfg::kHalves; ++h)
              tma_load_2d(smem + Cfg::kOffV + vs * Cfg::kStage + h * Cfg::kKTile, &tm_v, &v_full[vs],
                          it.kvh * HD + 64 * h, it.start + j * kKeys, keep);
          }
          if (ok) v_loads = t + 1;
        }
      }
      // copies in flight land before the CTA ends, also where a wait ran out
      if (Cfg::kOneRing) {
        const int loads = k_loads + v_loads;  // in turn
        for (int n = max(0, loads - 3); n < loads; ++n) wait(&k_full[n % 3], n / 3);
      } else {
        for (int n = max(0, k_loads - 2); n < k_loads; ++n) wait(&k_full[n % 2], n / 2);
        for (int n = max(0, v_loads - 2); n < v_loads; ++n) wait(&v_full[n % 2], n / 2);
      }
    } else {
      // ---- the MMAs of group g, a warp each (so that neither group waits for the other's softmax),
      // one lane elected at each issue. Two cursors walk the CTA's tiles: S runs ahead of P V by one tile,
      // across items too.
      const int g = warp - 1;
      constexpr uint32_t ID_S = idesc_attn(kKeys, 0);
      constexpr uint32_t ID_O = idesc_attn(64, 1);
      const uint32_t d0 = tmem + g * Cfg::kGroupCols;
      struct Cursor {
        int item, j, t, mine, tiles, own;  // item, tile of it, tile of the CTA; this group's tiles of the item, all; own tiles so far
      } cs = {-1, 0, -1, 0, 0, 0}, cp = {-1, 0, -1, 0, 0, 0};
      int n_items = 0;  // items that this group had rows in (of the P V cursor)
      auto pv_done = [&](int n) { return wait(&o_full[g], n); };  // this group's n-th P V
      // To the next tile; false past the last item.
      auto step = [&](Cursor& c) {
        ++c.t;
        if (c.item < 0 || ++c.j == c.tiles) {
          ++c.item;
          const PackedItem it = item_at(c.item);
          c.j = 0;
          c.mine = it.tiles_of(g);
          c.tiles = it.all_tiles();
        }
        return c.tiles > 0;
      };
      // S of the cursor's tile (the K stage freed where the group has no rows for it)
      auto issue_s = [&]() {
        const int st = Cfg::k_slot(cs.t), qb = cs.item % kQBufs;
        const bool has = cs.j < cs.mine;
        // (q_full[0]'s first use is for item kQBufs)
        const bool queries = cs.j > 0 || (cs.item == 0 ? wait(q_first, 0) : wait(&q_full[2 * qb + g], cs.item / kQBufs - (qb == 0 ? 1 : 0)));
        if (!queries || !wait(&k_full[st], Cfg::k_use(cs.t))) return false;
        // the S before is in registers; where P took its place, P V has read that
        if (has && cs.own > 0 && !(Cfg::kAlias ? pv_done(cs.own - 1) : wait(&s_free[g], cs.own - 1))) return false;
        tc_fence_after();
        if (elect_one()) {
          if (has) {
#pragma unroll
            for (int h = 0; h < Cfg::kHalves; ++h) {
              const uint64_t qd = sw128_desc(smem_u32(smem + Cfg::kOffQ + (2 * qb + g) * Cfg::kQGroup + h * Cfg::kQTile));
              const uint64_t kd = sw128_desc(smem_u32(smem + Cfg::kOffK + st * Cfg::kStage + h * Cfg::kKTile));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                mma_f16(d0 + Cfg::kColS, qd + 2 * k, kd + 2 * k, ID_S, h + k > 0 ? 1u : 0u);
              if (parted) {
                const uint64_t rd = qd + (Cfg::kHalves * Cfg::kQTile >> 4);
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16(d0 + Cfg::kColS, rd + 2 * k, kd + 2 * k, ID_S, 1u);
              }
            }
            mma_commit(&s_full[g]);
            mma_commit(&k_empty[st]);
          } else {
            mbar_arrive(&k_empty[st]);
          }
          if (cs.j + 1 == cs.tiles) {
            if (has || cs.mine > 0) mma_commit(&q_empty[qb]);
            else mbar_arrive(&q_empty[qb]);
          }
        }
        if (has) ++cs.own;
        return true;
      };
      auto issue_pv = [&]() {
        const int st = Cfg::v_slot(cp.t);
        const bool has = cp.j < cp.mine;
        if (!wait(&v_full[st], Cfg::v_use(cp.t)) || (has && !wait(&p_full[g], cp.own))) return false;
        if (has && cp.j == 0 && n_items > 0 && !wait(&o_free[g], n_items - 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          if (has) {
            const uint32_t p = d0 + Cfg::kColP;
#pragma unroll
            for (int h = 0; h < Cfg::kHalves; ++h) {
              const uint64_t vd = sw128_desc(smem_u32(smem + Cfg::kOffV + st * Cfg::kStage + h * Cfg::kKTile));
#pragma unroll
              for (int k = 0; k < kKeys / 16; ++k)  // 16 keys = 8 columns of P; of V, 16 rows = 2048 bytes
                mma_f16_ta(d0 + Cfg::kColO + 64 * h, p + 8 * k, vd + static_cast<uint64_t>(k) * (2048 >> 4), ID_O,
                           (cp.j > 0 || k > 0) ? 1u : 0u);
            }
            mma_commit(&o_full[g]);
            mma_commit(&v_empty[st]);
          } else {
            mbar_arrive(&v_empty[st]);
          }
        }
        if (has) {
          ++cp.own;
          if (cp.j == 0) ++n_items;
        }
        return true;
      };
      bool s_more = step(cs);
      bool ok = s_more && issue_s();
      if (ok) s_more = step(cs);
      while (ok && step(cp)) {
        // head_dim 64: the next S of the item as soon as this one is in registers, beside the softmax; then P V.
        // 128 (where it follows P V), and another item's first S (whose queries may not be there yet): P V first
        const bool first = !Cfg::kAlias && s_more && cs.j > 0;
        if (first) ok = issue_s();
        if (ok) ok = issue_pv();
        if (ok && !first && s_more) ok = issue_s();
        if (ok && s_more) s_more = step(cs);
      }
      // MMAs in flight end before TMEM is given back, also where a wait ran out
      if (cs.own > 0) wait(&s_full[g], cs.own - 1);
      if (cp.own > 0) wait(&o_full[g], cp.own - 1);
    }
  } else if (warp < 4 + Cfg::kQWarps) {
    // ---- the queries: 16-byte pieces copied into their swizzled places (all of an item's in flight together),
    // then, with rotary tables and head_dim 64, 8 dims and their partners (HD / 2 later) at a time turned in place
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsQuery));
    constexpr int kPieces = HD / 8, kPairs = HD / 16;
    // the softmax threads bring the first item's queries: at the start they have nothing else to do
    bool ok = item_at(0).rows > 0;
    for (int item = 1; ok; ++item) {
      const PackedItem it = item_at(item);
      if (it.rows == 0) break;
      const int qb = item % kQBufs;
      // the used groups' rows shared out to the warps, padding rows as zeros
      const int rows = (it.rows <= kPkRows ? kPkRows : 2 * kPkRows) / Cfg::kQWarps, row0 = (warp - 4) * rows;
      const int real = min(max(it.rows - row0, 0), rows);
      if (item >= kQBufs) ok = wait(&q_empty[qb], item / kQBufs - 1);  // the buffer's last item has been read
      if (!ok) break;
      uint8_t* base = smem + Cfg::kOffQ + 2 * qb * Cfg::kQGroup;
      // row r of the item is token tok0 + (rem0 + r) / group, head (rem0 + r) % group
      const int tok0 = it.start + it.tok, rem0 = it.lead;
      auto token = [&](int r) { return (rem0 + r) * a.group_inv >> 16; };
      // piece c of row r
      auto at = [&](int r, int c) {
        return base + (r >= kPkRows ? Cfg::kQGroup : 0) + c / 8 * Cfg::kQTile + r % kPkRows * 128 + ((c % 8 ^ (r & 7)) << 4);
      };
      const __nv_bfloat16* q0 = a.q + tok0 * a.ldq + it.kvh * a.group * HD;
#pragma unroll 4
      for (int p = lane; p < rows * kPieces; p += 32) {
        const int r = row0 + p / kPieces, c = p % kPieces, t = r < it.rows ? token(r) : 0;
        const __nv_bfloat16* src = q0 + t * a.ldq + (r < it.rows ? rem0 + r - t * a.group : 0) * HD + 8 * c;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(at(r, c))), "l"(src),
                     "r"(r < it.rows ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if (PARTS == 2 && a.cos && !Cfg::kSoftTurns) {
        // a lane takes 8 dims (and their partners) of a token at a time, for all its heads; the next token's
        // angles are asked for before this one's are used, the first ones beside the copies
        const int first = real > 0 ? token(row0) : 0, tasks = real > 0 ? (token(row0 + real - 1) - first + 1) * kPairs : 0;
        float4 ang[4], next[4];
        auto ask = [&](int p, float4 (&x)[4]) {
          if (p >= tasks) return;
          const long long t = static_cast<long long>(tok0 + first + p / kPairs) * (HD / 2) + p % kPairs * 8;
          x[0] = __ldg(reinterpret_cast<const float4*>(a.cos + t));
          x[1] = __ldg(reinterpret_cast<const float4*>(a.cos + t + 4));
          x[2] = __ldg(reinterpret_cast<const float4*>(a.sin + t));
          x[3] = __ldg(reinterpret_cast<const float4*>(a.sin + t + 4));
        };
        ask(lane, next);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();  // every lane's pieces are there
        for (int p = lane; p < tasks; p += 32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) ang[i] = next[i];
          ask(p + 32, next);
          const int c = p % kPairs, t = first + p / kPairs;
          const int lo = max(row0, t * a.group - rem0), hi = min(row0 + real, (t + 1) * a.group - rem0);
          const float* cv = reinterpret_cast<const float*>(ang);
          const float* sv = cv + 8;
          for (int r = lo; r < hi; ++r) {
            uint4* u1 = reinterpret_cast<uint4*>(at(r, c));
            uint4* u2 = reinterpret_cast<uint4*>(at(r, c + kPairs));
            uint4 x1 = *u1, x2 = *u2, l1, l2;
            packed_turn<PARTS>(x1, x2, l1, l2, cv, sv);
            *u1 = x1;
            *u2 = x2;
            if (PARTS == 2) {
              *reinterpret_cast<uint4*>(at(r, c) + Cfg::kHalves * Cfg::kQTile) = l1;
              *reinterpret_cast<uint4*>(at(r, c + kPairs) + Cfg::kHalves * Cfg::kQTile) = l2;
            }
          }
        }
        if (PARTS == 2)  // the second part of padding rows
          for (int p = real * kPieces + lane; p < rows * kPieces; p += 32)
            *reinterpret_cast<uint4*>(at(row0 + p / kPieces, p % kPieces) + Cfg::kHalves * Cfg::kQTile) = make_uint4(0u, 0u, 0u, 0u);
      } else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        if (a.cos && Cfg::kSoftTurns) {
          mbar_arrive(&q_raw[qb]);
        } else {
          mbar_arrive(&q_full[2 * qb]);
          mbar_arrive(&q_full[2 * qb + 1]);
        }
      }
    }
  } else {
    // ---- softmax of group g: row rl of its 128 (one TMEM lane) by two threads, half hf of every tile's keys
    // each, in warps of the same scheduler. One warp alone cannot keep the exponentials' pipe busy (its
    // instructions wait for one another), four per scheduler can.
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoft));
    constexpr int kMine = kKeys / 2;  // keys of a tile per thread
    const int g = (warp - 4 - Cfg::kQWarps) >> 3, hf = (warp >> 2) & 1;
    const int quad = warp & 3;
    const int rl = quad * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16) + g * Cfg::kGroupCols;
    const uint32_t s_addr = lane_base + Cfg::kColS + hf * kMine, p_addr = lane_base + Cfg::kColP + hf * (kMine / 2);
    const uint32_t o_addr = lane_base + Cfg::kColO + hf * (HD / 2);  // half of the row's O is this thread's too
    using Swap = typename std::conditional<Cfg::kOneRing, unsigned short, unsigned>::type;
    Swap* swap = reinterpret_cast<Swap*>(smem + Cfg::kOffSwap) + g * 256 + rl;  // + 512 per buffer, 128 per half
    const float sc = a.scale_log2;
    auto pv_done = [&](int n) { return wait(&o_full[g], n); };  // this group's n-th P V
    int n_swap = 0;
    // what the other half of the row has. The two buffers take turns: a value is read before the next but one is written.
    auto other_bits = [&](unsigned x) -> unsigned {
      Swap* at = swap + (n_swap++ & 1) * 512;
      at[hf * 128] = static_cast<Swap>(x);
      asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + quad) : "memory");
      return at[(hf ^ 1) * 128];
    };
    auto other = [&](float x) {
      const unsigned u = __float_as_uint(x);
      if (!Cfg::kOneRing) return __uint_as_float(other_bits(u));
      const unsigned high = other_bits(u >> 16);
      return __uint_as_float(high << 16 | other_bits(u & 0xFFFFu));
    };
    {  // the first item's queries: half of row rl's pairs of pieces
      const PackedItem it = item_at(0, true);
      const int r = g * kPkRows + rl;
      if (g * kPkRows < it.rows) {
        const int row = it.lead + (r < it.rows ? r : 0), t = row * a.group_inv >> 16, tok = it.tok + t;
        const uint4* qr = reinterpret_cast<const uint4*>(a.q + (it.start + tok) * a.ldq +
                                                         (it.kvh * a.group + row - t * a.group) * HD);
        constexpr int kPairs = HD / 16;
        uint8_t* to = smem + Cfg::kOffQ + g * Cfg::kQGroup + rl * 128;
#pragma unroll
        for (int i = 0; i < kPairs / 2; ++i) {
          const int c = hf * (kPairs / 2) + i;
          uint4 x1 = make_uint4(0u, 0u, 0u, 0u), x2 = x1, l1 = x1, l2 = x1;
          if (r < it.rows) {
            x1 = __ldg(qr + c);
            x2 = __ldg(qr + c + kPairs);
            if (PARTS == 2 && a.cos) {
              const long long at = static_cast<long long>(it.start + tok) * (HD / 2) + 8 * c;
              float4 ang[4];
              ang[0] = __ldg(reinterpret_cast<const float4*>(a.cos + at));
              ang[1] = __ldg(reinterpret_cast<const float4*>(a.cos + at + 4));
              ang[2] = __ldg(reinterpret_cast<const float4*>(a.sin + at));
              ang[3] = __ldg(reinterpret_cast<const float4*>(a.sin + at + 4));
              const float* cv = reinterpret_cast<const float*>(ang);
              packed_turn<PARTS>(x1, x2, l1, l2, cv, cv + 8);
            }
          }
          uint8_t* d1 = to + c / 8 * Cfg::kQTile + ((c % 8 ^ (rl & 7)) << 4);
          uint8_t* d2 = to + (c + kPairs) / 8 * Cfg::kQTile + (((c + kPairs) % 8 ^ (rl & 7)) << 4);
          *reinterpret_cast<uint4*>(d1) = x1;
          *reinterpret_cast<uint4*>(d2) = x2;
          if (parted) {
            *reinterpret_cast<uint4*>(d1 + Cfg::kHalves * Cfg::kQTile) = l1;
            *reinterpret_cast<uint4*>(d2 + Cfg::kHalves * Cfg::kQTile) = l2;
          }
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_first);
    }
    // Item i's queries of row rl turned: half of its pairs of pieces, in place (head_dim 128).
    auto turn = [&](int i) {
      const PackedItem it = item_at(i, true);
      if (it.rows == 0) return true;
      const int qb = i % kQBufs, r = it.lead + g * kPkRows + rl;
      const bool live = g * kPkRows + rl < it.rows;
      const long long at = (it.start + it.tok + (live ? r * a.group_inv >> 16 : 0)) * static_cast<long long>(HD / 2);
      constexpr int kPairs = HD / 16;
      uint8_t* to = smem + Cfg::kOffQ + (2 * qb + g) * Cfg::kQGroup + rl * 128;
      bool there = true;
#pragma unroll
      for (int c0 = hf * (kPairs / 2); c0 < (hf + 1) * (kPairs / 2); c0 += 2) {
        float4 ang[2][4];
#pragma unroll
        for (int z = 0; z < 2; ++z) {  // asked for before the wait
          const long long x = at + 8 * (c0 + z);
          ang[z][0] = __ldg(reinterpret_cast<const float4*>(a.cos + x));
          ang[z][1] = __ldg(reinterpret_cast<const float4*>(a.cos + x + 4));
          ang[z][2] = __ldg(reinterpret_cast<const float4*>(a.sin + x));
          ang[z][3] = __ldg(reinterpret_cast<const float4*>(a.sin + x + 4));
        }
        if (c0 == hf * (kPairs / 2)) there = wait(&q_raw[qb], i / kQBufs - (qb == 0 ? 1 : 0));
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const int c = c0 + z;
          uint4* u1 = reinterpret_cast<uint4*>(to + c / 8 * Cfg::kQTile + ((c % 8 ^ (rl & 7)) << 4));
          uint4* u2 = reinterpret_cast<uint4*>(to + (c + kPairs) / 8 * Cfg::kQTile + (((c + kPairs) % 8 ^ (rl & 7)) << 4));
          uint4 x1 = *u1, x2 = *u2, l1, l2;
          const float* cv = reinterpret_cast<const float*>(ang[z]);
          packed_turn<PARTS>(x1, x2, l1, l2, cv, cv + 8);
          *u1 = x1;
          *u2 = x2;
          *(u1 + Cfg::kHalves * Cfg::kQTile / 16) = l1;
          *(u2 + Cfg::kHalves * Cfg::kQTile / 16) = l2;
        }
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[2 * qb + g]);
      return there;
    };
    int t = 0;  // this group's key tiles so far
    bool ok = true;
    for (int item = 0; ok; ++item) {
      const PackedItem it = item_at(item);
      // the two warps of a row meet at every exchange, so they leave together (also after a wait ran out)
      if (fminf(it.rows, other(it.rows)) == 0.f) break;
      const int n_tiles = it.tiles_of(g);
      if (n_tiles == 0) {
        if (Cfg::kSoftTurns && a.cos && ok) ok = turn(item + 1);
        continue;
      }
      const bool live = g * kPkRows + rl < it.rows;
      const bool idle = g * kPkRows + quad * 32 >= it.rows;  // a warp of padding rows: nobody reads its P
      const int r = it.lead + (live ? g * kPkRows + rl : 0), past = r * a.group_inv >> 16;
      const int tok = it.tok + past, head = it.kvh * a.group + r - past * a.group;
      const int vis = (live ? tok + 1 : 1) - hf * kMine;  // of its half's keys, [0, vis) are visible to this row
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n_tiles; ++j, ++t) {
        if (ok) ok = wait(&s_full[g], t);
        tc_fence_after();
        if (idle) {
          if (j > 0 && ok) ok = pv_done(t - 1);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (!Cfg::kAlias) mbar_arrive(&s_free[g]);
            mbar_arrive(&p_full[g]);
          }
          continue;
        }
        uint32_t sv[kMine];
#pragma unroll
        for (int c = 0; c < kMine; c += 32) tmem_ld32(s_addr + c, sv + c);
        tmem_ld_wait();
        if (!Cfg::kAlias) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&s_free[g]);
        }
        const int nvis = vis - j * kKeys;
        if (nvis < kMine) {  // by bits: several become predicates in one instruction
#pragma unroll
          for (int c = 0; c < kMine; c += 32) {
            const int n = nvis - c;
            const uint32_t seen = n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(seen & 1u << e)) sv[c + e] = __float_as_uint(-INFINITY);
          }
        }
        auto tile_max = [&]() {
          float mx[4];  // three operands at a time
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = max3(__uint_as_float(sv[c]), __uint_as_float(sv[4 + c]), __uint_as_float(sv[8 + c]));
#pragma unroll
          for (int e = 12; e + 8 <= kMine; e += 8)
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = max3(mx[c], __uint_as_float(sv[e + c]), __uint_as_float(sv[e + 4 + c]));
          if ((kMine - 12) % 8)
#pragma unroll
            for (int c = 0; c < 4; ++c) mx[c] = fmaxf(mx[c], __uint_as_float(sv[kMine - 4 + c]));
          return fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]) * sc;
        };
        float m_tile = tile_max();
        m_tile = fmaxf(m_tile, other(m_tile));  // (head_dim 128: both halves have read S, P may take its place)
        const bool raise = m_tile > m + kPkStaleMax;
        const float alpha = raise ? ex2(m - m_tile) : 1.f;
        if (raise) m = m_tile;
        const float neg_m = m == -INFINITY ? 0.f : -m;
        float ls[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kMine; c += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            fma2(x0, x1, __uint_as_float(sv[c + e]), __uint_as_float(sv[c + e + 1]), sc, neg_m);
            const float p0 = ex2(x0), p1 = ex2(x1);
            const int k = (e >> 1) & 3;
            add2(ls[2 * k], ls[2 * k + 1], p0, p1);
            pk[e >> 1] = bf16x2(p0, p1);
          }
          if (c == 0 && j > 0) {  // the P V before has read P, and O is stable
            if (ok) ok = pv_done(t - 1);
            tc_fence_after();
          }
          tmem_st16(p_addr + c / 2, pk);
        }
        if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int c = 0; c < HD / 2; c += 32) {
            uint32_t ov[32];
            tmem_ld32(o_addr + c, ov);
            tmem_ld_wait();
#pragma unroll
            for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
            tmem_st16(o_addr + c, ov);
            tmem_st16(o_addr + c + 16, ov + 16);
          }
        }
        l = l * alpha + (((ls[0] + ls[2]) + (ls[4] + ls[6])) + ((ls[1] + ls[3]) + (ls[5] + ls[7])));
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[g]);
      }
      if (Cfg::kSoftTurns && a.cos && ok) ok = turn(item + 1);  // while the last P V runs
      l += other(l);
      if (ok) ok = pv_done(t - 1);
      tc_fence_after();
      const float inv = 1.f / l;
      uint32_t worst = 0u;
      const long long row_at = (it.start + tok) * a.ldo + head * HD + hf * (HD / 2);
#pragma unroll
      for (int h = 0; h < HD / 2; h += 32) {
        uint32_t ov[32];
        tmem_ld32(o_addr + h, ov);
        tmem_ld_wait();
        if (h + 32 == HD / 2) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&o_free[g]);  // the next item's P V may overwrite O
        }
        uint4 y[4];  // 8 dims each
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float f[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            f[e] = __uint_as_float(ov[8 * c + e]) * inv;
            worst = max(worst, __float_as_uint(f[e]) & 0x7FFFFFFFu);
          }
          y[c] = make_uint4(bf16x2(f[0], f[1]), bf16x2(f[2], f[3]), bf16x2(f[4], f[5]), bf16x2(f[6], f[7]));
        }
        // 4 x 4 pieces of four lanes' rows transposed, so that a store covers eight rows of 64 bytes, not 32 of 16
        auto swap4 = [&](uint4& lo, uint4& hi, int d) {  // the lane with bit d keeps hi, the other lo
          const bool up = lane & d;
          uint4 give = up ? lo : hi;
          give.x = __shfl_xor_sync(0xffffffffu, give.x, d);
          give.y = __shfl_xor_sync(0xffffffffu, give.y, d);
          give.z = __shfl_xor_sync(0xffffffffu, give.z, d);
          give.w = __shfl_xor_sync(0xffffffffu, give.w, d);
          (up ? lo : hi) = give;
        };
        swap4(y[0], y[1], 1);
        swap4(y[2], y[3], 1);
        swap4(y[0], y[2], 2);
        swap4(y[1], y[3], 2);
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // y[c]: piece lane % 4 of row lane / 4 * 4 + c
          const int w = (lane & ~3) + c;
          const long long to = __shfl_sync(0xffffffffu, row_at, w);
          if (g * kPkRows + quad * 32 + w < it.rows) *(reinterpret_cast<uint4*>(a.o + to + h) + (lane & 3)) = y[c];
        }
      }
      // rows that are not finite, again: whole, every other one by either warp
      if (!ok) worst = 0xFFFFFFFFu;
      worst = max(worst, __float_as_uint(other(__uint_as_float(worst))));
      if (__any_sync(0xffffffffu, worst == 0xFFFFFFFFu)) break;
      unsigned again = __ballot_sync(0xffffffffu, live && worst >= 0x7F800000u);
      for (int n = 0; again; ++n) {
        const int x = __ffs(again) - 1;
        again &= again - 1;
        if ((n & 1) != hf) continue;
        packed_row_alone<HD>(a, it.start, __shfl_sync(0xffffffffu, tok, x), __shfl_sync(0xffffffffu, head, x), it.kvh);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

namespace {

using PkEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// 128-row x 64-column boxes over `rows` rows of `cols` bf16 columns, row stride ld elements.
int packed_map(CUtensorMap* m, const void* base, long long rows, long long cols, long long ld) {
  static const PkEncodeFn enc = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<PkEncodeFn>(p);
    return static_cast<PkEncodeFn>(nullptr);
  }();
  if (!enc) return SO101_ERR_DRIVER;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  cuuint32_t box[2] = {64, 128};
  cuuint32_t estr[2] = {1, 1};
  return enc(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
             ? SO101_OK
             : SO101_ERR_ARG;
}

template <int HD, int PARTS>
int launch_packed(const CUtensorMap& tk, const CUtensorMap& tv, PackedArgs a, cudaStream_t stream) {
  static std::atomic<int> sms[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return SO101_ERR_DRIVER;
  int full = sms[dev].load();
  if (!full) {
    cudaError_t e = cudaFuncSetAttribute(attention_packed_kernel<HD, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         PkCfg<HD, PARTS>::kSmem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&full, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return launch_error(e);
    sms[dev].store(full);
  }
  // items, at most: the sequences' blocks, one part-filled each, of every kv head. Blocks of 128 rows where all of
  // them still run at once: a single prompt of 241 tokens takes 10.6 us so, 13.0 with 256.
  const int64_t part = a.n_seqs < a.rows ? a.n_seqs : a.rows, stacked = static_cast<int64_t>(a.rows) * a.group;
  const int64_t fine = (stacked / kPkRows + part) * a.n_kv;
  a.block = fine <= full ? kPkRows : 2 * kPkRows;
  const int64_t items = (stacked / a.block + part) * a.n_kv;
  if (items > (1 << 30)) return SO101_ERR_ARG;
  const dim3 grid(static_cast<unsigned>(items < full ? items : full));
  return launch_kernel(attention_packed_kernel<HD, PARTS>, grid, dim3(PkCfg<HD, PARTS>::kThreads), PkCfg<HD, PARTS>::kSmem, stream, tk, tv, a);
}

}  // namespace

}  // namespace so101

using namespace so101;

extern "C" int so101_attention_packed(const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                                      int64_t ldv, void* o, int64_t ldo, int64_t rows, const int* starts, int n_seqs,
                                      int64_t max_len, int nq, int nkv, int hd, float scale, const float* cos,
                                      const float* sin, cudaStream_t stream) {
  if (rows < 0 || n_seqs < 0 || max_len < 0 || nq < 1 || nkv < 1 || nq % nkv ||
      (hd != 64 && hd != 128) || (cos == nullptr) != (sin == nullptr) || !(scale > 0.f && scale < INFINITY))
    return SO101_ERR_ARG;
  if (nq / nkv > 128 || nkv > 65535 || n_seqs > (1 << 24) || rows * (nq / nkv) > (1LL << 30)) return SO101_ERR_ARG;
  if (rows == 0 || n_seqs == 0 || max_len == 0) return SO101_OK;
  if (!q || !k || !v || !o || !starts) return SO101_ERR_ARG;
  const auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!a16(q) || !a16(k) || !a16(v) || !a16(o) || ldq % 8 || ldk % 8 || ldv % 8 || ldo % 8) return SO101_ERR_ARG;
  if (cos && (!a16(cos) || !a16(sin))) return SO101_ERR_ARG;
  const int64_t wq = static_cast<int64_t>(nq) * hd, wk = static_cast<int64_t>(nkv) * hd;
  if (ldq < wq || ldo < wq || ldk < wk || ldv < wk) return SO101_ERR_ARG;
  CUtensorMap tk, tv;
  int rc = packed_map(&tk, k, rows, wk, ldk);
  if (!rc) rc = packed_map(&tv, v, rows, wk, ldv);
  if (rc) return rc;
  PackedArgs a;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.k = static_cast<const __nv_bfloat16*>(k);
  a.v = static_cast<const __nv_bfloat16*>(v);
  a.o = static_cast<__nv_bfloat16*>(o);
  a.ldq = ldq;
  a.ldk = ldk;
  a.ldv = ldv;
  a.ldo = ldo;
  a.starts = starts;
  a.n_seqs = n_seqs;
  a.rows = static_cast<int>(rows);
  a.group = nq / nkv;
  a.cos = cos;
  a.sin = sin;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.status = status_ptr();
  a.n_kv = nkv;
  a.group_inv = 65536 / a.group + 1;
  if (hd == 64) return launch_packed<64, 2>(tk, tv, a, stream);
  return cos ? launch_packed<128, 2>(tk, tv, a, stream) : launch_packed<128, 1>(tk, tv, a, stream);
}
