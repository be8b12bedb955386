// Attention of each sequence's last tokens over its 8-bit pages (so101_attention_pages): a decoding
// step's single tokens, a chunk of action tokens, drafted tokens.
//
//   o_r = sum_j p_rj s_v[page(j)] c_v[j] / sum_j p_rj,  p_rj = 2^(f s_k[page(j)] (q_r . c_k[j]) - m_r)
//
// with c the int8 codes, s the pages' scales, f = scale * log2(e). The codes are read once: at one
// token per sequence that is 2 * hd bytes per cached token and kv head against 4 * hd * group
// operations, far under the ridge, so the bytes in flight decide. Each warp streams its keys through
// a ring of its own in shared memory with bulk copies (a page's slots of one head are contiguous), and
// works on them alone:
//   S = Q K^T   mma.m16n8k16 f16: 16 query rows (heads of the group x tokens), 8 keys, 16 dims
//   O += s_v (P V)
// A code c becomes an f16 operand in units of 2^-24: the byte with its top bit flipped IS the subnormal f16
// (c + 128) 2^-24, so a mask and a flip (one LOP3) make two operands. For V a packed subtraction takes
// the 128 off again, exactly. For K it is left in: the MMA sums q (c + 128), and 128 times the row's sum of q (of
// its rounded f16 values, from MMAs against ones) comes off the fp32 S; that costs a logit 2^-24 of
// 128 sum |q|, far below the 2^-11 that rounding q to f16 does. (In O the same short cut would leave 2^-24 of 128
// steps beside values that are zero.) Against a prmt under the exponent of 1024 and a subtraction for
// both, a 32-key tile of 128 dims takes about 250 instructions less of 837.
// Measured: one sequence of 131071 tokens (32 heads on 8 of 128) 61-64 us, of which about
// 15 are the start and the join of its parts and the rest runs at the copy rate; 64 ragged sequences, 15 on 5 heads
// of 64, 46 us, bounded by the latency of the few-row tiles with three warps per scheduler.
// Which of a head's dims is which k index of the MMA is free as long as Q and K agree, and so is
// the order of the keys between S and V, so both are laid out to make a thread's codes contiguous: 16
// dims of a key row, 8 of a value row, and the pairs of V come from byte permutes of two rows. Q is
// scaled by a power of two per row and rounded to f16 (11 bits; the row's factor goes back in with f), P
// is rounded to f16.
#pragma once

#include <atomic>
#include <cmath>

#include "kv_pages.cuh"

namespace so101 {

struct PagesArgs {
  KvPages c;
  const __nv_bfloat16* q;
  __nv_bfloat16* o;
  long long ldq, ldo, rows;
  const int* starts;
  const int* seqs;
  const float* cos;
  const float* sin;
  float* partials;
  int* tickets;
  float scale_log2;
  int layer, nq, group, causal;
  uint32_t group_inv;  // 2^32 / group rounded up: x / group is the high word of x * group_inv (x < group + 256)
  bool o_wide;         // rows of o are 16-byte aligned
  int n_seqs, max_q;
  int* status;
};

constexpr float kCode = 1.f / (1 << 24);  // a code's unit as an operand
constexpr uint32_t kOnes = 0x3C003C00u;     // two f16 ones
constexpr int kPgWarps = 4;
constexpr int kPgThreads = 32 * kPgWarps;

// ROWS query rows per CTA: 8 or 16 (each warp works on its own keys), 32 (two warps' rows on each
// of two key groups) or 64 (four warps' rows on the same keys).
template <int HD, int ROWS>
struct PgCfg {
  static constexpr int kRowWarps = ROWS <= 16 ? 1 : ROWS / 16;
  static constexpr int kRings = kPgWarps / kRowWarps;  // key groups, a ring of tiles each
  static constexpr int kKeys = HD == 64 ? 64 : 32;     // keys per tile: 4 KB of K and of V
  static constexpr int kStep = kRings * kKeys;         // keys that the CTA takes at a time
  static constexpr int kTile = kKeys * HD;
  static constexpr int kStages = kRings == 4 ? 2 : 4;
  // tiles asked for ahead: where several warps read a ring, a stage is filled again only a tile's work after its
  // own, so that they need not run in step
  static constexpr int kAhead = kRowWarps == 1 ? kStages - 1 : kStages - 2;
  static constexpr int kMaxPages = kKeys / 16;
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kSlot = ROWS * (HD + 2);        // floats of a part: its rows of O, then their (m, l)
  static constexpr int kJoinRow = HD + 4;              // a row of O in shared memory
  static constexpr int kJoin = kPgWarps * 16 * (kJoinRow + 2) * 4;  // the rings' buffers serve the join too
  static constexpr int kOffScale = kRings * kRing > kJoin ? kRings * kRing : kJoin;
  static constexpr int kOffBar = kOffScale + kRings * kStages * 2 * kMaxPages * 4;
  static constexpr int kOffPlan = kOffBar + 2 * kRings * kStages * 8;
  static constexpr int kSmem = kOffPlan + 64;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// D = A B, and D = A B with B all ones (the rows' sums of A).
__device__ __forceinline__ void mma_16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%10, %10, %10, %10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

// Bytes 0 and 2 of w (codes), and bytes 1 and 3, as f16 pairs (c + 128) 2^-24.
__device__ __forceinline__ uint32_t codes_even(uint32_t w) {
  uint32_t r;  // (w & mask) ^ flip in one instruction
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(r) : "r"(w), "r"(0x00FF00FFu), "r"(0x00800080u));
  return r;
}
__device__ __forceinline__ uint32_t codes_odd(uint32_t w) { return codes_even(w >> 8); }
// The 128 off such a pair.
__device__ __forceinline__ uint32_t centred(uint32_t h) {
  uint32_t r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x00800080u));
  return r;
}

__device__ __forceinline__ void add_scaled(float4& y, float w, const float4& x) {
  y.x = fmaf(w, x.x, y.x);
  y.y = fmaf(w, x.y, y.y);
  y.z = fmaf(w, x.z, y.z);
  y.w = fmaf(w, x.w, y.w);
}

// Where the CTAs' work lies. A problem is (list entry, tile of ROWS query rows, kv head); its keys make
// steps of kStep, at least one, counted by the sequence's length. All problems' steps, end to end, are dealt
// out in equal runs, one per CTA: whatever the lengths, every CTA reads about as many keys. A cut within an
// eighth of a run, or two steps, of a problem's end moves there: a part costs its rows written and read again and
// the wait for the last of them, about as long as two steps (64 sequences of 1000 keys, runs of three
// steps: 16.0 us, 20.1 with every cut where it falls; longer sequences take the same time either way).
struct PagesPlan {
  int entry, first;  // the entry that holds the CTA's first step, and the step at which it begins
  int run, slack, total;
  int begin, end;    // the CTA's steps
};

// The cut b * run, moved to an end of the problem [p0, p0 + steps) that holds it if one is near.
__device__ __forceinline__ int snap_cut(const PagesPlan& p, int cut, int p0, int steps) {
  const int down = cut - p0, up = p0 + steps - cut;
  return min(down, up) > p.slack ? cut : down <= up ? p0 : p0 + steps;
}

// Steps of STEP keys per (row tile, kv head) and row tiles of entry i.
template <int STEP, int ROWS>
__device__ __forceinline__ void entry_size(const PagesArgs& a, int i, int& steps, int& tiles) {
  const int seq = a.seqs ? __ldg(a.seqs + i) : i;
  const int n = a.starts ? __ldg(a.starts + i + 1) - __ldg(a.starts + i) : 1;
  const int len = seq >= 0 && seq < a.c.max_seqs ? a.c.lengths[seq] : 0;
  const int most = a.c.max_pages * a.c.page;
  steps = max(1, (min(max(len, 0), most) + STEP - 1) / STEP);
  tiles = (min(max(n, 0), a.max_q) * a.group + ROWS - 1) / ROWS;
}

// Whole CTA: the sum of all entries' steps, then the entry in which the CTA's first step falls. The
// sums are kept in 32 bits (the host refuses what could pass them).
template <int STEP, int ROWS, int THREADS>
__device__ __forceinline__ PagesPlan pages_plan(const PagesArgs& a, int* shared) {
  constexpr int kWarps = THREADS / 32;
  int* at_cut = shared + 2 * kWarps;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto first_warps = [&](int n) {  // the sum of the first n warps' counts
    return static_cast<int>(__reduce_add_sync(0xffffffffu, lane < n ? shared[lane] : 0));
  };
  int longest = 1;  // most steps of a problem (ROWS > 64)
  auto size = [&](int i) {
    if (i >= a.n_seqs) return 0;
    int steps, tiles;
    entry_size<STEP, ROWS>(a, i, steps, tiles);
    if (tiles > 0) longest = max(longest, steps);
    return steps * tiles * a.c.n_kv;
  };
  const int mine = size(threadIdx.x);  // all entries of a short list
  int sum = mine;
  for (int i = threadIdx.x + THREADS; i < a.n_seqs; i += THREADS) sum += size(i);
  sum = __reduce_add_sync(0xffffffffu, sum);
  if (lane == 0) shared[warp] = sum;
  if (ROWS > 64) {
    longest = __reduce_max_sync(0xffffffffu, longest);
    if (lane == 0) shared[kWarps + warp] = longest;
  }
  __syncthreads();
  PagesPlan p;
  p.total = first_warps(kWarps);
  p.run = max(1, (p.total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x));
  p.slack = max(p.run / 8, min(2, p.run - 1));
  if (ROWS > 64) {
    // Parts of up to 256 rows: written by each and read again by one SM, about half a step's time each, so that the
    // square root of half the steps is the best run for a problem alone; and a cut costs the time of four steps
    // (one sequence of 16384 keys, 50 tokens, 32 heads on 8 of 128: 93 us, 108 with runs of total / CTAs).
    longest = __reduce_max_sync(0xffffffffu, lane < kWarps ? shared[kWarps + lane] : 1);
    p.run = max(p.run, static_cast<int>(ceilf(sqrtf(0.5f * longest))));
    p.slack = min(4, p.run / 2);
  }
  p.entry = p.first = p.begin = p.end = 0;
  const int cut0 = static_cast<int>(blockIdx.x) * p.run, cut1 = cut0 + p.run;
  __syncthreads();
  if (cut0 >= p.total) return p;
  int before = 0;
  for (int i0 = 0; i0 < a.n_seqs; i0 += THREADS) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    const int x = i0 ? size(i) : mine;
    int inc = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += y;
    }
    if (lane == 31) shared[warp] = inc;
    __syncthreads();
    const int first = before + first_warps(warp) + inc - x;
    before += first_warps(kWarps);
    if (x > 0) {  // the entries that hold the CTA's two cuts
      if (first <= cut0 && cut0 < first + x) {
        int steps, tiles;
        entry_size<STEP, ROWS>(a, i, steps, tiles);
        at_cut[0] = i;
        at_cut[1] = first;
        at_cut[2] = snap_cut(p, cut0, first + (cut0 - first) / steps * steps, steps);
      }
      if (cut1 < p.total && first <= cut1 && cut1 < first + x) {
        int steps, tiles;
        entry_size<STEP, ROWS>(a, i, steps, tiles);
        at_cut[3] = snap_cut(p, cut1, first + (cut1 - first) / steps * steps, steps);
      }
    }
    __syncthreads();
    if (cut1 < before) break;
  }
  p.entry = at_cut[0];
  p.first = at_cut[1];
  p.begin = at_cut[2];
  p.end = cut1 < p.total ? at_cut[3] : p.total;
  return p;
}

// Which CTAs share a problem of `steps` steps from p_first on: cuts b * run inside it, further than the slack from both of
// its ends, b = low .. high; part 0 is CTA low - 1's, part k CTA low - 1 + k's.
__device__ __forceinline__ void problem_parts(const PagesPlan& p, int p_first, int steps, int& cta_first, int& parts) {
  const int low = (p_first + p.slack) / p.run + 1, last = p_first + steps - p.slack - 1;
  cta_first = low - 1;
  parts = last > 0 ? max(0, last / p.run - low + 1) + 1 : 1;
}

// GRAN: slots of a page that a tile holds (a tile is one page, several, or a part of one). Three CTAs per SM (four of the
// 64-row kernel of head_dim 64) at the price of a few spilled registers: 64 x 50 tokens of three heads per kv head, in
// tiles of 64 rows over 291 keys, take 46 us, 57 with two.
template <int HD, int ROWS, int GRAN>
__global__ void __launch_bounds__(kPgThreads, HD == 64 && ROWS == 64 ? 4 : 3) attention_pages_kernel(const PagesArgs a) {
  using Cfg = PgCfg<HD, ROWS>;
  constexpr int kKeys = Cfg::kKeys, kStages = Cfg::kStages, kTile = Cfg::kTile;
  constexpr int kRings = Cfg::kRings, kRowWarps = Cfg::kRowWarps;
  constexpr int kHalfRows = ROWS == 8 ? 1 : 2;  // 8-row halves of the MMA's 16 rows that hold queries
  constexpr int kNT = kKeys / 8;                // 8-key tiles of S
  constexpr int kQK = HD / 16;                  // k steps of S
  constexpr int kHalves = HD / 64;              // 64-dim halves of a head
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  int* shared = reinterpret_cast<int*>(smem + Cfg::kOffPlan);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int ring = warp / kRowWarps, roww = warp % kRowWarps;
  const KvPages& c = a.c;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRings * kStages; ++i) {
      mbar_init(&bars[i], kRowWarps == 1 ? 1 : 2);  // the copies (and, for other warps, the scales)
      mbar_init(&bars[kRings * kStages + i], kRowWarps);  // read by every warp of the ring
    }
    fence_mbar_init();
  }
  grid_dep_launch();
  grid_dep_wait();
  const PagesPlan plan = pages_plan<Cfg::kStep, ROWS, kPgThreads>(a, shared);
  if (plan.begin >= plan.end) return;

  uint8_t* my_ring = smem + ring * Cfg::kRing;
  float* my_scales = reinterpret_cast<float*>(smem + Cfg::kOffScale) + ring * kStages * 2 * Cfg::kMaxPages;
  uint64_t* my_bars = bars + ring * kStages;
  uint64_t* my_empty = my_bars + kRings * kStages;
  const int page_log2 = __ffs(c.page) - 1;
  constexpr int per_tile = kKeys / GRAN;  // copies of K (and of V) per tile
  int entry = plan.entry, entry_first = plan.first;
  int at = plan.begin;  // the next step of this CTA's run
  int used = 0;         // tiles that this ring has taken (stages and phases)
  int issued = 0;       // and asked for
  bool ok = true;
  while (at < plan.end && entry < a.n_seqs) {
    // ---- the problem that step `at` belongs to, and the part of it in this CTA's run
    int steps, tiles_of;
    entry_size<Cfg::kStep, ROWS>(a, entry, steps, tiles_of);
    const int entry_end = entry_first + steps * tiles_of * c.n_kv;
    if (at >= entry_end) {
      entry_first = entry_end;
      ++entry;
      continue;
    }
    const int p = (at - entry_first) / steps;
    const int head = p % c.n_kv, rt = p / c.n_kv;
    const int p_first = entry_first + p * steps;
    const int from = at - p_first, to = min(steps, plan.end - p_first);  // its steps here
    at = p_first + to;
    int cta_first, parts;
    problem_parts(plan, p_first, steps, cta_first, parts);
    const int part_no = static_cast<int>(blockIdx.x) - cta_first;

    int seq, row0, n_q;
    if (!kv_rows(c, a.starts, a.seqs, entry, a.rows, seq, row0, n_q, a.status)) continue;
    if (n_q > a.max_q) {  // more rows than the host planned for
      record_error(a.status, SO101_ERR_PAGES);
      n_q = a.max_q;
    }
    const int rows = n_q * a.group;  // rows of this kv head: token r / group, head r % group
    const int tile_row = rt * ROWS;
    const int len = kv_length(c, seq, a.status);
    const int* table = c.table + static_cast<long long>(seq) * c.max_pages;
    // keys of this part that the tile's rows can see
    const int last_row = min(rows, tile_row + ROWS) - 1;
    const int q_len = a.starts ? __ldg(a.starts + entry + 1) - row0 : 1;
    const int key_end = a.causal ? max(0, min(len, len - q_len + last_row / a.group + 1)) : len;
    const int key0 = from * Cfg::kStep, key1 = min(key_end, to * Cfg::kStep);
    const int all_tiles = key1 > key0 ? (key1 - key0 + kKeys - 1) / kKeys : 0;
    const int tiles = all_tiles > ring ? (all_tiles - ring + kRings - 1) / kRings : 0;

    // ---- tile i of this ring: keys [key0 + (i * kRings + ring) * kKeys, + kKeys); lane l < per_tile
    // brings its l-th run of slots. Page numbers are fetched a tile ahead of the copies, scales go to
    // shared memory a tile's work after they were asked for.
    auto run_key = [&](int i) { return key0 + (i * kRings + ring) * kKeys + lane * GRAN; };
    auto page_of = [&](int i) {
      const int key = run_key(i);
      return i < tiles && lane < per_tile && key < key1 ? table[key >> page_log2] : -1;
    };
    float k_sc = 0.f, v_sc = 0.f;
    auto issue = [&](int i, int id) {
      const int n = used + i, key = run_key(i), st = n % kStages;
      if (kRowWarps > 1 && n >= kStages)
        ok = __all_sync(0xffffffffu, mbar_wait(&my_empty[st], static_cast<uint32_t>(n / kStages - 1) & 1u, a.status));
      if (!ok) return;
      bool mine = lane < per_tile && key < key1;
      if (mine && (id < 0 || id >= c.n_pages)) {
        record_error(a.status, SO101_ERR_PAGES);
        mine = false;
      }
      issued = used + i + 1;
      const int runs = __popc(__ballot_sync(0xffffffffu, mine));
      const uint32_t bytes = static_cast<uint32_t>(GRAN * HD);
      if (lane == 0) mbar_arrive_expect_tx(&my_bars[st], 2u * bytes * runs);
      __syncwarp();
      k_sc = v_sc = 0.f;
      if (mine) {
        const long long off = kv_code_at(c, a.layer, id, head) + (key & (c.page - 1)) * HD;
        const uint32_t dst = smem_u32(my_ring + st * 2 * kTile) + lane * bytes;
        bulk_load(dst, c.k + off, bytes, &my_bars[st]);
        bulk_load(dst + kTile, c.v + off, bytes, &my_bars[st]);
        const long long sc = kv_scale_at(c, a.layer, id, head);
        k_sc = c.k_scale[sc];
        v_sc = c.v_scale[sc];
      }
    };
    auto put_scales = [&](int i) {
      const int st = (used + i) % kStages;
      if (lane < per_tile) {
        my_scales[st * 2 * Cfg::kMaxPages + lane] = k_sc;
        my_scales[st * 2 * Cfg::kMaxPages + Cfg::kMaxPages + lane] = v_sc;
      }
      __syncwarp();
      if (kRowWarps > 1 && lane == 0) mbar_arrive(&my_bars[st]);
    };
    int next_id = -1;
    if (roww == 0) {
      next_id = page_of(0);
      for (int i = 0; i < Cfg::kAhead && i < tiles; ++i) {
        const int id = next_id;
        next_id = page_of(i + 1);
        if (ok) issue(i, id);
        if (ok) put_scales(i);
      }
    }

    // ---- this warp's query rows g and g + 8, dims 16 t .. 16 t + 15 of each 64, as f16 fragments
    const int wrow = tile_row + roww * 16;
    uint32_t qf[kQK][4];
    float factor[2] = {0.f, 0.f};  // S to log2 units, without the page's scale
    float q_sum[2] = {0.f, 0.f};   // what the 128 adds to S
    int vis[2] = {0, 0};  // keys [0, vis) are visible to the row
    int vis_low = 0x7FFFFFFF;  // the fewest of this lane's rows (padding rows may hold anything)
    {
      float x[2][kHalves][16];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = wrow + g + 8 * i;
        const bool live = i < kHalfRows && r < rows;
        const int tok = live ? r / a.group : 0;
        vis[i] = !live ? 0 : a.causal ? max(0, min(len, len - q_len + tok + 1)) : len;
        if (live) vis_low = min(vis_low, vis[i]);
        const __nv_bfloat16* qr = a.q + (row0 + tok) * a.ldq + (head * a.group + (live ? r % a.group : 0)) * HD;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 16; e += 8) {
            const uint4 u =
                live ? __ldg(reinterpret_cast<const uint4*>(qr + 64 * h + 16 * t + e)) : make_uint4(0, 0, 0, 0);
            const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 f = __bfloat1622float2(b[w]);
              x[i][h][e + 2 * w] = f.x;
              x[i][h][e + 2 * w + 1] = f.y;
            }
          }
        if (i < kHalfRows && a.cos) {
          // the partner of dim d is d + HD / 2: another half of this thread's (HD 128), or the same
          // place of the thread two lanes on (HD 64)
          const long long pos = static_cast<long long>(row0 + tok) * (HD / 2);
          const float* cs = a.cos + pos + (HD == 128 ? 16 * t : 16 * (t & 1));
          const float* sn = a.sin + pos + (HD == 128 ? 16 * t : 16 * (t & 1));
#pragma unroll
          for (int e = 0; e < 16; e += 4) {
            const float4 c4 = __ldg(reinterpret_cast<const float4*>(cs + e));
            const float4 s4 = __ldg(reinterpret_cast<const float4*>(sn + e));
            const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
            for (int z = 0; z < 4; ++z) {
              const float u = x[i][0][e + z];
              if (HD == 128) {
                const float w = x[i][kHalves - 1][e + z];
                x[i][0][e + z] = __fsub_rn(__fmul_rn(u, cv[z]), __fmul_rn(w, sv[z]));
                x[i][kHalves - 1][e + z] = __fadd_rn(__fmul_rn(w, cv[z]), __fmul_rn(u, sv[z]));
              } else {
                const float w = __shfl_xor_sync(0xffffffffu, u, 2);
                x[i][0][e + z] = t < 2 ? __fsub_rn(__fmul_rn(u, cv[z]), __fmul_rn(w, sv[z]))
                                       : __fadd_rn(__fmul_rn(u, cv[z]), __fmul_rn(w, sv[z]));
              }
            }
          }
        }
        // the row's largest exponent: x / 2^e is below 2
        uint32_t big = 0u;
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 16; ++e) big = max(big, __float_as_uint(x[i][h][e]) & 0x7FFFFFFFu);
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        const uint32_t ef = min(max(big >> 23, 1u), 253u);
        const float down = __uint_as_float((254u - ef) << 23);
        factor[i] = __uint_as_float(ef << 23) * a.scale_log2 * (1.f / kCode);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[i][h][e] *= down;
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          qf[4 * h + s][0] = f16x2(x[0][h][4 * s], x[0][h][4 * s + 2]);
          qf[4 * h + s][1] = f16x2(x[1][h][4 * s], x[1][h][4 * s + 2]);
          qf[4 * h + s][2] = f16x2(x[0][h][4 * s + 1], x[0][h][4 * s + 3]);
          qf[4 * h + s][3] = f16x2(x[1][h][4 * s + 1], x[1][h][4 * s + 3]);
        }
      float sums[4];
      mma_16816_first(sums, qf[0], kOnes, kOnes);
#pragma unroll
      for (int k = 1; k < kQK; ++k) mma_16816(sums, qf[k], kOnes, kOnes);
#pragma unroll
      for (int i = 0; i < kHalfRows; ++i) q_sum[i] = sums[2 * i] * 128.f * kCode;
    }

    float o[kHalves][8][4];
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[h][n][e] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (int i = 0; i < tiles; ++i) {
      const int st = (used + i) % kStages;
      const bool more = ok && roww == 0 && i + Cfg::kAhead < tiles;
      if (more) {
        const int id = next_id;
        next_id = page_of(i + Cfg::kAhead + 1);
        issue(i + Cfg::kAhead, id);
      }
      // after a wait that ran out the loop goes on without loads or waits, so that the CTA's warps still
      // meet; the result is void and the status word says so
      if (ok) ok = mbar_wait(&my_bars[st], static_cast<uint32_t>((used + i) / kStages) & 1u, a.status);
      ok = __all_sync(0xffffffffu, ok);
      if (wrow >= rows) {  // padding rows only
        if (more && ok) put_scales(i + Cfg::kAhead);
        if (kRowWarps > 1 && lane == 0) mbar_arrive(&my_empty[st]);
        continue;
      }
      const uint8_t* kt = my_ring + st * 2 * kTile;
      const uint8_t* vt = kt + kTile;
      const float* ks = my_scales + st * 2 * Cfg::kMaxPages;
      const float* vs = ks + Cfg::kMaxPages;
      const int tile_key = key0 + (i * kRings + ring) * kKeys;

      // S: key of (n tile j, column 2 t + e) = 8 j + 4 e + t
      float s[kNT][4];
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const uint8_t* row = kt + (8 * j + 4 * (g & 1) + (g >> 1)) * HD + 16 * t;
#pragma unroll
        for (int h = 0; h < kHalves; ++h) {
          const uint4 u = *reinterpret_cast<const uint4*>(row + 64 * h);
          const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (h + k == 0) mma_16816_first(s[j], qf[0], codes_even(w[0]), codes_odd(w[0]));
            else mma_16816(s[j], qf[4 * h + k], codes_even(w[k]), codes_odd(w[k]));
          }
        }
      }
      // logits in units of log2; masked by the key's place where the tile passes what a row sees
#pragma unroll
      for (int j = 0; j < kNT; ++j) {
        const float sk = ks[8 * j / GRAN];
        float mul[2], add[2];  // (S - q_sum) * factor * scale
#pragma unroll
        for (int r = 0; r < kHalfRows; ++r) {
          mul[r] = sk * factor[r];
          add[r] = -q_sum[r] * mul[r];
        }
#pragma unroll
        for (int e = 0; e < 2 * kHalfRows; ++e) s[j][e] = fmaf(s[j][e], mul[e >> 1], add[e >> 1]);
      }
      if (__any_sync(0xffffffffu, tile_key + kKeys > vis_low)) {
#pragma unroll
        for (int j = 0; j < kNT; ++j)
#pragma unroll
          for (int e = 0; e < 2 * kHalfRows; ++e)
            if (tile_key + 8 * j + 4 * (e & 1) + t >= vis[e >> 1]) s[j][e] = -INFINITY;
      }
      float alpha[2] = {1.f, 1.f}, sub[2];
#pragma unroll
      for (int r = 0; r < kHalfRows; ++r) {
        float mx = m[r];
#pragma unroll
        for (int j = 0; j < kNT; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * r], s[j][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        sub[r] = mx == -INFINITY ? 0.f : mx;  // a row that has seen no key yet
        alpha[r] = ex2(m[r] - sub[r]);
        m[r] = mx;
#pragma unroll
        for (int j = 0; j < kNT; ++j) {
          s[j][2 * r] = ex2(s[j][2 * r] - sub[r]);
          s[j][2 * r + 1] = ex2(s[j][2 * r + 1] - sub[r]);
        }
        l[r] *= alpha[r];
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
#pragma unroll
          for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 2 * kHalfRows; ++e) o[h][n][e] *= alpha[e >> 1];
      }
      // O += s_v (P V), page by page; a page that the row does not see adds nothing (its scale may be NaN)
      uint32_t pa[kKeys / 16][4];
#pragma unroll
      for (int k = 0; k < kKeys / 16; ++k) {
        pa[k][0] = f16x2(s[2 * k][0], s[2 * k][1]);
        pa[k][1] = kHalfRows == 2 ? f16x2(s[2 * k][2], s[2 * k][3]) : 0u;
        pa[k][2] = f16x2(s[2 * k + 1][0], s[2 * k + 1][1]);
        pa[k][3] = kHalfRows == 2 ? f16x2(s[2 * k + 1][2], s[2 * k + 1][3]) : 0u;
      }
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        float d[8][4], sums[4];
#pragma unroll
        for (int k = 0; k < kKeys / 16; ++k) {
          uint2 u[4];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            u[x] = *reinterpret_cast<const uint2*>(vt + (16 * k + 4 * x + t) * HD + 64 * h + 8 * g);
          const bool begins = 16 * k % GRAN == 0, ends = 16 * (k + 1) % GRAN == 0;
          auto mma = [&](float (&acc)[4], uint32_t b0, uint32_t b1) {
            if (begins) mma_16816_first(acc, pa[k], b0, b1);
            else mma_16816(acc, pa[k], b0, b1);
          };
          if (h == 0) mma(sums, kOnes, kOnes);
#pragma unroll
          for (int n = 0; n < 8; n += 2) {
            // dims 8 g + n, 8 g + n + 1 of keys x = 0, 1 and 2, 3: two rows' bytes side by side
            const uint32_t pick = (n & 2) ? 0x7632u : 0x5410u;
            const uint32_t p0 = n < 4 ? __byte_perm(u[0].x, u[1].x, pick) : __byte_perm(u[0].y, u[1].y, pick);
            const uint32_t p1 = n < 4 ? __byte_perm(u[2].x, u[3].x, pick) : __byte_perm(u[2].y, u[3].y, pick);
            mma(d[n], centred(codes_even(p0)), centred(codes_even(p1)));
            mma(d[n + 1], centred(codes_odd(p0)), centred(codes_odd(p1)));
          }
          if (ends) {  // the page ends here
            const int first = tile_key + 16 * k / GRAN * GRAN;
            const float sv = vs[16 * k / GRAN];
#pragma unroll
            for (int r = 0; r < kHalfRows; ++r) {
              const float f = first < vis[r] ? sv * (1.f / kCode) : 0.f;
              if (h == 0) l[r] += sums[2 * r];
#pragma unroll
              for (int n = 0; n < 8; ++n) {
                o[h][n][2 * r] = fmaf(d[n][2 * r], f, o[h][n][2 * r]);
                o[h][n][2 * r + 1] = fmaf(d[n][2 * r + 1], f, o[h][n][2 * r + 1]);
              }
            }
          }
        }
      }
      if (more && ok) put_scales(i + Cfg::kAhead);
      __syncwarp();  // the stage is read: a later load may fill it
      if (kRowWarps > 1 && lane == 0) mbar_arrive(&my_empty[st]);
    }
    if (!ok && roww == 0)  // copies in flight land before the ring's memory is used otherwise
      for (int n = max(0, issued - kStages); n < issued; ++n)
        mbar_wait(&my_bars[n % kStages], static_cast<uint32_t>(n / kStages) & 1u, a.status);
    used += tiles;
    __syncthreads();  // every ring's tiles have landed and been read

    // ---- join the rings: O, and (m, l), of each warp into shared memory (over the rings' buffers)
    float* part = reinterpret_cast<float*>(smem);
    float2* part_ml = reinterpret_cast<float2*>(part + kPgWarps * 16 * Cfg::kJoinRow);
#pragma unroll
    for (int r = 0; r < kHalfRows; ++r) {
      float* row = part + (warp * 16 + g + 8 * r) * Cfg::kJoinRow;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int n = 0; n < 8; n += 4)
            *reinterpret_cast<float4*>(row + 64 * h + 16 * t + 8 * x + n) =
                make_float4(o[h][n][2 * r + x], o[h][n + 1][2 * r + x], o[h][n + 2][2 * r + x], o[h][n + 3][2 * r + x]);
      if (t == 0) part_ml[warp * 16 + g + 8 * r] = make_float2(m[r], l[r]);
    }
    __syncthreads();
    // row r of the tile lies in the row warp r / 16 of every ring; a thread takes four dims of a row
    const int tile_rows = min(rows - tile_row, ROWS);
    constexpr int kQuads = HD / 4;
    auto put = [&](int r, int d, const float4& y, float ll) {
      const float inv = ll == 0.f ? 0.f : 1.f / ll;  // a row that sees nothing: O is 0
      const int tok = (tile_row + r) / a.group, hq = head * a.group + (tile_row + r) % a.group;
      const __nv_bfloat162 lo = __floats2bfloat162_rn(y.x * inv, y.y * inv), hi = __floats2bfloat162_rn(y.z * inv, y.w * inv);
      *reinterpret_cast<uint2*>(a.o + (row0 + tok) * a.ldo + hq * HD + d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    };
    float* mine = a.partials + (2LL * blockIdx.x + (part_no == 0 ? 1 : 0)) * Cfg::kSlot;
    for (int e = threadIdx.x; e < tile_rows * kQuads; e += kPgThreads) {
      const int r = e / kQuads, d = e % kQuads * 4;
      float2 ml[kRings];
      float mm = -INFINITY;
#pragma unroll
      for (int k = 0; k < kRings; ++k) {
        ml[k] = part_ml[k * kRowWarps * 16 + r];
        mm = fmaxf(mm, ml[k].x);
      }
      const float base = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < kRings; ++k) {
        const float w = ex2(ml[k].x - base);
        ll = fmaf(w, ml[k].y, ll);
        add_scaled(y, w, *reinterpret_cast<const float4*>(part + (k * kRowWarps * 16 + r) * Cfg::kJoinRow + d));
      }
      if (parts == 1) {
        put(r, d, y, ll);
      } else {
        *reinterpret_cast<float4*>(mine + r * HD + d) = y;
        if (d == 0) *reinterpret_cast<float2*>(mine + ROWS * HD + 2 * r) = make_float2(mm, ll);
      }
    }
    if (parts > 1) {
      // the last of the problem's CTAs to arrive joins their parts in order: part k > 0 lies in CTA
      // cta_first + k's first slot, part 0 in its CTA's second
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0) shared[0] = atomicAdd(a.tickets + cta_first, 1) == parts - 1 ? 1 : 0;
      __syncthreads();
      if (shared[0]) {
        __threadfence();
        auto part_at = [&](int k) { return a.partials + (2LL * (cta_first + k) + (k == 0 ? 1 : 0)) * Cfg::kSlot; };
        // per row the largest maximum and the sum: a warp per row, its lanes over the parts
        for (int r = warp; r < tile_rows; r += kPgWarps) {
          float mm = -INFINITY, ll = 0.f;
          for (int k = lane; k < parts; k += 32) {
            const float2 x = __ldcg(reinterpret_cast<const float2*>(part_at(k) + ROWS * HD + 2 * r));
            const float mn = fmaxf(mm, x.x), base = mn == -INFINITY ? 0.f : mn;
            ll = ll * ex2(mm - base) + x.y * ex2(x.x - base);
            mm = mn;
          }
          float top = mm;
#pragma unroll
          for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          ll *= ex2(mm - (top == -INFINITY ? 0.f : top));
#pragma unroll
          for (int d = 16; d; d >>= 1) ll += __shfl_xor_sync(0xffffffffu, ll, d);
          if (lane == 0) part_ml[r] = make_float2(top == -INFINITY ? 0.f : top, ll);
        }
        __syncthreads();
        // all loads of sixteen parts in flight together
        for (int e = threadIdx.x; e < tile_rows * kQuads; e += kPgThreads) {
          const int r = e / kQuads, d = e % kQuads * 4;
          const float2 ml = part_ml[r];
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int k0 = 0; k0 < parts; k0 += 16) {
            float4 v[16];
            float mk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float* from_part = part_at(min(k0 + k, parts - 1));
              v[k] = __ldcg(reinterpret_cast<const float4*>(from_part + r * HD + d));
              mk[k] = __ldcg(from_part + ROWS * HD + 2 * r);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k)
              if (k0 + k < parts) add_scaled(y, ex2(mk[k] - ml.x), v[k]);
          }
          put(r, d, y, ml.y);
        }
        if (threadIdx.x == 0) a.tickets[cta_first] = 0;
      }
    }
    // the join's reads and writes come before the copies of the next problem's tiles
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
  }
}

// CTAs that fit the GPU at once, looked up once per device (the kernel's registers and shared memory
// decide how many an SM takes).
template <int HD, int ROWS, int GRAN>
int launch_pages(const PagesArgs& a, int64_t most_steps, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream) {
  using Cfg = PgCfg<HD, ROWS>;
  static std::atomic<int> resident[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return SO101_ERR_DRIVER;
  int full = resident[dev].load();
  if (!full) {
    cudaError_t e = cudaFuncSetAttribute(attention_pages_kernel<HD, ROWS, GRAN>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         Cfg::kSmem);
    int per_sm = 0, sms = 0;
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, attention_pages_kernel<HD, ROWS, GRAN>, kPgThreads, Cfg::kSmem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return launch_error(e);
    if (per_sm < 1) return SO101_ERR_DRIVER;
    resident[dev].store(full = per_sm * sms);
  }
  // two slots of partial rows and a ticket per CTA
  const int64_t slots = workspace_bytes / (2LL * Cfg::kSlot * 4);
  int64_t grid = most_steps < full ? most_steps : full;
  if (grid > slots) grid = slots;
  if (grid > n_tickets) grid = n_tickets;
  if (grid < 1) return SO101_ERR_WORKSPACE;
  return launch_kernel(attention_pages_kernel<HD, ROWS, GRAN>, dim3(static_cast<unsigned>(grid)), dim3(kPgThreads), Cfg::kSmem,
                       stream, a);
}

template <int HD, int ROWS>
int dispatch_pages(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream) {
  using Cfg = PgCfg<HD, ROWS>;
  // steps of all problems, at most (they are counted in 32 bits)
  const int64_t tiles = (static_cast<int64_t>(a.max_q) * a.group + ROWS - 1) / ROWS;
  const int64_t problems = tiles * a.c.n_kv * a.n_seqs;
  const int64_t capacity = static_cast<int64_t>(a.c.max_pages) * a.c.page;
  const int64_t most = problems * ((capacity + Cfg::kStep - 1) / Cfg::kStep);
  if (problems > (1 << 24) || most > (1LL << 30)) return SO101_ERR_ARG;
  if (a.c.page == 16) return launch_pages<HD, ROWS, 16>(a, most, workspace_bytes, n_tickets, stream);
  if (a.c.page == 32 || Cfg::kKeys == 32) return launch_pages<HD, ROWS, 32>(a, most, workspace_bytes, n_tickets, stream);
  return launch_pages<HD, ROWS, Cfg::kKeys>(a, most, workspace_bytes, n_tickets, stream);
}

// rows per CTA: as few as hold a sequence's, up to 64, so that one pass over the keys serves them all (more rows go to
// the tcgen05 kernel)
template <int HD>
int attention_pages_run(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream) {
  const int64_t most_rows = static_cast<int64_t>(a.max_q) * a.group;
  if (most_rows <= 8) return dispatch_pages<HD, 8>(a, workspace_bytes, n_tickets, stream);
  if (most_rows <= 16) return dispatch_pages<HD, 16>(a, workspace_bytes, n_tickets, stream);
  if (most_rows <= 32) return dispatch_pages<HD, 32>(a, workspace_bytes, n_tickets, stream);
  return dispatch_pages<HD, 64>(a, workspace_bytes, n_tickets, stream);
}

}  // namespace so101
