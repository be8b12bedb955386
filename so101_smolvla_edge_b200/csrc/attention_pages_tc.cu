// Attention over the 8-bit pages on tcgen05, for many query rows per sequence and kv head (a chunk of action
// tokens, the rest of a prompt): the arithmetic of attention_pages.cuh in the structure of attention_packed.cu.
//
// A work item is a part of a problem's keys (the plan of attention_pages.cuh, in steps of 128) for up to 256 stacked
// query rows of one list entry and kv head, in two groups of 128. One CTA per SM walks its items:
//   warp 0      the pages: codes of 128 keys by bulk copies into a ring, their scales beside them
//   warps 1, 2  the MMAs of group 0 / 1 in f16: S = Q K^T -> TMEM, O += P V with P read from TMEM
//   warp 3      the items
//   warps 4-7   the queries: rotated in fp32, scaled by a power of two per row, rounded to f16
//   warps 8-11  per tile the codes as f16 (exact) into swizzled K and V tiles, once for all rows of the item
//   warps 12-27 with them the first item's queries; the softmax, two threads per row, and the result
// A page's key scale multiplies its 16-key groups of S. Its value scale goes into the V operand: code * 2^(8 + e - E)
// is exact in f16 for e, the page's exponent, within 32 of E, the largest of the item's pages, and 2^(E - 8) comes off
// with 1 / l. Items whose pages are further apart (or hold scales that are no power of two) go key by key in fp32.
// A page whose value scale is NaN multiplies S by NaN, so that rows that do not see it stay as they are;
// masked places are cut before the scales come in, and groups of them keep clear of it. P is 2^(x - m + 7): below
// 2^15, and no weight down to 2^-21 of the largest is rounded to fewer than 11 bits.
// K and V operands hold the dims of each four in the order 0, 2, 1, 3 (what a mask and a shift of a code word give);
// the queries are written, and O is read, in that order.
// Measured (us, the mma.sync kernel's in parentheses): 64 chunks of 50 tokens over 291 keys, 15 on 5 heads of 64, 39
// (45); over 2000 keys 123 (213); 64 x 128 tokens over 2000 keys, 32 on 8 heads of 128, 549 (1571); 64 x 24 tokens
// over 291 keys, 72 rows each, 34 (38). Up to 64 rows the mma.sync kernel reads the keys once too and is faster (48
// rows over 291 keys 21, here 33). Few tiles: the latency of a CTA's two or three items bounds it, 8 us of start and
// 9 us each; many: the exponentials and issue slots of the schedulers that hold two of the five row quarters.
#include <atomic>
#include <cmath>

#include "attention_pages.cuh"
#include "tc_attn.cuh"

namespace so101 {

constexpr int kPtRows = 128, kPtKeys = 128, kPtThreads = 896;
constexpr float kPtStaleMax = 8.f, kPtHead = 7.f;  // log2: a stale maximum's slack, P's factor
constexpr int kPtGroups = kPtKeys / 16;            // 16-key groups of a tile (no page is shorter)
constexpr int kPtSlots = 8;                        // tiles whose scales are held
constexpr int kPtItems = 8;

template <int HD>
struct PtCfg {
  static constexpr int kHalves = HD / 64;
  static constexpr int kTile = kPtRows * 128;          // 128 rows x 64 f16 dims
  static constexpr int kStage = kHalves * kTile;       // an operand tile of K or V; a group's queries
  static constexpr int kRaw = 2 * kPtKeys * HD;        // codes of K and V
  static constexpr int kQBufs = HD == 64 ? 2 : 1;
  static constexpr int kStages = HD == 64 ? 2 : 1;     // operand tiles of K and of V
  static constexpr int kRaws = HD == 64 ? 3 : 2;
  static constexpr bool kAlias = HD == 128;            // P in the place of S
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kQBufs * 2 * kStage;
  static constexpr int kOffV = kOffK + kStages * kStage;
  static constexpr int kOffRaw = kOffV + kStages * kStage;
  static constexpr int kOffSwap = kOffRaw + kRaws * kRaw;   // [2][2 groups][2 halves][128] floats between half rows
  static constexpr int kOffFactor = kOffSwap + 4096;        // [kPtItems][256] floats: what scaling a query took off
  // [kPtSlots][2][kPtGroups]: key scale, 2^(8 + e - E) twice
  static constexpr int kOffScale = kOffFactor + kPtItems * 1024;
  static constexpr int kOffBar = kOffScale + kPtSlots * 2 * kPtGroups * 4;
  static constexpr int kSlot = 32 * (HD + 2);               // floats of a part of 32 rows: O, then their (m, l)
  static constexpr int kSmem = kOffBar + 1024 + 1024;
  static constexpr uint32_t kColS = 0, kColP = HD == 64 ? 128 : 0, kColO = HD == 64 ? 192 : 128, kGroupCols = 256;
  static constexpr int kRegsLoad = 40, kRegsQuery = 64, kRegsOps = 48, kRegsSoft = 88;
  // together 64512: the 72 each that the threads start with
  static constexpr int kItemReaders = 1 + 2 + 4 + 4 + 16;  // reads of each item: codes, MMAs, queries, operands, softmax
};
static_assert(kPtSlots >= PtCfg<64>::kRaws + PtCfg<64>::kStages && kPtSlots >= PtCfg<128>::kRaws + PtCfg<128>::kStages,
              "a tile's scales are written while operands up to kRaws + kStages - 1 tiles back may be in use");
static_assert(PtCfg<64>::kSmem <= 232448 && PtCfg<128>::kSmem <= 232448, "227 KB of shared memory per CTA");

struct PtItem {
  int row0, row_first, rows, kvh;  // the entry's first packed row; its stacked rows; 0 rows: no more items
  int seq, len, n_q, exp_max;      // sequence, cached tokens, query tokens, E
  int from, to;                    // its key tiles
  int parts, part, cta_first;      // of the problem: items, which this is, the CTA of the first
  int alone;                       // key by key
  int tok, lead;                   // token and head of row row_first
  int tiles[2];                    // key tiles that some row of the group sees
};

// Four codes as f16: (bytes 0, 2) and (bytes 1, 3), by the byte under the exponent of 1024, less 1024 + 128.
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t& even, uint32_t& odd) {
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(even) : "r"(w), "r"(0x00FF00FFu), "r"(0x64806480u));
  asm("lop3.b32 %0, %1, %2, %3, 0x6A;" : "=r"(odd) : "r"(w >> 8), "r"(0x00FF00FFu), "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(even) : "r"(0x64806480u));
  asm("sub.rn.f16x2 %0, %0, %1;" : "+r"(odd) : "r"(0x64806480u));
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// Row r of the item's: its token and head.
__device__ __forceinline__ void pt_row(const PagesArgs& a, const PtItem& it, int r, int& tok, int& head) {
  const int x = it.lead + r, t = a.group == 1 ? x : __umulhi(x, a.group_inv);
  tok = it.tok + t;
  head = it.kvh * a.group + x - t * a.group;
}

// keys [0, seen) are visible to token `tok` of the item's entry
__device__ __forceinline__ int pt_seen(const PtItem& it, int tok, int causal) {
  return causal ? max(0, min(it.len, it.len - it.n_q + tok + 1)) : it.len;
}

__device__ __forceinline__ uint32_t timer_low() {  // (4.3 s around)
  uint32_t t;
  asm volatile("mov.u32 %0, %globaltimer_lo;" : "=r"(t));
  return t;
}

// Row r of the item over the item's keys in fp32, key by key, by a whole warp (lane l: dims l, l + 32, ...):
// o / l, and the logarithm of l in m (-infinity where it sees none). The time goes to `alive` every 256 keys.
template <int HD>
__device__ __forceinline__ void pt_row_alone(const PagesArgs& a, const PtItem& it, int r, float (&o)[HD / 32], float& m,
                                             uint32_t* alive) {
  const KvPages& c = a.c;
  const int lane = threadIdx.x & 31;
  int tok, head;
  pt_row(a, it, r, tok, head);
  constexpr int N = HD / 32;
  float q[N];
  const __nv_bfloat16* qr = a.q + (it.row0 + tok) * a.ldq + head * HD;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 32 * i;
    q[i] = __bfloat162float(qr[d]);
    if (a.cos) {
      const long long p = static_cast<long long>(it.row0 + tok) * (HD / 2) + d % (HD / 2);
      const float y = __bfloat162float(qr[(d + HD / 2) % HD]);
      q[i] = d < HD / 2 ? q[i] * a.cos[p] - y * a.sin[p] : q[i] * a.cos[p] + y * a.sin[p];
    }
    o[i] = 0.f;
  }
  m = -INFINITY;
  float l = 0.f;
  const int end = min(pt_seen(it, tok, a.causal), it.to * kPtKeys);
  const int* table = c.table + static_cast<long long>(it.seq) * c.max_pages;
  for (int j = it.from * kPtKeys; j < end; ++j) {
    if (lane == 0 && j % 256 == 0) *reinterpret_cast<volatile uint32_t*>(alive) = timer_low();
    const int id = table[j / c.page];
    if (id < 0 || id >= c.n_pages) {
      record_error(a.status, SO101_ERR_PAGES);
      continue;
    }
    const long long sc = kv_scale_at(c, a.layer, id, it.kvh), at = kv_code_at(c, a.layer, id, it.kvh) + j % c.page * HD;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], static_cast<float>(c.k[at + lane + 32 * i]), s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= c.k_scale[sc] * a.scale_log2;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = ex2(m - base), p = ex2(s - base), ps = p * c.v_scale[sc];
    m = mn;
    l = fmaf(l, alpha, p);
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = fmaf(o[i], alpha, ps * static_cast<float>(c.v[at + lane + 32 * i]));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) o[i] = l == 0.f ? 0.f : o[i] / l;
  m = l == 0.f ? -INFINITY : m + log2f(l);
}

// 4 x 4 pieces of four lanes' rows transposed, so that a store covers eight rows of 64 bytes, not 32 of 16.
__device__ __forceinline__ void transpose4(uint4 (&y)[4]) {
  const int lane = threadIdx.x & 31;
  auto swap = [&](uint4& lo, uint4& hi, int d) {  // the lane with bit d keeps hi, the other lo
    const bool up = lane & d;
    uint4 give = up ? lo : hi;
    give.x = __shfl_xor_sync(0xffffffffu, give.x, d);
    give.y = __shfl_xor_sync(0xffffffffu, give.y, d);
    give.z = __shfl_xor_sync(0xffffffffu, give.z, d);
    give.w = __shfl_xor_sync(0xffffffffu, give.w, d);
    (up ? lo : hi) = give;
  };
  swap(y[0], y[1], 1);
  swap(y[2], y[3], 1);
  swap(y[0], y[2], 2);
  swap(y[1], y[3], 2);
}

// As mbar_wait (2 s of the timer), but not while the time in `alive` is younger than that: items that go key by key note
// it there, and can hold the others up for longer. (The differences are of 32 bits, 4.3 s: at some time in each turn
// both are past the limit. The timer is left alone in short waits: 39.1 us for 64 chunks of 50 tokens, 39.6 with it
// looked at every 256 polls in a loop that tells the first look by its number, 38.6 with polls counted and no timer.)
__device__ __forceinline__ bool pt_wait(uint64_t* bar, uint32_t parity, int* status, const uint32_t* alive) {
  uint32_t t0 = 0;
#pragma unroll 1
  for (uint32_t i = 0; !mbar_try_wait(bar, parity); ++i) {
    if (i != 4096u) continue;
    i = 0;
    const uint32_t other = *reinterpret_cast<const volatile uint32_t*>(alive), now = timer_low();
    if (t0 == 0u) {
      t0 = now | 1u;
    } else if (now - t0 > kWaitLimitNs && now - other > kWaitLimitNs) {
      record_error(status, SO101_ERR_TIMEOUT);
      return false;
    }
  }
  return true;
}

// The largest of three (NaN only if all are).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int HD>
__global__ void __launch_bounds__(kPtThreads, 1) attention_pages_tc_kernel(const PagesArgs a) {
  using Cfg = PtCfg<HD>;
  constexpr int kStages = Cfg::kStages, kQBufs = Cfg::kQBufs, kRaws = Cfg::kRaws;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  PtItem* items = reinterpret_cast<PtItem*>(smem + Cfg::kOffBar);
  uint64_t* item_full = reinterpret_cast<uint64_t*>(items + kPtItems);
  uint64_t* item_empty = item_full + kPtItems;
  uint64_t* q_full = item_empty + kPtItems;
  uint64_t* q_empty = q_full + kQBufs;
  uint64_t* r_full = q_empty + kQBufs;     // [kRaws] codes landed, scales written
  uint64_t* r_empty = r_full + kRaws;      // [kRaws] codes converted
  uint64_t* k_full = r_empty + kRaws;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;    // [2] per group, as the rest
  uint64_t* s_free = s_full + 2;
  uint64_t* p_full = s_free + 2;
  uint64_t* o_full = p_full + 2;
  uint64_t* o_free = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_free + 2);
  int* last = reinterpret_cast<int*>(tmem_slot + 1);  // [8] whether two warps' part came last
  uint32_t* alive = reinterpret_cast<uint32_t*>(last + 8);  // when a warp last went on key by key
  static_assert(kPtItems * sizeof(PtItem) + (2 * kPtItems + 4 + 6 + 8 + 10) * 8 + 40 <= 1024, "barrier region");
  float* factors = reinterpret_cast<float*>(smem + Cfg::kOffFactor);
  float* scales = reinterpret_cast<float*>(smem + Cfg::kOffScale);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const KvPages& c = a.c;
  if (warp == 0) {
    if (lane < kPtItems) {
      mbar_init(&item_full[lane], 1);
      mbar_init(&item_empty[lane], Cfg::kItemReaders);
    }
    if (lane < kQBufs) {
      mbar_init(&q_full[lane], 20);
      mbar_init(&q_empty[lane], 2);
    }
    if (lane < kRaws) {
      mbar_init(&r_full[lane], 2);  // the copies and the scales
      mbar_init(&r_empty[lane], 4);
    }
    if (lane < kStages) {
      mbar_init(&k_full[lane], 4);
      mbar_init(&k_empty[lane], 2);
      mbar_init(&v_full[lane], 4);
      mbar_init(&v_empty[lane], 2);
    }
    if (lane < 2) {
      mbar_init(&s_full[lane], 1);
      mbar_init(&s_free[lane], 8);
      mbar_init(&p_full[lane], 8);
      mbar_init(&o_full[lane], 1);
      mbar_init(&o_free[lane], 8);
    }
    if (lane == 0) *alive = timer_low();
    fence_mbar_init();
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
  const PagesPlan plan = pages_plan<kPtKeys, 2 * kPtRows, kPtThreads>(a, reinterpret_cast<int*>(smem + Cfg::kOffSwap));
  __syncthreads();

  auto wait = [&](uint64_t* b, int n) {  // the n-th use (from 0) of a barrier; the same outcome for the whole warp
    return __all_sync(0xffffffffu, pt_wait(b, static_cast<uint32_t>(n) & 1u, a.status, alive));
  };
  auto item_at = [&](int i) {
    PtItem it = {};
    if (wait(&item_full[i % kPtItems], i / kPtItems)) it = items[i % kPtItems];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[i % kPtItems]);
    return it;
  };
  auto tiles_all = [](const PtItem& it) { return max(it.tiles[0], it.tiles[1]); };

  // the queries of item i (number `with` of those with tiles) by warp w of n_w
  auto put_queries = [&](const PtItem& it, int i, int with, int w, int n_w) {
    constexpr int kPairs = HD / 16;       // lanes of a row: 8 dims and their partners HD / 2 later each
    constexpr int kRowsAt = 32 / kPairs;  // rows of a warp at a time
    const int qb = with % kQBufs;
    const int rows = (min(it.rows, 2 * kPtRows) + 31) / 32 * 32, p = lane % kPairs;
    for (int r0 = w * kRowsAt; r0 < rows; r0 += n_w * kRowsAt) {
      const int r = r0 + lane / kPairs;
      float x[2][8];
#pragma unroll
      for (int e = 0; e < 8; ++e) x[0][e] = x[1][e] = 0.f;
      if (r < it.rows) {
        int tok, head;
        pt_row(a, it, r, tok, head);
        const uint4* qr = reinterpret_cast<const uint4*>(a.q + (it.row0 + tok) * a.ldq + head * HD);
        const uint4 u[2] = {__ldg(qr + p), __ldg(qr + p + kPairs)};
        float4 ang[4] = {};
        if (a.cos) {
          const long long at = static_cast<long long>(it.row0 + tok) * (HD / 2) + 8 * p;
          ang[0] = __ldg(reinterpret_cast<const float4*>(a.cos + at));
          ang[1] = __ldg(reinterpret_cast<const float4*>(a.cos + at + 4));
          ang[2] = __ldg(reinterpret_cast<const float4*>(a.sin + at));
          ang[3] = __ldg(reinterpret_cast<const float4*>(a.sin + at + 4));
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&u[z]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = __bfloat1622float2(b[e]);
            x[z][2 * e] = f.x;
            x[z][2 * e + 1] = f.y;
          }
        }
        if (a.cos) {
          const float* cv = reinterpret_cast<const float*>(ang);
          const float* sv = cv + 8;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = x[0][e], z = x[1][e];
            x[0][e] = __fsub_rn(__fmul_rn(y, cv[e]), __fmul_rn(z, sv[e]));
            x[1][e] = __fadd_rn(__fmul_rn(z, cv[e]), __fmul_rn(y, sv[e]));
          }
        }
      }
      // the row's largest exponent: x / 2^e is below 2
      uint32_t big = 0u;
#pragma unroll
      for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(x[z][e]) & 0x7FFFFFFFu);
#pragma unroll
      for (int d = 1; d < kPairs; d <<= 1) big = max(big, __shfl_xor_sync(0xffffffffu, big, d));
      const uint32_t ef = min(max(big >> 23, 1u), 253u);
      const float down = __uint_as_float((254u - ef) << 23);
      if (p == 0) factors[i % kPtItems * 256 + r] = __uint_as_float(ef << 23) * a.scale_log2;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const float* y = x[z];
        const uint4 packed = make_uint4(f16x2(y[0] * down, y[2] * down), f16x2(y[1] * down, y[3] * down),
                                   f16x2(y[4] * down, y[6] * down), f16x2(y[5] * down, y[7] * down));
        const int piece = p + z * kPairs;
        uint8_t* to = smem + Cfg::kOffQ + (2 * qb + r / kPtRows) * Cfg::kStage + piece / 8 * Cfg::kTile +
                      r % kPtRows * 128 + ((piece % 8 ^ (r & 7)) << 4);
        *reinterpret_cast<uint4*>(to) = packed;
      }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane < 20 / n_w) mbar_arrive(&q_full[qb]);
  };

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsLoad));
    if (warp == 3) {
      // ---- the items: the parts of problems in the CTA's run of steps
      int entry = plan.entry, entry_first = plan.first, at = plan.begin;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        PtItem it = {};
        while (at < plan.end && entry < a.n_seqs) {
          int steps, row_tiles;
          entry_size<kPtKeys, 2 * kPtRows>(a, entry, steps, row_tiles);
          const int entry_end = entry_first + steps * row_tiles * c.n_kv;
          if (at >= entry_end) {
            entry_first = entry_end;
            ++entry;
            continue;
          }
          const int p = (at - entry_first) / steps, p_first = entry_first + p * steps;
          it.kvh = p % c.n_kv;
          it.row_first = p / c.n_kv * 2 * kPtRows;
          it.from = at - p_first;
          it.to = min(steps, plan.end - p_first);
          at = p_first + it.to;
          problem_parts(plan, p_first, steps, it.cta_first, it.parts);
          it.part = static_cast<int>(blockIdx.x) - it.cta_first;
          int n;
          if (!kv_rows(c, a.starts, a.seqs, entry, a.rows, it.seq, it.row0, n, a.status)) continue;
          it.n_q = n;
          if (n > a.max_q) {  // more rows than the host planned for
            if (lane == 0) record_error(a.status, SO101_ERR_PAGES);
            n = a.max_q;
          }
          it.rows = min(2 * kPtRows, n * a.group - it.row_first);
          break;
        }
        if (it.rows > 0) {
          it.len = kv_length(c, it.seq, a.status);
          // exponents of the value scales, the smallest apart (pages of zeros hold it; others with it hold next to nothing)
          int top = 1, low = 255;
          bool odd = false;
          const int* table = c.table + static_cast<long long>(it.seq) * c.max_pages;
          const int end = min(it.to * kPtKeys, it.len);
          for (int key = it.from * kPtKeys + lane * c.page; key < end; key += 32 * c.page) {
            const int id = table[key / c.page];
            if (id < 0 || id >= c.n_pages) continue;
            const float x = c.v_scale[kv_scale_at(c, a.layer, id, it.kvh)];
            if (x != x) continue;
            const int f = static_cast<int>(__float_as_uint(x) >> 23);
            odd = odd || f > 254 || (__float_as_uint(x) & 0x7FFFFF);
            if (f > 1) {
              top = max(top, f);
              low = min(low, f);
            }
          }
          top = __reduce_max_sync(0xffffffffu, top);
          low = __reduce_min_sync(0xffffffffu, low);
          it.exp_max = top - 127;
          it.alone = __any_sync(0xffffffffu, odd) || top - low > 32 ? 1 : 0;
          it.tok = it.row_first / a.group;
          it.lead = it.row_first - it.tok * a.group;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            const int here = min(it.rows - g * kPtRows, kPtRows);
            if (here <= 0 || it.alone) continue;
            int tok, head;
            pt_row(a, it, g * kPtRows + here - 1, tok, head);
            it.tiles[g] = max(0, min(it.to, (pt_seen(it, tok, a.causal) + kPtKeys - 1) / kPtKeys) - it.from);
          }
        }
        if (i >= kPtItems) ok = wait(&item_empty[i % kPtItems], i / kPtItems - 1);
        if (ok && lane == 0) {
          items[i % kPtItems] = it;
          mbar_arrive(&item_full[i % kPtItems]);
        }
        __syncwarp();
        if (it.rows == 0) break;
      }
    } else if (warp == 0) {
      // ---- codes: lane l < 128 / page brings the l-th page's slots of a tile, its scales for 16-key groups
      const int per_tile = kPtKeys / c.page, page_log2 = __ffs(c.page) - 1;
      const uint32_t bytes = static_cast<uint32_t>(c.page * HD);
      int t = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        const PtItem it = item_at(i);
        if (it.rows == 0) break;
        const int n_tiles = tiles_all(it);
        const int* table = c.table + static_cast<long long>(it.seq) * c.max_pages;
        constexpr int kNone = -0x7FFFFFFF;  // no page there
        auto page_of = [&](int j) {
          const int key = (it.from + j) * kPtKeys + (lane << page_log2);
          return j < n_tiles && lane < per_tile && key < it.len ? table[key >> page_log2] : kNone;
        };
        int next = page_of(0);
        for (int j = 0; j < n_tiles && ok; ++j, ++t) {
          const int st = t % kRaws, id = next;
          next = page_of(j + 1);
          const bool mine = id >= 0 && id < c.n_pages;
          if (!mine && id != kNone) record_error(a.status, SO101_ERR_PAGES);
          float ks = 1.f, vs = 0.f;
          if (mine) {
            const long long sc = kv_scale_at(c, a.layer, id, it.kvh);
            ks = c.k_scale[sc];
            vs = c.v_scale[sc];
          }
          if (t >= kRaws) ok = wait(&r_empty[st], t / kRaws - 1);
          if (!ok) break;
          const int runs = __popc(__ballot_sync(0xffffffffu, mine));
          if (lane == 0) mbar_arrive_expect_tx(&r_full[st], 2u * bytes * runs);
          __syncwarp();
          if (mine) {
            const long long at = kv_code_at(c, a.layer, id, it.kvh);
            const uint32_t dst = smem_u32(smem + Cfg::kOffRaw + st * Cfg::kRaw) + lane * bytes;
            bulk_load(dst, c.k + at, bytes, &r_full[st]);
            bulk_load(dst + kPtKeys * HD, c.v + at, bytes, &r_full[st]);
          }
          if (lane < per_tile) {  // by 16 keys (a page is one to four groups)
            float* to = scales + t % kPtSlots * 2 * kPtGroups;
            const bool lost = vs != vs;
            const int x = 8 + static_cast<int>(__float_as_uint(vs) >> 23) - 127 - it.exp_max;
            const uint32_t h = lost || x < -24 ? 0u : x < -14 ? 1u << (x + 24) : static_cast<uint32_t>(x + 15) << 10;
            const uint32_t hh = h << 16 | h;
            for (int y = lane << (page_log2 - 4); y < (lane + 1) << (page_log2 - 4); ++y) {
              to[y] = lost ? vs : ks;
              to[kPtGroups + y] = __uint_as_float(hh);
            }
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&r_full[st]);
        }
      }
      // copies in flight land before the CTA ends, also where a wait ran out
      for (int n = max(0, t - kRaws); n < t; ++n) wait(&r_full[n % kRaws], n / kRaws);
    } else {
      // ---- the MMAs of group g, a warp each; S runs ahead of P V by one tile (as attention_packed.cu)
      const int g = warp - 1;
      constexpr uint32_t kF16 = ~((1u << 7) | (1u << 10));  // f16 operands, not bf16
      constexpr uint32_t ID_S = idesc_attn(kPtKeys, 0) & kF16;
      constexpr uint32_t ID_O = idesc_attn(64, 1) & kF16;
      const uint32_t d0 = tmem + g * Cfg::kGroupCols;
      // Both cursors are in one item: the next is looked for when the last P V of this one is issued.
      struct Cursor {
        int j, t, own;  // tile of the item, of the CTA; own tiles so far
      } cs = {0, -1, 0}, cp = {0, -1, 0};
      int item = -1, with = -1, mine = 0, tiles = 0;  // with: items that had tiles, before this; this group's tiles, all
      int n_items = 0;
      auto pv_done = [&](int n) { return wait(&o_full[g], n); };
      // To the next item that has tiles; false past the last. The list's slots go round only as the softmax ends items,
      // and a row of items without tiles can be longer than the list: so each is read once, with no P V outstanding.
      auto seek = [&]() {
        do {
          const PtItem it = item_at(++item);
          if (it.rows == 0) return false;
          mine = g ? it.tiles[1] : it.tiles[0];
          tiles = tiles_all(it);
        } while (tiles == 0);
        cs.j = cp.j = 0;
        ++with;
        return true;
      };
      auto issue_s = [&]() {
        const int st = ++cs.t % kStages, qb = with % kQBufs;
        const bool has = cs.j < mine;
        if (!((cs.j > 0 || wait(&q_full[qb], with / kQBufs)) && wait(&k_full[st], cs.t / kStages))) return false;
        if (has && cs.own > 0 && !(Cfg::kAlias ? pv_done(cs.own - 1) : wait(&s_free[g], cs.own - 1))) return false;
        tc_fence_after();
        if (elect_one()) {
          if (has) {
#pragma unroll
            for (int h = 0; h < Cfg::kHalves; ++h) {
              const uint64_t qd = sw128_desc(smem_u32(smem + Cfg::kOffQ + (2 * qb + g) * Cfg::kStage + h * Cfg::kTile));
              const uint64_t kd = sw128_desc(smem_u32(smem + Cfg::kOffK + st * Cfg::kStage + h * Cfg::kTile));
#pragma unroll
              for (int k = 0; k < 4; ++k) mma_f16(d0 + Cfg::kColS, qd + 2 * k, kd + 2 * k, ID_S, h + k > 0 ? 1u : 0u);
            }
            mma_commit(&s_full[g]);
            mma_commit(&k_empty[st]);
          } else {
            mbar_arrive(&k_empty[st]);
          }
          if (cs.j + 1 == tiles) {
            if (mine > 0) mma_commit(&q_empty[qb]);
            else mbar_arrive(&q_empty[qb]);
          }
        }
        if (has) ++cs.own;
        ++cs.j;
        return true;
      };
      auto issue_pv = [&]() {
        const int st = ++cp.t % kStages;
        const bool has = cp.j < mine;
        if (!wait(&v_full[st], cp.t / kStages) || (has && !wait(&p_full[g], cp.own))) return false;
        if (has && cp.j == 0 && n_items > 0 && !wait(&o_free[g], n_items - 1)) return false;
        tc_fence_after();
        if (elect_one()) {
          if (has) {
#pragma unroll
            for (int h = 0; h < Cfg::kHalves; ++h) {
              const uint64_t vd = sw128_desc(smem_u32(smem + Cfg::kOffV + st * Cfg::kStage + h * Cfg::kTile));
#pragma unroll
              for (int k = 0; k < kPtKeys / 16; ++k)
                mma_f16_ta(d0 + Cfg::kColO + 64 * h, d0 + Cfg::kColP + 8 * k, vd + static_cast<uint64_t>(k) * (2048 >> 4),
                           ID_O, (cp.j > 0 || k > 0) ? 1u : 0u);
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
        ++cp.j;
        return true;
      };
      // S runs a tile ahead of P V; after it, an item's first S (whose queries may not be there yet) and S in the
      // place of P
      bool ok = true;
      while (ok && seek()) {
        while (ok && cp.j < tiles) {
          const int ahead = cs.j - cp.j;
          if (cs.j < tiles && (ahead == 0 || (ahead == 1 && !Cfg::kAlias)))
            ok = issue_s();
          else
            ok = issue_pv();
        }
      }
      // MMAs in flight end before TMEM is given back, also where a wait ran out
      if (cs.own > 0) wait(&s_full[g], cs.own - 1);
      if (cp.own > 0) wait(&o_full[g], cp.own - 1);
    }
  } else if (warp < 8) {
    // ---- queries (the first item's with the softmax warps, which wait for them)
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsQuery));
    int with = 0;
    for (int i = 0;; ++i) {
      const PtItem it = item_at(i);
      if (it.rows == 0) break;
      if (tiles_all(it) == 0) continue;
      if (with >= kQBufs && !wait(&q_empty[with % kQBufs], with / kQBufs - 1)) break;
      put_queries(it, i, with, with ? warp - 4 : warp + 12, with ? 4 : 20);
      ++with;
    }
  } else if (warp < 12) {
    // ---- operands
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsOps));
    int t = 0;
    bool ok = true;
    for (int i = 0; ok; ++i) {
      const PtItem it = item_at(i);
      if (it.rows == 0) break;
      const int n_tiles = tiles_all(it);
      for (int j = 0; j < n_tiles && ok; ++j, ++t) {
        const int st = t % kStages, rs = t % kRaws;
        ok = wait(&r_full[rs], t / kRaws);
#pragma unroll 1
        for (int z = 0; z < 2 && ok; ++z) {  // K, then V
          if (t >= kStages) ok = wait(z ? &v_empty[st] : &k_empty[st], t / kStages - 1);
          if (!ok) break;
          const uint8_t* raw = smem + Cfg::kOffRaw + rs * Cfg::kRaw + z * kPtKeys * HD;
          uint8_t* out = smem + (z ? Cfg::kOffV : Cfg::kOffK) + st * Cfg::kStage;
          constexpr int kPieces = HD / 16;  // of 16 codes in a row
#pragma unroll 2
          for (int n = 0; n < kPieces; ++n) {
            const int x = n * 128 + (static_cast<int>(threadIdx.x) & 127);
            const int r = x / kPieces, p = x % kPieces;
            const uint4 u = *reinterpret_cast<const uint4*>(raw + r * HD + 16 * p);
            uint4 lo, hi;
            codes_to_f16(u.x, lo.x, lo.y);
            codes_to_f16(u.y, lo.z, lo.w);
            codes_to_f16(u.z, hi.x, hi.y);
            codes_to_f16(u.w, hi.z, hi.w);
            if (z) {
              const uint32_t f = __float_as_uint(scales[(t % kPtSlots * 2 + 1) * kPtGroups + r / 16]);
              lo = make_uint4(mul_f16x2(lo.x, f), mul_f16x2(lo.y, f), mul_f16x2(lo.z, f), mul_f16x2(lo.w, f));
              hi = make_uint4(mul_f16x2(hi.x, f), mul_f16x2(hi.y, f), mul_f16x2(hi.z, f), mul_f16x2(hi.w, f));
            }
            uint8_t* row = out + p / 4 * Cfg::kTile + r * 128;
            const int piece = 2 * (p % 4);
            *reinterpret_cast<uint4*>(row + ((piece ^ (r & 7)) << 4)) = lo;
            *reinterpret_cast<uint4*>(row + ((piece + 1 ^ (r & 7)) << 4)) = hi;
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(z ? &v_full[st] : &k_full[st]);
        }
        if (ok && lane == 0) mbar_arrive(&r_empty[rs]);
      }
    }
  } else {
    // ---- softmax of group g: row rl of its 128 by two threads, half hf of every tile's keys each
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsSoft));
    constexpr int kMine = kPtKeys / 2;
    const int g = (warp - 12) >> 3, hf = (warp >> 2) & 1;
    const int quad = warp & 3;
    const int rl = quad * 32 + lane;
    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16) + g * Cfg::kGroupCols;
    const uint32_t s_addr = lane_base + Cfg::kColS + hf * kMine, p_addr = lane_base + Cfg::kColP + hf * (kMine / 2);
    const uint32_t o_addr = lane_base + Cfg::kColO + hf * (HD / 2);
    float* swap = reinterpret_cast<float*>(smem + Cfg::kOffSwap) + g * 256 + rl;
    auto pv_done = [&](int n) { return wait(&o_full[g], n); };
    auto pair_sync = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(1 + g * 4 + quad) : "memory"); };
    int n_swap = 0;
    auto other = [&](float x) {  // what the other half of the row has
      float* at = swap + (n_swap++ & 1) * 512;
      at[hf * 128] = x;
      pair_sync();
      return at[(hf ^ 1) * 128];
    };
    auto slot_at = [&](int cta, int part) {  // of the two warps' rows
      return a.partials + (16LL * cta + (part == 0 ? 8 : 0) + g * 4 + quad) * Cfg::kSlot;
    };
    // The part of the item's rows that two warps share is written; the last to arrive joins the problem's parts in order.
    auto join = [&](const PtItem& it) {
      const int row0 = g * kPtRows + quad * 32;
      __threadfence();
      pair_sync();
      int* ticket = a.tickets + 8 * it.cta_first + g * 4 + quad;
      if (hf == 0 && lane == 0) last[g * 4 + quad] = atomicAdd(ticket, 1) == it.parts - 1 ? 1 : 0;
      pair_sync();
      if (!last[g * 4 + quad]) return;
      __threadfence();
      // a row per lane: the largest m, and l
      const int rows = min(32, it.rows - row0);
      auto part_at = [&](int k) { return slot_at(it.cta_first + k, k); };
      float top = -INFINITY, sum = 0.f;
      for (int k0 = 0; k0 < it.parts; k0 += 8) {
        float2 x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          x[k] = k0 + k < it.parts && lane < rows
                     ? __ldcg(reinterpret_cast<const float2*>(part_at(k0 + k) + 32 * HD + 2 * lane))
                     : make_float2(-INFINITY, 0.f);
        float now = top;
#pragma unroll
        for (int k = 0; k < 8; ++k) now = fmaxf(now, x[k].x);
        const float base = now == -INFINITY ? 0.f : now;
        sum *= ex2(top - base);
#pragma unroll
        for (int k = 0; k < 8; ++k) sum = fmaf(x[k].y, ex2(x[k].x - base), sum);
        top = now;
      }
      top = top == -INFINITY ? 0.f : top;
      sum = sum == 0.f ? 0.f : 1.f / sum;
      // four dims of two rows per thread, four parts in flight
      constexpr int kQuads = HD / 4, kRowsAt = 32 / kQuads;  // rows of a warp at a time
      const int sub = lane / kQuads, d = lane % kQuads * 4;
      for (int r0 = hf * 2 * kRowsAt; r0 < rows; r0 += 4 * kRowsAt) {
        float4 y[2];
        float base[2], inv[2];
        int r[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          r[z] = r0 + z * kRowsAt + sub;
          base[z] = __shfl_sync(0xffffffffu, top, r[z] & 31);
          inv[z] = __shfl_sync(0xffffffffu, sum, r[z] & 31);
          y[z] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int k0 = 0; k0 < it.parts; k0 += 4) {
          float4 v[2][4];
          float w[2][4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              v[z][k] = make_float4(0.f, 0.f, 0.f, 0.f);
              w[z][k] = -INFINITY;
              if (k0 + k < it.parts && r[z] < rows) {
                const float* from = part_at(k0 + k);
                v[z][k] = __ldcg(reinterpret_cast<const float4*>(from + r[z] * HD + d));
                w[z][k] = __ldcg(from + 32 * HD + 2 * r[z]);
              }
            }
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int z = 0; z < 2; ++z) add_scaled(y[z], ex2(w[z][k] - base[z]), v[z][k]);
        }
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          if (r[z] >= rows) continue;
          int tok, head;
          pt_row(a, it, row0 + r[z], tok, head);
          *reinterpret_cast<uint2*>(a.o + (it.row0 + tok) * a.ldo + head * HD + d) =
              make_uint2(bf16x2(y[z].x * inv[z], y[z].y * inv[z]), bf16x2(y[z].z * inv[z], y[z].w * inv[z]));
        }
      }
      if (hf == 0 && lane == 0) *ticket = 0;
    };
    int own = 0, t0 = 0;  // this group's key tiles so far, and the CTA's before this item
    bool ok = true;
    for (int item = 0;; ++item) {
      const PtItem& it = items[item % kPtItems];  // held till the item's end: its fields need no registers
      if (ok) ok = wait(&item_full[item % kPtItems], item / kPtItems);
      // the two warps of a row meet in barriers, so they leave together (also after a wait ran out)
      if (fminf(ok ? 1.f : 0.f, other(ok ? 1.f : 0.f)) == 0.f || it.rows == 0) break;
      if (t0 == 0 && tiles_all(it) > 0) put_queries(it, item, 0, warp - 12, 20);
      const int n_tiles = it.tiles[g], all = tiles_all(it);
      auto release = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&item_empty[item % kPtItems]);
      };
      const bool idle = g * kPtRows + quad * 32 >= it.rows;  // two warps of padding rows: nobody reads their P
      if (n_tiles == 0) {  // no row of the group sees a key of the item, or each goes alone
        for (int x = hf; x < min(32, it.rows - g * kPtRows - quad * 32); x += 2) {
          const int r = g * kPtRows + quad * 32 + x;
          float o[HD / 32], top;
          pt_row_alone<HD>(a, it, r, o, top, alive);
          int tok, head;
          pt_row(a, it, r, tok, head);
          float* mine = slot_at(it.cta_first + it.part, it.part);
#pragma unroll
          for (int e = 0; e < HD / 32; ++e) {
            if (it.parts == 1) a.o[(it.row0 + tok) * a.ldo + head * HD + lane + 32 * e] = __float2bfloat16(o[e]);
            else mine[x * HD + lane + 32 * e] = o[e];
          }
          if (it.parts > 1 && lane == 0)
            *reinterpret_cast<float2*>(mine + 32 * HD + 2 * x) = make_float2(top, top == -INFINITY ? 0.f : 1.f);
        }
      } else {
        const bool live = g * kPtRows + rl < it.rows;
        int tok, head;
        pt_row(a, it, live ? g * kPtRows + rl : 0, tok, head);
        const int vis = (live ? pt_seen(it, tok, a.causal) : 0) - hf * kMine - it.from * kPtKeys;
        float factor = 0.f;
        float m = -INFINITY, l = 0.f;
        for (int j = 0; j < n_tiles; ++j, ++own) {
          if (ok) ok = wait(&s_full[g], own);
          tc_fence_after();
          // S is there, so its queries' factors are
          if (j == 0) factor = factors[item % kPtItems * 256 + g * kPtRows + rl];
          if (idle) {
            if (j > 0 && ok) ok = pv_done(own - 1);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (!Cfg::kAlias) mbar_arrive(&s_free[g]);
              mbar_arrive(&p_full[g]);
            }
            continue;
          }
          const float* sc = scales + (t0 + j) % kPtSlots * 2 * kPtGroups + hf * (kPtGroups / 2);
          uint32_t sv[kMine];
#pragma unroll
          for (int x = 0; x < kMine; x += 32) tmem_ld32(s_addr + x, sv + x);
          tmem_ld_wait();
          if (!Cfg::kAlias) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&s_free[g]);
          }
          const int nvis = vis - j * kPtKeys;
          const bool edge = __any_sync(0xffffffffu, nvis < kMine);
          if (edge) {
#pragma unroll
            for (int c = 0; c < kMine; c += 32) {
              const int n = nvis - c;
              const uint32_t seen = n >= 32 ? 0xFFFFFFFFu : n <= 0 ? 0u : (1u << n) - 1u;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen & 1u << e)) sv[c + e] = __float_as_uint(-INFINITY);
            }
          }
          float m_tile = -INFINITY, mul[kMine / 16];
#pragma unroll
          for (int x = 0; x < kMine / 16; ++x) {
            // where the row sees none of a group, and for a product that underflows: no NaN from -infinity times it
            const float f = sc[x] * factor;
            mul[x] = (edge && 16 * x >= nvis) || f == 0.f ? 1e-30f : f;
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
              mx[0] = max3(mx[0], __uint_as_float(sv[16 * x + e]), __uint_as_float(sv[16 * x + e + 1]));
              mx[1] = max3(mx[1], __uint_as_float(sv[16 * x + e + 2]), __uint_as_float(sv[16 * x + e + 3]));
            }
            m_tile = fmaxf(m_tile, fmaxf(mx[0], mx[1]) * mul[x]);
          }
          m_tile = fmaxf(m_tile, other(m_tile));  // (head_dim 128: both halves have read S, P may take its place)
          const bool raise = m_tile > m + kPtStaleMax;
          const float alpha = raise ? ex2(m - m_tile) : 1.f;
          if (raise) m = m_tile;
          const float add = (m == -INFINITY ? 0.f : -m) + kPtHead;
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x0 = 0; x0 < kMine; x0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float v0, v1;
              fma2(v0, v1, __uint_as_float(sv[x0 + e]), __uint_as_float(sv[x0 + e + 1]), mul[(x0 + e) / 16], add);
              const float p0 = ex2(v0), p1 = ex2(v1);
              add2(ls[e & 2], ls[(e & 2) + 1], p0, p1);
              pk[e >> 1] = f16x2(p0, p1);
            }
            if (x0 == 0 && j > 0) {  // the P V before has read P, and O is stable
              if (ok) ok = pv_done(own - 1);
              tc_fence_after();
            }
            tmem_st16(p_addr + x0 / 2, pk);
          }
          if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll
            for (int x = 0; x < HD / 2; x += 32) {
              uint32_t ov[32];
              tmem_ld32(o_addr + x, ov);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
              tmem_st16(o_addr + x, ov);
              tmem_st16(o_addr + x + 16, ov + 16);
            }
          }
          l = fmaf(l, alpha, (ls[0] + ls[1]) + (ls[2] + ls[3]));
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_full[g]);
        }
        l += other(l);
        if (ok) ok = pv_done(own - 1);
        tc_fence_after();
        // O / l and the factors of V; a row that sees nothing is 0 (its P are)
        const float inv = l == 0.f ? 0.f : __fdividef(1.f / 256.f, l);
        const float back = __uint_as_float(static_cast<uint32_t>(it.exp_max + 127) << 23);
        pt_row(a, it, live ? g * kPtRows + rl : 0, tok, head);
        const long long row_at = (it.row0 + tok) * a.ldo + head * HD + hf * (HD / 2);
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
          float f[32];
#pragma unroll
          for (int e = 0; e < 32; ++e)  // in order again
            f[e] = __uint_as_float(ov[(e & ~3) + ((e & 3) >> 1 | (e & 1) << 1)]) * inv * back;
          if (it.parts > 1) {
            float* mine = slot_at(it.cta_first + it.part, it.part);
            if (live)
#pragma unroll
              for (int x = 0; x < 32; x += 4)
                *reinterpret_cast<float4*>(mine + lane * HD + hf * (HD / 2) + h + x) =
                    make_float4(f[x], f[x + 1], f[x + 2], f[x + 3]);
            continue;
          }
          uint4 y[4];  // 8 dims each
#pragma unroll
          for (int x = 0; x < 4; ++x)
            y[x] = make_uint4(bf16x2(f[8 * x], f[8 * x + 1]), bf16x2(f[8 * x + 2], f[8 * x + 3]),
                              bf16x2(f[8 * x + 4], f[8 * x + 5]), bf16x2(f[8 * x + 6], f[8 * x + 7]));
          transpose4(y);
#pragma unroll
          for (int x = 0; x < 4; ++x) {  // y[x]: piece lane % 4 of row lane / 4 * 4 + x
            const int w = (lane & ~3) + x;
            const long long to = __shfl_sync(0xffffffffu, row_at, w);
            if (g * kPtRows + quad * 32 + w >= it.rows) continue;
            uint2* out = reinterpret_cast<uint2*>(a.o + to + h + 8 * (lane & 3));
            if (a.o_wide) {
              *reinterpret_cast<uint4*>(out) = y[x];
            } else {
              out[0] = make_uint2(y[x].x, y[x].y);
              out[1] = make_uint2(y[x].z, y[x].w);
            }
          }
        }
        if (it.parts > 1 && live && hf == 0)  // the part's logarithm of l: parts weigh by it
          *reinterpret_cast<float2*>(slot_at(it.cta_first + it.part, it.part) + 32 * HD + 2 * lane) =
              l == 0.f ? make_float2(-INFINITY, 0.f) : make_float2(m - kPtHead + log2f(l), 1.f);
      }
      t0 += all;
      if (it.parts > 1 && !idle) join(it);
      release();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

template <int HD>
int launch_pages_tc(const PagesArgs& a, int64_t most_steps, int64_t workspace_bytes, int64_t n_tickets,
                    cudaStream_t stream) {
  static std::atomic<int> sms[64];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return SO101_ERR_DRIVER;
  int full = sms[dev].load();
  if (!full) {
    cudaError_t e = cudaFuncSetAttribute(attention_pages_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         PtCfg<HD>::kSmem);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&full, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return launch_error(e);
    sms[dev].store(full);
  }
  // per CTA: two slots and a ticket for each 32 rows
  const int64_t slots = workspace_bytes / (16LL * PtCfg<HD>::kSlot * 4);
  int64_t grid = most_steps < full ? most_steps : full;
  if (grid > slots) grid = slots;
  if (grid > n_tickets / 8) grid = n_tickets / 8;
  if (grid < 1) return SO101_ERR_WORKSPACE;
  return launch_kernel(attention_pages_tc_kernel<HD>, dim3(static_cast<unsigned>(grid)), dim3(kPtThreads),
                       PtCfg<HD>::kSmem, stream, a);
}

// The tcgen05 kernel where it is the faster one: false where the mma.sync kernel is, whose CTA holds up to 64 rows.
// (group: what group_inv is exact for.)
bool attention_pages_tc(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream, int* rc) {
  const int64_t rows = static_cast<int64_t>(a.max_q) * a.group;  // of an entry and kv head, at most
  if (rows <= 64 || a.group > 32768) return false;
  const int64_t problems = (rows + 2 * kPtRows - 1) / (2 * kPtRows) * a.c.n_kv * a.n_seqs;
  const int64_t capacity = static_cast<int64_t>(a.c.max_pages) * a.c.page;
  const int64_t most = problems * ((capacity + kPtKeys - 1) / kPtKeys);  // steps are counted in 32 bits
  if (problems > (1 << 24) || most > (1LL << 30)) {
    *rc = SO101_ERR_ARG;
    return true;
  }
  *rc = a.c.hd == 64 ? launch_pages_tc<64>(a, most, workspace_bytes, n_tickets, stream)
                     : launch_pages_tc<128>(a, most, workspace_bytes, n_tickets, stream);
  return true;
}

}  // namespace so101
