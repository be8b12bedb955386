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
// Codes become f16 exactly (a byte under the exponent of 1024, minus 1152). Which of a head's dims is
// which k index of the MMA is free as long as Q and K agree, and so is the order of the keys between
// S and V, so both are laid out to make a thread's codes contiguous: 16 dims of a key row, 8 of a
// value row, and the packed pairs of V come from byte permutes of two rows. Q is scaled by a power of
// two per row and rounded to f16 (11 bits; the row's factor goes back in with f), P is rounded to f16.
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
  int chunk;      // keys per CTA (a multiple of its step)
  int splits;     // chunks per sequence in the grid
  int row_tiles;  // tiles of 16 * ROWW rows in the grid
  int* status;
};

constexpr int kPgWarps = 4;
constexpr int kPgThreads = 32 * kPgWarps;

template <int HD, int ROWW>
struct PgCfg {
  static constexpr int kKeys = HD == 64 ? 64 : 32;  // keys per tile: 4 KB of K and of V
  static constexpr int kTile = kKeys * HD;
  static constexpr int kStages = 3;
  static constexpr int kMaxPages = kKeys / 16;
  static constexpr int kRing = kStages * 2 * kTile;
  static constexpr int kRings = kPgWarps / ROWW;
  static constexpr int kJoin = kPgWarps * 16 * (HD + 2) * 4;  // the rings' buffers serve the join too
  static constexpr int kOffScale = kRings * kRing > kJoin ? kRings * kRing : kJoin;
  static constexpr int kOffBar = kOffScale + kRings * kStages * 2 * kMaxPages * 4;
  static constexpr int kOffFlag = kOffBar + kRings * kStages * 8;
  static constexpr int kSmem = kOffFlag + 16;
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

// Two bytes (biased by 128) to two f16 codes: the byte under the exponent of 1024, minus 1024 + 128.
__device__ __forceinline__ uint32_t codes_f16(uint32_t bytes, uint32_t sel) {
  uint32_t h = __byte_perm(bytes, 0x64646464u, sel), r;
  asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(h), "r"(0x64806480u));
  return r;
}

// Grid: (splits * row tiles, kv heads, list entries). ROWW of the CTA's warps take 16 query rows each
// of the same keys (one ring for them all), the others take other keys of the chunk.
template <int HD, int ROWW>
__global__ void __launch_bounds__(kPgThreads) attention_pages_kernel(const PagesArgs a) {
  using Cfg = PgCfg<HD, ROWW>;
  constexpr int kKeys = Cfg::kKeys, kStages = Cfg::kStages, kTile = Cfg::kTile;
  constexpr int kRings = Cfg::kRings;      // key groups of the CTA
  constexpr int kNT = kKeys / 8;           // 8-key tiles of S
  constexpr int kQK = HD / 16;             // k steps of S
  constexpr int kHalves = HD / 64;         // 64-dim halves of a head
  extern __shared__ __align__(128) uint8_t smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  int* flag = reinterpret_cast<int*>(smem + Cfg::kOffFlag);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, t = lane & 3;
  const int ring = warp / ROWW, roww = warp % ROWW;
  const KvPages& c = a.c;
  const int head = blockIdx.y;
  const int split = blockIdx.x % a.splits, rt = blockIdx.x / a.splits;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRings * kStages; ++i) mbar_init(&bars[i], 1);
    fence_mbar_init();
  }
  grid_dep_launch();
  grid_dep_wait();
  int seq, row0, n_q;
  const bool good = kv_rows(c, a.starts, a.seqs, blockIdx.z, a.rows, seq, row0, n_q, a.status);
  const int rows = good ? n_q * a.group : 0;  // rows of this kv head: token r / group, head r % group
  const int tile_row = rt * 16 * ROWW;
  if (rt == a.row_tiles - 1 && rows > tile_row + 16 * ROWW && threadIdx.x == 0)
    record_error(a.status, SO101_ERR_PAGES);  // more rows than max_q said
  if (tile_row >= rows) return;
  const int len = kv_length(c, seq, a.status);
  // keys that this CTA's rows can see
  const int last_row = min(rows, tile_row + 16 * ROWW) - 1;
  const int key_end = a.causal ? max(0, min(len, len - n_q + last_row / a.group + 1)) : len;
  const int n_chunks = max(1, (key_end + a.chunk - 1) / a.chunk);
  if (split >= n_chunks) return;
  const int key0 = split * a.chunk, key1 = min(key_end, key0 + a.chunk);
  __syncthreads();  // the barriers are set up

  // ---- this warp's query rows g and g + 8, dims 16 t .. 16 t + 15 of each 64, as f16 fragments
  const int wrow = tile_row + roww * 16;
  uint32_t qf[kQK][4];
  float factor[2];
  int vis[2];  // keys [0, vis) are visible to the row
  {
    float x[2][kHalves][16];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = wrow + g + 8 * i;
      const bool live = r < rows;
      const int tok = live ? r / a.group : 0;
      vis[i] = !live ? 0 : a.causal ? max(0, min(len, len - n_q + tok + 1)) : len;
      const __nv_bfloat16* qr = a.q + (row0 + tok) * a.ldq + (head * a.group + (live ? r % a.group : 0)) * HD;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int e = 0; e < 16; e += 8) {
          const uint4 u = live ? __ldg(reinterpret_cast<const uint4*>(qr + 64 * h + 16 * t + e)) : make_uint4(0, 0, 0, 0);
          const __nv_bfloat162* b = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 f = __bfloat1622float2(b[w]);
            x[i][h][e + 2 * w] = f.x;
            x[i][h][e + 2 * w + 1] = f.y;
          }
        }
      if (a.cos) {
        // the partner of dim d is d + HD / 2: another half of this thread's (HD 128), or the same
        // place of the thread two lanes on (HD 64)
        const long long p = static_cast<long long>(row0 + tok) * (HD / 2);
        if (HD == 128) {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float cs = __ldg(a.cos + p + 16 * t + e), sn = __ldg(a.sin + p + 16 * t + e);
            const float u = x[i][0][e], w = x[i][kHalves - 1][e];
            x[i][0][e] = __fsub_rn(__fmul_rn(u, cs), __fmul_rn(w, sn));
            x[i][kHalves - 1][e] = __fadd_rn(__fmul_rn(w, cs), __fmul_rn(u, sn));
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const int d = 16 * (t & 1) + e;
            const float cs = __ldg(a.cos + p + d), sn = __ldg(a.sin + p + d);
            const float u = x[i][0][e], w = __shfl_xor_sync(0xffffffffu, u, 2);
            x[i][0][e] = t < 2 ? __fsub_rn(__fmul_rn(u, cs), __fmul_rn(w, sn))
                               : __fadd_rn(__fmul_rn(u, cs), __fmul_rn(w, sn));
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
      factor[i] = __uint_as_float(ef << 23) * a.scale_log2;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int e = 0; e < 16; ++e) x[i][h][e] *= down;
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        qf[4 * h + s][0] = f16x2(x[0][h][4 * s], x[0][h][4 * s + 1]);
        qf[4 * h + s][1] = f16x2(x[1][h][4 * s], x[1][h][4 * s + 1]);
        qf[4 * h + s][2] = f16x2(x[0][h][4 * s + 2], x[0][h][4 * s + 3]);
        qf[4 * h + s][3] = f16x2(x[1][h][4 * s + 2], x[1][h][4 * s + 3]);
      }
  }

  // ---- the key tiles of this ring: tile i covers keys [key0 + (i * kRings + ring) * kKeys, + kKeys)
  uint8_t* my_ring = smem + ring * Cfg::kRing;
  float* my_scales = reinterpret_cast<float*>(smem + Cfg::kOffScale) + ring * kStages * 2 * Cfg::kMaxPages;
  uint64_t* my_bars = bars + ring * kStages;
  const int span = key1 - key0;
  const int all_tiles = (span + kKeys - 1) / kKeys;
  const int tiles = all_tiles > ring ? (all_tiles - ring + kRings - 1) / kRings : 0;
  const int gran = min(c.page, kKeys);        // slots per copy (a power of two)
  const int gran_log2 = __ffs(gran) - 1;
  const int per_tile = kKeys / gran;          // copies of K (and of V) per tile
  const int* table = c.table + static_cast<long long>(seq) * c.max_pages;
  // lane l < per_tile brings the l-th run of slots of tile i, its scales beside it (whole warp calls)
  auto load_tile = [&](int i) {
    const int key = key0 + (i * kRings + ring) * kKeys + lane * gran;
    const int st = i % kStages;
    bool mine = lane < per_tile && key < key1;
    int id = 0;
    if (mine) {
      id = table[key / c.page];
      if (id < 0 || id >= c.n_pages) {
        record_error(a.status, SO101_ERR_PAGES);
        mine = false;
      }
    }
    const int runs = __popc(__ballot_sync(0xffffffffu, mine));
    const uint32_t bytes = static_cast<uint32_t>(gran * HD);
    if (lane == 0) mbar_arrive_expect_tx(&my_bars[st], 2u * bytes * runs);
    __syncwarp();
    if (mine) {
      const long long at = kv_code_at(c, a.layer, id, head) + (key % c.page) * HD;
      const uint32_t dst = smem_u32(my_ring + st * 2 * kTile) + lane * bytes;
      bulk_load(dst, c.k + at, bytes, &my_bars[st]);
      bulk_load(dst + kTile, c.v + at, bytes, &my_bars[st]);
    }
    if (lane < per_tile) {
      const long long at = mine ? kv_scale_at(c, a.layer, id, head) : 0;
      my_scales[st * 2 * Cfg::kMaxPages + lane] = mine ? c.k_scale[at] : 0.f;
      my_scales[st * 2 * Cfg::kMaxPages + Cfg::kMaxPages + lane] = mine ? c.v_scale[at] : 0.f;
    }
    __syncwarp();
  };
  // ROWW > 1: the ring's first warp loads, the others wait for it by name at each tile
  auto ring_sync = [&]() {
    if (ROWW == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + ring), "r"(32 * ROWW) : "memory");
  };
  if (roww == 0)
    for (int i = 0; i < kStages - 1 && i < tiles; ++i) load_tile(i);
  ring_sync();

  float o[kHalves][8][4];
#pragma unroll
  for (int h = 0; h < kHalves; ++h)
#pragma unroll
    for (int n = 0; n < 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[h][n][e] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  bool ok = true;

  for (int i = 0; i < tiles; ++i) {
    const int st = i % kStages;
    if (ok && roww == 0 && i + kStages - 1 < tiles) load_tile(i + kStages - 1);
    // after a wait that ran out the loop goes on without loads or waits, so that the warps of a ring
    // still meet; the result is void and the status word says so
    if (ok) ok = mbar_wait(&my_bars[st], static_cast<uint32_t>(i / kStages) & 1u, a.status);
    ok = __all_sync(0xffffffffu, ok);
    const uint8_t* kt = my_ring + st * 2 * kTile;
    const uint8_t* vt = kt + kTile;
    const float* ks = my_scales + st * 2 * Cfg::kMaxPages;
    const float* vs = ks + Cfg::kMaxPages;
    const int tile_key = key0 + (i * kRings + ring) * kKeys;

    // S: key of (n tile j, column 2 t + e) = 16 (j / 2) + 8 (j % 2) + 4 e + t
    float s[kNT][4];
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
      const uint8_t* row = kt + (8 * j + 4 * (g & 1) + (g >> 1)) * HD + 16 * t;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        const uint4 u = *reinterpret_cast<const uint4*>(row + 64 * h);
        const uint32_t w[4] = {u.x ^ 0x80808080u, u.y ^ 0x80808080u, u.z ^ 0x80808080u, u.w ^ 0x80808080u};
#pragma unroll
        for (int k = 0; k < 4; ++k) mma_16816(s[j], qf[4 * h + k], codes_f16(w[k], 0x4140u), codes_f16(w[k], 0x4342u));
      }
    }
    // logits in units of log2, masked by the key's place; the row maximum
    float mx[2] = {m[0], m[1]};
#pragma unroll
    for (int j = 0; j < kNT; ++j) {
      const float sk = ks[(8 * j) >> gran_log2];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = tile_key + 8 * j + 4 * (e & 1) + t, r = e >> 1;
        s[j][e] = key < vis[r] ? s[j][e] * (sk * factor[r]) : -INFINITY;
        mx[r] = fmaxf(mx[r], s[j][e]);
      }
    }
    float alpha[2], sub[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
      mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
      sub[r] = mx[r] == -INFINITY ? 0.f : mx[r];  // a row that has seen no key yet
      alpha[r] = exp2f(m[r] - sub[r]);
      m[r] = mx[r];
      l[r] *= alpha[r];
    }
#pragma unroll
    for (int h = 0; h < kHalves; ++h)
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        o[h][n][0] *= alpha[0];
        o[h][n][1] *= alpha[0];
        o[h][n][2] *= alpha[1];
        o[h][n][3] *= alpha[1];
      }
#pragma unroll
    for (int j = 0; j < kNT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2(s[j][e] - sub[e >> 1]);
        l[e >> 1] += s[j][e];
      }
    // O += s_v (P V), 16 keys at a time; a page that the row does not see adds nothing (its scale
    // may be NaN)
#pragma unroll
    for (int k = 0; k < kKeys / 16; ++k) {
      const uint32_t pa[4] = {f16x2(s[2 * k][0], s[2 * k][1]), f16x2(s[2 * k][2], s[2 * k][3]),
                              f16x2(s[2 * k + 1][0], s[2 * k + 1][1]), f16x2(s[2 * k + 1][2], s[2 * k + 1][3])};
      const int first = tile_key + 16 * k;
      const float sv = vs[(16 * k) >> gran_log2];
      const float f0 = first < vis[0] ? sv : 0.f, f1 = first < vis[1] ? sv : 0.f;
#pragma unroll
      for (int h = 0; h < kHalves; ++h) {
        uint2 u[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          u[x] = *reinterpret_cast<const uint2*>(vt + (16 * k + 4 * x + t) * HD + 64 * h + 8 * g);
          u[x].x ^= 0x80808080u;
          u[x].y ^= 0x80808080u;
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          // dim 8 g + n of keys x = 0, 1 and 2, 3: bytes of two rows side by side, then f16
          const uint32_t pick = (n & 2) ? 0x7362u : 0x5140u;
          const uint32_t p0 = n < 4 ? __byte_perm(u[0].x, u[1].x, pick) : __byte_perm(u[0].y, u[1].y, pick);
          const uint32_t p1 = n < 4 ? __byte_perm(u[2].x, u[3].x, pick) : __byte_perm(u[2].y, u[3].y, pick);
          const uint32_t sel = (n & 1) ? 0x4342u : 0x4140u;
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          mma_16816(d, pa, codes_f16(p0, sel), codes_f16(p1, sel));
          o[h][n][0] = fmaf(d[0], f0, o[h][n][0]);
          o[h][n][1] = fmaf(d[1], f0, o[h][n][1]);
          o[h][n][2] = fmaf(d[2], f1, o[h][n][2]);
          o[h][n][3] = fmaf(d[3], f1, o[h][n][3]);
        }
      }
    }
    ring_sync();  // the stage is read: the next load may fill it
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
  }
  // a wait ran out: the copies in flight must land before this CTA's shared memory goes away
  if (!ok && roww == 0)
    for (int i = max(0, tiles - kStages); i < tiles; ++i)
      mbar_wait(&my_bars[i % kStages], static_cast<uint32_t>(i / kStages) & 1u, a.status);
  __syncthreads();

  // ---- join the rings: (m, l, O) of each warp into shared memory (over the rings' buffers)
  constexpr int kRow = HD + 2;  // O, m, l
  float* part = reinterpret_cast<float*>(smem);
  {
    float* w = part + (ring * ROWW + roww) * 16 * kRow;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float* row = w + (g + 8 * r) * kRow;
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int n = 0; n < 8; ++n) {
          row[64 * h + 16 * t + n] = o[h][n][2 * r];
          row[64 * h + 16 * t + 8 + n] = o[h][n][2 * r + 1];
        }
      if (t == 0) {
        row[HD] = m[r];
        row[HD + 1] = l[r];
      }
    }
  }
  __syncthreads();
  // rows of this CTA, one (row, dim) at a time: over its rings, then (the last CTA of a sequence's
  // chunks to arrive) over the chunks in order
  const int tile_rows = min(rows - tile_row, 16 * ROWW);
  const long long slot = (static_cast<long long>(blockIdx.z) * a.row_tiles + rt) * c.n_kv + head;
  float* mine = n_chunks > 1 ? a.partials + (slot * a.splits + split) * (16 * ROWW * kRow) : nullptr;
  for (int e = threadIdx.x; e < tile_rows * HD; e += kPgThreads) {
    const int r = e / HD, d = e % HD;
    float mm = -INFINITY;
    for (int k = 0; k < kRings; ++k) mm = fmaxf(mm, part[(k * ROWW * 16 + r) * kRow + HD]);
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, oo = 0.f;
    for (int k = 0; k < kRings; ++k) {
      const float* row = part + (k * ROWW * 16 + r) * kRow;
      const float w = exp2f(row[HD] - base);
      ll = fmaf(w, row[HD + 1], ll);
      oo = fmaf(w, row[d], oo);
    }
    if (mine) {
      mine[r * kRow + d] = oo;
      if (d == 0) {
        mine[r * kRow + HD] = mm;
        mine[r * kRow + HD + 1] = ll;
      }
    } else {
      const int tok = (tile_row + r) / a.group, hq = head * a.group + (tile_row + r) % a.group;
      a.o[(row0 + tok) * a.ldo + hq * HD + d] = __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
    }
  }
  if (!mine) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) *flag = atomicAdd(a.tickets + slot, 1) == n_chunks - 1 ? 1 : 0;
  __syncthreads();
  if (!*flag) return;
  __threadfence();
  const float* all = a.partials + slot * a.splits * (16 * ROWW * kRow);
  for (int e = threadIdx.x; e < tile_rows * HD; e += kPgThreads) {
    const int r = e / HD, d = e % HD;
    float mm = -INFINITY;
    for (int k = 0; k < n_chunks; ++k) mm = fmaxf(mm, __ldcg(all + (k * 16 * ROWW + r) * kRow + HD));
    const float base = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f, oo = 0.f;
    for (int k = 0; k < n_chunks; ++k) {
      const float* row = all + (k * 16 * ROWW + r) * kRow;
      const float w = exp2f(__ldcg(row + HD) - base);
      ll = fmaf(w, __ldcg(row + HD + 1), ll);
      oo = fmaf(w, __ldcg(row + d), oo);
    }
    const int tok = (tile_row + r) / a.group, hq = head * a.group + (tile_row + r) % a.group;
    a.o[(row0 + tok) * a.ldo + hq * HD + d] = __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
  }
  if (threadIdx.x == 0) a.tickets[slot] = 0;
}

namespace {

template <int HD, int ROWW>
int launch_pages(const PagesArgs& a, dim3 grid, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};  // a bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && !(configured.load() >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(attention_pages_kernel<HD, ROWW>,
                                               cudaFuncAttributeMaxDynamicSharedMemorySize, PgCfg<HD, ROWW>::kSmem);
    if (e != cudaSuccess) return launch_error(e);
    configured.fetch_or(1ull << dev);
  }
  return launch_kernel(attention_pages_kernel<HD, ROWW>, grid, dim3(kPgThreads), PgCfg<HD, ROWW>::kSmem, stream, a);
}

}  // namespace

}  // namespace so101

using namespace so101;

extern "C" int so101_attention_pages(const void* q, int64_t ldq, void* o, int64_t ldo, int64_t rows,
                                     const so101_kv_pages* c, int layer, int nq, const int* starts, const int* seqs,
                                     int n_seqs, int64_t max_q, int causal, float scale, const float* cos,
                                     const float* sin, void* workspace, int64_t workspace_bytes, int* tickets,
                                     int64_t n_tickets, cudaStream_t stream) {
  if (!kv_pages_ok(c) || layer < 0 || layer >= c->n_layers || nq < 1 || nq % c->n_kv || n_seqs < 0 ||
      n_seqs > 65535 || rows < 0 || rows > (1 << 30) || max_q < 1 || (cos == nullptr) != (sin == nullptr) ||
      !(scale > 0.f && scale < INFINITY))
    return SO101_ERR_ARG;
  if (!starts && (rows != n_seqs || max_q != 1)) return SO101_ERR_ARG;
  if (n_seqs == 0 || rows == 0) return SO101_OK;
  if (!q || !o) return SO101_ERR_ARG;
  const int64_t width = static_cast<int64_t>(nq) * c->hd;
  if (reinterpret_cast<uintptr_t>(q) % 16 || ldq % 8 || reinterpret_cast<uintptr_t>(o) % 2 ||
      (rows > 1 && (ldq < width || ldo < width)) || nq > 65535)
    return SO101_ERR_ARG;
  PagesArgs a;
  a.c = *c;
  a.q = static_cast<const __nv_bfloat16*>(q);
  a.o = static_cast<__nv_bfloat16*>(o);
  a.ldq = ldq;
  a.ldo = ldo;
  a.rows = rows;
  a.starts = starts;
  a.seqs = seqs;
  a.cos = cos;
  a.sin = sin;
  a.partials = static_cast<float*>(workspace);
  a.tickets = tickets;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.layer = layer;
  a.nq = nq;
  a.group = nq / c->n_kv;
  a.causal = causal;
  a.status = status_ptr();
  // rows per CTA: one warp's 16 where they suffice, up to 64 so that one pass over the keys serves more
  const int64_t most_rows = (max_q < rows ? max_q : rows) * a.group;
  const int roww = most_rows <= 16 ? 1 : most_rows <= 32 ? 2 : 4;
  a.row_tiles = static_cast<int>((most_rows + 16 * roww - 1) / (16 * roww));
  // chunks: enough CTAs for every SM twice over, none under 256 keys, as the workspace allows
  const int64_t capacity = static_cast<int64_t>(c->max_pages) * c->page;
  const int64_t problems = static_cast<int64_t>(n_seqs) * c->n_kv * a.row_tiles;
  const int64_t slot_bytes = static_cast<int64_t>(16) * roww * (c->hd + 2) * 4;
  int64_t splits = problems > 0 ? (2 * 148 + problems - 1) / problems : 1;
  if (!workspace || !tickets || problems > n_tickets) splits = 1;
  if (splits > 1 && splits * problems * slot_bytes > workspace_bytes) splits = workspace_bytes / (problems * slot_bytes);
  if (splits < 1) splits = 1;
  int64_t chunk = ((capacity + splits - 1) / splits + 255) / 256 * 256;
  a.chunk = static_cast<int>(chunk);
  a.splits = static_cast<int>((capacity + chunk - 1) / chunk);
  if (static_cast<int64_t>(a.splits) * a.row_tiles > (1 << 30) || c->n_kv > 65535) return SO101_ERR_ARG;
  const dim3 grid(static_cast<unsigned>(a.splits * a.row_tiles), static_cast<unsigned>(c->n_kv),
                  static_cast<unsigned>(n_seqs));
  if (c->hd == 64)
    return roww == 1 ? launch_pages<64, 1>(a, grid, stream)
                     : roww == 2 ? launch_pages<64, 2>(a, grid, stream) : launch_pages<64, 4>(a, grid, stream);
  return roww == 1 ? launch_pages<128, 1>(a, grid, stream)
                   : roww == 2 ? launch_pages<128, 2>(a, grid, stream) : launch_pages<128, 4>(a, grid, stream);
}
