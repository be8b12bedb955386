// Causal grouped-query attention over prompts packed end to end (so101_attention_packed), on tcgen05.
//
//   o_i = sum_{j <= i} 2^(f q_i . k_j - m_i) v_j / sum_{j <= i} 2^(f q_i . k_j - m_i),  f = scale * log2(e)
//
// The query heads of a kv head are stacked: row r of (sequence, kv head) is token r / group, head
// r % group of the group, so 128 MMA rows span few tokens (43 at three heads per kv head) and little of
// a 128-key tile is masked at the diagonal; a sequence of one token still fills `group` rows.
// One CTA takes 128 such rows:
//   warp 0 (one thread)  TMA: K_j and V_j (128 keys) into rings
//   warp 1 (one thread)  S = Q K_j^T -> TMEM; O += P V_j, P read from TMEM
//   warps 2-5            first the queries: each thread loads its row, rotates it in fp32, rounds it to
//                        bf16 once and writes the swizzled Q tile; then the softmax of its row (one TMEM
//                        lane), at the end O / l to the output row.
// The row maximum is only raised when a tile exceeds it by more than 2^8 (as in the SigLIP kernel).
// Keys past the row's own token are masked by their index. Their values still meet P = 0 in the MMA, where an
// infinity or a NaN in a value the row must not see would make the row NaN, so a row whose result is
// not finite is computed again key by key over what it sees (never with finite values).
#include <atomic>
#include <cmath>

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
  int n_seqs, rows, group;
  const float* cos;
  const float* sin;
  float scale_log2;
  int* status;
};

constexpr int kPkRows = 128, kPkKeys = 128;
constexpr int kPkThreads = 32 * 6;
constexpr float kPkStaleMax = 8.f;

// head_dim 64: S, P and O side by side in 256 TMEM columns. 128: P takes the place of the S it came
// from, so the next S waits for P V (the other CTA of the SM runs meanwhile).
template <int HD>
struct PkCfg {
  static constexpr int kHalves = HD / 64;                 // 64-dim (128-byte) tiles of a row
  static constexpr int kTile = kPkRows * 128;             // 16 KB: 128 rows x 64 dims
  static constexpr int kStage = kHalves * kTile;
  static constexpr int kStages = HD == 64 ? 2 : 1;
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = kStage;
  static constexpr int kOffV = kOffK + kStages * kStage;
  static constexpr int kOffBar = kOffV + kStages * kStage;
  static constexpr int kSmem = kOffBar + 256 + 1024;
  static constexpr bool kAlias = HD == 128;
  static constexpr uint32_t kCols = 256;
  static constexpr uint32_t kColS = 0, kColP = kAlias ? 0 : 128, kColO = kAlias ? 128 : 192;
};

// One output row in plain fp32 over the keys it may see, by a whole warp: lane l holds dims
// l, l + 32, ... Only for rows that came out not finite.
template <int HD>
__device__ __noinline__ void packed_row_alone(const PackedArgs& a, const uint8_t* q_tile, int tile_row, int start, int tok,
                                              int kvh, long long o_at) {
  const int lane = threadIdx.x & 31;
  constexpr int N = HD / 32;
  float q[N], o[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int d = lane + 32 * i;
    const uint8_t* row = q_tile + (d / 64) * (kPkRows * 128) + tile_row * 128;
    const int piece = (d % 64) / 8;
    q[i] = __bfloat162float(
        reinterpret_cast<const __nv_bfloat16*>(row + ((piece ^ (tile_row & 7)) << 4))[d % 8]);
    o[i] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  for (int j = 0; j <= tok; ++j) {
    const __nv_bfloat16* kr = a.k + (start + j) * a.ldk + kvh * HD;
    const __nv_bfloat16* vr = a.v + (start + j) * a.ldv + kvh * HD;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(q[i], __bfloat162float(kr[lane + 32 * i]), s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= a.scale_log2;
    const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
    const float alpha = exp2f(m - base), p = exp2f(s - base);
    m = mn;
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * alpha + p * __bfloat162float(vr[lane + 32 * i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) a.o[o_at + lane + 32 * i] = __float2bfloat16(l == 0.f ? 0.f : o[i] / l);
}

template <int HD>
__global__ void __launch_bounds__(kPkThreads, 2)
    attention_packed_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const PackedArgs a) {
  using Cfg = PkCfg<HD>;
  constexpr int kStages = Cfg::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ int plan[4];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bar = reinterpret_cast<uint64_t*>(smem + Cfg::kOffBar);
  uint64_t* q_full = bar;
  uint64_t* k_full = bar + 1;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;
  uint64_t* s_free = s_full + 1;
  uint64_t* p_full = s_free + 1;
  uint64_t* o_full = p_full + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(o_full + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_launch();
  grid_dep_wait();
  // block blockIdx.x of all sequences' 128-row blocks, the sequence's last block first (most keys):
  // warp 0 walks the sequences 32 at a time
  if (warp == 0) {
    int before = 0, seq = -1, start = 0, len = 0, block = 0;
    const int want = static_cast<int>(blockIdx.x);
    for (int s0 = 0; s0 < a.n_seqs && seq < 0; s0 += 32) {
      const int s = s0 + lane;
      int b = 0, at = 0, n = 0;
      if (s < a.n_seqs) {
        at = __ldg(a.starts + s);
        n = __ldg(a.starts + s + 1) - at;
        if (at < 0 || n < 0 || static_cast<long long>(at) + n > a.rows) {
          record_error(a.status, SO101_ERR_PAGES);
          n = 0;
        }
        b = static_cast<int>((static_cast<long long>(n) * a.group + kPkRows - 1) / kPkRows);
      }
      int inc = b;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += y;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + inc > want);
      if (hit) {
        const int w = __ffs(hit) - 1;
        seq = s0 + w;
        start = __shfl_sync(0xffffffffu, at, w);
        len = __shfl_sync(0xffffffffu, n, w);
        const int end = before + __shfl_sync(0xffffffffu, inc, w);
        block = end - 1 - want;  // last block first
      }
      before += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) {
      plan[0] = seq;
      plan[1] = start;
      plan[2] = len;
      plan[3] = block;
    }
  }
  if (threadIdx.x == 32) {
    mbar_init(q_full, 4);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    mbar_init(s_full, 1);
    mbar_init(s_free, 4);
    mbar_init(p_full, 4);
    mbar_init(o_full, 1);
    fence_mbar_init();
  }
  __syncthreads();
  if (plan[0] < 0) return;  // past the last block: nothing was allocated
  const int start = plan[1], len = plan[2], row_first = plan[3] * kPkRows;
  const int kvh = blockIdx.y;
  const int rows = min(kPkRows, len * a.group - row_first);
  const int last_tok = (row_first + rows - 1) / a.group;
  const int n_tiles = last_tok / kPkKeys + 1;
  if (warp == 1) {
    tmem_alloc(tmem_slot, Cfg::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tm_k);
      tma_prefetch_desc(&tm_v);
      const uint64_t keep = policy_evict_normal();
      for (int j = 0; j < n_tiles; ++j) {
        const int st = j % kStages;
        const uint32_t back = static_cast<uint32_t>(j / kStages - 1) & 1u;
        if (j >= kStages && !mbar_wait(&k_empty[st], back, a.status)) break;
        mbar_arrive_expect_tx(&k_full[st], Cfg::kStage);
        for (int h = 0; h < Cfg::kHalves; ++h)
          tma_load_2d(smem + Cfg::kOffK + st * Cfg::kStage + h * Cfg::kTile, &tm_k, &k_full[st], kvh * HD + 64 * h,
                      start + j * kPkKeys, keep);
        if (j >= kStages && !mbar_wait(&v_empty[st], back, a.status)) break;
        mbar_arrive_expect_tx(&v_full[st], Cfg::kStage);
        for (int h = 0; h < Cfg::kHalves; ++h)
          tma_load_2d(smem + Cfg::kOffV + st * Cfg::kStage + h * Cfg::kTile, &tm_v, &v_full[st], kvh * HD + 64 * h,
                      start + j * kPkKeys, keep);
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t ID_S = idesc_attn(kPkKeys, 0);
      constexpr uint32_t ID_O = idesc_attn(64, 1);
      auto issue_s = [&](int j) {
        const int st = j % kStages;
#pragma unroll
        for (int h = 0; h < Cfg::kHalves; ++h) {
          const uint64_t qd = sw128_desc(smem_u32(smem + Cfg::kOffQ + h * Cfg::kTile));
          const uint64_t kd = sw128_desc(smem_u32(smem + Cfg::kOffK + st * Cfg::kStage + h * Cfg::kTile));
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_f16(tmem + Cfg::kColS, qd + 2 * k, kd + 2 * k, ID_S, h + k > 0 ? 1u : 0u);
        }
        mma_commit(s_full);
        mma_commit(&k_empty[st]);
      };
      auto issue_pv = [&](int j) {
        const int st = j % kStages;
#pragma unroll
        for (int h = 0; h < Cfg::kHalves; ++h) {
          const uint64_t vd = sw128_desc(smem_u32(smem + Cfg::kOffV + st * Cfg::kStage + h * Cfg::kTile));
#pragma unroll
          for (int k = 0; k < kPkKeys / 16; ++k)
            mma_f16_ta(tmem + Cfg::kColO + 64 * h, tmem + Cfg::kColP + 8 * k, vd + static_cast<uint64_t>(k) * (2048 >> 4),
                       ID_O, (j > 0 || k > 0) ? 1u : 0u);
        }
        mma_commit(o_full);
        mma_commit(&v_empty[st]);
      };
      auto k_ready = [&](int j) { return mbar_wait(&k_full[j % kStages], static_cast<uint32_t>(j / kStages) & 1u, a.status); };
      bool ok = mbar_wait(q_full, 0, a.status) && k_ready(0);
      if (ok) {
        tc_fence_after();
        issue_s(0);
      }
      for (int j = 0; j < n_tiles && ok; ++j) {
        if (!Cfg::kAlias && j + 1 < n_tiles) {  // the next S beside this tile's P V
          ok = k_ready(j + 1) && mbar_wait(s_free, j & 1u, a.status);
          if (!ok) break;
          tc_fence_after();
          issue_s(j + 1);
        }
        ok = mbar_wait(&v_full[j % kStages], static_cast<uint32_t>(j / kStages) & 1u, a.status) &&
             mbar_wait(p_full, j & 1u, a.status);
        if (!ok) break;
        tc_fence_after();
        issue_pv(j);
        if (Cfg::kAlias && j + 1 < n_tiles) {  // over P, once P V (issued before it) has read it
          ok = k_ready(j + 1);
          if (!ok) break;
          tc_fence_after();
          issue_s(j + 1);
        }
      }
    }
  } else {
    const int quad = warp & 3;
    const int rl = quad * 32 + lane;
    const bool live = rl < rows;
    const int r = row_first + (live ? rl : 0);
    const int tok = r / a.group, head = kvh * a.group + r % a.group;
    uint8_t* q_tile = smem + Cfg::kOffQ;
    {
      const __nv_bfloat16* qr = a.q + (start + tok) * a.ldq + head * HD;
      uint4 u[HD / 8];
#pragma unroll
      for (int c = 0; c < HD / 8; ++c) u[c] = live ? __ldg(reinterpret_cast<const uint4*>(qr) + c) : make_uint4(0, 0, 0, 0);
      if (a.cos) {
        const long long p = static_cast<long long>(start + tok) * (HD / 2);
#pragma unroll
        for (int c = 0; c < HD / 16; ++c) {
          __nv_bfloat162* h1 = reinterpret_cast<__nv_bfloat162*>(&u[c]);
          __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&u[c + HD / 16]);
          float cv[8], sv[8];
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float4 x = __ldg(reinterpret_cast<const float4*>(a.cos + p + 8 * c + e));
            const float4 y = __ldg(reinterpret_cast<const float4*>(a.sin + p + 8 * c + e));
            cv[e] = x.x, cv[e + 1] = x.y, cv[e + 2] = x.z, cv[e + 3] = x.w;
            sv[e] = y.x, sv[e + 1] = y.y, sv[e + 2] = y.z, sv[e + 3] = y.w;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 x1 = __bfloat1622float2(h1[e]), x2 = __bfloat1622float2(h2[e]);
            h1[e] = __floats2bfloat162_rn(__fsub_rn(__fmul_rn(x1.x, cv[2 * e]), __fmul_rn(x2.x, sv[2 * e])),
                                          __fsub_rn(__fmul_rn(x1.y, cv[2 * e + 1]), __fmul_rn(x2.y, sv[2 * e + 1])));
            h2[e] = __floats2bfloat162_rn(__fadd_rn(__fmul_rn(x2.x, cv[2 * e]), __fmul_rn(x1.x, sv[2 * e])),
                                          __fadd_rn(__fmul_rn(x2.y, cv[2 * e + 1]), __fmul_rn(x1.y, sv[2 * e + 1])));
          }
        }
      }
#pragma unroll
      for (int c = 0; c < HD / 8; ++c)
        *reinterpret_cast<uint4*>(q_tile + (c / 8) * Cfg::kTile + rl * 128 + (((c % 8) ^ (rl & 7)) << 4)) = u[c];
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }

    const uint32_t lane_base = tmem + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t s_addr = lane_base + Cfg::kColS;
    const uint32_t p_addr = lane_base + Cfg::kColP;
    const uint32_t o_addr = lane_base + Cfg::kColO;
    const float sc = a.scale_log2;
    const int vis = live ? tok + 1 : 1;  // keys [0, vis) are visible to this row
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      if (!mbar_wait(s_full, j & 1u, a.status)) {
        ok = false;
        break;
      }
      tc_fence_after();
      uint32_t sv[kPkKeys];
#pragma unroll
      for (int c = 0; c < kPkKeys; c += 32) tmem_ld32(s_addr + c, sv + c);
      tmem_ld_wait();
      if (!Cfg::kAlias) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_free);
      }
      const int nvis = vis - j * kPkKeys;
      if (nvis < kPkKeys) {
#pragma unroll
        for (int e = 0; e < kPkKeys; ++e)
          if (e >= nvis) sv[e] = __float_as_uint(-INFINITY);
      }
      float mx[8];
#pragma unroll
      for (int t = 0; t < 8; ++t) mx[t] = __uint_as_float(sv[t]);
#pragma unroll
      for (int e = 8; e < kPkKeys; e += 8)
#pragma unroll
        for (int t = 0; t < 8; ++t) mx[t] = fmaxf(mx[t], __uint_as_float(sv[e + t]));
      const float m_tile =
          fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7]))) * sc;
      const bool raise = m_tile > m + kPkStaleMax;
      const float alpha = raise ? ex2(m - m_tile) : 1.f;
      if (raise) m = m_tile;
      const float neg_m = m == -INFINITY ? 0.f : -m;
      uint32_t pk[kPkKeys / 2];
      float ls[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < kPkKeys; e += 2) {
        float x0, x1;
        fma2(x0, x1, __uint_as_float(sv[e]), __uint_as_float(sv[e + 1]), sc, neg_m);
        const float p0 = ex2(x0), p1 = ex2(x1);
        const int t = (e >> 1) & 3;
        add2(ls[2 * t], ls[2 * t + 1], p0, p1);
        pk[e >> 1] = bf16x2(p0, p1);
      }
      const float s0 = (ls[0] + ls[2]) + (ls[4] + ls[6]), s1 = (ls[1] + ls[3]) + (ls[5] + ls[7]);
      if (j > 0) {
        if (!mbar_wait(o_full, (j - 1) & 1u, a.status)) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
#pragma unroll
      for (int c = 0; c < kPkKeys / 2; c += 16) tmem_st16(p_addr + c, pk + c);
      if (j > 0 && __any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int c = 0; c < HD; c += 32) {
          uint32_t ov[32];
          tmem_ld32(o_addr + c, ov);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 32; ++e) ov[e] = __float_as_uint(__uint_as_float(ov[e]) * alpha);
          tmem_st16(o_addr + c, ov);
          tmem_st16(o_addr + c + 16, ov + 16);
        }
      }
      l = l * alpha + (s0 + s1);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    if (ok && mbar_wait(o_full, (n_tiles - 1) & 1u, a.status)) {
      tc_fence_after();
      const float inv = 1.f / l;
      const long long o_at = (start + tok) * a.ldo + head * HD;
      uint4* dst = reinterpret_cast<uint4*>(a.o + o_at);
      uint32_t worst = 0u;
#pragma unroll
      for (int c = 0; c < HD; c += 32) {
        uint32_t ov[32];
        tmem_ld32(o_addr + c, ov);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const float y = __uint_as_float(ov[e]) * inv;
          ov[e] = __float_as_uint(y);
          worst = max(worst, ov[e] & 0x7FFFFFFFu);
        }
        if (live) {
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* y = reinterpret_cast<const float*>(ov) + 8 * q;
            dst[c / 8 + q] = make_uint4(bf16x2(y[0], y[1]), bf16x2(y[2], y[3]), bf16x2(y[4], y[5]), bf16x2(y[6], y[7]));
          }
        }
      }
      __syncwarp();
      unsigned again = __ballot_sync(0xffffffffu, live && worst >= 0x7F800000u);
      while (again) {
        const int w = __ffs(again) - 1;
        again &= again - 1;
        packed_row_alone<HD>(a, q_tile, quad * 32 + w, start, __shfl_sync(0xffffffffu, tok, w), kvh,
                             __shfl_sync(0xffffffffu, o_at, w));
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, Cfg::kCols);
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

template <int HD>
int launch_packed(const CUtensorMap& tk, const CUtensorMap& tv, const PackedArgs& a, dim3 grid, cudaStream_t stream) {
  static std::atomic<uint64_t> configured{0};  // a bit per device
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && !(configured.load() >> dev & 1)) {
    const cudaError_t e = cudaFuncSetAttribute(attention_packed_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               PkCfg<HD>::kSmem);
    if (e != cudaSuccess) return launch_error(e);
    configured.fetch_or(1ull << dev);
  }
  return launch_kernel(attention_packed_kernel<HD>, grid, dim3(kPkThreads), PkCfg<HD>::kSmem, stream, tk, tv, a);
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
  // the blocks of all sequences: at most one part-filled block each
  const int64_t full = rows * a.group / kPkRows;
  const int64_t blocks = full + (n_seqs < rows ? n_seqs : rows);
  const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(nkv));
  return hd == 64 ? launch_packed<64>(tk, tv, a, grid, stream) : launch_packed<128>(tk, tv, a, grid, stream);
}
