// New tokens into the 8-bit pages (so101_kv_append) and cached tokens back as rows (so101_kv_read).
//
// Per (page, kv head), for keys and values apart, with a = max |x| over the page's new tokens:
//   s = 2^e, e = ceil(log2(a / 127)) in [-126, 121];  s' = max(s_old, s);  code = rint(x / s')
//   older codes of a part-filled page: rint(code * s_old / s')
// A power of two costs at most one bit of the scale's fit (the steps are up to twice as wide as with
// a / 127 itself), and makes every product exact: codes do not depend on how the division is
// computed, and re-rounding an older code when a later token raises the scale halves its precision
// at most log2 times, so that all re-roundings together stay under one step of the last scale.
// (With s = a / 127 each small rise would round every older code again, by half a step each time.)
#include "kv_pages.cuh"

namespace so101 {

struct AppendArgs {
  KvPages c;
  const __nv_bfloat16* x[2];  // new keys, new values
  long long ld[2];
  long long rows;
  const int* starts;
  const int* seqs;
  const int* refused;
  const float* cos;
  const float* sin;
  int layer;
  int* status;
};

// The scale's exponent field for the largest magnitude (its bit pattern, finite): 2^e with
// a <= 127 * 2^e. 127 = 1.984375 * 2^6, so e is a's exponent - 6, and one more where a's mantissa is
// past 1.984375 (0x7E0000). A zero or subnormal a lands on the lowest scale, 2^-126.
__device__ __forceinline__ uint32_t scale_bits(uint32_t amax) {
  const int e = static_cast<int>(amax >> 23) - 6 + ((amax & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, 1), 121 + 127)) << 23;
}

__device__ __forceinline__ void unpack8(const uint4& u, float (&f)[8]) {
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float2 p = __bfloat1622float2(h[e]);
    f[2 * e] = p.x;
    f[2 * e + 1] = p.y;
  }
}

__device__ __forceinline__ uint2 codes8(const float (&f)[8], float inv) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int q = min(max(__float2int_rn(f[e] * inv), -127), 127);
    w[e >> 2] |= (static_cast<uint32_t>(q) & 0xFFu) << (8 * (e & 3));
  }
  return make_uint2(w[0], w[1]);
}

constexpr int kAppendThreads = 128;

// One CTA per (touched page, kv head, keys or values, sequence): the page's new rows are read once
// into registers (at most 64 x 128 elements: four pairs of 8-element pieces a thread at head_dim 64,
// eight at 128), the maximum taken over the CTA, then the codes written. A piece and its rotary
// partner hd / 2 later belong to one thread.
template <int HD>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const AppendArgs a) {
  constexpr int kPairs = HD / 16;                                // pairs of pieces in a row
  constexpr int kMost = 64 * kPairs / kAppendThreads;            // pairs per thread
  __shared__ uint32_t warp_max[kAppendThreads / 32];
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = a.c;
  const int head = blockIdx.y >> 1, which = blockIdx.y & 1;
  int seq, row0, n;
  if (!kv_rows(c, a.starts, a.seqs, blockIdx.z, a.rows, seq, row0, n, a.status)) return;
  const int refused = a.refused[seq];  // there is no room for these rows: the length does not count them
  const int len = kv_length(c, seq, a.status);
  const int old = len - n;
  if (old < 0 || (refused && n > 0)) {
    if (threadIdx.x == 0) record_error(a.status, SO101_ERR_PAGES);
    return;
  }
  const int at = old / c.page + static_cast<int>(blockIdx.x);  // the page's place in the sequence
  const int lo = max(old, at * c.page), hi = min(len, (at + 1) * c.page);
  if (lo >= hi) {
    // more new tokens than the grid covers (its last CTA of the sequence sees them left over)
    return;
  }
  if (blockIdx.x == gridDim.x - 1 && len > (at + 1) * c.page && threadIdx.x == 0)
    record_error(a.status, SO101_ERR_PAGES);
  const int held = lo - at * c.page;  // older tokens of the page
  const __nv_bfloat16* src = a.x[which] + static_cast<long long>(row0 + lo - old) * a.ld[which] + head * HD;
  const long long ld = a.ld[which];
  const bool turn = which == 0 && a.cos != nullptr;
  const int pairs = (hi - lo) * kPairs;
  // the page's number is looked up while the rows are on their way
  uint4 u[kMost][2];
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int p = threadIdx.x + i * kAppendThreads;
    if (p < pairs) {
      const __nv_bfloat16* row = src + p / kPairs * ld + p % kPairs * 8;
      u[i][0] = __ldg(reinterpret_cast<const uint4*>(row));
      u[i][1] = __ldg(reinterpret_cast<const uint4*>(row + HD / 2));
    }
  }
  const int id = c.table[static_cast<long long>(seq) * c.max_pages + at];
  if (id < 0 || id >= c.n_pages) {
    if (threadIdx.x == 0) record_error(a.status, SO101_ERR_PAGES);
    return;
  }
  float* scale = (which ? c.v_scale : c.k_scale) + kv_scale_at(c, a.layer, id, head);
  const float was = held ? *scale : 0.f;
  float x[kMost][2][8];
  uint32_t big = 0u;
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int p = threadIdx.x + i * kAppendThreads;
    if (p < pairs) {
      unpack8(u[i][0], x[i][0]);
      unpack8(u[i][1], x[i][1]);
      if (turn) {
        const long long t = static_cast<long long>(row0 + lo - old + p / kPairs) * (HD / 2) + p % kPairs * 8;
#pragma unroll
        for (int e0 = 0; e0 < 8; e0 += 4) {
          const float4 c4 = __ldg(reinterpret_cast<const float4*>(a.cos + t + e0));
          const float4 s4 = __ldg(reinterpret_cast<const float4*>(a.sin + t + e0));
          const float cv[4] = {c4.x, c4.y, c4.z, c4.w}, sv[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u0 = x[i][0][e0 + e], u1 = x[i][1][e0 + e];
            x[i][0][e0 + e] = __fsub_rn(__fmul_rn(u0, cv[e]), __fmul_rn(u1, sv[e]));
            x[i][1][e0 + e] = __fadd_rn(__fmul_rn(u1, cv[e]), __fmul_rn(u0, sv[e]));
          }
        }
      }
      // magnitudes compare as integers; a NaN is past infinity
#pragma unroll
      for (int e = 0; e < 8; ++e)
        big = max(big, max(__float_as_uint(x[i][0][e]) & 0x7FFFFFFFu, __float_as_uint(x[i][1][e]) & 0x7FFFFFFFu));
    }
  }
  big = __reduce_max_sync(0xffffffffu, big);
  if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = big;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kAppendThreads / 32; ++w) big = max(big, warp_max[w]);
  const bool lost = big >= 0x7F800000u || was != was;
  float s = __uint_as_float(scale_bits(big));
  if (was > s) s = was;
  const float inv = lost ? 0.f : 1.f / s;  // a power of two: exact
  int8_t* codes = (which ? c.v : c.k) + kv_code_at(c, a.layer, id, head);
  if (threadIdx.x == 0 && (held == 0 || lost || s != was)) *scale = lost ? __uint_as_float(0x7FC00000u) : s;
  if (held && !lost && s != was) {  // older codes to the wider step
    const float ratio = was * inv;
    for (int p = threadIdx.x; p < held * (HD / 8); p += kAppendThreads) {
      uint2* w = reinterpret_cast<uint2*>(codes) + p;
      const uint2 u = *w;
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        f[e] = static_cast<float>(static_cast<int8_t>((e < 4 ? u.x : u.y) >> (8 * (e & 3))));
      *w = codes8(f, ratio);
    }
  }
#pragma unroll
  for (int i = 0; i < kMost; ++i) {
    const int p = threadIdx.x + i * kAppendThreads;
    if (p < pairs) {
      const int r = p / kPairs, d = p % kPairs * 8;
      int8_t* dst = codes + (held + r) * HD + d;
      *reinterpret_cast<uint2*>(dst) = codes8(x[i][0], inv);
      *reinterpret_cast<uint2*>(dst + HD / 2) = codes8(x[i][1], inv);
    }
  }
}

struct ReadArgs {
  KvPages c;
  const int* starts;
  const int* seqs;
  const int* first;
  __nv_bfloat16* out[2];
  long long ld[2];
  int n_seqs, rows, layer;
  int* status;
};

constexpr int kReadRows = 8, kReadThreads = 256;

// 8 rows per CTA. Where the rows lie is worked out once, a thread per row (the sequence by counting the
// starts at or before it, in one barrier per 256 of them); then a thread takes 16 codes of a row at a
// time: one 16-byte load, two 16-byte stores. Latency bounds a small call (one token of each of 64 sequences appended
// and read back, five heads of 64: 6.9 us for both kernels; 10.7 when each piece looked its sequence, length and page
// up again), the stores' bandwidth a large one.
template <int HD>
__global__ void __launch_bounds__(kReadThreads) kv_read_kernel(const ReadArgs a) {
  __shared__ int page_of[kReadRows], slot_of[kReadRows];
  grid_dep_launch();
  grid_dep_wait();
  const KvPages& c = a.c;
  const int r0 = blockIdx.x * kReadRows;
  int s0 = -1;
  for (int i0 = 0; i0 <= a.n_seqs; i0 += kReadThreads) {
    const int i = i0 + static_cast<int>(threadIdx.x);
    s0 += __syncthreads_count(i <= a.n_seqs && __ldg(a.starts + i) <= r0);
  }
  if (threadIdx.x < kReadRows) {
    const int row = r0 + static_cast<int>(threadIdx.x);
    int id = -1, slot = 0;
    int i = s0;
    while (i < a.n_seqs && (i < 0 || __ldg(a.starts + i + 1) <= row)) ++i;
    if (row < a.rows && i >= 0 && i < a.n_seqs) {  // else a row outside every sequence
      const int seq = a.seqs ? __ldg(a.seqs + i) : i;
      const int tok = (a.first ? __ldg(a.first + i) : 0) + row - __ldg(a.starts + i);
      const bool there = seq >= 0 && seq < c.max_seqs && tok >= 0 && tok < c.max_pages * c.page;
      if (there) {
        const int len = c.lengths[seq];
        id = c.table[static_cast<long long>(seq) * c.max_pages + tok / c.page];
        slot = tok % c.page;
        if (tok >= len || id >= c.n_pages) id = -1;
      }
      if (id < 0) record_error(a.status, SO101_ERR_PAGES);
    }
    page_of[threadIdx.x] = id;
    slot_of[threadIdx.x] = slot;
  }
  __syncthreads();
  constexpr int kPieces = HD / 16;
  const int per_row = 2 * c.n_kv * kPieces;
#pragma unroll 2
  for (int p = threadIdx.x; p < kReadRows * per_row; p += kReadThreads) {
    const int r = p / per_row;
    int q = p - r * per_row;
    const int d = q % kPieces * 16;
    q /= kPieces;
    const int which = q >= c.n_kv ? 1 : 0, head = q - which * c.n_kv;
    const int id = page_of[r];
    if (id < 0) continue;
    const float s = (which ? c.v_scale : c.k_scale)[kv_scale_at(c, a.layer, id, head)];
    const int8_t* src = (which ? c.v : c.k) + kv_code_at(c, a.layer, id, head) + slot_of[r] * HD + d;
    const uint4 u = *reinterpret_cast<const uint4*>(src);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
    uint32_t y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t h = w[e >> 1] >> (16 * (e & 1));
      const __nv_bfloat162 b = __floats2bfloat162_rn(static_cast<float>(static_cast<int8_t>(h)) * s,
                                                     static_cast<float>(static_cast<int8_t>(h >> 8)) * s);
      y[e] = *reinterpret_cast<const uint32_t*>(&b);
    }
    uint4* dst = reinterpret_cast<uint4*>(a.out[which] + static_cast<long long>(r0 + r) * a.ld[which] + head * HD + d);
    dst[0] = make_uint4(y[0], y[1], y[2], y[3]);
    dst[1] = make_uint4(y[4], y[5], y[6], y[7]);
  }
}

}  // namespace so101

using namespace so101;

extern "C" int so101_kv_append(const so101_kv_pages* c, int layer, const void* k, int64_t ldk, const void* v,
                               int64_t ldv, int64_t rows, const int* starts, const int* seqs, int n_seqs,
                               int64_t max_new, const float* cos, const float* sin, cudaStream_t stream) {
  if (!kv_pages_ok(c) || layer < 0 || layer >= c->n_layers || n_seqs < 0 || n_seqs > 65535 || rows < 0 ||
      rows > (1 << 30) || max_new < 1 || (cos == nullptr) != (sin == nullptr))
    return SO101_ERR_ARG;
  if (!starts && (rows != n_seqs || max_new != 1)) return SO101_ERR_ARG;
  if (n_seqs == 0 || rows == 0) return SO101_OK;
  if (!k || !v) return SO101_ERR_ARG;
  const int width = c->n_kv * c->hd;
  const auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!a16(k) || !a16(v) || ldk % 8 || ldv % 8 || (cos && (!a16(cos) || !a16(sin))) || (rows > 1 && (ldk < width || ldv < width))) return SO101_ERR_ARG;
  AppendArgs a;
  a.c = *c;
  a.x[0] = static_cast<const __nv_bfloat16*>(k);
  a.x[1] = static_cast<const __nv_bfloat16*>(v);
  a.ld[0] = ldk;
  a.ld[1] = ldv;
  a.rows = rows;
  a.starts = starts;
  a.seqs = seqs;
  a.refused = c->scratch + kv_refused_at(*c);
  a.cos = cos;
  a.sin = sin;
  a.layer = layer;
  a.status = status_ptr();
  // n new tokens touch at most ceil((n - 1) / page) + 1 pages
  const int64_t most = max_new < rows ? max_new : rows;
  const dim3 grid(static_cast<unsigned>((most - 1 + c->page - 1) / c->page + 1), static_cast<unsigned>(2 * c->n_kv),
                  static_cast<unsigned>(n_seqs));
  return c->hd == 64 ? launch_kernel(kv_append_kernel<64>, grid, dim3(kAppendThreads), 0, stream, a)
                     : launch_kernel(kv_append_kernel<128>, grid, dim3(kAppendThreads), 0, stream, a);
}

extern "C" int so101_kv_read(const so101_kv_pages* c, int layer, const int* starts, const int* seqs, const int* first,
                             int n_seqs, int64_t rows, void* k_out, int64_t ldk, void* v_out, int64_t ldv,
                             cudaStream_t stream) {
  if (!kv_pages_ok(c) || layer < 0 || layer >= c->n_layers || n_seqs < 0 || rows < 0 ||
      rows > (1 << 30))
    return SO101_ERR_ARG;
  if (n_seqs == 0 || rows == 0) return SO101_OK;
  if (!starts || !k_out || !v_out) return SO101_ERR_ARG;
  const int width = c->n_kv * c->hd;
  const auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  if (!a16(k_out) || !a16(v_out) || ldk % 8 || ldv % 8 || ldk < width || ldv < width) return SO101_ERR_ARG;
  ReadArgs a;
  a.c = *c;
  a.starts = starts;
  a.seqs = seqs;
  a.first = first;
  a.out[0] = static_cast<__nv_bfloat16*>(k_out);
  a.out[1] = static_cast<__nv_bfloat16*>(v_out);
  a.ld[0] = ldk;
  a.ld[1] = ldv;
  a.n_seqs = n_seqs;
  a.rows = static_cast<int>(rows);
  a.layer = layer;
  a.status = status_ptr();
  const dim3 grid(static_cast<unsigned>((rows + kReadRows - 1) / kReadRows));
  return c->hd == 64 ? launch_kernel(kv_read_kernel<64>, grid, dim3(kReadThreads), 0, stream, a)
                     : launch_kernel(kv_read_kernel<128>, grid, dim3(kReadThreads), 0, stream, a);
}
