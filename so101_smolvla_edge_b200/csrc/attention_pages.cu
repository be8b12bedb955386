// Entry point of the attention over 8-bit pages (attention_pages.cuh), and its head_dim 64 kernels.
#include "attention_pages.cuh"

namespace so101 {

int attention_pages_64(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream) {
  return attention_pages_run<64>(a, workspace_bytes, n_tickets, stream);
}
int attention_pages_128(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream);
// attention_pages_tc.cu
bool attention_pages_tc(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream, int* rc);

}  // namespace so101

using namespace so101;

extern "C" int so101_attention_pages(const void* q, int64_t ldq, void* o, int64_t ldo, int64_t rows,
                                     const so101_kv_pages* c, int layer, int nq, const int* starts, const int* seqs,
                                     int n_seqs, int64_t max_q, int causal, float scale, const float* cos,
                                     const float* sin, void* workspace, int64_t workspace_bytes, int* tickets,
                                     int64_t n_tickets, cudaStream_t stream) {
  if (!kv_pages_ok(c) || layer < 0 || layer >= c->n_layers || nq < 1 || nq % c->n_kv || n_seqs < 0 ||
      n_seqs > (1 << 24) || rows < 0 || rows > (1 << 30) || max_q < 1 || (cos == nullptr) != (sin == nullptr) ||
      !(scale > 0.f && scale < INFINITY))
    return SO101_ERR_ARG;
  if (!starts && (rows != n_seqs || max_q != 1)) return SO101_ERR_ARG;
  if (n_seqs == 0 || rows == 0) return SO101_OK;
  if (!q || !o) return SO101_ERR_ARG;
  if (!workspace || !tickets) return SO101_ERR_WORKSPACE;
  const auto a16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const int64_t width = static_cast<int64_t>(nq) * c->hd;
  if (!a16(q) || ldq % 8 || reinterpret_cast<uintptr_t>(o) % 8 || (rows > 1 && (ldq < width || ldo < width)) ||
      nq > 65535 || ldo % 4 || (cos && (!a16(cos) || !a16(sin))))
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
  a.group_inv = static_cast<uint32_t>(((1ULL << 32) + a.group - 1) / a.group);
  a.o_wide = a16(o) && ldo % 8 == 0;
  a.n_seqs = n_seqs;
  a.max_q = static_cast<int>(max_q < rows ? max_q : rows);
  a.status = status_ptr();
  int rc = SO101_OK;
  if (attention_pages_tc(a, workspace_bytes, n_tickets, stream, &rc)) return rc;
  return c->hd == 64 ? attention_pages_64(a, workspace_bytes, n_tickets, stream)
                     : attention_pages_128(a, workspace_bytes, n_tickets, stream);
}
