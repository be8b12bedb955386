// The head_dim 128 kernels of attention_pages.cuh (a source of their own: they compile beside the others).
#include "attention_pages.cuh"

namespace so101 {

int attention_pages_128(const PagesArgs& a, int64_t workspace_bytes, int64_t n_tickets, cudaStream_t stream) {
  return attention_pages_run<128>(a, workspace_bytes, n_tickets, stream);
}

}  // namespace so101
