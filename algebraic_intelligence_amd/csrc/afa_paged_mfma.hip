// The attention of a step's tokens over the paged cache on the matrix cores: the instances for the requests' own keys
// (afa_paged_attend.h), and what their plans need.
#include "afa_paged_attend.h"

namespace afa {

bool paged_fast_supported(const afa_paged_plan& p) {
  const int64_t d = p.head_dim;
  return p.dtype != AFA_F64 && (d == 32 || d == 48 || d == 64 || d == 96 || d == 128 || d == 256) && p.page_size >= 8 &&
         (p.page_size & (p.page_size - 1)) == 0;
}

size_t paged_fast_workspace(const afa_paged_plan& p, const PagedCut& c) {
  return (size_t)(p.kv_heads * 2 * c.slots * c.rows) * (size_t)(p.head_dim + 2) * 4;
}

hipError_t paged_fwd_fast_launch(const PagedFwdArgs& a, const PagedCut& c, const PrefixSums& shared, void* ws, hipStream_t st) {
  return fast_launch<false>(paged_fast_args(a, c, a.ps, shared, ws), c.rows, st);
}

}  // namespace afa
