// A prefix that all requests share, met once by the rows of all the step's tokens: sum_j w_ij v_j and sum_j w_ij over its
// keys in fp32 (afa_paged_attend.h, PREFIX), for the attention of the requests' own keys to start from.  The sums are
// additive, so that nothing else passes between the two launches.
#include "afa_paged_attend.h"

namespace afa {

PagedCut prefix_cut(const afa_paged_plan& p, int cus) {
  afa_paged_plan all = p;
  all.max_new = p.max_tokens;  // the rows of one key head are those of all tokens
  return paged_cut(all, cus);
}

hipError_t prefix_sums_launch(const PagedFwdArgs& a, const PagedCut& c, const PrefixSums& shared, void* ws, hipStream_t st) {
  const PrefixKeys& x = a.prefix;
  return fast_launch<true>(paged_fast_args(a, c, PageStrides{0, x.k_head, x.k_key, 0, x.v_head, x.v_key}, shared, ws), c.rows, st);
}

}  // namespace afa
