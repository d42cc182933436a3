// What each token of the cache was given by a step's rows, added up:
//
//   W[r][j] += sum over the step's tokens i of request r that see j, and heads h, of  rho(s_ihj)^8 / d_ih
//
// with d the denominators that the step's attention returned, sink and prefix included.  A token of the step
// itself has no weight yet: its place is set, not added to.
#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

constexpr int KEYS = 256;

template <int DT, typename A>
__device__ __forceinline__ A elem_of(const void* p, int64_t i) {
  if constexpr (DT == AFA_F64) return ((const double*)p)[i];
  else return Elem<DT>::load(p, i);
}

// Any head_dim, type, stride and page size: a key a thread, its rows one after the other.
template <int DT>
__global__ __launch_bounds__(KEYS) void afa_paged_weight_key_kernel(const WeightArgs a, int64_t blocks, int64_t total) {
  using A = typename std::conditional<DT == AFA_F64, double, float>::type;
  const afa_paged_plan& p = a.plan;
  const int D = (int)p.head_dim, H = (int)p.heads, W = (int)(p.max_tree / 64);
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int r = (int)(item / blocks);
    const int pos = (int)(item % blocks) * KEYS + (int)threadIdx.x;
    const int start = p.starts[r], n = p.starts[r + 1] - start, c = a.sched.cached[r];
    if (p.status[r] != AFA_PAGED_OK || n <= 0 || pos >= c + n) continue;
    const int page = p.block_tables[r * p.table_width + pos / p.page_size];
    double sum = 0;  // of rows * heads terms, one after the other
    if (page >= 0 && page < p.num_pages) {
      const bool tree = a.masks != nullptr && n <= p.max_tree;
      const int j = pos - c;
      for (int i = j < 0 || tree ? 0 : j; i < n; ++i) {
        if (j >= 0 && tree && !((a.masks[(int64_t)(start + i) * W + j / 64] >> (j & 63)) & 1)) continue;
        for (int h = 0; h < H; ++h) {
          const int64_t t = start + i;
          const A d = ((const A*)a.denom)[t * H + h];
          if (d == 0) continue;  // the row saw no key
          const int64_t q = t * a.q_t + h * a.q_h;
          const int64_t k = page * a.k_page + h / a.group * a.k_head + pos % p.page_size * a.k_slot;
          A s = 0;
          for (int e = 0; e < D; ++e) s += elem_of<DT, A>(a.q, q + e) * elem_of<DT, A>(a.k_pages, k + e);
          if constexpr (DT == AFA_F64) sum += rho8_f64(s * a.scale) / d;
          else sum += (double)(rho8_ref(s * (float)a.scale) / d);
        }
      }
    }
    float* w = a.weights + r * a.row + pos;
    *w = (float)(pos < c ? *w + sum : sum);
  }
}

template <int DT>
hipError_t weight_keys_go(const WeightArgs& a, int cus, hipStream_t st) {
  const int64_t blocks = (a.plan.table_width * a.plan.page_size + KEYS - 1) / KEYS, total = a.plan.requests * blocks;
  const int64_t most = 16 * (int64_t)cus;
  hipLaunchKernelGGL((afa_paged_weight_key_kernel<DT>), dim3((unsigned)(total < most ? total : most)), dim3(KEYS), 0, st, a,
                     blocks, total);
  return hipGetLastError();
}

}  // namespace

hipError_t paged_weights_launch(const WeightArgs& a, int cus, hipStream_t st) {
  switch ((int)a.plan.dtype) {
    case AFA_F32: return weight_keys_go<AFA_F32>(a, cus, st);
    case AFA_BF16: return weight_keys_go<AFA_BF16>(a, cus, st);
    case AFA_F16: return weight_keys_go<AFA_F16>(a, cus, st);
    default: return weight_keys_go<AFA_F64>(a, cus, st);
  }
}

}  // namespace afa
