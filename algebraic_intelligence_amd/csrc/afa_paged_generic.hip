// AFA of a serving step's tokens over the paged cache, for any head_dim up to 1024, page size, stride
// and type: one workgroup for a token's row of one head.
//
//   out = sum_j w_j v_j / (sum_j w_j + Omega),  w_j = rho(q.k_j / sqrt(D))^8
//
// over the keys of a prefix that all requests share, where there is one, the cached keys and the drafted ones that
// the token's mask shows.  The sums are additive, so keys
// go by in blocks of one key a thread with no running maximum; a masked key is left out of both sums,
// whatever its page holds.  Latency bounds it (a key row a thread, 126 us for one token over 700 in 12 heads of
// 64); it is here for the calls that the matrix-core kernel does not take, and to check that one.
#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

constexpr int ROW_KEYS = 256, MAX_DIM = 1024;

template <int DT, typename A>
__device__ __forceinline__ A elem(const void* p, int64_t i) {
  if constexpr (DT == AFA_F64) return ((const double*)p)[i];
  else return Elem<DT>::load(p, i);
}

template <int DT>
__global__ __launch_bounds__(ROW_KEYS) void afa_paged_row_kernel(const PagedFwdArgs a) {
  using A = typename std::conditional<DT == AFA_F64, double, float>::type;
  constexpr int ESZ = DT == AFA_F64 ? 8 : DT == AFA_F32 ? 4 : 2;
  __shared__ A q_row[MAX_DIM], weight[ROW_KEYS];
  __shared__ const char* row[ROW_KEYS];  // the key's v row, nullptr where it is masked
  const afa_paged_plan& p = a.plan;
  const int D = (int)p.head_dim, H = (int)p.heads, tid = threadIdx.x;
  const int64_t t = blockIdx.x / H;
  const int h = blockIdx.x % H, hk = h / a.group, r = p.token_request[t];
  A* den = (A*)a.denom;
  if (r < 0 && !a.zero_tail) return;
  const bool live = r >= 0 && p.status[r] == AFA_PAGED_OK;
  const int start = live ? p.starts[r] : 0, n = live ? p.starts[r + 1] - start : 0, i = (int)t - start;
  const int c = live ? a.sched.cached[r] : 0, keys = live ? c + n : 0;
  const int W = (int)(p.max_tree / 64);
  const bool tree = a.masks != nullptr && n <= p.max_tree;
  for (int d = tid; d < D; d += ROW_KEYS) q_row[d] = elem<DT, A>(a.q, t * a.q_t + h * a.q_h + d);
  A acc[MAX_DIM / ROW_KEYS] = {}, sum = 0;
  // `count` keys, of which locate(pos, k, v) gives the rows, or leaves nullptr
  auto meet = [&](int count, auto locate) {
    for (int base = 0; base < count; base += ROW_KEYS) {
      __syncthreads();
      const int pos = base + tid;
      const char *k = nullptr, *v = nullptr;
      if (pos < count) locate(pos, k, v);
      A w = 0;
      if (k != nullptr) {
        A s = 0;
        for (int d = 0; d < D; ++d) s += q_row[d] * elem<DT, A>(k, d);
        w = rho8_above_0(s, a.scale);
        sum += w;
      }
      row[tid] = v;
      weight[tid] = w;
      __syncthreads();
      const int m = min(ROW_KEYS, count - base);
      for (int d = tid, u = 0; d < D; d += ROW_KEYS, ++u)
        for (int j = 0; j < m; ++j)
          if (row[j] != nullptr) acc[u] += weight[j] * elem<DT, A>(row[j], d);
    }
  };
  if (live && a.prefix.len > 0) {
    const PrefixKeys& x = a.prefix;
    meet(x.len, [&](int pos, const char*& k, const char*& v) {
      k = (const char*)x.k + (hk * x.k_head + pos * x.k_key) * ESZ;
      v = (const char*)x.v + (hk * x.v_head + pos * x.v_key) * ESZ;
    });
  }
  meet(keys, [&](int pos, const char*& k, const char*& v) {
    bool sees = true;
    if (pos >= c) {
      const int j = pos - c;
      sees = tree ? (a.masks[t * W + j / 64] >> (j & 63)) & 1 : j <= i;
    }
    const int page = sees ? p.block_tables[r * p.table_width + pos / p.page_size] : -1;
    if (page < 0 || page >= p.num_pages) return;
    const int64_t at = pos % p.page_size;
    k = (const char*)a.k_pages + (page * a.ps.k_page + hk * a.ps.k_head + at * a.ps.k_slot) * ESZ;
    v = (const char*)a.v_pages + (page * a.ps.v_page + hk * a.ps.v_head + at * a.ps.v_slot) * ESZ;
  });
  __syncthreads();
  weight[tid] = sum;
  __syncthreads();
  for (int o = ROW_KEYS / 2; o > 0; o >>= 1) {
    if (tid < o) weight[tid] += weight[tid + o];
    __syncthreads();
  }
  const A total = weight[0] + (A)a.omega;
  const int64_t to = t * H + h;
  if (den != nullptr && tid == 0) den[to] = r < 0 ? (A)0 : total;
  for (int d = tid, u = 0; d < D; d += ROW_KEYS, ++u) {
    // no key seen: 0, also where there is no sink
    const A y = total == 0 ? (A)0 : acc[u] / total;
    if constexpr (DT == AFA_F64) ((double*)a.out)[to * D + d] = y;
    else Elem<DT>::store(a.out, to * D + d, y);
  }
}

}  // namespace

hipError_t paged_fwd_generic_launch(const PagedFwdArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.plan.max_tokens * a.plan.heads)), block(ROW_KEYS);
  switch ((int)a.plan.dtype) {
    case AFA_F32: hipLaunchKernelGGL((afa_paged_row_kernel<AFA_F32>), grid, block, 0, st, a); break;
    case AFA_BF16: hipLaunchKernelGGL((afa_paged_row_kernel<AFA_BF16>), grid, block, 0, st, a); break;
    case AFA_F16: hipLaunchKernelGGL((afa_paged_row_kernel<AFA_F16>), grid, block, 0, st, a); break;
    default: hipLaunchKernelGGL((afa_paged_row_kernel<AFA_F64>), grid, block, 0, st, a); break;
  }
  return hipGetLastError();
}

}  // namespace afa
