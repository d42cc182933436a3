// Requests of more than `budget` cached tokens cut back to it: their `first` oldest tokens stay, their `recent`
// newest, and of the others those of the largest weight, the lower index among equal ones.  What stays keeps its
// order: token kept[i] moves to place i, in k, in v and in the weights.
//
// Two launches.  The first finds, one workgroup a request, the weight from which on tokens stay, by its bits from
// the top (four passes over the weights, eight bits each, in LDS), and lists the tokens that do.  The second moves
// rows in place: kept[i] >= i and both rise, so that one workgroup that goes through a head's rows in order, reads a
// batch of them, waits and writes it, never writes over a row that it has still to read.
#include <initializer_list>

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

constexpr int PICK = 1024, BINS = 256;

// Bits whose unsigned order is that of the weights: -0 and 0 alike, NaN above infinity.
__device__ __forceinline__ unsigned order_bits(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sums of x over the threads before this one; all: over the workgroup.
__device__ __forceinline__ int before(int x, int* lds, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s, o);
    if (lane >= o) s += u;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < PICK / 64; ++w) {
    if (w == wave) base = all;
    all += lds[w];
  }
  return base + s - x;
}

__global__ __launch_bounds__(PICK) void afa_paged_pick_kernel(const EvictArgs a) {
  __shared__ int bins[BINS], scan[PICK / 64], found[2];
  const int r = blockIdx.x, tid = threadIdx.x;
  const int64_t width = a.table_width * a.page_size;
  const int held = (int)min(max((int64_t)a.held[r], (int64_t)0) * a.page_size, width);
  const int c = min(max(a.cached[r], 0), held), budget = a.budget, m = min(c, budget);
  const float* w = a.weights + r * a.row;
  float* left = a.left + r * width;
  int32_t* kept = a.kept + (int64_t)r * budget;
  int32_t* moved = a.kept + a.requests * budget + r;
  if (tid == 0) a.lens[r] = m;
  for (int64_t i = m + tid; i < width; i += PICK) left[i] = 0.0f;
  if (c <= budget) {
    for (int i = tid; i < m; i += PICK) left[i] = w[i];
    if (tid == 0) *moved = m;
    return;
  }
  // tokens [lo, hi) are chosen from; `need` of them stay
  const int lo = a.first, hi = c - a.recent;
  int need = budget - a.first - a.recent;
  unsigned prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < BINS; i += PICK) bins[i] = 0;
    __syncthreads();
    for (int i = lo + tid; i < hi; i += PICK) {
      const unsigned u = order_bits(w[i]);
      if (shift == 24 || u >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&bins[u >> shift & 255], 1);
    }
    __syncthreads();
    // the bin in which the need-th largest lies
    if (tid == 0) {
      int b = BINS - 1, above = 0;
      while (b > 0 && above + bins[b] < need) above += bins[b--];
      found[0] = b;
      found[1] = above;
    }
    __syncthreads();
    prefix |= (unsigned)found[0] << shift;
    need -= found[1];
    __syncthreads();
  }
  // above `prefix` all stay, and the first `need` that equal it
  int at = 0, equal = 0, start = budget;
  for (int base = 0; base < c; base += PICK) {
    const int i = base + tid;
    const bool in = i < c, sure = in && (i < lo || i >= hi);
    const unsigned u = in && !sure ? order_bits(w[i]) : 0;
    const bool same = in && !sure && u == prefix;
    int all;
    const int rank = equal + before(same, scan, all);
    equal += all;
    const bool stays = sure || (in && !sure && (u > prefix || (same && rank < need)));
    const int to = at + before(stays, scan, all);
    at += all;
    if (stays) {
      kept[to] = i;
      left[to] = w[i];
      if (to != i) start = min(start, to);
    }
  }
  // the first place whose token moves
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) start = min(start, __shfl_xor(start, o));
  __syncthreads();
  if ((tid & 63) == 0) scan[tid >> 6] = start;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < PICK / 64; ++k) start = min(start, scan[k]);
    *moved = start;
  }
}

// Rows as `units` of type T each; U of them a thread and batch.
template <typename T>
__global__ __launch_bounds__(256) void afa_paged_move_kernel(const EvictArgs a, int units) {
  constexpr int U = 8;
  int64_t item = blockIdx.x;
  const bool is_v = item & 1;
  item >>= 1;
  const int hk = (int)(item % a.kv_heads), r = (int)(item / a.kv_heads);
  const int m = a.lens[r], start = a.kept[a.requests * a.budget + r];
  const int32_t *kept = a.kept + (int64_t)r * a.budget, *table = a.block_tables + (int64_t)r * a.table_width;
  char* pages = (char*)(is_v ? a.v_pages : a.k_pages);
  const int64_t page = (is_v ? a.ps.v_page : a.ps.k_page) * a.esz, slot = (is_v ? a.ps.v_slot : a.ps.k_slot) * a.esz;
  pages += hk * (is_v ? a.ps.v_head : a.ps.k_head) * a.esz;
  auto place = [&](int pos) -> char* {
    const int at = (int)(pos / a.page_size), id = table[at];
    return id < 0 || id >= a.num_pages ? nullptr : pages + id * page + (pos - at * a.page_size) * slot;
  };
  const int64_t all = (int64_t)(m - start) * units;
  for (int64_t base = 0; base < all; base += 256 * U) {
    T x[U];
    char* to[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t e = base + u * 256 + threadIdx.x;
      to[u] = nullptr;
      if (e >= all) continue;
      const int i = start + (int)(e / units), in = (int)(e % units);
      const char* from = place(kept[i]);
      if (from == nullptr) continue;
      to[u] = place(i);
      if (to[u] == nullptr) continue;
      to[u] += in * sizeof(T);
      x[u] = *(const T*)(from + in * sizeof(T));
    }
    // read by all before any is written
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (to[u] != nullptr) *(T*)to[u] = x[u];
  }
}

}  // namespace

size_t paged_evict_workspace(int64_t requests, int64_t budget) { return (size_t)(requests * (budget + 1)) * 4; }

hipError_t paged_evict_launch(const EvictArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(afa_paged_pick_kernel, dim3((unsigned)a.requests), dim3(PICK), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((unsigned)(2 * a.requests * a.kv_heads)), block(256);
  int64_t unit = 16;
  const int64_t bytes = a.head_dim * a.esz;
  for (int64_t v : {(int64_t)(uintptr_t)a.k_pages, (int64_t)(uintptr_t)a.v_pages, bytes, a.ps.k_page * a.esz, a.ps.k_head * a.esz,
                    a.ps.k_slot * a.esz, a.ps.v_page * a.esz, a.ps.v_head * a.esz, a.ps.v_slot * a.esz})
    while (v % unit != 0) unit /= 2;
  const int units = (int)(bytes / unit);
  switch (unit) {
    case 16: hipLaunchKernelGGL((afa_paged_move_kernel<u32x4_t>), grid, block, 0, st, a, units); break;
    case 8: hipLaunchKernelGGL((afa_paged_move_kernel<u32x2_t>), grid, block, 0, st, a, units); break;
    case 4: hipLaunchKernelGGL((afa_paged_move_kernel<unsigned>), grid, block, 0, st, a, units); break;
    default: hipLaunchKernelGGL((afa_paged_move_kernel<unsigned short>), grid, block, 0, st, a, units); break;
  }
  return hipGetLastError();
}

}  // namespace afa
