// Requests of more than `budget` cached tokens cut back to it: their `first` oldest tokens stay, their `recent`
// newest, and of the others those of the largest weight, the lower index among equal ones.  What stays keeps its
// order: token kept[i] moves to place i, in k, in v and in the weights.
//
// Two launches.  The first finds, one workgroup a request, the weight from which on tokens stay, by its bits from
// the top (three passes over the weights, up to eleven bits each, counted in LDS), and lists the tokens that do.
//
// The second moves rows in place.  A workgroup has one chunk of ROWS places of one head's k or v; its sources are behind its
// places, in places of later chunks, so it reads all of them, says so, and writes only once the chunks that read from
// its own places (earlier ones, two at most, as ROWS places hold at most ROWS sources) have said so too.  Chunks are handed
// out in their order by a counter, and a workgroup reads and says so before it waits: whatever one waits for has begun and
// waits for nothing before it says so, so every wait ends.
//
// HBM bounds the second launch: every row that moves is read and written once.
#include <algorithm>
#include <initializer_list>

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

constexpr int PICK = 1024, PICK_WAVES = PICK / 64;
constexpr int DIGIT = 11, BINS = 1 << DIGIT, COPIES = 8;  // of a bin, in banks of their own: neighbours often share one
constexpr int LOADS = 8;                                  // weights of a thread in flight
constexpr int MOVE = 256, BATCH = 8;                      // threads of a mover, and units that each holds

// The workspace: slots of the tokens that stay, page * page_size + offset, or -1 for a page of no pool (requests, budget); the first place that moves (requests,); sources before each chunk's
// places, and behind the last's (requests, chunks + 1); chunks handed out (requests, streams) and chunks that are read (requests, streams, chunks), a
// stream being one head's k or v.
struct EvictSpace {
  int32_t *kept, *moved, *before, *next, *read;
};
__host__ __device__ inline EvictSpace evict_space(const EvictArgs& a) {
  const int64_t streams = a.requests * 2 * a.kv_heads;
  EvictSpace s;
  s.kept = a.space;
  s.moved = s.kept + a.requests * a.budget;
  s.before = s.moved + a.requests;
  s.next = s.before + a.requests * (a.chunks + 1);
  s.read = s.next + streams;
  return s;
}

// Bits whose unsigned order is that of the weights: -0 and 0 alike, NaN above infinity.
__device__ __forceinline__ unsigned order_bits(float w) {
  const unsigned u = __builtin_bit_cast(unsigned, w + 0.0f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Slot of a request's token.
__device__ __forceinline__ int slot_of(const EvictArgs& a, const int32_t* table, int pos) {
  const unsigned P = (unsigned)a.page_size, at = a.log_page >= 0 ? (unsigned)pos >> a.log_page : (unsigned)pos / P;
  const int page = table[at];
  return page < 0 || page >= a.num_pages ? -1 : page * (int)P + (int)((unsigned)pos - at * P);
}

// Inclusive sums of x over the lanes up to this one.
__device__ __forceinline__ int lanes_up_to(int x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(x, o);
    if ((int)(threadIdx.x & 63) >= o) x += u;
  }
  return x;
}

__global__ __launch_bounds__(PICK) void afa_paged_pick_kernel(const EvictArgs a) {
  __shared__ int bins[COPIES * BINS], wave_sum[PICK_WAVES], found[2];
  __shared__ int2 counts[LOADS * PICK_WAVES];
  const EvictSpace s = evict_space(a);
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t width = a.table_width * a.page_size;
  const int held = (int)min(max((int64_t)a.held[r], (int64_t)0) * a.page_size, width);
  const int c = min(max(a.cached[r], 0), held), budget = a.budget, m = min(c, budget);
  const float* w = a.weights + r * a.row;
  float* left = a.left + r * width;
  int32_t* kept = s.kept + (int64_t)r * budget;
  const int streams = (int)(2 * a.kv_heads);
  for (int i = tid; i < streams; i += PICK) s.next[(int64_t)r * streams + i] = 0;
  for (int64_t i = tid; i < (int64_t)streams * a.chunks; i += PICK) s.read[(int64_t)r * streams * a.chunks + i] = 0;
  if (tid == 0) a.lens[r] = m;
  for (int64_t i = m + tid; i < width; i += PICK) left[i] = 0.0f;
  if (c <= budget) {
    for (int i = tid; i < m; i += PICK) left[i] = w[i];
    if (tid == 0) s.moved[r] = m;
    return;
  }
  const int32_t* table = a.block_tables + (int64_t)r * a.table_width;
  const int log_rows = __builtin_ctz((unsigned)a.rows);
  int32_t* before = s.before + (int64_t)r * (a.chunks + 1);
  for (int i = tid; i <= a.chunks; i += PICK)
    if ((int64_t)i * a.rows >= c) before[i] = m;
  // tokens [lo, hi) are chosen from; `need` of them stay
  const int lo = a.first, hi = c - a.recent;
  int need = budget - a.first - a.recent;
  unsigned top = 0;  // the bits of the least weight that stays, as far as they are known
  for (int shift = 32 - DIGIT; ; shift = shift > DIGIT ? shift - DIGIT : 0) {
    const int above = shift == 32 - DIGIT ? 32 : shift == 0 ? 32 - 2 * DIGIT : 32 - DIGIT;
    const unsigned mask = (1u << (above - shift)) - 1;
    for (int i = tid; i < COPIES * BINS; i += PICK) bins[i] = 0;
    __syncthreads();
    // the next batch comes while this one is counted
    float v[LOADS], next[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) next[k] = w[min(lo + k * PICK + tid, hi - 1)];
    for (int base = lo; base < hi; base += LOADS * PICK) {
#pragma unroll
      for (int k = 0; k < LOADS; ++k) {
        v[k] = next[k];
        next[k] = w[min(base + (LOADS + k) * PICK + tid, hi - 1)];
      }
#pragma unroll
      for (int k = 0; k < LOADS; ++k) {
        const unsigned u = order_bits(v[k]);
        if (base + k * PICK + tid < hi && (above == 32 || u >> above == top >> above))
          atomicAdd(&bins[(u >> shift & mask) * COPIES + lane % COPIES], 1);
      }
    }
    __syncthreads();
    // the bin in which the need-th largest lies: thread t has bins of rank 2 t and 2 t + 1 from the top
    static_assert(BINS == 2 * PICK, "two bins a thread");
    int n[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      n[k] = 0;
#pragma unroll
      for (int i = 0; i < COPIES; ++i) n[k] += bins[(BINS - 1 - 2 * tid - k) * COPIES + i];
    }
    const int upto = lanes_up_to(n[0] + n[1]);
    if (lane == 63) wave_sum[wave] = upto;
    if (tid == 0) found[0] = -1;
    __syncthreads();
    int earlier = upto - n[0] - n[1];
    for (int v = 0; v < wave; ++v) earlier += wave_sum[v];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (earlier < need && need <= earlier + n[k]) {
        found[0] = BINS - 1 - 2 * tid - k;
        found[1] = earlier;
      }
      earlier += n[k];
    }
    __syncthreads();
    if (found[0] < 0) {  // none is needed
      top = 0xffffffffu;
      need = 0;
      break;
    }
    top |= (unsigned)found[0] << shift;
    need -= found[1];
    if (shift == 0) break;
    __syncthreads();
  }
  // those above `top` stay, and the first `need` that equal it
  int over = 0, equal = 0, start = budget;  // of the tokens before this batch: above and sure ones, and equal ones
  float v[LOADS], next[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) next[k] = w[min(k * PICK + tid, c - 1)];
  for (int base = 0; base < c; base += LOADS * PICK) {
    int kind[LOADS];  // 2: stays, 1: equal, 0: neither
    unsigned long long overs[LOADS], equals[LOADS];
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      v[k] = next[k];
      next[k] = w[min(base + (LOADS + k) * PICK + tid, c - 1)];
    }
    __syncthreads();  // counts is free
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = base + k * PICK + tid;
      const unsigned u = order_bits(v[k]);
      kind[k] = i >= c ? 0 : i < lo || i >= hi || u > top ? 2 : u == top ? 1 : 0;
      overs[k] = __ballot(kind[k] == 2);
      equals[k] = __ballot(kind[k] == 1);
      if (lane == 0) counts[k * PICK_WAVES + wave] = int2{__popcll(overs[k]), __popcll(equals[k])};
    }
    __syncthreads();
    // sums before each wave's, in place; the last two entries' sums are the batch's
    static_assert(LOADS * PICK_WAVES == 128, "two entries a lane");
    if (wave == 0) {
      const int2 x = counts[2 * lane], y = counts[2 * lane + 1];
      const int o = lanes_up_to(x.x + y.x), e = lanes_up_to(x.y + y.y);
      counts[2 * lane] = int2{o - x.x - y.x, e - x.y - y.y};
      counts[2 * lane + 1] = int2{o - y.x, e - y.y};
      if (lane == 63) {
        found[0] = o;
        found[1] = e;
      }
    }
    __syncthreads();
    const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      const int i = base + k * PICK + tid;
      const int2 b = counts[k * PICK_WAVES + wave];
      const int o = over + b.x + __popcll(overs[k] & below), e = equal + b.y + __popcll(equals[k] & below);
      const int to = o + min(e, need);
      if (i < c && (i & (a.rows - 1)) == 0 && i >> log_rows <= a.chunks) before[i >> log_rows] = to;
      if (kind[k] == 2 || (kind[k] == 1 && e < need)) {
        kept[to] = slot_of(a, table, i);
        left[to] = v[k];
        if (to != i) start = min(start, to);
      }
    }
    over += found[0];
    equal += found[1];
  }
  // the first place whose token moves
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) start = min(start, __shfl_xor(start, o));
  if (lane == 0) wave_sum[wave] = start;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < PICK_WAVES; ++k) start = min(start, wave_sum[k]);
    s.moved[r] = start;
  }
}

// Rows as `units` of type T each; a chunk is BATCH units a thread, a.rows rows.
template <typename T>
__global__ __launch_bounds__(MOVE, 5) void afa_paged_move_kernel(const EvictArgs a, int units) {
  __shared__ int ticket;
  const EvictSpace s = evict_space(a);
  const int64_t streams = a.requests * 2 * a.kv_heads, stream = blockIdx.x % streams;
  const int r = (int)(stream / (2 * a.kv_heads)), which = (int)(stream % (2 * a.kv_heads)), hk = which >> 1;
  const bool is_v = which & 1;
  const int32_t *kept = s.kept + (int64_t)r * a.budget, *table = a.block_tables + (int64_t)r * a.table_width;
  const int32_t* before = s.before + (int64_t)r * (a.chunks + 1);
  int32_t* read = s.read + stream * a.chunks;
  char* pages = (char*)(is_v ? a.v_pages : a.k_pages) + hk * (is_v ? a.ps.v_head : a.ps.k_head) * a.esz;
  const int64_t page = (is_v ? a.ps.v_page : a.ps.k_page) * a.esz, step = (is_v ? a.ps.v_slot : a.ps.k_slot) * a.esz;
  const unsigned P = (unsigned)a.page_size;
  const int log_rows = __builtin_ctz((unsigned)a.rows);
  auto row = [&](int slot) {
    const unsigned at = a.log_page >= 0 ? (unsigned)slot >> a.log_page : (unsigned)slot / P;
    return pages + at * page + ((unsigned)slot - at * P) * step;
  };
  const int m = a.lens[r], start = s.moved[r];  // from place `start` on every token moves
  const int begin = start >> log_rows, end = start < m ? (m + a.rows - 1) >> log_rows : 0;
  for (;;) {
    // begin and end come with the counter, not before it: what a workgroup reads one after the other is what bounds it
    if (threadIdx.x == 0) ticket = atomicAdd(s.next + stream, 1);
    __syncthreads();
    const int chunk = begin + ticket;
    if (chunk >= end) return;
    const int first = chunk << log_rows, count = min(a.rows, m - first) * units;
    // sources [low, high) lie in this chunk's places: the first's chunk and the last's have to be read
    int other = -1;
    if (threadIdx.x < 2) {
      const int low = before[chunk], high = before[chunk + 1];
      if (low < high) other = (threadIdx.x == 0 ? low : high - 1) >> log_rows;
      if (other >= chunk || other < begin) other = -1;
    }
    T x[BATCH];
    unsigned moves = 0;
    int from[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int e = u * MOVE + (int)threadIdx.x, i = e / units;
      from[u] = e < count && first + i >= start ? kept[first + i] : -1;
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int e = u * MOVE + (int)threadIdx.x, i = e / units;
      if (from[u] < 0) continue;
      moves |= 1u << u;
      x[u] = *(const T*)(row(from[u]) + (e - i * units) * sizeof(T));
    }
    bool ready = other < 0 || __hip_atomic_load(read + other, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    // every read of the chunk is done
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) __hip_atomic_store(read + chunk, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    while (!ready) {
      __builtin_amdgcn_s_sleep(1);
      ready = __hip_atomic_load(read + other, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      if (!(moves >> u & 1)) continue;
      const int e = u * MOVE + (int)threadIdx.x, i = e / units, to = slot_of(a, table, first + i);
      if (to >= 0) *(T*)(row(to) + (e - i * units) * sizeof(T)) = x[u];
    }
  }
}

}  // namespace

// Chunks are shortest where units are elements.
size_t paged_evict_workspace(int64_t requests, int64_t budget, int64_t kv_heads, int64_t head_dim) {
  int64_t rows = 1;
  while (2 * rows * head_dim <= MOVE * BATCH) rows *= 2;
  const int64_t chunks = (budget + rows - 1) / rows;
  return (size_t)(requests * (budget + 2 + chunks + 2 * kv_heads * (1 + chunks))) * 4;
}

hipError_t paged_evict_launch(EvictArgs a, hipStream_t st) {
  int64_t unit = 16;
  const int64_t bytes = a.head_dim * a.esz;
  for (int64_t v : {(int64_t)(uintptr_t)a.k_pages, (int64_t)(uintptr_t)a.v_pages, bytes, a.ps.k_page * a.esz, a.ps.k_head * a.esz,
                    a.ps.k_slot * a.esz, a.ps.v_page * a.esz, a.ps.v_head * a.esz, a.ps.v_slot * a.esz})
    while (v % unit != 0) unit /= 2;
  const int units = (int)(bytes / unit);
  a.rows = 1;  // a power of two
  while (2 * a.rows * units <= MOVE * BATCH) a.rows *= 2;
  a.log_page = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)a.page_size) : -1;
  a.chunks = (a.budget + a.rows - 1) / a.rows;
  hipLaunchKernelGGL(afa_paged_pick_kernel, dim3((unsigned)a.requests), dim3(PICK), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t streams = 2 * a.requests * a.kv_heads, most = std::max<int64_t>(1, (int64_t(1) << 20) / streams);
  const dim3 grid((unsigned)(streams * std::min<int64_t>(a.chunks, most))), block(MOVE);
  switch (unit) {
    case 16: hipLaunchKernelGGL((afa_paged_move_kernel<u32x4_t>), grid, block, 0, st, a, units); break;
    case 8: hipLaunchKernelGGL((afa_paged_move_kernel<u32x2_t>), grid, block, 0, st, a, units); break;
    case 4: hipLaunchKernelGGL((afa_paged_move_kernel<unsigned>), grid, block, 0, st, a, units); break;
    default: hipLaunchKernelGGL((afa_paged_move_kernel<unsigned short>), grid, block, 0, st, a, units); break;
  }
  return hipGetLastError();
}

}  // namespace afa
