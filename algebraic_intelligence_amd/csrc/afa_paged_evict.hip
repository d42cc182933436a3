// Requests of more than `budget` cached tokens cut back to it: their `first` oldest tokens stay, their `recent`
// newest, and of the others those of the largest weight, the lower index among equal ones.  What stays keeps its
// order: token kept[i] moves to place i, in k, in v and in the weights.
//
// First the weight is found from which on tokens stay, by its bits from the top (three passes over the weights, up to eleven
// bits each, counted in LDS), and the tokens that stay are listed: in one launch of a workgroup a request, or, where caches are
// long, in five launches of a workgroup for every 8192 tokens.
//
// The last launch moves rows in place.  A workgroup has one chunk of ROWS places of one head's k or v; its sources are behind its
// places, in places of later chunks, so it reads all of them, says so, and writes only once the chunks that read from
// its own places (earlier ones, two at most, as ROWS places hold at most ROWS sources) have said so too.  Chunks are handed
// out in their order by a counter, and a workgroup reads and says so before it waits: whatever one waits for has begun and
// waits for nothing before it says so, so every wait ends.
//
// HBM bounds the last launch: every row that moves is read and written once.  64 requests of up to 8192 tokens cut back to 2048, 4 heads
// of 128 in bf16: 18 us for the choice and 104 for the rows (4.6 TB/s); 4 of up to 131072 cut back to 32768: 33 and 100.  Short
// requests, 2 of 124 tokens: 11 and 6, a chain of barriers and of code that is fetched once.
#include <algorithm>
#include <initializer_list>

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

constexpr int PICK = 1024, PICK_WAVES = PICK / 64;
constexpr int DIGIT = 11, BINS = 1 << DIGIT, COPIES = 8;  // of a bin, in banks of their own: neighbours often share one
constexpr int LOADS = 8;                                  // weights of a thread in flight
constexpr int MOVE = 1024, FEW = 256, BATCH = 8;          // threads of a mover, or of one for short streams, and units that each holds

constexpr int SLICE = LOADS * PICK;                       // tokens of a workgroup where a request has several
constexpr int PASSES = 3;

// The workspace: slots of the tokens that stay, page * page_size + offset, or -1 for a page of no pool (requests, budget); the
// first place that moves (requests,); sources before each chunk's places, and behind the last's (requests, chunks + 1); chunks
// handed out (requests, streams) and chunks that are read (requests, streams, chunks), a stream being one head's k or v.
// With slices: counts of the digits (requests, PASSES, BINS), the digits found before each but the first pass and how many
// tokens of the last are needed (requests, PASSES - 1, 2), slices handed out (requests,), and each one's counts (requests, slices).
struct EvictSpace {
  int64_t* counted;
  int32_t *kept, *moved, *before, *next, *read, *bins, *state, *slice;
};
__host__ __device__ inline EvictSpace evict_space(const EvictArgs& a) {
  const int64_t streams = a.requests * 2 * a.kv_heads;
  EvictSpace s;
  s.counted = (int64_t*)a.space;
  s.kept = a.space + 2 * a.requests * a.slices;
  s.moved = s.kept + a.requests * a.budget;
  s.before = s.moved + a.requests;
  s.next = s.before + a.requests * (a.chunks + 1);
  s.read = s.next + streams;
  s.bins = s.read + streams * a.chunks;
  s.state = s.bins + a.requests * PASSES * BINS;
  s.slice = s.state + 2 * (PASSES - 1) * a.requests;
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

// What a request asks for: its tokens, those that are chosen from, and how many of them stay.
struct Choice {
  int c, m, lo, hi, need;
  bool over;  // more than the budget
};
__device__ __forceinline__ Choice choice(const EvictArgs& a, int r) {
  const int held = (int)min(max((int64_t)a.held[r], (int64_t)0) * a.page_size, a.table_width * a.page_size);
  const int c = min(max(a.cached[r], 0), held);
  return Choice{c, min(c, a.budget), a.first, c - a.recent, a.budget - a.first - a.recent, c > a.budget};
}

// Digit `pass` of the weights: its lowest bit, and the lowest of the digits above it.
__device__ __forceinline__ int shift_of(int pass) { return pass == 0 ? 32 - DIGIT : pass == 1 ? 32 - 2 * DIGIT : 0; }
__device__ __forceinline__ int above_of(int pass) { return pass == 0 ? 32 : shift_of(pass - 1); }

__device__ __forceinline__ void clear(int* bins) {
  for (int i = threadIdx.x; i < COPIES * BINS; i += PICK) bins[i] = 0;
}
// Counts weights [base, base + SLICE) of [lo, hi), of which v are this thread's, whose digits above are those of `top`.
__device__ __forceinline__ void count_digits(const float (&v)[LOADS], int base, int hi, int pass, unsigned top, int* bins) {
  const int shift = shift_of(pass), above = above_of(pass);
  const unsigned mask = (1u << (above - shift)) - 1;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    if (base + k * PICK >= hi) break;  // code that is not run is not fetched, which short requests wait for
    const unsigned u = order_bits(v[k]);
    if (base + k * PICK + (int)threadIdx.x < hi && (above == 32 || u >> above == top >> above))
      atomicAdd(&bins[(u >> shift & mask) * COPIES + threadIdx.x % COPIES], 1);
  }
}
// The bin in which the need-th largest lies, from the counts n of bins BINS - 1 - 2 t and the one below, t this thread: found =
// {bin, those above it}, bin -1 where none is needed.
__device__ __forceinline__ void find_digit(const int (&n)[2], int need, int* wave_sum, int* found) {
  static_assert(BINS == 2 * PICK, "two bins a thread");
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, upto = lanes_up_to(n[0] + n[1]);
  if (lane == 63) wave_sum[wave] = upto;
  if (tid == 0) found[0] = -1;
  __syncthreads();
  int earlier = upto - n[0] - n[1];
#pragma unroll
  for (int v = 0; v < PICK_WAVES; ++v) earlier += v < wave ? wave_sum[v] : 0;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if (earlier < need && need <= earlier + n[k]) {
      found[0] = BINS - 1 - 2 * tid - k;
      found[1] = earlier;
    }
    earlier += n[k];
  }
  __syncthreads();
}

// Lists those of tokens [base, base + SLICE) that stay: those above `top`, and of those that equal it the first `need` of the
// request.  before(over, equal), called by all threads with the batch's counts, gives those of the tokens before it.
struct Lists {
  float* left;
  int32_t *kept, *before;
  const int32_t* table;
};
template <typename B>
__device__ __forceinline__ void list_tokens(const EvictArgs& a, const Choice& q, const Lists& to, const float (&v)[LOADS], int base,
                                            unsigned top, int need, int2* counts, int* found, int& first_gone, const B& before) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, log_rows = __builtin_ctz((unsigned)a.rows);
  int kind[LOADS];  // 2: stays, 1: equal, 0: neither
  unsigned long long overs[LOADS], equals[LOADS];
  __syncthreads();  // counts is free
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    kind[k] = 0;
    overs[k] = equals[k] = 0;
    if (base + k * PICK >= q.c) continue;
    const int i = base + k * PICK + tid;
    const unsigned u = order_bits(v[k]);
    kind[k] = i >= q.c ? 0 : i < q.lo || i >= q.hi || u > top ? 2 : u == top ? 1 : 0;
    overs[k] = __ballot(kind[k] == 2);
    equals[k] = __ballot(kind[k] == 1);
    if (lane == 0) counts[k * PICK_WAVES + wave] = int2{__popcll(overs[k]), __popcll(equals[k])};
  }
  __syncthreads();
  // sums before each wave's, in place, and the batch's
  static_assert(LOADS * PICK_WAVES == 128, "two entries a lane");
  if (wave == 0) {
    const bool some = base + 2 * lane / PICK_WAVES * PICK < q.c;
    const int2 x = some ? counts[2 * lane] : int2{0, 0}, y = some ? counts[2 * lane + 1] : int2{0, 0};
    const int o = lanes_up_to(x.x + y.x), e = lanes_up_to(x.y + y.y);
    counts[2 * lane] = int2{o - x.x - y.x, e - x.y - y.y};
    counts[2 * lane + 1] = int2{o - y.x, e - y.y};
    if (lane == 63) {
      found[0] = o;
      found[1] = e;
    }
  }
  __syncthreads();
  const int2 earlier = before(found[0], found[1]);
  const unsigned long long below = (1ull << lane) - 1;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    if (base + k * PICK >= q.c) break;
    const int i = base + k * PICK + tid;
    const int2 b = counts[k * PICK_WAVES + wave];
    const int o = earlier.x + b.x + __popcll(overs[k] & below), e = earlier.y + b.y + __popcll(equals[k] & below);
    const int at = o + min(e, need);
    if (i < q.c && (i & (a.rows - 1)) == 0 && i >> log_rows <= a.chunks) to.before[i >> log_rows] = at;
    if (kind[k] == 2 || (kind[k] == 1 && e < need)) {
      to.kept[at] = slot_of(a, to.table, i);
      to.left[at] = v[k];
    } else if (i < q.c) {
      first_gone = min(first_gone, i);
    }
  }
}

__device__ __forceinline__ Lists lists_of(const EvictArgs& a, const EvictSpace& s, int r) {
  return Lists{a.left + r * a.table_width * a.page_size, s.kept + (int64_t)r * a.budget, s.before + (int64_t)r * (a.chunks + 1),
               a.block_tables + (int64_t)r * a.table_width};
}

__global__ __launch_bounds__(PICK) void afa_paged_pick_kernel(const EvictArgs a) {
  __shared__ __attribute__((aligned(16))) int bins[COPIES * BINS];
  __shared__ int wave_sum[PICK_WAVES], found[2];
  __shared__ int2 counts[LOADS * PICK_WAVES];
  static_assert(COPIES == 8, "pieces of 16 bytes");
  const EvictSpace s = evict_space(a);
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t width = a.table_width * a.page_size;
  const Choice q = choice(a, r);
  const Lists to = lists_of(a, s, r);
  const float* w = a.weights + r * a.row;
  const int streams = (int)(2 * a.kv_heads);
  for (int i = tid; i < streams; i += PICK) s.next[(int64_t)r * streams + i] = 0;
  for (int64_t i = tid; i < (int64_t)streams * a.chunks; i += PICK) s.read[(int64_t)r * streams * a.chunks + i] = 0;
  if (tid == 0) a.lens[r] = q.m;
  for (int64_t i = q.m + tid; i < width; i += PICK) to.left[i] = 0.0f;
  if (!q.over) {
    for (int i = tid; i < q.m; i += PICK) to.left[i] = w[i];
    if (tid == 0) s.moved[r] = q.m;
    return;
  }
  for (int i = tid; i <= a.chunks; i += PICK)
    if ((int64_t)i * a.rows >= q.c) to.before[i] = q.m;
  int need = q.need;
  unsigned top = 0;  // the bits of the least weight that stays, as far as they are known
  float v[LOADS], next[LOADS] = {};  // the next batch comes while this one is counted
  auto load = [&](int base, int end) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) {
      if (base + k * PICK >= end) break;
      next[k] = w[min(base + k * PICK + tid, end - 1)];
    }
  };
  auto take = [&](int base, int end) {
#pragma unroll
    for (int k = 0; k < LOADS; ++k) v[k] = next[k];
    load(base + SLICE, end);
  };
  for (int pass = 0; pass < PASSES; ++pass) {
    clear(bins);
    load(q.lo, q.hi > q.lo ? q.hi : q.lo + 1);
    __syncthreads();
    for (int base = q.lo; base < q.hi; base += SLICE) {
      take(base, q.hi);
      count_digits(v, base, q.hi, pass, top, bins);
    }
    __syncthreads();
    // two bins are 64 bytes, four pieces of 16; lanes four apart, which would meet in their banks, begin with another piece
    int n[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int piece = (i + (lane >> 2)) & 3;
      const int4 x = *(const int4*)&bins[(BINS - 2 - 2 * tid) * COPIES + 4 * piece];
      n[0] += piece >= 2 ? (x.x + x.y) + (x.z + x.w) : 0;
      n[1] += piece >= 2 ? 0 : (x.x + x.y) + (x.z + x.w);
    }
    find_digit(n, need, wave_sum, found);
    if (found[0] < 0) {  // none is needed
      top = 0xffffffffu;
      need = 0;
      break;
    }
    top |= (unsigned)found[0] << shift_of(pass);
    need -= found[1];
    __syncthreads();
  }
  int2 earlier = {0, 0};
  int gone = q.m;
  load(0, q.c);
  for (int base = 0; base < q.c; base += SLICE) {
    take(base, q.c);
    list_tokens(a, q, to, v, base, top, need, counts, found, gone, [&](int over, int equal) {
      const int2 was = earlier;
      earlier.x += over;
      earlier.y += equal;
      return was;
    });
  }
  // the first place whose token moves: that of the first token that does not stay
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) gone = min(gone, __shfl_xor(gone, o));
  if (lane == 0) wave_sum[wave] = gone;
  __syncthreads();
  if (tid == 0) {
    for (int k = 1; k < PICK_WAVES; ++k) gone = min(gone, wave_sum[k]);
    s.moved[r] = gone;
  }
}

// ------------------------------------------------------------------ a workgroup for every SLICE tokens
// What the other launches count in is cleared, and the lengths and first places set.
__global__ __launch_bounds__(256) void afa_paged_slice_clear_kernel(const EvictArgs a) {
  const EvictSpace s = evict_space(a);
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const int64_t streams = a.requests * 2 * a.kv_heads;
  for (int64_t i = i0; i < streams * (a.chunks + 1); i += step) s.next[i] = 0;  // read lies behind it
  for (int64_t i = i0; i < a.requests * PASSES * BINS; i += step) s.bins[i] = 0;
  for (int64_t i = i0; i < a.requests * a.slices; i += step) s.counted[i] = 0;
  for (int64_t r = i0; r < a.requests; r += step) {
    const Choice q = choice(a, (int)r);
    a.lens[r] = s.moved[r] = q.m;
    s.slice[r] = 0;
  }
}

// The digits of the passes before `pass`, from their counts: top and need.
__device__ __forceinline__ bool digits_before(const EvictArgs& a, const EvictSpace& s, int r, int pass, const Choice& q, unsigned& top,
                                              int& need, int* wave_sum, int* found) {
  top = 0;
  need = q.need;
  if (pass >= 2) {
    const int32_t* state = s.state + 2 * ((PASSES - 1) * r + pass - 2);
    top = (unsigned)state[0];
    need = state[1];
  }
  if (pass >= 1 && need > 0) {
    const int* bins = s.bins + ((int64_t)r * PASSES + pass - 1) * BINS;
    const int n[2] = {bins[BINS - 1 - 2 * (int)threadIdx.x], bins[BINS - 2 - 2 * (int)threadIdx.x]};
    find_digit(n, need, wave_sum, found);
    top |= (unsigned)found[0] << shift_of(pass - 1);
    need -= found[1];
    __syncthreads();  // found is free
  }
  if (need <= 0) {  // none is needed
    top = 0xffffffffu;
    need = 0;
  }
  return need > 0;
}

__global__ __launch_bounds__(PICK) void afa_paged_slice_count_kernel(const EvictArgs a, int pass) {
  __shared__ int bins[COPIES * BINS], wave_sum[PICK_WAVES], found[2];
  const EvictSpace s = evict_space(a);
  const int r = blockIdx.x / a.slices, slice = blockIdx.x % a.slices, tid = threadIdx.x;
  const Choice q = choice(a, r);
  const int base = slice * SLICE;
  if (!q.over || (base >= q.hi && slice > 0)) return;
  const float* w = a.weights + r * a.row;
  float v[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) v[k] = w[min(base + k * PICK + tid, q.c - 1)];
  clear(bins);
  unsigned top;
  int need;
  const bool some = digits_before(a, s, r, pass, q, top, need, wave_sum, found);
  // for the next pass, which reads it in another launch
  if (slice == 0 && tid == 0 && pass >= 1) {
    int32_t* state = s.state + 2 * ((PASSES - 1) * r + pass - 1);
    state[0] = (int)top;
    state[1] = need;
  }
  if (!some) return;
  __syncthreads();
  const int shift = shift_of(pass), above = above_of(pass);
  const unsigned mask = (1u << (above - shift)) - 1;
#pragma unroll
  for (int k = 0; k < LOADS; ++k) {
    const int i = base + k * PICK + tid;
    const unsigned u = order_bits(v[k]);
    if (i >= q.lo && i < q.hi && (above == 32 || u >> above == top >> above))
      atomicAdd(&bins[(u >> shift & mask) * COPIES + tid % COPIES], 1);
  }
  __syncthreads();
  int* to = s.bins + ((int64_t)r * PASSES + pass) * BINS;
  for (int b = tid; b < BINS; b += PICK) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < COPIES; ++i) n += bins[b * COPIES + i];
    if (n > 0) atomicAdd(to + b, n);
  }
}

// A request's slices are handed out in their order; each says what it counts before it waits for the earlier ones' counts,
// so every wait ends.
__global__ __launch_bounds__(PICK) void afa_paged_slice_list_kernel(const EvictArgs a) {
  __shared__ int wave_sum[PICK_WAVES], wave_more[PICK_WAVES], found[2], ticket;
  __shared__ int2 counts[LOADS * PICK_WAVES];
  const EvictSpace s = evict_space(a);
  const int r = blockIdx.x / a.slices, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const Choice q = choice(a, r);
  const Lists to = lists_of(a, s, r);
  const float* w = a.weights + r * a.row;
  if (tid == 0) ticket = atomicAdd(s.slice + r, 1);
  __syncthreads();
  const int slice = ticket, base = slice * SLICE;
  const int64_t width = a.table_width * a.page_size, end = min((int64_t)base + SLICE, width);
  for (int64_t i = max((int64_t)base, (int64_t)q.m) + tid; i < end; i += PICK) to.left[i] = 0.0f;
  if (!q.over) {
    for (int64_t i = base + tid; i < min(end, (int64_t)q.m); i += PICK) to.left[i] = w[i];
    return;
  }
  if (slice == 0)
    for (int i = tid; i <= a.chunks; i += PICK)
      if ((int64_t)i * a.rows >= q.c) to.before[i] = q.m;
  if (base >= q.c) return;
  float v[LOADS];
#pragma unroll
  for (int k = 0; k < LOADS; ++k) v[k] = w[min(base + k * PICK + tid, q.c - 1)];
  unsigned top;
  int need;
  digits_before(a, s, r, PASSES, q, top, need, wave_sum, found);
  int gone = q.m;
  list_tokens(a, q, to, v, base, top, need, counts, found, gone, [&](int over, int equal) {
    int64_t* counted = s.counted + (int64_t)r * a.slices;
    if (tid == 0)
      __hip_atomic_store(counted + slice, (int64_t)1 << 62 | (int64_t)over << 31 | equal, __ATOMIC_RELAXED,
                         __HIP_MEMORY_SCOPE_AGENT);
    int2 sum = {0, 0};
    for (int j = tid; j < slice; j += PICK) {
      int64_t x;
      while ((x = __hip_atomic_load(counted + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == 0) __builtin_amdgcn_s_sleep(1);
      sum.x += (int)(x >> 31 & 0x7fffffff);
      sum.y += (int)(x & 0x7fffffff);
    }
    const int o = lanes_up_to(sum.x), e = lanes_up_to(sum.y);
    if (lane == 63) {
      wave_sum[wave] = o;
      wave_more[wave] = e;
    }
    __syncthreads();
    sum = int2{0, 0};
    for (int k = 0; k < PICK_WAVES; ++k) {
      sum.x += wave_sum[k];
      sum.y += wave_more[k];
    }
    return sum;
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) gone = min(gone, __shfl_xor(gone, o));
  if (lane == 0 && gone < q.m) atomicMin(s.moved + r, gone);
}

// Rows as `units` of type T each; a chunk is up to BATCH units a thread, a.rows rows.  Long chunks wait for one another less: with
// 256, 512 and 1024 threads 4 requests of up to 131072 tokens take 170, 142 and 133 us in all, 64 of up to 8192 126, 124 and 124.
// A stream that one chunk of 256 threads holds has no more of them: 68 requests of 23 tokens, 8 heads of 48, take 7 us and not 20.
// Rows pass by the caches (5 us less in each): what is moved is not read again soon.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void afa_paged_move_kernel(const EvictArgs a, int units) {
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
      const int e = u * THREADS + (int)threadIdx.x, i = e / units;
      from[u] = e < count && first + i >= start ? kept[first + i] : -1;
    }
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      const int e = u * THREADS + (int)threadIdx.x, i = e / units;
      if (from[u] < 0) continue;
      moves |= 1u << u;
      x[u] = __builtin_nontemporal_load((const T*)(row(from[u]) + (e - i * units) * sizeof(T)));
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
      const int e = u * THREADS + (int)threadIdx.x, i = e / units, to = slot_of(a, table, first + i);
      if (to >= 0) __builtin_nontemporal_store(x[u], (T*)(row(to) + (e - i * units) * sizeof(T)));
    }
  }
}

template <typename T>
void move_go(const EvictArgs& a, int units, bool few, dim3 grid, hipStream_t st) {
  if (few) hipLaunchKernelGGL((afa_paged_move_kernel<T, FEW>), grid, dim3(FEW), 0, st, a, units);
  else hipLaunchKernelGGL((afa_paged_move_kernel<T, MOVE>), grid, dim3(MOVE), 0, st, a, units);
}

// Slices of a request, 0 where one workgroup has all of its tokens.  With the rows' launch that takes about 16 us and 8 for every slice,
// requests side by side; five launches 35, and 0.1 for a request and 0.04 for its every slice.  48 requests in three slices (up to
// 16384 tokens and a page) take 32 us and 38, in four 40 and 39, in five 49 and 39; 80 in five 49 and 54; 84 in nine 82 and 69, in 17 146 and 96.
int64_t slices_of(int64_t requests, int64_t max_len) {
  const int64_t slices = (max_len + SLICE - 1) / SLICE;
  return requests * (3 + 2 * slices) < 385 * slices - 1285 ? slices : 0;
}

}  // namespace

// Chunks are shortest where units are elements.
size_t paged_evict_workspace(int64_t requests, int64_t max_len, int64_t budget, int64_t kv_heads, int64_t head_dim) {
  int64_t rows = 1;
  while (2 * rows * head_dim <= MOVE * BATCH) rows *= 2;
  const int64_t chunks = (budget + rows - 1) / rows, slices = slices_of(requests, max_len);
  return (size_t)(requests * (budget + 2 + chunks + 2 * kv_heads * (1 + chunks) +
                              (slices > 0 ? 2 * slices + PASSES * BINS + 2 * (PASSES - 1) + 1 : 0))) * 4;
}

hipError_t paged_evict_launch(EvictArgs a, hipStream_t st) {
  int64_t unit = 16;
  const int64_t bytes = a.head_dim * a.esz;
  for (int64_t v : {(int64_t)(uintptr_t)a.k_pages, (int64_t)(uintptr_t)a.v_pages, bytes, a.ps.k_page * a.esz, a.ps.k_head * a.esz,
                    a.ps.k_slot * a.esz, a.ps.v_page * a.esz, a.ps.v_head * a.esz, a.ps.v_slot * a.esz})
    while (v % unit != 0) unit /= 2;
  const int units = (int)(bytes / unit);
  auto rows_of = [&](int threads) {  // a power of two
    int rows = 1;
    while (2 * rows * units <= threads * BATCH) rows *= 2;
    return rows;
  };
  const bool few = a.budget <= rows_of(FEW);  // one chunk
  a.rows = rows_of(few ? FEW : MOVE);
  a.log_page = (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctzll((unsigned long long)a.page_size) : -1;
  a.chunks = (a.budget + a.rows - 1) / a.rows;
  a.slices = (int)slices_of(a.requests, a.table_width * a.page_size);
  if (a.slices == 0) {
    hipLaunchKernelGGL(afa_paged_pick_kernel, dim3((unsigned)a.requests), dim3(PICK), 0, st, a);
  } else {
    const dim3 grid((unsigned)(a.requests * a.slices)), block(PICK);
    const int64_t ints = a.requests * (PASSES * BINS + a.slices + 2 * a.kv_heads * (a.chunks + 1));
    hipLaunchKernelGGL(afa_paged_slice_clear_kernel, dim3((unsigned)std::min<int64_t>((ints + 1023) / 1024, 4096)), dim3(256), 0, st,
                       a);
    for (int pass = 0; pass < PASSES; ++pass) hipLaunchKernelGGL(afa_paged_slice_count_kernel, grid, block, 0, st, a, pass);
    hipLaunchKernelGGL(afa_paged_slice_list_kernel, grid, block, 0, st, a);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t streams = 2 * a.requests * a.kv_heads, most = std::max<int64_t>(1, (int64_t(1) << 20) / streams);
  const dim3 grid((unsigned)(streams * std::min<int64_t>(a.chunks, most)));
  switch (unit) {
    case 16: move_go<u32x4_t>(a, units, few, grid, st); break;
    case 8: move_go<u32x2_t>(a, units, few, grid, st); break;
    case 4: move_go<unsigned>(a, units, few, grid, st); break;
    default: move_go<unsigned short>(a, units, few, grid, st); break;
  }
  return hipGetLastError();
}

}  // namespace afa
