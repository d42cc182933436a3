// A serving step's plan from request lengths: pages taken and given back, block tables, the new tokens'
// slots, positions and tree masks, and the items that the attention's workgroups take.
//
// With c cached and n new tokens of request r and pages of P tokens:
//   need = ceil((c + n) / P);  pages popped from the ring: max(need - held, 0), at the sum of the same
//   over the earlier requests; pages pushed behind its end: max(held - need, 0), likewise.
//   Token i of r: cache index c + i, slot table[(c + i) / P] * P + (c + i) % P.
//   A tree's mask: bit i and the parent's mask; position c + depth.
// Popped places lie within the ring's free pages and pushed ones outside them, so that the two never
// meet and each request can be served by its own workgroup, once the sums are known.
//
// The amounts of data are small and launches bound the work: one workgroup forms the sums over the
// requests, then one workgroup per request does the rest.
#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

PagedCut paged_cut(const afa_paged_plan& p, int cus) {
  PagedCut c;
  const int64_t group = p.heads / p.kv_heads, most = p.max_new * group;
  // as many rows as a wave's registers hold beside a tile of K and V
  const int64_t bytes = p.head_dim * (p.dtype == AFA_F32 ? 4 : 2), limit = bytes <= 256 ? 64 : bytes <= 512 ? 32 : 16;
  c.rows = most <= 16 || limit == 16 ? 16 : most <= 32 || limit == 32 ? 32 : 64;
  const int64_t want = 2 * (int64_t)cus;
  c.target = (want + p.kv_heads - 1) / p.kv_heads;
  // Keys are cut into chunks of at least total / target tiles, total the sum of tiles over the row blocks.
  // A block cut in two or more has at most 2 tiles / chunk parts, all blocks together 2 target.
  c.max_parts = 2 * c.target;
  c.max_items = c.max_parts + (p.max_tokens * group + c.rows - 1) / c.rows + p.requests;
  return c;
}

size_t paged_schedule_bytes(const afa_paged_plan& p, const PagedCut& c) {
  const int64_t ints = (PS_INTS + 6 * p.requests + 3) & ~(int64_t)3;
  return (size_t)ints * 4 + (size_t)c.max_items * sizeof(PagedItem);
}

namespace {

constexpr int SCAN = 1024;
// Fewest tiles of a chunk: one for each wave of the attention's workgroups.
constexpr int kMinChunk = 4;

// Inclusive sum of v over the workgroup's threads, in thread order; `total` the sum of all.
__device__ int64_t block_scan(int64_t v, int64_t* lds, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();  // earlier reads of lds are over
  if (lane == 63) lds[wave] = v;
  __syncthreads();
  total = 0;
  int64_t before = 0;
  for (int w = 0; w < SCAN / 64; ++w) {
    if (w == wave) before = total;
    total += lds[w];
  }
  return before + v;
}

__global__ __launch_bounds__(SCAN) void afa_paged_scan_kernel(const afa_paged_plan p, const int rows, const int64_t target,
                                                              const int32_t* cached, const int32_t* fresh) {
  __shared__ int64_t lds[SCAN / 64];
  const PagedSchedule s = paged_schedule(p);
  const int R = (int)p.requests, P = (int)p.page_size, group = (int)(p.heads / p.kv_heads);
  // within the ring whatever the arrays hold
  const int NP = (int)p.num_pages, count = min(max(p.ring_state[1], 0), NP);
  const int head = (int)((unsigned)p.ring_state[0] % (unsigned)NP);
  int64_t tokens = 0, grown = 0, shrunk = 0, taken = 0, tiles = 0;
  for (int base = 0; base < R; base += SCAN) {
    const int r = base + threadIdx.x;
    int c = 0, n = 0, held = 0, status = AFA_PAGED_OK;
    if (r < R) {
      c = cached[r];
      n = fresh[r];
      held = min(max(p.held[r], 0), (int)p.table_width);
      if (c < 0 || n < 0) status = AFA_PAGED_NEGATIVE;
      else if (n > p.max_new) status = AFA_PAGED_TOO_MANY;
      else if ((int64_t)c + n > p.table_width * P) status = AFA_PAGED_TOO_LONG;
    }
    int64_t all;
    const int64_t end = tokens + block_scan(max(n, 0), lds, all);
    tokens += all;
    if (status == AFA_PAGED_OK && n > 0 && end > p.max_tokens) status = AFA_PAGED_PAST_END;
    int need = status == AFA_PAGED_OK ? (int)(((int64_t)c + n + P - 1) / P) : held;
    const int grow = max(need - held, 0), shrink = max(held - need, 0);
    const int64_t grow_end = grown + block_scan(grow, lds, all);
    grown += all;
    const int64_t shrink_end = shrunk + block_scan(shrink, lds, all);
    shrunk += all;
    if (grow > 0 && grow_end > count) {
      status = AFA_PAGED_NO_PAGES;
      need = held;
    }
    // the pages that are taken: the sum up to the last request that is served
    block_scan(status == AFA_PAGED_OK ? grow : 0, lds, all);
    taken += all;
    const bool live = r < R && status == AFA_PAGED_OK && n > 0;
    const int64_t blocks = live ? ((int64_t)n * group + rows - 1) / rows : 0;
    block_scan(live ? blocks * ((c + n + kPagedTile - 1) / kPagedTile) : 0, lds, all);
    tiles += all;
    if (r < R) {
      s.pop[r] = (int)((head + grow_end - grow) % NP);
      s.push[r] = (int)((head + count + shrink_end - shrink) % NP);
      s.held[r] = held;
      p.held[r] = need;
      p.status[r] = status;
      p.starts[r + 1] = (int)min(end, p.max_tokens);
      if (r == 0) p.starts[0] = 0;
    }
  }
  const int64_t even = (tiles + target - 1) / target;
  const int chunk = (int)max(even, (int64_t)kMinChunk);
  int64_t items = 0, parts = 0;
  for (int base = 0; base < R; base += SCAN) {
    const int r = base + threadIdx.x;
    int64_t blocks = 0, chunks = 0;
    if (r < R && p.status[r] == AFA_PAGED_OK && fresh[r] > 0) {
      blocks = ((int64_t)fresh[r] * group + rows - 1) / rows;
      chunks = ((cached[r] + fresh[r] + kPagedTile - 1) / kPagedTile + chunk - 1) / chunk;
    }
    int64_t all;
    const int64_t mine = blocks * chunks, split = chunks > 1 ? mine : 0;
    const int64_t item_end = items + block_scan(mine, lds, all);
    items += all;
    const int64_t part_end = parts + block_scan(split, lds, all);
    parts += all;
    if (r < R) {
      s.item[r] = (int)(item_end - mine);
      s.part[r] = (int)(part_end - split);
      s.chunks[r] = (int)chunks;
    }
  }
  if (threadIdx.x == 0) {
    s.header[PS_ITEMS] = (int)items;
    s.header[PS_CHUNK] = chunk;
    s.header[PS_HEAD] = head;
    s.header[PS_COUNT] = count;
    p.ring_state[0] = (int)((head + taken) % NP);
    p.ring_state[1] = (int)(count - taken + shrunk);
  }
}

// Workgroups (r, y) of request r share its tokens, pages and items; r = requests: the rows behind the
// last request's.
__global__ __launch_bounds__(kMaxTree) void afa_paged_fill_kernel(const afa_paged_plan p, const int rows,
                                                                  const int32_t* cached, const int32_t* fresh,
                                                                  const int32_t* parents) {
  const PagedSchedule s = paged_schedule(p);
  const int R = (int)p.requests, P = (int)p.page_size, r = blockIdx.x, words = (int)(p.max_tree / 64);
  const int tid = threadIdx.x, step = gridDim.y * kMaxTree, first = blockIdx.y * kMaxTree + tid;
  if (r == R) {
    for (int64_t t = p.starts[R] + first; t < p.max_tokens; t += step) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      p.token_request[t] = -1;
      for (int w = 0; w < words; ++w) p.masks[t * words + w] = 0;
    }
    return;
  }
  const int start = p.starts[r], status = p.status[r];
  if (status != AFA_PAGED_OK) {
    for (int64_t t = start + first; t < p.starts[r + 1]; t += step) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      p.token_request[t] = r;
      for (int w = 0; w < words; ++w) p.masks[t * words + w] = 0;
    }
    return;
  }
  const int c = cached[r], n = fresh[r], held = s.held[r], need = p.held[r];
  int32_t* table = p.block_tables + (int64_t)r * p.table_width;
  // page b of the request, also before this launch has written it into the table
  auto page = [&](int b) { return b < held ? table[b] : p.ring[(s.pop[r] + (int64_t)(b - held)) % p.num_pages]; };
  for (int b = held + first; b < need; b += step) table[b] = page(b);
  for (int b = need + first; b < held; b += step) {
    p.ring[(s.push[r] + (int64_t)(b - need)) % p.num_pages] = table[b];
    table[b] = -1;
  }
  const bool tree = n <= p.max_tree;  // masks are written; a chain's where there are no parents
  for (int i = first; i < n; i += step) {
    const int64_t t = start + i;
    const int at = c + i;
    p.slots[t] = page(at / P) * P + at % P;
    p.token_request[t] = r;
    if (!tree) {
      p.positions[t] = at;
      for (int w = 0; w < words; ++w) p.masks[t * words + w] = 0;
    }
  }
  if (tree && blockIdx.y == 0) {
    // Ancestors by doubling: after k rounds a node's set holds its 2^k nearest ancestors and `up` is the
    // one behind them.
    __shared__ int up[kMaxTree];
    __shared__ uint64_t set[kMaxTree / 64][kMaxTree];
    int mine = -1;
    uint64_t seen[kMaxTree / 64];
#pragma unroll
    for (int w = 0; w < kMaxTree / 64; ++w) seen[w] = tid >> 6 == w ? uint64_t(1) << (tid & 63) : 0;
    if (tid < n) {
      mine = parents != nullptr ? parents[start + tid] : tid - 1;
      if (mine < 0 || mine >= tid) mine = -1;
    }
    for (int span = 1; span < n; span <<= 1) {
      up[tid] = mine;
#pragma unroll
      for (int w = 0; w < kMaxTree / 64; ++w) set[w][tid] = seen[w];
      __syncthreads();
      if (mine >= 0) {
#pragma unroll
        for (int w = 0; w < kMaxTree / 64; ++w) seen[w] |= set[w][mine];
        mine = up[mine];
      }
      __syncthreads();
    }
    if (tid < n) {
      int depth = -1;
#pragma unroll
      for (int w = 0; w < kMaxTree / 64; ++w) {
        depth += __popcll(seen[w]);
        if (w < words) p.masks[(int64_t)(start + tid) * words + w] = (int64_t)seen[w];
      }
      p.positions[start + tid] = c + depth;
    }
  }
  if (n == 0) return;
  const int group = (int)(p.heads / p.kv_heads), chunk = s.header[PS_CHUNK], chunks = s.chunks[r];
  const int blocks = (int)(((int64_t)n * group + rows - 1) / rows), all = (c + n + kPagedTile - 1) / kPagedTile;
  for (int64_t j = first; j < (int64_t)blocks * chunks; j += step) {
    // row blocks run fastest: those that read the same keys follow one another
    const int block = (int)(j % blocks), ch = (int)(j / blocks);
    int end = all;
    if (!tree || p.max_tree == 0) {
      // a chain's rows see no key behind their own token
      const int last = min(n - 1, (int)(((int64_t)block * rows + rows - 1) / group));
      end = (c + last + kPagedTile) / kPagedTile;
    }
    PagedItem it;
    it.request = r;
    it.row0 = block * rows;
    it.tile0 = ch * chunk;
    it.tile1 = min(it.tile0 + chunk, end);
    it.part = chunks > 1 ? s.part[r] + block * chunks + ch : -1;
    it.cached = c;
    it.fresh = n;
    it.start = start;
    s.items[s.item[r] + j] = it;
  }
}

}  // namespace

hipError_t paged_build_launch(const afa_paged_plan& p, const PagedCut& c, const int32_t* cached, const int32_t* fresh,
                              const int32_t* parents, hipStream_t st) {
  hipLaunchKernelGGL(afa_paged_scan_kernel, dim3(1), dim3(SCAN), 0, st, p, c.rows, c.target, cached, fresh);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t y = (p.max_new + 1023) / 1024;
  hipLaunchKernelGGL(afa_paged_fill_kernel, dim3((unsigned)(p.requests + 1), (unsigned)(y < 64 ? y : 64)),
                     dim3(kMaxTree), 0, st, p, c.rows, cached, fresh, parents);
  return hipGetLastError();
}

}  // namespace afa
