// A serving step's plan from request lengths: pages taken and given back, block tables, the new tokens'
// slots, positions and tree masks, and how the attention's workgroups share the work.
//
// With c cached and n new tokens of request r and pages of P tokens:
//   need = ceil((c + n) / P);  pages popped from the ring: max(need - held, 0), at the sum of the same
//   over the earlier requests; pages pushed behind its end: max(held - need, 0), likewise.
//   Token i of r: cache index c + i, slot table[(c + i) / P] * P + (c + i) % P.
//   A tree's mask: bit i and the parent's mask; position c + depth.
// Popped places lie within the ring's free pages and pushed ones outside them, so that the two never
// meet and each request can be served by its own workgroup, once the sums are known.
//
// The amounts of data are small and launches bound the work: one launch, in which every request's
// workgroup forms the sums over all requests again (two launches beyond 1024 requests).  24 requests of one
// token: 5.8 us, 512 with trees of up to 48 nodes: 8.8 us, of which a launch is about 4.
#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

PagedCut paged_cut(const afa_paged_plan& p, int cus) {
  PagedCut c;
  const int64_t group = p.heads / p.kv_heads, most = p.max_new * group;
  // rows of a segment: 16, or up to 128 (64 where a row takes 512 bytes and more) as its workgroup has waves
  const int64_t bytes = p.head_dim * (p.dtype == AFA_F32 ? 4 : 2), limit = bytes <= 256 ? 128 : 64;
  c.rows = 16;
  while (c.rows < most && c.rows < limit) c.rows *= 2;
  // Workgroups that fit the device's registers at once: two a CU, or one where rows are that long.  Three and
  // four a CU, in turn, are slower: 172 and 178 us for 132 (32 requests, trees, heads of 128), 163 and 175 for 161.
  const int64_t want = (bytes >= 512 ? 1 : 2) * (int64_t)cus;
  c.slots = want > p.kv_heads ? want / p.kv_heads : 1;
  return c;
}

size_t paged_schedule_bytes(const afa_paged_plan& p, const PagedCut& c) {
  return (size_t)((int64_t)sizeof(PagedHeader) + p.requests * (int64_t)(sizeof(PagedLive) + 8 + 20) +
                  c.slots * (int64_t)sizeof(PagedSlot) + p.kv_heads * c.slots * 16);
}

namespace {

// Most requests whose sums every workgroup forms for itself, four a thread at most, and most workgroups that
// do: as many as the device holds at once.  24 requests take 5.8 us this way and 512 with trees 8.8, for which two
// launches, the first of one workgroup, took 11.4 and 13.4 when tried.  At the border of the rule, one token a
// request, 1024 take 12.8 us in one launch and 1025 14.0 in two; 2000 take 17.8, 64 prompts of 32768 tokens 18.6.
constexpr int kOwnSums = 4 * kMaxTree, kOwnGroups = 2048;

// The attention's cut as the kernels take it: rows of a segment (a power of two), query heads of a key head, and
// slots.
struct Cut {
  int log_rows, group, slots;
  __device__ int blocks(int n) const { return (n * group + (1 << log_rows) - 1) >> log_rows; }
};

struct Sums {
  int64_t v[3];
};

// Sums of x over the threads before this one; `all` over all THREADS of the workgroup.
template <int THREADS, int N>
__device__ Sums block_before(Sums x, int64_t (*lds)[3], Sums& all) {
  constexpr int WAVES = THREADS / 64;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  Sums s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int64_t u = __shfl_up(s.v[k], o);
      if (lane >= o) s.v[k] += u;
    }
  __syncthreads();  // earlier reads of lds are over
  if (lane == 63)
#pragma unroll
    for (int k = 0; k < N; ++k) lds[wave][k] = s.v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) {
    int64_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w == wave) before = total;
      total += lds[w][k];
    }
    s.v[k] += before - x.v[k];
    all.v[k] = total;
  }
  return s;
}

// One request: what it asks for, and in the end what it gets.
struct Request {
  int c, n, held, need, status;
};

__device__ __forceinline__ Request request(const afa_paged_plan& p, int c, int n, int held) {
  Request q{c, n, min(max(held, 0), (int)p.table_width), 0, AFA_PAGED_OK};
  if (c < 0 || n < 0) q.status = AFA_PAGED_NEGATIVE;
  else if (n > p.max_new) q.status = AFA_PAGED_TOO_MANY;
  else if ((unsigned)c + (unsigned)n > (unsigned)p.table_width * (unsigned)p.page_size) q.status = AFA_PAGED_TOO_LONG;
  const unsigned P = (unsigned)p.page_size;
  q.need = q.status == AFA_PAGED_OK ? (int)(((unsigned)(c + n) + P - 1) / P) : q.held;
  return q;
}

// Places in the ring, from sums below three times its length.
__device__ __forceinline__ int ring_place(int64_t i, int pages) {
  if (i >= pages) i -= pages;
  if (i >= pages) i -= pages;
  return (int)i;
}

// What request r's workgroup has to know.
struct Mine {
  Request q;
  int start, pop, push, place;
  int64_t flat, stretch;
};

// The sums over all requests, formed by a whole workgroup; thread i has requests [i k, i k + k).  `mine` is that
// of request `which`; where `store` is set all requests' values go to the plan and the schedule.  The
// pages held and the ring's state are brought up to date only by `finish`.  K: the most requests of a thread,
// which keeps them; 0: any number, read again in every pass.
template <int THREADS, int K>
struct PlanSums {
  const afa_paged_plan& p;
  const Cut& cut;
  const int32_t *cached, *fresh;
  int64_t (*lds)[3];
  int pages, head, count, r0, r1, end;
  Request own[K > 0 ? K : 1];
  Sums all, first;  // of all requests, and of those before this thread's
  int64_t taken;

  __device__ Request read(int r) const { return request(p, cached[r], fresh[r], p.held[r]); }
  template <typename F>
  __device__ void each_request(const F& f) {
    if constexpr (K > 0) {
#pragma unroll
      for (int u = 0; u < K; ++u)
        if (r0 + u < r1) f(r0 + u, own[u]);
    } else {
      for (int r = r0; r < r1; ++r) f(r, read(r));
    }
  }

  // Calls f(r, request, sums before it) of this thread's requests, in order, with status and need as they end.
  // free: the pages that there are to have.
  template <typename F>
  __device__ void each(Sums before, int64_t free, const F& f) {
    each_request([&](int r, Request q) {
      const int64_t stop = before.v[0] + max(q.n, 0);
      if (q.status == AFA_PAGED_OK && q.n > 0 && stop > p.max_tokens) {
        q.status = AFA_PAGED_PAST_END;
        q.need = q.held;
      }
      const int grow = max(q.need - q.held, 0), shrink = max(q.held - q.need, 0);
      const Sums at = before;
      before.v[0] = stop;
      before.v[1] += grow;
      before.v[2] += shrink;
      if (grow > 0 && before.v[1] > free) {
        q.status = AFA_PAGED_NO_PAGES;
        q.need = q.held;
      }
      f(r, q, at);
    });
  }

  // Two scans: the pages that are asked for depend on where the tokens end.
  __device__ void prepare() {
    const int R = (int)p.requests, k = (R + THREADS - 1) / THREADS;
    pages = (int)p.num_pages;
    count = min(max(p.ring_state[1], 0), pages);
    head = (int)((unsigned)p.ring_state[0] % (unsigned)pages);
    r0 = min((int)threadIdx.x * k, R);
    r1 = min(r0 + k, R);
    if constexpr (K > 0) {
#pragma unroll
      for (int u = 0; u < K; ++u)
        if (r0 + u < r1) own[u] = read(r0 + u);
    }
    Sums x = {{0, 0, 0}}, total;
    each_request([&](int, const Request& q) { x.v[0] += max(q.n, 0); });
    first = block_before<THREADS, 1>(x, lds, total);
    all.v[0] = total.v[0];
    first.v[1] = first.v[2] = 0;
    Sums change = {{0, 0, 0}};
    each(first, INT64_MAX, [&](int, const Request& q, const Sums&) {
      change.v[0] += max(q.need - q.held, 0);
      change.v[1] += max(q.held - q.need, 0);
    });
    const Sums pg = block_before<THREADS, 2>(change, lds, total);
    all.v[1] = total.v[0];
    all.v[2] = total.v[1];
    first.v[1] = pg.v[0];
    first.v[2] = pg.v[1];
  }

  static __device__ bool live(const Request& q) { return q.status == AFA_PAGED_OK && q.n > 0; }
  static __device__ int cost(const Request& q) { return kPagedLead + (q.c + q.n + kPagedTile - 1) / kPagedTile; }

  __device__ Mine run(int which, bool store, Mine* shared) {
    const PagedSchedule s = paged_schedule(p, cut.slots);
    prepare();
    Sums work = {{0, 0, 0}}, total;
    each(first, count, [&](int, const Request& q, const Sums&) {
      if (live(q)) {
        work.v[0] += (int64_t)cut.blocks(q.n) * cost(q);
        work.v[1] += 1;
      }
      if (q.status == AFA_PAGED_OK) work.v[2] += max(q.need - q.held, 0);
    });
    Sums at = block_before<THREADS, 3>(work, lds, total);
    taken = total.v[2];
    end = (int)min(all.v[0], p.max_tokens);
    // an equal share, by a division that may be one too long; slots behind the line's end stay empty
    const int64_t share = (int64_t)((double)total.v[0] / (double)cut.slots) + 1, stretch = max(share, (int64_t)kPagedMin);
    each(first, count, [&](int r, const Request& q, const Sums& b) {
      Mine m;
      m.q = q;
      m.start = (int)min(b.v[0], p.max_tokens);
      m.pop = ring_place(head + b.v[1], pages);
      m.push = ring_place(head + count + b.v[2], pages);
      m.flat = at.v[0];
      m.place = (int)at.v[1];
      m.stretch = stretch;
      if (live(q)) {
        at.v[0] += (int64_t)cut.blocks(q.n) * cost(q);
        at.v[1] += 1;
      }
      if (r == which) *shared = m;
      if (store || r == which) {
        s.cached[r] = q.c;
        p.status[r] = q.status;
        p.starts[r + 1] = (int)min(b.v[0] + max(q.n, 0), p.max_tokens);
      }
      if (store) {
        s.pop[r] = m.pop;
        s.push[r] = m.push;
        s.held[r] = q.held;
        s.flat[r] = m.flat;
        s.place[r] = m.place;
      }
    });
    if (threadIdx.x == 0 && (store || which == 0)) {
      s.header->slots = (int)((total.v[0] + stretch - 1) / stretch);
      s.header->stretch = stretch;
      s.header->end = total.v[0];
      p.starts[0] = 0;
    }
    __syncthreads();
    return *shared;
  }

  // Only once no workgroup reads held and ring_state any more.
  __device__ void finish() {
    each(first, count, [&](int r, const Request& q, const Sums&) { p.held[r] = q.need; });
    if (threadIdx.x == 0) {
      p.ring_state[0] = ring_place(head + taken, pages);
      p.ring_state[1] = (int)(count - taken + all.v[2]);
    }
  }
};

// Request r's tokens, pages and stretches by one or more workgroups (gridDim.y); r = requests: the rows behind
// the last request's, from row `end` on.
__device__ void fill(const afa_paged_plan& p, const Cut& cut, const int32_t* parents, const int r, const Mine& mine,
                     const int end) {
  const PagedSchedule s = paged_schedule(p, cut.slots);
  const int P = (int)p.page_size, words = (int)(p.max_tree / 64), pages = (int)p.num_pages;
  const int tid = threadIdx.x, step = gridDim.y * kMaxTree, first = blockIdx.y * kMaxTree + tid;
  const int c = mine.q.c, n = mine.q.n, held = mine.q.held, need = mine.q.need, start = mine.start;
  const bool rest = r == (int)p.requests;
  if (rest || mine.q.status != AFA_PAGED_OK) {
    const int64_t from = rest ? end : start, to = rest ? p.max_tokens : min((int64_t)start + max(n, 0), p.max_tokens);
    for (int64_t t = from + first; t < to; t += step) {
      p.slots[t] = -1;
      p.positions[t] = 0;
      p.token_request[t] = rest ? -1 : r;
      for (int w = 0; w < words; ++w) p.masks[t * words + w] = 0;
    }
    return;
  }
  int32_t* table = p.block_tables + (int64_t)r * p.table_width;
  // page b of the request, also before it is written into the table
  auto page = [&](int b) { return b < held ? table[b] : p.ring[ring_place((int64_t)mine.pop + (b - held), pages)]; };
  for (int b = held + first; b < need; b += step) table[b] = page(b);
  for (int b = need + first; b < held; b += step) {
    p.ring[ring_place((int64_t)mine.push + (b - need), pages)] = table[b];
    table[b] = -1;
  }
  const bool tree = n <= p.max_tree;  // masks are written; a chain's where there are no parents
  for (int i = first; i < n; i += step) {
    const int64_t t = start + i;
    const unsigned at = c + i;
    p.slots[t] = page((int)(at / (unsigned)P)) * P + (int)(at % (unsigned)P);
    p.token_request[t] = r;
    if (!tree) {
      p.positions[t] = (int)at;
      for (int w = 0; w < words; ++w) p.masks[t * words + w] = 0;
    }
  }
  if (tree && blockIdx.y == 0 && n > 0) {
    // Ancestors by doubling: after k rounds a node's set holds its 2^k nearest ancestors and `up` is the
    // one behind them.
    __shared__ int up[kMaxTree];
    __shared__ uint64_t set[kMaxTree / 64][kMaxTree];
    int above = -1;
    uint64_t seen[kMaxTree / 64];
#pragma unroll
    for (int w = 0; w < kMaxTree / 64; ++w) seen[w] = tid >> 6 == w ? uint64_t(1) << (tid & 63) : 0;
    if (tid < n) {
      above = parents != nullptr ? parents[start + tid] : tid - 1;
      if (above < 0 || above >= tid) above = -1;
    }
    for (int span = 1; span < n; span <<= 1) {
      up[tid] = above;
#pragma unroll
      for (int w = 0; w < kMaxTree / 64; ++w) set[w][tid] = seen[w];
      __syncthreads();
      if (above >= 0) {
#pragma unroll
        for (int w = 0; w < kMaxTree / 64; ++w) seen[w] |= set[w][above];
        above = up[above];
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
  const int blocks = cut.blocks(n), cost = kPagedLead + (c + n + kPagedTile - 1) / kPagedTile;
  if (first == 0) s.live[mine.place] = PagedLive{r, c, n, start, mine.flat, blocks, cost};
  const int64_t stop = mine.flat + (int64_t)blocks * cost;
  for (int64_t i = (mine.flat + mine.stretch - 1) / mine.stretch + first; i * mine.stretch < stop; i += step) {
    const int64_t at = i * mine.stretch - mine.flat;
    const int block = (int)(at / cost);
    s.slot[i] = PagedSlot{mine.place, block, (int)(at - (int64_t)block * cost), 0};
  }
}

// Every workgroup forms the sums over all requests for itself and fills in its own request.  The last
// one to have read the lengths held brings them up to date.
template <int K>
__global__ __launch_bounds__(kMaxTree) void afa_paged_plan_kernel(const afa_paged_plan p, const Cut cut, const int32_t* cached,
                                                                  const int32_t* fresh, const int32_t* parents) {
  __shared__ int64_t lds[kMaxTree / 64][3];
  __shared__ Mine shared;
  __shared__ bool last;
  PlanSums<kMaxTree, K> sums{p, cut, cached, fresh, lds};
  const Mine mine = sums.run(blockIdx.x, false, &shared);
  if (threadIdx.x == 0) {
    // the last of all by two steps: several hundred counts of one address would take longer than the rest
    int (*ticket)[16] = paged_schedule(p, cut.slots).header->ticket;
    const int all = (int)(gridDim.x * gridDim.y), id = (int)(blockIdx.y * gridDim.x + blockIdx.x), set = id % kTickets;
    last = true;
    if (all > kTickets) {
      last = atomicAdd(ticket[set], 1) == (all - set + kTickets - 1) / kTickets - 1;
      if (last) *ticket[set] = 0;
    }
    if (last) {
      last = atomicAdd(ticket[kTickets], 1) == min(all, kTickets) - 1;
      if (last) *ticket[kTickets] = 0;
    }
  }
  fill(p, cut, parents, blockIdx.x, mine, sums.end);
  __syncthreads();
  if (last) sums.finish();
}

// The same in two launches, for more requests.
constexpr int SCAN = 1024;
__global__ __launch_bounds__(SCAN) void afa_paged_scan_kernel(const afa_paged_plan p, const Cut cut, const int32_t* cached,
                                                              const int32_t* fresh) {
  __shared__ int64_t lds[SCAN / 64][3];
  __shared__ Mine shared;
  PlanSums<SCAN, 0> sums{p, cut, cached, fresh, lds};
  sums.run(-1, true, &shared);
  sums.finish();
}

__global__ __launch_bounds__(kMaxTree) void afa_paged_fill_kernel(const afa_paged_plan p, const Cut cut, const int32_t* cached,
                                                                  const int32_t* fresh, const int32_t* parents) {
  const PagedSchedule s = paged_schedule(p, cut.slots);
  const int r = blockIdx.x, R = (int)p.requests;
  Mine m = {};
  if (r < R) {
    m.start = p.starts[r];
    m.pop = s.pop[r];
    m.push = s.push[r];
    m.flat = s.flat[r];
    m.place = s.place[r];
    m.stretch = s.header->stretch;
    m.q = Request{cached[r], fresh[r], s.held[r], p.held[r], p.status[r]};
  }
  fill(p, cut, parents, r, m, p.starts[R]);
}

}  // namespace

hipError_t paged_build_launch(const afa_paged_plan& p, const PagedCut& c, const int32_t* cached, const int32_t* fresh,
                              const int32_t* parents, hipStream_t st) {
  // a workgroup of long prompts takes about 1024 of their tokens
  const int64_t y = (p.max_new + 1023) / 1024;
  const dim3 grid((unsigned)(p.requests + 1), (unsigned)(y < 64 ? y : 64));
  const Cut cut{__builtin_ctz((unsigned)c.rows), (int)(p.heads / p.kv_heads), (int)c.slots};
  if (p.requests <= kOwnSums && (int64_t)grid.x * grid.y <= kOwnGroups) {
    if (p.requests <= kMaxTree)
      hipLaunchKernelGGL((afa_paged_plan_kernel<1>), grid, dim3(kMaxTree), 0, st, p, cut, cached, fresh, parents);
    else
      hipLaunchKernelGGL((afa_paged_plan_kernel<4>), grid, dim3(kMaxTree), 0, st, p, cut, cached, fresh, parents);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(afa_paged_scan_kernel, dim3(1), dim3(SCAN), 0, st, p, cut, cached, fresh);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(afa_paged_fill_kernel, grid, dim3(kMaxTree), 0, st, p, cut, cached, fresh, parents);
  return hipGetLastError();
}

}  // namespace afa
