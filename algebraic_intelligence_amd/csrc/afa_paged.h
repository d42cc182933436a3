// Argument blocks and launchers of the paged-cache serving operators (afa_paged_*.hip, ago_axes.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/afa.h"

namespace afa {

constexpr int kPagedTile = 32;   // keys of a tile, the unit in which a request's keys are split
constexpr int kMaxTree = 256;    // nodes of a drafted tree
constexpr int kMaxAxes = 4;

// How the attention of a plan is cut, a function of its sizes and the device alone.
//
// A segment is one request's query rows of one block (up to `rows` of its new tokens * group) over all of its
// keys.  Laid end to end, a segment taking kPagedLead units and one for each of its key tiles, the segments
// of a key/value head form a line that is cut into `slots` even stretches, one for each workgroup.  Every
// workgroup so has the same units.  Trees and rows of one block have a tile of work in each.  In a chain of
// several blocks (a prompt) the units of a block behind its last token's keys are empty, on an empty cache about
// half of them: there the workgroups of the last blocks have up to twice the mean work.  A segment that a cut
// crosses ends as partial sums, at most two of a slot: of a segment that began earlier and of one that goes on.
struct PagedCut {
  int rows;
  int64_t slots;  // per key/value head
};
// What a segment costs beside its tiles, in tiles (its start, the join of its waves).  2, 4, 8 and 16 take 98, 96,
// 96 and 100 us for 32 requests of up to 32 drafted tokens over up to 8192, and 40, 38, 38 and 40 for 40 of up to
// 13 over up to 3001 in fp32.
constexpr int kPagedLead = 4;
constexpr int kPagedMin = 4;  // shortest stretch: a tile for each wave

// A request with attention to do: its place on the line, and `cost` units for each of `blocks` row blocks.
struct PagedLive {
  int request, cached, fresh, start;
  int64_t flat;
  int blocks, cost;
};
// Where slot s begins: unit `at` of row block `block` of live request `live`.
struct PagedSlot {
  int live, block, at, unused;
};

// plan->schedule.  The tickets and the counters are 0 between calls.
constexpr int kTickets = 32;  // of groups of workgroups, each on a cache line of its own, then one of the groups
struct PagedHeader {
  int64_t stretch, end;  // of a slot, and of the line
  int slots, unused[11];
  int ticket[kTickets + 1][16];
};
struct PagedSchedule {
  PagedHeader* header;
  PagedLive* live;
  PagedSlot* slot;
  int* count;                        // (kv_heads, 2, 2 slots): parts that have arrived, and groups of them
  int *pop, *push, *held, *cached;   // per request
  int64_t* flat;                     // per request, then its place among the live ones
  int* place;
};

PagedCut paged_cut(const afa_paged_plan& p, int cus);
size_t paged_schedule_bytes(const afa_paged_plan& p, const PagedCut& c);

__host__ __device__ inline PagedSchedule paged_schedule(const afa_paged_plan& p, int64_t slots) {
  PagedSchedule s;
  char* at = (char*)p.schedule;
  const int64_t R = p.requests;
  s.header = (PagedHeader*)at;
  at += sizeof(PagedHeader);
  s.live = (PagedLive*)at;
  at += R * sizeof(PagedLive);
  s.slot = (PagedSlot*)at;
  at += slots * sizeof(PagedSlot);
  s.flat = (int64_t*)at;
  at += R * 8;
  s.count = (int*)at;
  s.pop = s.count + p.kv_heads * 4 * slots;
  s.push = s.pop + R;
  s.held = s.push + R;
  s.cached = s.held + R;
  s.place = s.cached + R;
  return s;
}

// Key tiles that row block `block` of a request's n new tokens sees: all, or in a chain those up to the
// block's last token.
__host__ __device__ inline int paged_block_tiles(int c, int n, bool tree, int block, int rows, int group) {
  const unsigned last = (unsigned)(block * rows + rows - 1) / (unsigned)group;
  return (int)((unsigned)(c + (tree || last >= (unsigned)n ? n - 1 : (int)last) + kPagedTile) / kPagedTile);
}

hipError_t paged_build_launch(const afa_paged_plan& p, const PagedCut& c, const int32_t* cached, const int32_t* fresh,
                              const int32_t* parents, hipStream_t st);

struct PageStrides {
  int64_t k_page, k_head, k_slot, v_page, v_head, v_slot;
};

// Tables and positions of a rotation by several axes.
struct AxisRotation {
  const void *rc, *rs;   // (len, pairs); nullptr: none
  int64_t len;
  int pairs;
  const void* positions;
  int pos64;             // positions are int64
  int wide;              // aligned runs of four fp32 table entries are 16-byte aligned
  int axes;
  int end[kMaxAxes];     // first pair behind each axis's section
};

struct AppendArgs {
  const void *q, *k, *v;
  void *q_out, *k_pages, *v_pages;
  int64_t q_t, q_h, k_t, k_h, v_t, v_h;
  PageStrides ps;
  AxisRotation rot;
  const int32_t* slots;
  int tokens, heads, kv_heads, dim, page_size;
  int64_t capacity;      // slots in the pool
};
hipError_t paged_append_launch(int dtype, const AppendArgs& a, hipStream_t st);

// Keys and values that all requests of a call see before their own: (kv_heads, len, head_dim).
struct PrefixKeys {
  const void *k, *v;
  int64_t k_head, k_key, v_head, v_key;
  int len;  // 0: none
};

struct PagedFwdArgs {
  afa_paged_plan plan;
  PagedSchedule sched;
  const void *q, *k_pages, *v_pages;
  const int64_t* masks;  // nullptr: no trees
  int64_t q_t, q_h;
  PageStrides ps;
  void* out;
  void* denom;           // nullable
  double scale, omega;
  int group, zero_tail;
  PrefixKeys prefix;
};
hipError_t paged_fwd_generic_launch(const PagedFwdArgs& a, hipStream_t st);
// Matrix-core path (afa_paged_mfma.hip): 16-byte aligned rows of q, pages and out.  ws: paged_fast_workspace bytes.
bool paged_fast_supported(const afa_paged_plan& p);
size_t paged_fast_workspace(const afa_paged_plan& p, const PagedCut& c);
// Sums over a shared prefix: (max_tokens, heads, head_dim) numerators and (max_tokens, heads) row sums; nullptr: none.
struct PrefixSums {
  float *top, *bottom;
};
hipError_t paged_fwd_fast_launch(const PagedFwdArgs& a, const PagedCut& c, const PrefixSums& shared, void* ws, hipStream_t st);
// The prefix's part (afa_prefix.hip), whose sums that call takes.  ws: paged_fast_workspace bytes of the cut.
PagedCut prefix_cut(const afa_paged_plan& p, int cus);
hipError_t prefix_sums_launch(const PagedFwdArgs& a, const PagedCut& c, const PrefixSums& shared, void* ws, hipStream_t st);

// What each cached token was given by the step's rows (afa_paged_weights.hip).
struct WeightArgs {
  afa_paged_plan plan;
  PagedSchedule sched;
  const void *q, *k_pages;
  const int64_t* masks;  // nullptr: no trees
  const void* denom;     // (max_tokens, heads), accumulation type
  int64_t q_t, q_h, k_page, k_head, k_slot;
  float* weights;        // (requests, row stride)
  int64_t row;
  double scale;
  int group;
};
// Whether the matrix-core kernel takes the call.  It has `ws`, the attention's workspace; nullptr: the other kernel.
bool paged_weights_fast(const WeightArgs& a);
hipError_t paged_weights_launch(const WeightArgs& a, const PagedCut& cut, int cus, void* ws, size_t ws_bytes, hipStream_t st);

// Requests cut back to a budget of tokens (afa_paged_evict.hip).
struct EvictArgs {
  int64_t num_pages, page_size, requests, table_width, kv_heads, head_dim;
  const int32_t *block_tables, *held, *cached;
  void *k_pages, *v_pages;
  PageStrides ps;
  const float* weights;  // (requests, row stride)
  int64_t row;
  float* left;           // (requests, table_width * page_size)
  int32_t* lens;
  int32_t* space;        // paged_evict_workspace bytes, 16-byte aligned
  int budget, first, recent, esz;
  int rows, chunks;      // set by the launch: places of a chunk, a power of two; chunks of a budget; and the
  int log_page, slices;  // logarithm of a page_size that is one, or -1; workgroups of a long request, or 0
};
size_t paged_evict_workspace(int64_t requests, int64_t max_len, int64_t budget, int64_t kv_heads, int64_t head_dim);
hipError_t paged_evict_launch(EvictArgs a, hipStream_t st);

struct RotateAxesArgs {
  const void *x[2];
  void* y[2];
  int64_t sx[2][3], sy[2][3];  // b, h, l
  int heads[2];
  int64_t batch, seq;
  int dim;
  AxisRotation rot;
  int64_t pos_b;
  float sign;
};
hipError_t rotate_axes_launch(int dtype, const RotateAxesArgs& a, hipStream_t st);

// Norm of q's and k's rows with their rotation (ago_norm.hip).  Scales are fp32 (fp64 for AFA_F64).
struct HeadNorm {
  const void* scale[2];  // of q and of k, (dim,)
  double eps;
};
struct NormArgs {
  const void *x[2];
  const void *g[2];        // backward: the results' cotangents
  void* y[2];              // results, or x's gradients
  int64_t sx[2][3], sg[2][3], sy[2][3];  // b, h, l
  int heads[2];
  int64_t batch, seq;
  int dim;
  HeadNorm norm;
  AxisRotation rot;
  int64_t pos_b;
};
hipError_t norm_rotate_launch(int dtype, const NormArgs& a, hipStream_t st);
// dscale: of q and of k, fp32 (fp64), (dim,); ws: norm_rotate_bwd_workspace bytes
size_t norm_rotate_bwd_workspace(int dtype, int dim, int cus);
hipError_t norm_rotate_bwd_launch(int dtype, const NormArgs& a, void* const dscale[2], void* ws, int cus, hipStream_t st);
hipError_t paged_append_norm_launch(int dtype, const AppendArgs& a, const HeadNorm& n, hipStream_t st);

// The axis whose section holds pair p, or -1 behind the last section.
__host__ __device__ inline int pair_axis(const AxisRotation& r, int p) {
  for (int a = 0; a < r.axes; ++a)
    if (p < r.end[a]) return a;
  return -1;
}

}  // namespace afa
