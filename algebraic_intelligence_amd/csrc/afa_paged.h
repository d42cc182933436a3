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
};
hipError_t paged_fwd_generic_launch(const PagedFwdArgs& a, hipStream_t st);
// Matrix-core path (afa_paged_mfma.hip): 16-byte aligned rows of q, pages and out.  ws: paged_fast_workspace bytes.
bool paged_fast_supported(const afa_paged_plan& p);
size_t paged_fast_workspace(const afa_paged_plan& p, const PagedCut& c);
hipError_t paged_fwd_fast_launch(const PagedFwdArgs& a, const PagedCut& c, void* ws, hipStream_t st);

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

// The axis whose section holds pair p, or -1 behind the last section.
__host__ __device__ inline int pair_axis(const AxisRotation& r, int p) {
  for (int a = 0; a < r.axes; ++a)
    if (p < r.end[a]) return a;
  return -1;
}

}  // namespace afa
