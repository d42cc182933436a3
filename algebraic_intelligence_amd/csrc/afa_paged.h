// Argument blocks and launchers of the paged-cache serving operators (afa_paged_*.hip, ago_axes.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/afa.h"

namespace afa {

constexpr int kPagedTile = 32;   // keys of a tile, the unit in which a request's keys are split
constexpr int kMaxTree = 256;    // nodes of a drafted tree
constexpr int kMaxAxes = 4;

// A part of one request's attention for one key/value head: query rows [row0, row0 + rows per item) of its
// new * group rows, key tiles [tile0, tile1).  part: the slot of its partial sums, -1 where the part is whole.
struct PagedItem {
  int request, row0, tile0, tile1, part, cached, fresh, start;
};

// Key tiles that row block `block` of a request's n new tokens sees: all, or in a chain those up to the
// block's last token.
__host__ __device__ inline int paged_block_tiles(int c, int n, bool tree, int block, int rows, int group) {
  const unsigned last = (unsigned)(block * rows + rows - 1) / (unsigned)group;
  return (int)((unsigned)(c + (tree || last >= (unsigned)n ? n - 1 : (int)last) + kPagedTile) / kPagedTile);
}

// plan->schedule: a header, six ints per request, the items, then a counter for each part of each key/value head.
// The ticket and the counters are 0 between calls.
enum { PS_ITEMS = 0, PS_CHUNK = 1, PS_TICKET = 2, PS_INTS = 16 };
struct PagedSchedule {
  int* header;
  int *pop, *push, *held, *chunks, *part, *item;  // per request
  PagedItem* items;
};

// How the attention of a plan is cut, a function of its sizes and the device alone.
struct PagedCut {
  int rows;            // query rows of an item
  int64_t target;      // items per head that fill the device
  int64_t max_items;   // per head
  int64_t max_parts;   // partial sums per head
};

PagedCut paged_cut(const afa_paged_plan& p, int cus);
size_t paged_schedule_bytes(const afa_paged_plan& p, const PagedCut& c);

__host__ __device__ inline PagedSchedule paged_schedule(const afa_paged_plan& p) {
  PagedSchedule s;
  const int64_t R = p.requests;
  s.header = p.schedule;
  int* at = p.schedule + PS_INTS;
  s.pop = at;
  s.push = at + R;
  s.held = at + 2 * R;
  s.chunks = at + 3 * R;
  s.part = at + 4 * R;
  s.item = at + 5 * R;
  // the items, two 16-byte words each, start at a multiple of 16 bytes
  s.items = (PagedItem*)(p.schedule + ((PS_INTS + 6 * R + 3) & ~(int64_t)3));
  return s;
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
hipError_t paged_fwd_fast_launch(const PagedFwdArgs& a, const PagedCut& c, int cus, void* ws, hipStream_t st);

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
