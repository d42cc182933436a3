// C ABI of the paged-cache serving operators (include/afa.h): argument checks and dispatch.
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <utility>

#include "../../include/afa.h"
#include "afa_launch.h"
#include "afa_paged.h"

namespace {

constexpr int64_t kLaunchThreads = int64_t(1) << 32;

bool aligned16(const void* p) { return ((uintptr_t)p & 15u) == 0; }
bool within(int64_t v, int64_t lo, int64_t hi) { return v >= lo && v <= hi; }

// The sizes of a plan, without its pointers.
int check_sizes(const afa_paged_plan& p) {
  if (!within(p.dtype, AFA_F32, AFA_F64)) return AFA_ERR_DTYPE;
  const int64_t most = int64_t(1) << 30;
  if (!within(p.num_pages, 1, most) || !within(p.page_size, 1, most) || !within(p.requests, 1, int64_t(1) << 22) ||
      !within(p.table_width, 1, most) || !within(p.max_tokens, 1, int64_t(1) << 26) ||
      !within(p.max_new, 1, p.max_tokens) || !within(p.heads, 1, 1 << 16) || !within(p.kv_heads, 1, p.heads))
    return AFA_ERR_SHAPE;
  // slots, cache indices and table rows by 32 bits
  if (p.num_pages > ((int64_t(1) << 31) - 1) / p.page_size || p.table_width > most / p.page_size) return AFA_ERR_SHAPE;
  if (p.heads % p.kv_heads != 0) return AFA_ERR_SHAPE;
  if (p.max_tree % 64 != 0 || !within(p.max_tree, 0, afa::kMaxTree)) return AFA_ERR_SHAPE;
  if (!within(p.head_dim, 1, 1024)) return AFA_ERR_HEAD_DIM;
  // rows of one key/value head, and items, by 32 bits
  const int64_t group = p.heads / p.kv_heads;
  if (p.max_tokens > ((int64_t(1) << 30) - 1) / group) return AFA_ERR_SHAPE;
  return AFA_OK;
}

int check_plan(const afa_paged_plan* p) {
  if (p == nullptr) return AFA_ERR_NULL;
  const int rc = check_sizes(*p);
  if (rc != AFA_OK) return rc;
  if (p->block_tables == nullptr || p->held == nullptr || p->ring == nullptr || p->ring_state == nullptr ||
      p->slots == nullptr || p->positions == nullptr || p->token_request == nullptr || p->starts == nullptr ||
      p->status == nullptr || p->schedule == nullptr || (p->max_tree > 0 && p->masks == nullptr))
    return AFA_ERR_NULL;
  return aligned16(p->schedule) ? AFA_OK : AFA_ERR_ALIGN;
}

// Tables, positions and sections of a rotation of head_dim features.
int check_rotation(afa::AxisRotation& r, const void* rc, const void* rs, int64_t len, int64_t head_dim, int axes,
                   const int32_t* sections, const void* positions, int pos64) {
  r = {};
  if (rc == nullptr && rs == nullptr) return AFA_OK;
  if (rc == nullptr || rs == nullptr || head_dim % 2 != 0 || len < 1) return AFA_ERR_ROTARY;
  if (positions == nullptr) return AFA_ERR_NULL;
  if (axes < 1 || axes > afa::kMaxAxes) return AFA_ERR_ROTARY;
  r.rc = rc;
  r.rs = rs;
  r.len = len;
  r.pairs = (int)(head_dim / 2);
  r.positions = positions;
  r.pos64 = pos64;
  r.wide = r.pairs % 4 == 0 && aligned16(rc) && aligned16(rs);
  r.axes = axes;
  if (sections == nullptr) {
    if (axes != 1) return AFA_ERR_NULL;
    r.end[0] = r.pairs;
    return AFA_OK;
  }
  int64_t end = 0;
  for (int a = 0; a < axes; ++a) {
    if (sections[a] < 0) return AFA_ERR_ROTARY;
    end += sections[a];
    if (end > r.pairs) return AFA_ERR_ROTARY;
    r.end[a] = (int)end;
  }
  return AFA_OK;
}

afa::PageStrides page_strides_of(const afa_paged_plan& p, const int64_t* s) {
  if (s != nullptr) return afa::PageStrides{s[0], s[1], s[2], s[3], s[4], s[5]};
  const int64_t head = p.page_size * p.head_dim, page = p.kv_heads * head;
  return afa::PageStrides{page, head, p.head_dim, page, head, p.head_dim};
}

// Whether `left` is a sum of the axes' steps (bytes), each taken between `least` and `most` times.  The axes come in falling order of
// their steps, and reach[i] is what those from i on come to at least and at most: of steps that each pass what the later ones
// come to, as strides of arrays whose elements lie apart do, two numbers at most are left to try of each.
struct Axis {
  int64_t step, least, most;
};
struct Reach {
  int64_t low, high;
};
bool sum_of_steps(const Axis* a, const Reach* reach, int count, int64_t left, int& tries) {
  if (left < reach[0].low || left > reach[0].high) return false;
  if (count == 0) return true;  // both are 0
  if (--tries < 0) return false;
  // multiples of the step that leave what the later axes reach
  auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  const int64_t low = std::max(-floor_div(reach[1].high - left, a->step), a->least);
  const int64_t high = std::min(floor_div(left - reach[1].low, a->step), a->most);
  for (int64_t n = low; n <= high && tries > 0; ++n)
    if (sum_of_steps(a + 1, reach + 1, count - 1, left - n * a->step, tries)) return true;
  return false;
}

// Whether k and v pages of these strides share a byte, as far as 4096 steps tell, which is to the end where an array's own
// elements lie apart and both have the same strides, in any order, or lie in places of their own altogether.
bool pages_share(const afa_paged_plan& p, const void* k_pages, const void* v_pages, const int64_t* strides) {
  const int64_t esz = p.dtype == AFA_F64 ? 8 : p.dtype == AFA_F32 ? 4 : 2;
  const int64_t sizes[4] = {p.num_pages, p.kv_heads, p.page_size, p.head_dim};
  Axis a[9];
  int count = 0;
  auto add = [&](int64_t step, int64_t least, int64_t most) {
    if (step < 0) {
      step = -step;
      std::swap(least, most);
      least = -least;
      most = -most;
    }
    if (step == 0 || least == most) return true;
    if (step >= int64_t(1) << 50 || (double)step * (double)(most - least) >= 0x1p58) return false;  // sums of them fit
    for (int i = 0; i < count; ++i)
      if (a[i].step == step) {  // also of k's and v's arrays in another order
        a[i].least += least;
        a[i].most += most;
        return true;
      }
    a[count++] = Axis{step, least, most};
    return true;
  };
  bool fits = add(1, 1 - esz, esz - 1);
  for (int i = 0; i < 4; ++i) {
    const int64_t k = (i < 3 ? strides[i] : 1), v = (i < 3 ? strides[3 + i] : 1), n = sizes[i] - 1;
    const int64_t most = int64_t(1) << 46;
    if (!within(k, -most, most) || !within(v, -most, most)) return false;
    if (k == v) {
      fits = fits && add(k * esz, -n, n);
    } else {
      fits = fits && add(k * esz, 0, n);
      fits = fits && add(v * esz, -n, 0);
    }
  }
  if (!fits) return false;
  std::sort(a, a + count, [](const Axis& x, const Axis& y) { return x.step > y.step; });
  Reach reach[10];
  reach[count] = Reach{0, 0};
  for (int i = count - 1; i >= 0; --i)
    reach[i] = Reach{reach[i + 1].low + a[i].step * a[i].least, reach[i + 1].high + a[i].step * a[i].most};
  int tries = 4096;
  return sum_of_steps(a, reach, count, (int64_t)((uintptr_t)v_pages - (uintptr_t)k_pages), tries);
}

// The arguments of a cache write; `turned`: q_out is written.
int check_append(afa::AppendArgs& a, const afa_paged_plan* plan, const void* q, const void* k, const void* v,
                 const int64_t* strides, void* q_out, void* k_pages, void* v_pages, const int64_t* page_strides,
                 const void* rot_cos, const void* rot_sin, int64_t rot_len, const int32_t* positions, int axes,
                 const int32_t* sections, bool turned) {
  int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr) return AFA_ERR_NULL;
  if (q_out == nullptr && (turned || rot_cos != nullptr)) return AFA_ERR_NULL;
  if (positions == nullptr && axes != 1) return AFA_ERR_NULL;
  const afa_paged_plan& p = *plan;
  a = {};
  rc = check_rotation(a.rot, rot_cos, rot_sin, rot_len, p.head_dim, axes, sections,
                      positions != nullptr ? positions : p.positions, 0);
  if (rc != AFA_OK) return rc;
  a.q = q; a.k = k; a.v = v;
  a.q_out = q_out; a.k_pages = k_pages; a.v_pages = v_pages;
  a.q_t = p.heads * p.head_dim;
  a.k_t = a.v_t = p.kv_heads * p.head_dim;
  a.q_h = a.k_h = a.v_h = p.head_dim;
  if (strides != nullptr) {
    a.q_t = strides[0]; a.q_h = strides[1];
    a.k_t = strides[2]; a.k_h = strides[3];
    a.v_t = strides[4]; a.v_h = strides[5];
  }
  if (page_strides != nullptr && pages_share(p, k_pages, v_pages, page_strides)) return AFA_ERR_OVERLAP;
  a.ps = page_strides_of(p, page_strides);
  a.slots = p.slots;
  a.tokens = (int)p.max_tokens; a.heads = (int)p.heads; a.kv_heads = (int)p.kv_heads; a.dim = (int)p.head_dim;
  a.page_size = (int)p.page_size;
  a.capacity = p.num_pages * p.page_size;
  if (p.max_tokens > (kLaunchThreads - 256) / ((p.heads + 2 * p.kv_heads) * ((p.head_dim + 1) / 2))) return AFA_ERR_SHAPE;
  return AFA_OK;
}

constexpr int64_t kMostPrefix = int64_t(1) << 29;

// The arguments of the attention of a plan's tokens, without a prefix.
int check_fwd(afa::PagedFwdArgs& a, const afa_paged_plan* plan, const void* q, const int64_t* q_strides, const void* k_pages,
              const void* v_pages, const int64_t* page_strides, const int64_t* masks, void* out, void* denom,
              double sink_omega, unsigned flags) {
  const int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || out == nullptr) return AFA_ERR_NULL;
  if (!(sink_omega >= 0.0 && sink_omega < INFINITY)) return AFA_ERR_SINK;
  const afa_paged_plan& p = *plan;
  if (masks != nullptr && p.max_tree == 0) return AFA_ERR_UNSUPPORTED;
  if (p.max_tokens > (kLaunchThreads - 1) / 256 / p.heads) return AFA_ERR_SHAPE;
  a = {};
  a.plan = p;
  a.sched = afa::paged_schedule(p, afa::paged_cut(p, afa::device_cus()).slots);
  a.q = q; a.k_pages = k_pages; a.v_pages = v_pages;
  a.masks = masks != nullptr ? masks : p.max_tree > 0 ? p.masks : nullptr;
  a.q_t = q_strides != nullptr ? q_strides[0] : p.heads * p.head_dim;
  a.q_h = q_strides != nullptr ? q_strides[1] : p.head_dim;
  a.ps = page_strides_of(p, page_strides);
  a.out = out; a.denom = denom;
  a.scale = 1.0 / std::sqrt((double)p.head_dim);
  a.omega = sink_omega;
  a.group = (int)(p.heads / p.kv_heads);
  a.zero_tail = (flags & AFA_FLAG_ZERO_TAIL) != 0;
  return AFA_OK;
}

// Whether the matrix-core kernel takes the call: 16-byte rows of q and of the pages; byte offsets within a page, and its
// stride, in 32 bits.
bool fast_rows(const afa::PagedFwdArgs& a, unsigned flags) {
  const afa_paged_plan& p = a.plan;
  const int64_t unit = p.dtype == AFA_F32 ? 4 : 8;
  bool fast = (flags & AFA_FLAG_GENERIC) == 0 && afa::paged_fast_supported(p) && aligned16(a.q) && aligned16(a.k_pages) &&
              aligned16(a.v_pages) && aligned16(a.out) && a.q_t % unit == 0 && a.q_h % unit == 0;
  for (int64_t v : {a.ps.k_page, a.ps.k_head, a.ps.k_slot, a.ps.v_page, a.ps.v_head, a.ps.v_slot})
    fast = fast && v % unit == 0 && v >= 0;
  const int64_t reach = (int64_t(1) << 30) / p.page_size;  // elements, of 4 bytes at most
  for (int64_t v : {a.ps.k_slot, a.ps.v_slot}) fast = fast && v < reach - p.head_dim;
  for (int64_t v : {a.ps.k_page, a.ps.v_page}) fast = fast && v < int64_t(1) << 30;
  return fast;
}

// A call behind a prefix: its sums, and the parts of the two launches, which come one after the other.
size_t prefix_sum_bytes(const afa_paged_plan& p) {
  return (size_t)((p.max_tokens * p.heads * (p.head_dim + 1) * 4 + 15) / 16 * 16);
}
size_t prefix_workspace(const afa_paged_plan& p, int cus) {
  const size_t a = afa::paged_fast_workspace(p, afa::paged_cut(p, cus)), b = afa::paged_fast_workspace(p, afa::prefix_cut(p, cus));
  return prefix_sum_bytes(p) + (a > b ? a : b);
}

// A norm's scales and eps.
int check_norm(afa::HeadNorm& n, const void* q_scale, const void* k_scale, bool has_k, double eps) {
  if (q_scale == nullptr || (has_k && k_scale == nullptr)) return AFA_ERR_NULL;
  if (!(eps >= 0.0 && eps < INFINITY)) return AFA_ERR_EPS;
  n.scale[0] = q_scale;
  n.scale[1] = k_scale;
  n.eps = eps;
  return AFA_OK;
}

// Workspace of `need` bytes: the caller's, or one of the stream's (`own`).
int workspace_of(void* given, size_t bytes, size_t need, hipStream_t s, void*& ws, bool& own) {
  own = given == nullptr;
  ws = given;
  if (own) {
    ws = afa::workspace_alloc(need, s);
    return ws != nullptr ? AFA_OK : afa::hip_status_code(hipErrorOutOfMemory);
  }
  if (bytes < need) return AFA_ERR_WORKSPACE;
  return aligned16(ws) ? AFA_OK : AFA_ERR_ALIGN;
}
int workspace_done(hipError_t e, void* ws, bool own, hipStream_t s) {
  if (own) {
    const hipError_t e2 = hipFreeAsync(ws, s);
    if (e == hipSuccess) e = e2;
  }
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

// Sizes, strides, positions and norms of ago_norm_rotate_axes and its gradient.
int check_norm_rows(afa::NormArgs& a, int dtype, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t seq_len,
                    int64_t head_dim, const void* q_scale, const void* k_scale, double eps, const void* rot_cos,
                    const void* rot_sin, int64_t rot_len, const void* positions, int pos_bytes, int64_t pos_b, int axes,
                    const int32_t* sections) {
  if (!within(dtype, AFA_F32, AFA_F64)) return AFA_ERR_DTYPE;
  if (batch < 1 || q_heads < 1 || k_heads < 0 || seq_len < 1 || head_dim < 1) return AFA_ERR_SHAPE;
  if (pos_bytes != 4 && pos_bytes != 8) return AFA_ERR_UNSUPPORTED;
  const int64_t most = kLaunchThreads - 256;
  if (head_dim > (1 << 24) || seq_len > most || batch > most / seq_len || q_heads > (1 << 30) || k_heads > (1 << 30) ||
      batch * seq_len > most / (q_heads + k_heads) ||
      batch * seq_len * (q_heads + k_heads) > most / ((head_dim + 1) / 2))
    return AFA_ERR_SHAPE;
  a = {};
  int rc = check_norm(a.norm, q_scale, k_scale, k_heads > 0, eps);
  if (rc != AFA_OK) return rc;
  // no positions: a row's index
  if (positions == nullptr && (axes != 1 || pos_b != 0)) return AFA_ERR_NULL;
  rc = check_rotation(a.rot, rot_cos, rot_sin, rot_len, head_dim, axes, sections, positions != nullptr ? positions : &axes,
                      pos_bytes == 8);
  if (rc != AFA_OK) return rc;
  if (positions == nullptr) a.rot.positions = nullptr;
  a.heads[0] = (int)q_heads; a.heads[1] = (int)k_heads;
  a.batch = batch; a.seq = seq_len; a.dim = (int)head_dim;
  a.pos_b = pos_b;
  return AFA_OK;
}
void row_strides(const afa::NormArgs& a, const int64_t* strides, int64_t (*q)[3]) {
  for (int i = 0; i < 2; ++i) {
    if (strides != nullptr) {
      for (int j = 0; j < 3; ++j) q[i][j] = strides[3 * i + j];
    } else {
      q[i][0] = a.heads[i] * a.seq * a.dim;
      q[i][1] = a.seq * a.dim;
      q[i][2] = a.dim;
    }
  }
}

}  // namespace

extern "C" {

size_t afa_paged_schedule_bytes(const afa_paged_plan* plan) {
  if (plan == nullptr || check_sizes(*plan) != AFA_OK) return 0;
  return afa::paged_schedule_bytes(*plan, afa::paged_cut(*plan, afa::device_cus()));
}

int afa_paged_build(const afa_paged_plan* plan, const int32_t* cached, const int32_t* fresh, const int32_t* parents,
                    void* stream) {
  const int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (cached == nullptr || fresh == nullptr) return AFA_ERR_NULL;
  const hipError_t e = afa::paged_build_launch(*plan, afa::paged_cut(*plan, afa::device_cus()), cached, fresh, parents,
                                               (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

int afa_paged_append(const afa_paged_plan* plan, const void* q, const void* k, const void* v, const int64_t* strides,
                     void* q_out, void* k_pages, void* v_pages, const int64_t* page_strides, const void* rot_cos,
                     const void* rot_sin, int64_t rot_len, const int32_t* positions, int axes, const int32_t* sections,
                     void* stream) {
  afa::AppendArgs a;
  const int rc = check_append(a, plan, q, k, v, strides, q_out, k_pages, v_pages, page_strides, rot_cos, rot_sin, rot_len,
                              positions, axes, sections, false);
  if (rc != AFA_OK) return rc;
  const hipError_t e = afa::paged_append_launch((int)plan->dtype, a, (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

int afa_paged_append_norm(const afa_paged_plan* plan, const void* q, const void* k, const void* v, const int64_t* strides,
                          void* q_out, void* k_pages, void* v_pages, const int64_t* page_strides, const void* q_scale,
                          const void* k_scale, double eps, const void* rot_cos, const void* rot_sin, int64_t rot_len,
                          const int32_t* positions, int axes, const int32_t* sections, void* stream) {
  afa::AppendArgs a;
  int rc = check_append(a, plan, q, k, v, strides, q_out, k_pages, v_pages, page_strides, rot_cos, rot_sin, rot_len, positions,
                        axes, sections, true);
  if (rc != AFA_OK) return rc;
  afa::HeadNorm n;
  rc = check_norm(n, q_scale, k_scale, true, eps);
  if (rc != AFA_OK) return rc;
  const hipError_t e = afa::paged_append_norm_launch((int)plan->dtype, a, n, (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

size_t afa_paged_workspace_size(const afa_paged_plan* plan) {
  if (plan == nullptr || check_sizes(*plan) != AFA_OK || !afa::paged_fast_supported(*plan)) return 0;
  return afa::paged_fast_workspace(*plan, afa::paged_cut(*plan, afa::device_cus()));
}

int afa_paged_fwd(const afa_paged_plan* plan, const void* q, const int64_t* q_strides, const void* k_pages,
                  const void* v_pages, const int64_t* page_strides, const int64_t* masks, void* out, void* denom,
                  double sink_omega, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  afa::PagedFwdArgs a;
  const int rc = check_fwd(a, plan, q, q_strides, k_pages, v_pages, page_strides, masks, out, denom, sink_omega, flags);
  if (rc != AFA_OK) return rc;
  const hipStream_t s = (hipStream_t)stream;
  if (!fast_rows(a, flags)) {
    const hipError_t e = afa::paged_fwd_generic_launch(a, s);
    return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
  }
  const afa::PagedCut cut = afa::paged_cut(*plan, afa::device_cus());
  void* ws;
  bool own;
  const int got = workspace_of(workspace, workspace_bytes, afa::paged_fast_workspace(*plan, cut), s, ws, own);
  if (got != AFA_OK) return got;
  return workspace_done(afa::paged_fwd_fast_launch(a, cut, afa::PrefixSums{}, ws, s), ws, own, s);
}

size_t afa_paged_prefix_workspace_size(const afa_paged_plan* plan, int64_t prefix_len) {
  if (plan == nullptr || check_sizes(*plan) != AFA_OK || !within(prefix_len, 1, kMostPrefix) ||
      !afa::paged_fast_supported(*plan))
    return 0;
  return prefix_workspace(*plan, afa::device_cus());
}

int afa_paged_prefix_fwd(const afa_paged_plan* plan, const void* q, const int64_t* q_strides, const void* k_prefix,
                         const void* v_prefix, int64_t prefix_len, const int64_t* prefix_strides, const void* k_pages,
                         const void* v_pages, const int64_t* page_strides, const int64_t* masks, void* out, void* denom,
                         double sink_omega, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  afa::PagedFwdArgs a;
  const int rc = check_fwd(a, plan, q, q_strides, k_pages, v_pages, page_strides, masks, out, denom, sink_omega, flags);
  if (rc != AFA_OK) return rc;
  if (k_prefix == nullptr || v_prefix == nullptr) return AFA_ERR_NULL;
  if (!within(prefix_len, 1, kMostPrefix)) return AFA_ERR_SHAPE;
  afa::PrefixKeys& x = a.prefix;
  x.k = k_prefix;
  x.v = v_prefix;
  x.len = (int)prefix_len;
  x.k_head = x.v_head = prefix_len * plan->head_dim;
  x.k_key = x.v_key = plan->head_dim;
  if (prefix_strides != nullptr) {
    x.k_head = prefix_strides[0]; x.k_key = prefix_strides[1];
    x.v_head = prefix_strides[2]; x.v_key = prefix_strides[3];
  }
  const hipStream_t s = (hipStream_t)stream;
  const afa_paged_plan& p = *plan;
  // a tile's 32 rows by 32-bit byte offsets
  const int64_t unit = p.dtype == AFA_F32 ? 4 : 8;
  bool fast = fast_rows(a, flags) && aligned16(k_prefix) && aligned16(v_prefix);
  for (int64_t v : {x.k_head, x.k_key, x.v_head, x.v_key}) fast = fast && v % unit == 0;
  for (int64_t v : {x.k_key, x.v_key}) fast = fast && v >= 0 && v < int64_t(1) << 24;
  if (!fast) {
    const hipError_t e = afa::paged_fwd_generic_launch(a, s);
    return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
  }
  const int cus = afa::device_cus();
  void* ws;
  bool own;
  const int got = workspace_of(workspace, workspace_bytes, prefix_workspace(p, cus), s, ws, own);
  if (got != AFA_OK) return got;
  // the sums, then the parts of either launch
  const int64_t rows = p.max_tokens * p.heads;
  const afa::PrefixSums sums{(float*)ws, (float*)ws + rows * p.head_dim};
  void* parts = (char*)ws + prefix_sum_bytes(p);
  hipError_t e = afa::prefix_sums_launch(a, afa::prefix_cut(p, cus), sums, parts, s);
  if (e == hipSuccess) e = afa::paged_fwd_fast_launch(a, afa::paged_cut(p, cus), sums, parts, s);
  return workspace_done(e, ws, own, s);
}

int afa_paged_weights(const afa_paged_plan* plan, const void* q, const int64_t* q_strides, const void* k_pages,
                      const int64_t* page_strides, const int64_t* masks, const void* denom, float* weights,
                      int64_t weights_stride, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || k_pages == nullptr || denom == nullptr || weights == nullptr) return AFA_ERR_NULL;
  const afa_paged_plan& p = *plan;
  if (masks != nullptr && p.max_tree == 0) return AFA_ERR_UNSUPPORTED;
  if (weights_stride < p.table_width * p.page_size && p.requests > 1) return AFA_ERR_SHAPE;
  afa::WeightArgs a = {};
  a.plan = p;
  const int cus = afa::device_cus();
  const afa::PagedCut cut = afa::paged_cut(p, cus);
  a.sched = afa::paged_schedule(p, cut.slots);
  a.q = q; a.k_pages = k_pages;
  a.masks = masks != nullptr ? masks : p.max_tree > 0 ? p.masks : nullptr;
  a.denom = denom;
  a.q_t = q_strides != nullptr ? q_strides[0] : p.heads * p.head_dim;
  a.q_h = q_strides != nullptr ? q_strides[1] : p.head_dim;
  a.k_head = p.page_size * p.head_dim;
  a.k_page = p.kv_heads * a.k_head;
  a.k_slot = p.head_dim;
  if (page_strides != nullptr) {
    a.k_page = page_strides[0]; a.k_head = page_strides[1]; a.k_slot = page_strides[2];
  }
  a.weights = weights;
  a.row = weights_stride;
  a.scale = 1.0 / std::sqrt((double)p.head_dim);
  a.group = (int)(p.heads / p.kv_heads);
  const hipStream_t s = (hipStream_t)stream;
  if ((flags & AFA_FLAG_GENERIC) != 0 || !afa::paged_weights_fast(a)) {
    const hipError_t e = afa::paged_weights_launch(a, cut, cus, nullptr, 0, s);
    return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
  }
  const size_t need = afa::paged_fast_workspace(p, cut);
  void* ws;
  bool own;
  const int got = workspace_of(workspace, workspace_bytes, need, s, ws, own);
  if (got != AFA_OK) return got;
  return workspace_done(afa::paged_weights_launch(a, cut, cus, ws, need, s), ws, own, s);
}

size_t afa_paged_evict_workspace_size(int64_t requests, int64_t max_len, int64_t budget, int64_t kv_heads, int64_t head_dim) {
  if (!within(requests, 1, int64_t(1) << 22) || !within(max_len, 1, int64_t(1) << 30) || !within(budget, 1, max_len) || !within(kv_heads, 1, 1 << 16) ||
      !within(head_dim, 1, 1024))
    return 0;
  return afa::paged_evict_workspace(requests, max_len, budget, kv_heads, head_dim);
}

int afa_paged_evict(int dtype, int64_t num_pages, int64_t page_size, int64_t requests, int64_t table_width, int64_t kv_heads,
                    int64_t head_dim, const int32_t* block_tables, const int32_t* held, void* k_pages, void* v_pages,
                    const int64_t* page_strides, const int32_t* cached, int64_t budget, int64_t first, int64_t recent,
                    const float* weights, int64_t weights_stride, float* left, int32_t* lens, void* workspace,
                    size_t workspace_bytes, void* stream) {
  afa_paged_plan p = {};
  p.num_pages = num_pages; p.page_size = page_size; p.requests = requests; p.table_width = table_width;
  p.max_tokens = p.max_new = 1;
  p.heads = p.kv_heads = kv_heads; p.head_dim = head_dim; p.dtype = dtype;
  const int rc = check_sizes(p);
  if (rc != AFA_OK) return rc;
  if (block_tables == nullptr || held == nullptr || k_pages == nullptr || v_pages == nullptr || cached == nullptr ||
      weights == nullptr || left == nullptr || lens == nullptr)
    return AFA_ERR_NULL;
  const int64_t width = table_width * page_size;
  if (!within(budget, 1, width) || first < 0 || recent < 0 || first > budget || recent > budget - first) return AFA_ERR_SHAPE;
  if (weights_stride < width && requests > 1) return AFA_ERR_SHAPE;
  if (page_strides != nullptr && pages_share(p, k_pages, v_pages, page_strides)) return AFA_ERR_OVERLAP;
  if (requests > (kLaunchThreads - 1) / 2048 / kv_heads || requests > (kLaunchThreads - 1) / 1024 / ((width + 8191) / 8192))
    return AFA_ERR_SHAPE;
  afa::EvictArgs a = {};
  a.num_pages = num_pages; a.page_size = page_size; a.requests = requests; a.table_width = table_width;
  a.kv_heads = kv_heads; a.head_dim = head_dim;
  a.block_tables = block_tables; a.held = held; a.cached = cached;
  a.k_pages = k_pages; a.v_pages = v_pages;
  a.ps = page_strides_of(p, page_strides);
  a.weights = weights; a.row = weights_stride;
  a.left = left; a.lens = lens;
  a.budget = (int)budget; a.first = (int)first; a.recent = (int)recent;
  a.esz = dtype == AFA_F64 ? 8 : dtype == AFA_F32 ? 4 : 2;
  const hipStream_t s = (hipStream_t)stream;
  void* ws;
  bool own;
  const int got = workspace_of(workspace, workspace_bytes, afa::paged_evict_workspace(requests, width, budget, kv_heads, head_dim), s,
                               ws, own);
  if (got != AFA_OK) return got;
  a.space = (int32_t*)ws;
  return workspace_done(afa::paged_evict_launch(a, s), ws, own, s);
}

int ago_norm_rotate_axes(int dtype, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t seq_len, int64_t head_dim,
                         const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, const void* q_scale,
                         const void* k_scale, double eps, const void* rot_cos, const void* rot_sin, int64_t rot_len,
                         const void* positions, int pos_bytes, int64_t pos_b, int axes, const int32_t* sections,
                         void* stream) {
  afa::NormArgs a;
  const int rc = check_norm_rows(a, dtype, batch, q_heads, k_heads, seq_len, head_dim, q_scale, k_scale, eps, rot_cos, rot_sin,
                                 rot_len, positions, pos_bytes, pos_b, axes, sections);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || q_out == nullptr || (k_heads > 0 && (k == nullptr || k_out == nullptr))) return AFA_ERR_NULL;
  a.x[0] = q; a.x[1] = k_heads > 0 ? k : q;
  a.y[0] = q_out; a.y[1] = k_heads > 0 ? k_out : q_out;
  row_strides(a, strides, a.sx);
  row_strides(a, strides != nullptr ? strides + 6 : nullptr, a.sy);
  const hipError_t e = afa::norm_rotate_launch(dtype, a, (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

size_t ago_norm_rotate_axes_bwd_workspace_size(int dtype, int64_t head_dim) {
  if (!within(dtype, AFA_F32, AFA_F64) || !within(head_dim, 1, 1 << 24)) return 0;
  return afa::norm_rotate_bwd_workspace(dtype, (int)head_dim, afa::device_cus());
}

int ago_norm_rotate_axes_bwd(int dtype, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t seq_len, int64_t head_dim,
                             const void* q, const void* k, const void* gq, const void* gk, void* dq, void* dk,
                             const int64_t* strides, const void* q_scale, const void* k_scale, void* dq_scale, void* dk_scale,
                             double eps, const void* rot_cos, const void* rot_sin, int64_t rot_len, const void* positions,
                             int pos_bytes, int64_t pos_b, int axes, const int32_t* sections, void* workspace,
                             size_t workspace_bytes, void* stream) {
  afa::NormArgs a;
  const int rc = check_norm_rows(a, dtype, batch, q_heads, k_heads, seq_len, head_dim, q_scale, k_scale, eps, rot_cos, rot_sin,
                                 rot_len, positions, pos_bytes, pos_b, axes, sections);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || gq == nullptr || dq == nullptr || dq_scale == nullptr ||
      (k_heads > 0 && (k == nullptr || gk == nullptr || dk == nullptr || dk_scale == nullptr)))
    return AFA_ERR_NULL;
  const bool two = k_heads > 0;
  a.x[0] = q; a.x[1] = two ? k : q;
  a.g[0] = gq; a.g[1] = two ? gk : gq;
  a.y[0] = dq; a.y[1] = two ? dk : dq;
  row_strides(a, strides, a.sx);
  row_strides(a, strides != nullptr ? strides + 6 : nullptr, a.sg);
  row_strides(a, strides != nullptr ? strides + 12 : nullptr, a.sy);
  const int cus = afa::device_cus();
  const hipStream_t s = (hipStream_t)stream;
  void* ws;
  bool own;
  const int got = workspace_of(workspace, workspace_bytes, afa::norm_rotate_bwd_workspace(dtype, a.dim, cus), s, ws, own);
  if (got != AFA_OK) return got;
  void* const dscale[2] = {dq_scale, dk_scale};
  return workspace_done(afa::norm_rotate_bwd_launch(dtype, a, dscale, ws, cus, s), ws, own, s);
}

int ago_rotate_axes(int dtype, int64_t batch, int64_t q_heads, int64_t k_heads, int64_t seq_len, int64_t head_dim,
                    const void* q, const void* k, void* q_out, void* k_out, const int64_t* strides, const void* rot_cos,
                    const void* rot_sin, int64_t rot_len, const void* positions, int pos_bytes, int64_t pos_b, int axes,
                    const int32_t* sections, int transpose, void* stream) {
  if (!within(dtype, AFA_F32, AFA_F64)) return AFA_ERR_DTYPE;
  if (batch < 1 || q_heads < 1 || k_heads < 0 || seq_len < 1 || head_dim < 1) return AFA_ERR_SHAPE;
  if (q == nullptr || q_out == nullptr || rot_cos == nullptr || rot_sin == nullptr || positions == nullptr ||
      (k_heads > 0 && (k == nullptr || k_out == nullptr)))
    return AFA_ERR_NULL;
  if (pos_bytes != 4 && pos_bytes != 8) return AFA_ERR_UNSUPPORTED;
  const int64_t most = kLaunchThreads - 256;
  if (head_dim > most || batch > most / seq_len || batch * seq_len > most / (q_heads + k_heads) ||
      batch * seq_len * (q_heads + k_heads) > most / ((head_dim + 1) / 2) || q_heads + k_heads > (1 << 30))
    return AFA_ERR_SHAPE;
  afa::RotateAxesArgs a = {};
  const int rc = check_rotation(a.rot, rot_cos, rot_sin, rot_len, head_dim, axes, sections, positions, pos_bytes == 8);
  if (rc != AFA_OK) return rc;
  a.x[0] = q; a.x[1] = k;
  a.y[0] = q_out; a.y[1] = k_out;
  a.heads[0] = (int)q_heads; a.heads[1] = (int)k_heads;
  for (int i = 0; i < 4; ++i) {
    int64_t* to = i < 2 ? a.sx[i] : a.sy[i - 2];
    if (strides != nullptr) {
      for (int j = 0; j < 3; ++j) to[j] = strides[3 * i + j];
    } else {
      to[0] = a.heads[i & 1] * seq_len * head_dim;
      to[1] = seq_len * head_dim;
      to[2] = head_dim;
    }
  }
  a.batch = batch; a.seq = seq_len; a.dim = (int)head_dim;
  a.pos_b = pos_b;
  a.sign = transpose ? -1.0f : 1.0f;
  const hipError_t e = afa::rotate_axes_launch(dtype, a, (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

}  // extern "C"
