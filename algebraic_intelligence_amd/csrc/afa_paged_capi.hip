// C ABI of the paged-cache serving operators (include/afa.h): argument checks and dispatch.
#include <cmath>
#include <cstdint>
#include <initializer_list>

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
  int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || k == nullptr || v == nullptr || k_pages == nullptr || v_pages == nullptr) return AFA_ERR_NULL;
  if (q_out == nullptr && rot_cos != nullptr) return AFA_ERR_NULL;
  if (positions == nullptr && axes != 1) return AFA_ERR_NULL;
  const afa_paged_plan& p = *plan;
  afa::AppendArgs a = {};
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
  a.ps = page_strides_of(p, page_strides);
  a.slots = p.slots;
  a.tokens = (int)p.max_tokens; a.heads = (int)p.heads; a.kv_heads = (int)p.kv_heads; a.dim = (int)p.head_dim;
  a.page_size = (int)p.page_size;
  a.capacity = p.num_pages * p.page_size;
  if (p.max_tokens > (kLaunchThreads - 256) / ((p.heads + 2 * p.kv_heads) * ((p.head_dim + 1) / 2))) return AFA_ERR_SHAPE;
  const hipError_t e = afa::paged_append_launch((int)p.dtype, a, (hipStream_t)stream);
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
}

size_t afa_paged_workspace_size(const afa_paged_plan* plan) {
  if (plan == nullptr || check_sizes(*plan) != AFA_OK || !afa::paged_fast_supported(*plan)) return 0;
  return afa::paged_fast_workspace(*plan, afa::paged_cut(*plan, afa::device_cus()));
}

int afa_paged_fwd(const afa_paged_plan* plan, const void* q, const int64_t* q_strides, const void* k_pages,
                  const void* v_pages, const int64_t* page_strides, const int64_t* masks, void* out, void* denom,
                  double sink_omega, unsigned flags, void* workspace, size_t workspace_bytes, void* stream) {
  const int rc = check_plan(plan);
  if (rc != AFA_OK) return rc;
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || out == nullptr) return AFA_ERR_NULL;
  if (!(sink_omega >= 0.0 && sink_omega < INFINITY)) return AFA_ERR_SINK;
  const afa_paged_plan& p = *plan;
  if (masks != nullptr && p.max_tree == 0) return AFA_ERR_UNSUPPORTED;
  if (p.max_tokens > (kLaunchThreads - 1) / 256 / p.heads) return AFA_ERR_SHAPE;
  afa::PagedFwdArgs a = {};
  a.plan = p;
  const int cus = afa::device_cus();
  const afa::PagedCut cut = afa::paged_cut(p, cus);
  a.sched = afa::paged_schedule(p, cut.slots);
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
  hipStream_t s = (hipStream_t)stream;
  // 16-byte rows of q and of the pages; byte offsets within a page, and its stride, in 32 bits
  const int64_t unit = p.dtype == AFA_F32 ? 4 : 8;
  bool fast = (flags & AFA_FLAG_GENERIC) == 0 && afa::paged_fast_supported(p) && aligned16(q) && aligned16(k_pages) &&
              aligned16(v_pages) && aligned16(out) && a.q_t % unit == 0 && a.q_h % unit == 0;
  for (int64_t v : {a.ps.k_page, a.ps.k_head, a.ps.k_slot, a.ps.v_page, a.ps.v_head, a.ps.v_slot})
    fast = fast && v % unit == 0 && v >= 0;
  const int64_t reach = (int64_t(1) << 30) / p.page_size;  // elements, of 4 bytes at most
  for (int64_t v : {a.ps.k_slot, a.ps.v_slot}) fast = fast && v < reach - p.head_dim;
  for (int64_t v : {a.ps.k_page, a.ps.v_page}) fast = fast && v < int64_t(1) << 30;
  if (!fast) {
    const hipError_t e = afa::paged_fwd_generic_launch(a, s);
    return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
  }
  const size_t need = afa::paged_fast_workspace(p, cut);
  void* ws = workspace;
  if (ws == nullptr) {
    ws = afa::workspace_alloc(need, s);
    if (ws == nullptr) return afa::hip_status_code(hipErrorOutOfMemory);
  } else if (workspace_bytes < need) {
    return AFA_ERR_WORKSPACE;
  } else if (!aligned16(ws)) {
    return AFA_ERR_ALIGN;
  }
  hipError_t e = afa::paged_fwd_fast_launch(a, cut, ws, s);
  if (workspace == nullptr) {
    const hipError_t e2 = hipFreeAsync(ws, s);
    if (e == hipSuccess) e = e2;
  }
  return e == hipSuccess ? AFA_OK : afa::hip_status_code(e);
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
