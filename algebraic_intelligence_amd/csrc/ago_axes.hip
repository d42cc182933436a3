// Cayley rotation by positions of several axes, and its VJP (the transposed rotation).
//
// Pair p of a row at (b, l) belongs to one axis a (time, height, width: the sections of the pairs, in
// order) and is turned by table row m = positions[b][l][a]: (x0, x1) -> (c x0 - s x1, s x0 + c x1), c and s
// the entries (m, p).  Pairs behind the last section stay as they are.  The tables enter in fp32 (fp64)
// and each result is rounded once.
#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

__device__ __forceinline__ int64_t position(const AxisRotation& r, int64_t i) {
  return r.pos64 ? ((const int64_t*)r.positions)[i] : ((const int32_t*)r.positions)[i];
}

// One pair by the table entries of position m of its axis; NaN where the tables have no such row.
template <typename T>
__device__ __forceinline__ void turn(const AxisRotation& r, int64_t m, int p, T sign, T x0, T x1, T& y0, T& y1) {
#pragma clang fp contract(off)
  T c, s;
  if (m >= 0 && m < r.len) {
    c = ((const T*)r.rc)[m * r.pairs + p];
    s = ((const T*)r.rs)[m * r.pairs + p] * sign;
  } else {
    c = s = (T)__builtin_nanf("");
  }
  y0 = c * x0 - s * x1;
  y1 = s * x0 + c * x1;
}

// One thread a pair, q's rows before k's.
template <int DT>
__global__ __launch_bounds__(256) void ago_axes_kernel(const RotateAxesArgs a, int64_t total) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  const int pairs = a.dim / 2, p = (int)(e % pairs);
  const int64_t row = e / pairs, token = row / (a.heads[0] + a.heads[1]);
  int h = (int)(row % (a.heads[0] + a.heads[1]));
  const int which = h >= a.heads[0];
  if (which) h -= a.heads[0];
  const int64_t b = token / a.seq, l = token % a.seq;
  const int64_t from = b * a.sx[which][0] + h * a.sx[which][1] + l * a.sx[which][2] + 2 * p;
  const int64_t to = b * a.sy[which][0] + h * a.sy[which][1] + l * a.sy[which][2] + 2 * p;
  const int axis = pair_axis(a.rot, p);
  const int64_t m = axis < 0 ? 0 : position(a.rot, b * a.pos_b + l * a.rot.axes + axis);
  if constexpr (DT == AFA_F64) {
    double y0 = ((const double*)a.x[which])[from], y1 = ((const double*)a.x[which])[from + 1];
    if (axis >= 0) turn<double>(a.rot, m, p, (double)a.sign, y0, y1, y0, y1);
    ((double*)a.y[which])[to] = y0;
    ((double*)a.y[which])[to + 1] = y1;
  } else {
    float y0 = Elem<DT>::load(a.x[which], from), y1 = Elem<DT>::load(a.x[which], from + 1);
    if (axis >= 0) turn<float>(a.rot, m, p, a.sign, y0, y1, y0, y1);
    Elem<DT>::store(a.y[which], to, y0);
    Elem<DT>::store(a.y[which], to + 1, y1);
  }
}

// The cache write: one thread a pair (or the last element of an odd head_dim) of a token's q, k and v
// heads, in this order.
template <int DT>
__global__ __launch_bounds__(256) void afa_paged_append_kernel(const AppendArgs a, int64_t total) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= total) return;
  const int pairs = (a.dim + 1) / 2, p = (int)(e % pairs);
  const int64_t row = e / pairs;
  const int all = a.heads + 2 * a.kv_heads, t = (int)(row / all);
  int h = (int)(row % all);
  const bool two = 2 * p + 1 < a.dim;
  const void* x;
  void* y;
  int64_t from, to;
  bool turned = a.rot.rc != nullptr;
  if (h < a.heads) {
    if (a.q_out == nullptr) return;
    x = a.q;
    y = a.q_out;
    from = t * a.q_t + h * a.q_h;
    to = ((int64_t)t * a.heads + h) * a.dim;
  } else {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.capacity) return;
    const int64_t page = slot / a.page_size, at = slot % a.page_size;
    h -= a.heads;
    if (h < a.kv_heads) {
      x = a.k;
      y = a.k_pages;
      from = t * a.k_t + h * a.k_h;
      to = page * a.ps.k_page + h * a.ps.k_head + at * a.ps.k_slot;
    } else {
      h -= a.kv_heads;
      x = a.v;
      y = a.v_pages;
      from = t * a.v_t + h * a.v_h;
      to = page * a.ps.v_page + h * a.ps.v_head + at * a.ps.v_slot;
      turned = false;
    }
  }
  from += 2 * p;
  to += 2 * p;
  const int axis = turned ? pair_axis(a.rot, p) : -1;
  const int64_t m = axis < 0 ? 0 : position(a.rot, (int64_t)t * a.rot.axes + axis);
  if constexpr (DT == AFA_F64) {
    double y0 = ((const double*)x)[from], y1 = two ? ((const double*)x)[from + 1] : 0.0;
    if (axis >= 0) turn<double>(a.rot, m, p, 1.0, y0, y1, y0, y1);
    ((double*)y)[to] = y0;
    if (two) ((double*)y)[to + 1] = y1;
  } else {
    float y0 = Elem<DT>::load(x, from), y1 = two ? Elem<DT>::load(x, from + 1) : 0.0f;
    if (axis >= 0) turn<float>(a.rot, m, p, 1.0f, y0, y1, y0, y1);
    Elem<DT>::store(y, to, y0);
    if (two) Elem<DT>::store(y, to + 1, y1);
  }
}

template <int DT>
hipError_t rotate_axes_go(const RotateAxesArgs& a, hipStream_t st) {
  const int64_t n = a.batch * a.seq * (a.heads[0] + a.heads[1]) * (a.dim / 2);
  hipLaunchKernelGGL((ago_axes_kernel<DT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, n);
  return hipGetLastError();
}

template <int DT>
hipError_t append_go(const AppendArgs& a, hipStream_t st) {
  const int64_t n = (int64_t)a.tokens * (a.heads + 2 * a.kv_heads) * ((a.dim + 1) / 2);
  hipLaunchKernelGGL((afa_paged_append_kernel<DT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, n);
  return hipGetLastError();
}

}  // namespace

hipError_t rotate_axes_launch(int dtype, const RotateAxesArgs& a, hipStream_t st) {
  switch (dtype) {
    case AFA_F32: return rotate_axes_go<AFA_F32>(a, st);
    case AFA_BF16: return rotate_axes_go<AFA_BF16>(a, st);
    case AFA_F16: return rotate_axes_go<AFA_F16>(a, st);
    default: return rotate_axes_go<AFA_F64>(a, st);
  }
}

hipError_t paged_append_launch(int dtype, const AppendArgs& a, hipStream_t st) {
  switch (dtype) {
    case AFA_F32: return append_go<AFA_F32>(a, st);
    case AFA_BF16: return append_go<AFA_BF16>(a, st);
    case AFA_F16: return append_go<AFA_F16>(a, st);
    default: return append_go<AFA_F64>(a, st);
  }
}

}  // namespace afa
