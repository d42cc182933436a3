// Cayley rotation by positions of several axes, and its VJP (the transposed rotation).
//
// Pair p of a row at (b, l) belongs to one axis a (time, height, width: the sections of the pairs, in
// order) and is turned by table row m = positions[b][l][a]: (x0, x1) -> (c x0 - s x1, s x0 + c x1), c and s
// the entries (m, p).  Pairs behind the last section stay as they are.  The tables enter in fp32 (fp64)
// and each result is rounded once.
//
// Every element is read and written once and HBM bounds the large calls: q and k of (8, 12, 2048, 64) bf16 21 us
// (4.8 TB/s), of (1, 16 and 4, 8189, 128) fp32 31 us (5.4 TB/s); the cache write of 16384 tokens of 16 heads of 64,
// fp16, 30 us (5.1 TB/s).  Calls of a few tokens take 4 us, three dependent reads (position, table entry, row).
#include <initializer_list>

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

// One thread a pair, q's rows before k's: fp64, rows that are no whole 16-byte chunks, and any alignment.
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

// The same in 16-byte chunks: a thread owns one chunk of a token's rows, holds its table entries and turns
// it in up to HG heads, `groups` apart, whose loads are in flight together.  Where the heads of a token lie
// nearer to one another than its neighbours do, lanes run over heads before tokens, so that a wave's
// accesses stay whole lines side by side either way.
template <int DT>
struct ChunkTurn {
  using R = RowChunk<DT>;
  static constexpr int NP = R::EPC / 2;
  float c[NP], s[NP];
  bool keep[NP];

  __device__ __forceinline__ void load(const AxisRotation& r, int64_t token, int p0, float sign) {
    const int first = pair_axis(r, p0), last = pair_axis(r, p0 + NP - 1);
    if (first == last && first >= 0 && r.wide) {
      const int64_t m = position(r, token + first), at = m * r.pairs + p0;
      const bool in = m >= 0 && m < r.len;
      typedef __attribute__((ext_vector_type(NP))) float vec;
      const vec nan = __builtin_nanf("");
      const vec cv = in ? *(const vec*)((const float*)r.rc + at) : nan, sv = in ? *(const vec*)((const float*)r.rs + at) : nan;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        c[p] = cv[p];
        s[p] = sv[p] * sign;
        keep[p] = false;
      }
      return;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int axis = pair_axis(r, p0 + p);
      const int64_t m = axis < 0 ? 0 : position(r, token + axis), at = m * r.pairs + p0 + p;
      const bool in = m >= 0 && m < r.len;
      keep[p] = axis < 0;
      c[p] = in ? ((const float*)r.rc)[at] : __builtin_nanf("");
      s[p] = in ? ((const float*)r.rs)[at] * sign : __builtin_nanf("");
    }
  }

  __device__ __forceinline__ u32x4_t turned(u32x4_t w) const {
#pragma clang fp contract(off)
    float v[R::EPC];
    R::unpack(w, v);
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const float x0 = v[2 * p], x1 = v[2 * p + 1];
      v[2 * p] = keep[p] ? x0 : c[p] * x0 - s[p] * x1;
      v[2 * p + 1] = keep[p] ? x1 : s[p] * x0 + c[p] * x1;
    }
    return R::pack(v);
  }
};

// Thread i of tokens * groups * chunks: its chunk of a row, its token and its first head.
struct ChunkPlace {
  uint32_t chunk, token, group;
};
struct ChunkGrid {
  uint32_t chunks, tokens, groups, total;
  int heads_inner;
};
__device__ __forceinline__ ChunkPlace chunk_place(const ChunkGrid& g, uint32_t i) {
  const uint32_t rest = i / g.chunks, inner = g.heads_inner ? g.groups : g.tokens;
  const uint32_t in = rest % inner, out = rest / inner;
  return ChunkPlace{i - rest * g.chunks, g.heads_inner ? out : in, g.heads_inner ? in : out};
}

template <int DT, int HG, bool STREAM>
__global__ __launch_bounds__(256) void ago_axes_chunk_kernel(const RotateAxesArgs a, const ChunkGrid g) {
  constexpr int EPC = RowChunk<DT>::EPC;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= g.total) return;
  const ChunkPlace at = chunk_place(g, i);
  const uint32_t b = at.token / (uint32_t)a.seq, l = at.token - b * (uint32_t)a.seq;
  const int all = a.heads[0] + a.heads[1];
  u32x4_t w[HG];
  int64_t to[HG];
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    const int h = (int)(at.group + u * g.groups);
    if (h >= all) break;
    const int which = h >= a.heads[0], hh = which ? h - a.heads[0] : h;
    w[u] = *(const u32x4_t*)((const typename Elem<DT>::storage*)a.x[which] + b * a.sx[which][0] + hh * a.sx[which][1] +
                             l * a.sx[which][2] + at.chunk * EPC);
    to[u] = b * a.sy[which][0] + hh * a.sy[which][1] + l * a.sy[which][2] + at.chunk * EPC;
  }
  ChunkTurn<DT> turn;
  turn.load(a.rot, b * a.pos_b + (int64_t)l * a.rot.axes, (int)(at.chunk * EPC / 2), a.sign);
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    const int h = (int)(at.group + u * g.groups);
    if (h >= all) break;
    u32x4_t* y = (u32x4_t*)((typename Elem<DT>::storage*)a.y[h >= a.heads[0]] + to[u]);
    if constexpr (STREAM) __builtin_nontemporal_store(turn.turned(w[u]), y);
    else *y = turn.turned(w[u]);
  }
}

template <int DT, int HG>
__global__ __launch_bounds__(256) void afa_paged_append_chunk_kernel(const AppendArgs a, const ChunkGrid g) {
  constexpr int EPC = RowChunk<DT>::EPC;
  using S = typename Elem<DT>::storage;
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= g.total) return;
  const ChunkPlace at = chunk_place(g, i);
  const int64_t t = at.token;
  const int d = (int)(at.chunk * EPC), H = a.heads, K = a.kv_heads, all = H + 2 * K;
  const int64_t slot = a.slots[t];
  u32x4_t w[HG];
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    const int h = (int)(at.group + u * g.groups);
    if (h >= all) break;
    const S* x = h < H ? (const S*)a.q + t * a.q_t + h * a.q_h
                 : h < H + K ? (const S*)a.k + t * a.k_t + (h - H) * a.k_h
                             : (const S*)a.v + t * a.v_t + (h - H - K) * a.v_h;
    w[u] = *(const u32x4_t*)(x + d);
  }
  ChunkTurn<DT> turn;
  if (a.rot.rc != nullptr) turn.load(a.rot, t * a.rot.axes, d / 2, 1.0f);
  const bool stored = slot >= 0 && slot < a.capacity;
  const uint32_t page = stored ? (uint32_t)slot / (uint32_t)a.page_size : 0, place = (uint32_t)slot - page * a.page_size;
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    const int h = (int)(at.group + u * g.groups);
    if (h >= all) break;
    if (h < H ? a.q_out == nullptr : !stored) continue;
    S* y = h < H ? (S*)a.q_out + (t * H + h) * a.dim
           : h < H + K ? (S*)a.k_pages + page * a.ps.k_page + (h - H) * a.ps.k_head + place * a.ps.k_slot
                       : (S*)a.v_pages + page * a.ps.v_page + (h - H - K) * a.ps.v_head + place * a.ps.v_slot;
    *(u32x4_t*)(y + d) = a.rot.rc != nullptr && h < H + K ? turn.turned(w[u]) : w[u];
  }
}

// Four heads a thread where that leaves threads enough to fill the device (about 2^17), else one.  2, 4 and 8
// heads take 22.9, 21.2 and 23.0 us for the bf16 call above and 33, 31 and 34 for the fp32 one.
constexpr int HEADS = 4;
inline ChunkGrid chunk_grid(int64_t tokens, int64_t heads, int64_t chunks, bool heads_inner, bool& four) {
  four = tokens * chunks * heads >= (int64_t(1) << 19);
  ChunkGrid g;
  g.chunks = (uint32_t)chunks;
  g.tokens = (uint32_t)tokens;
  g.groups = (uint32_t)(four ? (heads + HEADS - 1) / HEADS : heads);
  g.total = g.chunks * g.tokens * g.groups;
  g.heads_inner = heads_inner;
  return g;
}

// The cache write, as ago_axes_kernel: one thread a pair (or the last element of an odd head_dim) of a token's q, k and v
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
  if constexpr (DT != AFA_F64) {
    constexpr int EPC = RowChunk<DT>::EPC;
    bool whole = a.dim % EPC == 0;
    for (int i = 0; i < 2 && whole; ++i) {
      if (a.heads[i] == 0) continue;
      whole = (((uintptr_t)a.x[i] | (uintptr_t)a.y[i]) & 15u) == 0;
      for (int j = 0; j < 3; ++j) whole = whole && a.sx[i][j] % EPC == 0 && a.sy[i][j] % EPC == 0;
    }
    if (whole) {
      bool four;
      const ChunkGrid g = chunk_grid(a.batch * a.seq, a.heads[0] + a.heads[1], a.dim / EPC, a.sx[0][1] < a.sx[0][2], four);
      const dim3 grid((g.total + 255) / 256);
      // Results larger than all L2 caches are written past them: (1, 20, 8189, 128) fp32 31 us (5.4 TB/s), 50
      // without; (8, 24, 2048, 64) bf16 21 us, 23 without.  Smaller ones are left for the reader that comes next.
      const bool stream = a.batch * a.seq * (a.heads[0] + a.heads[1]) * a.dim / EPC * 16 > (int64_t(1) << 25);
      if (four && stream) hipLaunchKernelGGL((ago_axes_chunk_kernel<DT, HEADS, true>), grid, dim3(256), 0, st, a, g);
      else if (four) hipLaunchKernelGGL((ago_axes_chunk_kernel<DT, HEADS, false>), grid, dim3(256), 0, st, a, g);
      else hipLaunchKernelGGL((ago_axes_chunk_kernel<DT, 1, false>), grid, dim3(256), 0, st, a, g);
      return hipGetLastError();
    }
  }
  const int64_t n = a.batch * a.seq * (a.heads[0] + a.heads[1]) * (a.dim / 2);
  hipLaunchKernelGGL((ago_axes_kernel<DT>), dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a, n);
  return hipGetLastError();
}

template <int DT>
hipError_t append_go(const AppendArgs& a, hipStream_t st) {
  if constexpr (DT != AFA_F64) {
    constexpr int EPC = RowChunk<DT>::EPC;
    const uintptr_t bases = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q_out | (uintptr_t)a.k_pages |
                            (uintptr_t)a.v_pages;
    bool whole = a.dim % EPC == 0 && (bases & 15u) == 0;
    for (int64_t v : {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.ps.k_page, a.ps.k_head, a.ps.k_slot, a.ps.v_page,
                      a.ps.v_head, a.ps.v_slot})
      whole = whole && v % EPC == 0;
    if (whole) {
      bool four;
      const ChunkGrid g = chunk_grid(a.tokens, a.heads + 2 * a.kv_heads, a.dim / EPC, true, four);
      const dim3 grid((g.total + 255) / 256);
      if (four) hipLaunchKernelGGL((afa_paged_append_chunk_kernel<DT, HEADS>), grid, dim3(256), 0, st, a, g);
      else hipLaunchKernelGGL((afa_paged_append_chunk_kernel<DT, 1>), grid, dim3(256), 0, st, a, g);
      return hipGetLastError();
    }
  }
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
