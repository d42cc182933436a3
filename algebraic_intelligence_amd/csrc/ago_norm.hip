// Rows of q and k normalised head by head, scaled and rotated in one pass, and the gradients.
//
//   y = R(m) (w . xh),   xh = x r,   r = 1 / sqrt(mean(x^2) + eps)
//
// with R(m) the Cayley rotation by positions of several axes (ago_axes.hip) and w a scale per feature, one for q and
// one for k.  With the cotangent g and back = R(m)^T g:
//
//   dx = r (h - xh mean(h . xh)),  h = w . back;     dw = sum over all rows of back . xh
//
// Everything between the loads and the stores is fp32 (fp64), rounded once.  r is formed again from x in the
// backward, which reads x in any case.
//
// Every element is read and written once and HBM bounds the large calls.  A row is 2^k lanes side by side (LPR), one
// 16-byte chunk each, so that its mean takes k lane exchanges and no LDS.  dw is summed in registers over the
// rows that a lane meets, then over its workgroup, and a second launch adds the workgroups' sums in a fixed
// order: results repeat bit for bit, which atomics would not give.
//
// 8 sequences of 4096 tokens, 12 and 12 heads of 64 in bf16: 39 us and 60, 5.2 and 5.0 TB/s, as a large copy.  A prompt's way into
// the cache, 8 x 2048 tokens of 16 + 4 + 4 heads of 128 in fp16: 39 us, 5.1 TB/s.  Small calls are a launch: 4.2 us.
#include <initializer_list>
#include <type_traits>

#include "afa_common.h"
#include "afa_launch.h"
#include "afa_paged.h"
#include "ago_turn.h"

namespace afa {

namespace {

// 1 / sqrt(x) in fp32, the hardware's approximation refined by one Newton step.  Numbers below the normal ones, which it takes for 0, go
// through it times 2^80.
__device__ __forceinline__ float inverse_root(float x) {
  const bool small = x < 0x1p-100f;
  const float z = small ? x * 0x1p80f : x;
  const float r = __builtin_amdgcn_rsqf(z);
  const float y = r * __builtin_fmaf(-0.5f * z * r, r, 1.5f);
  return (r > 0.0f && r < __builtin_inff() ? y : r) * (small ? 0x1p40f : 1.0f);  // x = 0 and infinity
}
__device__ __forceinline__ double inverse_root(double x) { return 1.0 / sqrt(x); }

// Where the rows of a call lie: `which` is 0 for q, 1 for k and 2 for v.  A row without a place (dst nullptr) is not
// stored.  `at`: the token's first position.
struct RotateRows {
  NormArgs a;
  static constexpr int KINDS = 2;
  struct Token {
    int64_t b, l, at;
  };
  __device__ __forceinline__ int heads(int which) const { return a.heads[which]; }
  __device__ __forceinline__ Token token(uint32_t t) const {
    const uint32_t b = t / (uint32_t)a.seq, l = t - b * (uint32_t)a.seq;
    return Token{b, l, b * a.pos_b + (int64_t)l * a.rot.axes};
  }
  template <typename S>
  __device__ __forceinline__ const S* src(const Token& t, int which, int h) const {
    return (const S*)a.x[which] + (t.b * a.sx[which][0] + h * a.sx[which][1] + t.l * a.sx[which][2]);
  }
  template <typename S>
  __device__ __forceinline__ S* dst(const Token& t, int which, int h) const {
    return (S*)a.y[which] + (t.b * a.sy[which][0] + h * a.sy[which][1] + t.l * a.sy[which][2]);
  }
  __device__ __forceinline__ const AxisRotation& rotation() const { return a.rot; }
  __device__ __forceinline__ const HeadNorm& norm() const { return a.norm; }
  __device__ __forceinline__ int dim() const { return a.dim; }
};

struct AppendRows {
  // q, k and v.  k and v lie in pages; q's page is its token, and its place there 0
  const void* x[3];
  void* y[3];
  int64_t xt[3], xh[3], page[3], head[3], slot[3];
  int count[3];
  const int32_t* slots;
  int64_t capacity;
  int page_size, features;
  HeadNorm n;
  AxisRotation rot;
  static constexpr int KINDS = 3;
  struct Token {
    int64_t t, at, page, place;
    bool stored;
  };
  __device__ __forceinline__ int heads(int which) const { return count[which]; }
  __device__ __forceinline__ Token token(uint32_t t) const {
    const int64_t slot = slots[t];
    const bool stored = slot >= 0 && slot < capacity;
    const uint32_t page = stored ? (uint32_t)slot / (uint32_t)page_size : 0;
    return Token{t, (int64_t)t * rot.axes, page, stored ? slot - (int64_t)page * page_size : 0, stored};
  }
  template <typename S>
  __device__ __forceinline__ const S* src(const Token& t, int which, int h) const {
    return (const S*)x[which] + (t.t * xt[which] + h * xh[which]);
  }
  template <typename S>
  __device__ __forceinline__ S* dst(const Token& t, int which, int h) const {
    const bool in_pages = which > 0;
    if (in_pages && !t.stored) return nullptr;
    return (S*)y[which] + ((in_pages ? t.page : t.t) * page[which] + h * head[which] + (in_pages ? t.place : 0) * slot[which]);
  }
  __device__ __forceinline__ const AxisRotation& rotation() const { return rot; }
  __device__ __forceinline__ const HeadNorm& norm() const { return n; }
  __device__ __forceinline__ int dim() const { return features; }
};

// ------------------------------------------------------------------ rows in 16-byte chunks
// Groups of LPR lanes, each for up to HG heads of one token, `groups[which]` apart.  A workgroup has rows of one kind, that
// of the last of `begin` that it does not precede: what differs by kind stays in scalar registers.
struct NormGrid {
  uint32_t chunks, tokens, groups[3], begin[4];
  int heads_inner;
};

template <int DT>
struct ChunkScale {
  static constexpr int EPC = RowChunk<DT>::EPC;
  float v[EPC];
  __device__ __forceinline__ void load(const void* scale, int d) {
#pragma unroll
    for (int i = 0; i < EPC; ++i) v[i] = ((const float*)scale)[d + i];
  }
};

template <int DT, int LPR, int HG, bool STREAM, typename Rows>
__global__ __launch_bounds__(256) void ago_norm_chunk_kernel(const Rows rows, const NormGrid g) {
  using R = RowChunk<DT>;
  using S = typename Elem<DT>::storage;
  constexpr int EPC = R::EPC;
  int which = 0;
#pragma unroll
  for (int k = 1; k < Rows::KINDS; ++k) which += blockIdx.x >= g.begin[k];
  const uint32_t i = (blockIdx.x - g.begin[which]) * 256 + threadIdx.x, c = i % LPR, set = i / LPR, step = g.groups[which];
  if (set >= g.tokens * step) return;  // whole rows of lanes
  const uint32_t inner = g.heads_inner ? step : g.tokens, out = set / inner, in = set - out * inner;
  const uint32_t t = g.heads_inner ? out : in, first = g.heads_inner ? in : out;
  const typename Rows::Token token = rows.token(t);
  const int heads = rows.heads(which), d = (int)c * EPC;
  const bool mine = c < g.chunks;
  u32x4_t w[HG];
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    w[u] = u32x4_t{0, 0, 0, 0};
    const int h = (int)(first + u * step);
    if (mine && h < heads) w[u] = *(const u32x4_t*)(rows.template src<S>(token, which, h) + d);
  }
  ChunkTurn<DT> turn;
  ChunkScale<DT> scale;
  const bool turned = rows.rotation().rc != nullptr;
  if (which < 2 && mine) {
    scale.load(rows.norm().scale[which], d);
    if (turned) turn.load(rows.rotation(), token.at, d / 2, 1.0f);
  }
#pragma unroll
  for (int u = 0; u < HG; ++u) {
    const int h = (int)(first + u * step);
    if (h >= heads) break;
    if (which < 2) {
      float v[EPC], sum = 0.0f;
      R::unpack(w[u], v);
#pragma unroll
      for (int e = 0; e < EPC; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
      sum = group_sum<LPR>(sum);
      const float r = inverse_root(sum / (float)rows.dim() + (float)rows.norm().eps);
#pragma unroll
      for (int e = 0; e < EPC; ++e) v[e] = v[e] * r * scale.v[e];
      if (turned) turn.turn_values(v);
      w[u] = R::pack(v);
    }
    S* to = rows.template dst<S>(token, which, h);
    if (!mine || to == nullptr) continue;
    if constexpr (STREAM) __builtin_nontemporal_store(w[u], (u32x4_t*)(to + d));
    else *(u32x4_t*)(to + d) = w[u];
  }
}

// The gradients.  Workgroups below `parts[0]` have q's rows, the others k's; a group of lanes goes through every
// parts * (BWD / LPR)-th set of heads, and its sums of back . xh stay in registers.
struct NormParts {
  uint32_t parts[2];
  void* sums;  // (parts[0] + parts[1], dim)
};

constexpr int BWD = 512;
template <int DT, int LPR, int HG, bool STREAM>
__global__ __launch_bounds__(BWD) void ago_norm_bwd_chunk_kernel(const NormArgs a, const NormGrid g, const NormParts p) {
  using R = RowChunk<DT>;
  using S = typename Elem<DT>::storage;
  constexpr int EPC = R::EPC, SLOTS = BWD / LPR;
  __shared__ float sums[SLOTS][LPR * EPC];
  const int which = blockIdx.x >= p.parts[0];
  const uint32_t part = which ? blockIdx.x - p.parts[0] : blockIdx.x;
  const uint32_t c = threadIdx.x % LPR, slot = threadIdx.x / LPR, step = g.groups[which], sets = g.tokens * step;
  const int heads = a.heads[which], d = (int)c * EPC;
  const bool mine = c < g.chunks, turned = a.rot.rc != nullptr;
  const float over = 1.0f / (float)a.dim;
  ChunkScale<DT> scale;
  float acc[EPC];
#pragma unroll
  for (int e = 0; e < EPC; ++e) acc[e] = scale.v[e] = 0.0f;
  if (mine) scale.load(a.norm.scale[which], d);
  for (uint32_t i = part * SLOTS + slot; i < sets; i += p.parts[which] * SLOTS) {
    const uint32_t inner = g.heads_inner ? step : g.tokens, out = i / inner, in = i - out * inner;
    const uint32_t t = g.heads_inner ? out : in, first = g.heads_inner ? in : out;
    const uint32_t b = t / (uint32_t)a.seq, l = t - b * (uint32_t)a.seq;
    u32x4_t w[HG], q[HG];
#pragma unroll
    for (int u = 0; u < HG; ++u) {
      w[u] = q[u] = u32x4_t{0, 0, 0, 0};
      const int h = (int)(first + u * step);
      if (mine && h < heads) {
        w[u] = *(const u32x4_t*)((const S*)a.x[which] + (b * a.sx[which][0] + h * a.sx[which][1] + l * a.sx[which][2] + d));
        q[u] = *(const u32x4_t*)((const S*)a.g[which] + (b * a.sg[which][0] + h * a.sg[which][1] + l * a.sg[which][2] + d));
      }
    }
    ChunkTurn<DT> turn;
    if (mine && turned) turn.load(a.rot, b * a.pos_b + (int64_t)l * a.rot.axes, d / 2, -1.0f);
#pragma unroll
    for (int u = 0; u < HG; ++u) {
      const int h = (int)(first + u * step);
      if (h >= heads) break;
      float x[EPC], y[EPC], sum = 0.0f, dot = 0.0f;
      R::unpack(w[u], x);
      R::unpack(q[u], y);
      if (mine && turned) turn.turn_values(y);
#pragma unroll
      for (int e = 0; e < EPC; ++e) {
        sum = __builtin_fmaf(x[e], x[e], sum);
        dot = __builtin_fmaf(y[e] * scale.v[e], x[e], dot);
      }
      sum = group_sum<LPR>(sum);
      dot = group_sum<LPR>(dot);
      const float r = inverse_root(sum / (float)a.dim + (float)a.norm.eps);
      const float mean = r == 0.0f ? 0.0f : dot * r * over;  // of h . xh: 0 past the range, where dot may be infinite
#pragma unroll
      for (int e = 0; e < EPC; ++e) {
        const float xh = x[e] * r;
        acc[e] = __builtin_fmaf(y[e], xh, acc[e]);
        x[e] = r * __builtin_fmaf(-xh, mean, y[e] * scale.v[e]);
      }
      if (!mine) continue;
      S* to = (S*)a.y[which] + (b * a.sy[which][0] + h * a.sy[which][1] + l * a.sy[which][2] + d);
      if constexpr (STREAM) __builtin_nontemporal_store(R::pack(x), (u32x4_t*)to);
      else *(u32x4_t*)to = R::pack(x);
    }
  }
#pragma unroll
  for (int e = 0; e < EPC; ++e) sums[slot][d + e] = acc[e];
  __syncthreads();
  for (int e = threadIdx.x; e < a.dim; e += BWD) {
    float x = 0.0f;
#pragma unroll
    for (int s = 0; s < SLOTS; ++s) x += sums[s][e];
    ((float*)p.sums)[(int64_t)blockIdx.x * a.dim + e] = x;
  }
}

// The workgroups' sums, in their order.
constexpr int JOIN = 1024;
template <typename A>
__global__ __launch_bounds__(JOIN) void ago_norm_join_kernel(const NormParts p, int dim, A* q_scale, A* k_scale) {
  __shared__ A sums[JOIN / 64][64];
  const int which = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = blockIdx.x * 64 + lane;
  const A* from = (const A*)p.sums + (int64_t)(which ? p.parts[0] : 0) * dim;
  const uint32_t n = p.parts[which];
  constexpr int W = JOIN / 64, U = 8;
  A x = 0;
  if (d < dim) {
    for (uint32_t i0 = wave; i0 < n; i0 += W * U) {
      A y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) y[u] = i0 + u * W < n ? from[(int64_t)(i0 + u * W) * dim + d] : (A)0;
#pragma unroll
      for (int u = 0; u < U; ++u) x += y[u];
    }
  }
  sums[wave][lane] = x;
  __syncthreads();
  A* to = which ? k_scale : q_scale;
  if (wave != 0 || d >= dim || to == nullptr) return;
  A all = 0;
  for (int w = 0; w < W; ++w) all += sums[w][lane];
  to[d] = all;
}

// ------------------------------------------------------------------ any rows
// A wave a row, for fp64, odd and long head dims, and any alignment.
template <int DT>
using Wide = typename std::conditional<DT == AFA_F64, double, float>::type;

template <int DT>
__device__ __forceinline__ Wide<DT> take(const void* p, int64_t i) {
  if constexpr (DT == AFA_F64) return ((const double*)p)[i];
  else return Elem<DT>::load(p, i);
}
template <int DT>
__device__ __forceinline__ void give(void* p, int64_t i, Wide<DT> x) {
  if constexpr (DT == AFA_F64) ((double*)p)[i] = x;
  else Elem<DT>::store(p, i, x);
}
template <typename A>
__device__ __forceinline__ A wave_sum(A x) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) x += __shfl_xor(x, o);
  return x;
}
// Pair p of a row turned, or as it is.
template <typename A>
__device__ __forceinline__ void turn_pair(const AxisRotation& r, int64_t at, int p, A sign, A& y0, A& y1) {
  const int axis = r.rc != nullptr ? pair_axis(r, p) : -1;
  if (axis >= 0) turn<A>(r, position(r, at + axis), p, sign, y0, y1, y0, y1);
}
template <int DT>
struct ElemSize {
  typedef unsigned short type;
};
template <>
struct ElemSize<AFA_F32> {
  typedef float type;
};
template <>
struct ElemSize<AFA_F64> {
  typedef double type;
};

template <int DT, typename Rows>
__global__ __launch_bounds__(256) void ago_norm_row_kernel(const Rows rows, uint32_t tokens, int64_t total) {
  using A = Wide<DT>;
  using S = typename ElemSize<DT>::type;
  const int lane = threadIdx.x & 63, D = rows.dim();
  int all = 0;
  for (int w = 0; w < Rows::KINDS; ++w) all += rows.heads(w);
  for (int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); row < total; row += (int64_t)gridDim.x * 4) {
    const typename Rows::Token t = rows.token((uint32_t)(row / all));
    int h = (int)(row % all), which = 0;
    while (h >= rows.heads(which)) h -= rows.heads(which++);
    const S* x = rows.template src<S>(t, which, h);
    S* y = rows.template dst<S>(t, which, h);
    if (y == nullptr) continue;
    A r = 0;
    if (which < 2) {
      A sum = 0;
      for (int d = lane; d < D; d += 64) {
        const A v = take<DT>(x, d);
        sum += v * v;
      }
      r = inverse_root(wave_sum(sum) / (A)D + (A)rows.norm().eps);
    }
    for (int p = lane; 2 * p < D; p += 64) {
      const bool two = 2 * p + 1 < D;
      A y0 = take<DT>(x, 2 * p), y1 = two ? take<DT>(x, 2 * p + 1) : (A)0;
      if (which < 2) {
        const A* w = (const A*)rows.norm().scale[which];
        y0 = y0 * r * w[2 * p];
        if (two) y1 = y1 * r * w[2 * p + 1];
        turn_pair<A>(rows.rotation(), t.at, p, (A)1, y0, y1);
      }
      give<DT>(y, 2 * p, y0);
      if (two) give<DT>(y, 2 * p + 1, y1);
    }
  }
}

// A part is a wave here, which adds to its own sums in memory.
template <int DT>
__global__ __launch_bounds__(64) void ago_norm_bwd_row_kernel(const NormArgs a, const NormParts p) {
  using A = Wide<DT>;
  using S = typename ElemSize<DT>::type;
  const int which = blockIdx.x >= p.parts[0], lane = threadIdx.x, D = a.dim;
  const uint32_t part = which ? blockIdx.x - p.parts[0] : blockIdx.x;
  const int64_t total = a.batch * a.seq * a.heads[which];
  A* sums = (A*)p.sums + (int64_t)blockIdx.x * D;
  const A* w = (const A*)a.norm.scale[which];
  // a lane's features are those of its pairs all along
  for (int q = lane; 2 * q < D; q += 64) {
    sums[2 * q] = 0;
    if (2 * q + 1 < D) sums[2 * q + 1] = 0;
  }
  for (int64_t row = part; row < total; row += p.parts[which]) {
    const int64_t t = row / a.heads[which], b = t / a.seq, l = t - b * a.seq, at = b * a.pos_b + l * a.rot.axes;
    const int h = (int)(row % a.heads[which]);
    const S* x = (const S*)a.x[which] + (b * a.sx[which][0] + h * a.sx[which][1] + l * a.sx[which][2]);
    const S* g = (const S*)a.g[which] + (b * a.sg[which][0] + h * a.sg[which][1] + l * a.sg[which][2]);
    S* y = (S*)a.y[which] + (b * a.sy[which][0] + h * a.sy[which][1] + l * a.sy[which][2]);
    A sum = 0, dot = 0;
    for (int q = lane; 2 * q < D; q += 64) {
      const bool two = 2 * q + 1 < D;
      const A x0 = take<DT>(x, 2 * q), x1 = two ? take<DT>(x, 2 * q + 1) : (A)0;
      A g0 = take<DT>(g, 2 * q), g1 = two ? take<DT>(g, 2 * q + 1) : (A)0;
      turn_pair<A>(a.rot, at, q, (A)-1, g0, g1);
      sum += x0 * x0 + x1 * x1;
      dot += g0 * w[2 * q] * x0;
      if (two) dot += g1 * w[2 * q + 1] * x1;
    }
    const A r = inverse_root(wave_sum(sum) / (A)D + (A)a.norm.eps), all = wave_sum(dot);
    const A mean = r == 0 ? (A)0 : all * r / (A)D;
    for (int q = lane; 2 * q < D; q += 64) {
      const bool two = 2 * q + 1 < D;
      A x0 = take<DT>(x, 2 * q), x1 = two ? take<DT>(x, 2 * q + 1) : (A)0;
      A g0 = take<DT>(g, 2 * q), g1 = two ? take<DT>(g, 2 * q + 1) : (A)0;
      turn_pair<A>(a.rot, at, q, (A)-1, g0, g1);
      x0 *= r;
      x1 *= r;
      sums[2 * q] += g0 * x0;
      give<DT>(y, 2 * q, r * (g0 * w[2 * q] - x0 * mean));
      if (!two) continue;
      sums[2 * q + 1] += g1 * x1;
      give<DT>(y, 2 * q + 1, r * (g1 * w[2 * q + 1] - x1 * mean));
    }
  }
}

// ------------------------------------------------------------------ launches
constexpr int HEADS = 4;
constexpr uint32_t kMostRows = 1u << 20;  // workgroups of the row kernels

// Lanes of a row: the power of two that holds its chunks, 64 at most.
inline int lanes_of(int chunks) {
  int n = 4;
  while (n < chunks) n *= 2;
  return n;
}

// Groups of up to `per` heads, or of one where fewer than about 2^17 threads would be left: 512 tokens of 24 heads of 64 in bf16 take
// 4.3 us by ones and 6.0 by fours, 2730 as long either way, 10920 18.2 and 16.5, 32768 50 and 39 (by twos 44).
inline NormGrid norm_grid(int64_t tokens, std::initializer_list<int> heads, int chunks, bool heads_inner, int per, bool& many) {
  int64_t all = 0;
  for (int h : heads) all += h;
  many = tokens * chunks * all >= (int64_t(1) << 17) * per;
  NormGrid g = {};
  g.chunks = (uint32_t)chunks;
  g.tokens = (uint32_t)tokens;
  g.heads_inner = heads_inner;
  int i = 0;
  for (int h : heads) {
    g.groups[i] = (uint32_t)(many ? (h + per - 1) / per : h);
    g.begin[i + 1] = g.begin[i] + (uint32_t)((tokens * g.groups[i] * lanes_of(chunks) + 255) / 256);
    ++i;
  }
  for (; i < 3; ++i) g.begin[i + 1] = g.begin[i];
  return g;
}

template <int DT, int HG, bool STREAM, typename Rows>
hipError_t norm_chunks_go(const Rows& rows, const NormGrid& g, hipStream_t st) {
  const int lanes = lanes_of((int)g.chunks);
  const dim3 grid(g.begin[Rows::KINDS]), block(256);
  switch (lanes) {
    case 4: hipLaunchKernelGGL((ago_norm_chunk_kernel<DT, 4, HG, STREAM, Rows>), grid, block, 0, st, rows, g); break;
    case 8: hipLaunchKernelGGL((ago_norm_chunk_kernel<DT, 8, HG, STREAM, Rows>), grid, block, 0, st, rows, g); break;
    case 16: hipLaunchKernelGGL((ago_norm_chunk_kernel<DT, 16, HG, STREAM, Rows>), grid, block, 0, st, rows, g); break;
    case 32: hipLaunchKernelGGL((ago_norm_chunk_kernel<DT, 32, HG, STREAM, Rows>), grid, block, 0, st, rows, g); break;
    default: hipLaunchKernelGGL((ago_norm_chunk_kernel<DT, 64, HG, STREAM, Rows>), grid, block, 0, st, rows, g); break;
  }
  return hipGetLastError();
}

template <int DT, typename Rows>
hipError_t norm_rows_go(const Rows& rows, int64_t tokens, int64_t heads, hipStream_t st) {
  const int64_t total = tokens * heads, groups = (total + 3) / 4;
  hipLaunchKernelGGL((ago_norm_row_kernel<DT, Rows>), dim3((unsigned)(groups < kMostRows ? groups : kMostRows)), dim3(256), 0,
                     st, rows, (uint32_t)tokens, total);
  return hipGetLastError();
}

// Results larger than the L2 caches (8 of 4 MB) are written past them: 32768 tokens of 24 heads of 64 in bf16 take 39 us for 43, and
// backward 60 for 67; 8189 of 20 heads of 128 in fp32 33 for 35, and 51 for 50.
inline bool past_caches(int64_t chunks) { return chunks * 16 > (int64_t(1) << 25); }

// Whether rows go by in chunks: whole ones at 16-byte addresses, at most a wave of them, and threads by 32 bits.
template <int DT>
bool in_chunks(int dim, int64_t tokens, int64_t heads, std::initializer_list<const void*> bases,
               std::initializer_list<int64_t> strides) {
  if constexpr (DT == AFA_F64) return false;
  constexpr int EPC = DT == AFA_F32 ? 4 : 8;
  if (dim % EPC != 0 || dim / EPC > 64) return false;
  for (const void* p : bases)
    if (((uintptr_t)p & 15u) != 0) return false;
  for (int64_t s : strides)
    if (s % EPC != 0) return false;
  return tokens * heads <= ((int64_t(1) << 32) - 256) / lanes_of(dim / EPC);
}

template <int DT>
hipError_t norm_go(const NormArgs& a, hipStream_t st) {
  const RotateRows rows{a};
  const int64_t tokens = a.batch * a.seq, heads = (int64_t)a.heads[0] + a.heads[1];
  if constexpr (DT != AFA_F64) {
    constexpr int EPC = RowChunk<DT>::EPC;
    const auto &x = a.sx, &y = a.sy;
    if (in_chunks<DT>(a.dim, tokens, heads, {a.x[0], a.y[0], a.x[1], a.y[1]},
                      {x[0][0], x[0][1], x[0][2], x[1][0], x[1][1], x[1][2], y[0][0], y[0][1], y[0][2], y[1][0], y[1][1],
                       y[1][2]})) {
      bool many;
      const NormGrid g = norm_grid(tokens, {a.heads[0], a.heads[1]}, a.dim / EPC, a.sx[0][1] < a.sx[0][2], HEADS, many);
      if (many && past_caches(tokens * heads * a.dim / EPC)) return norm_chunks_go<DT, HEADS, true>(rows, g, st);
      if (many) return norm_chunks_go<DT, HEADS, false>(rows, g, st);
      return norm_chunks_go<DT, 1, false>(rows, g, st);
    }
  }
  return norm_rows_go<DT>(rows, tokens, heads, st);
}

template <int DT>
hipError_t append_norm_go(const AppendArgs& a, const HeadNorm& n, hipStream_t st) {
  const AppendRows rows{{a.q, a.k, a.v}, {a.q_out, a.k_pages, a.v_pages}, {a.q_t, a.k_t, a.v_t}, {a.q_h, a.k_h, a.v_h},
                        {(int64_t)a.heads * a.dim, a.ps.k_page, a.ps.v_page}, {a.dim, a.ps.k_head, a.ps.v_head},
                        {0, a.ps.k_slot, a.ps.v_slot}, {a.heads, a.kv_heads, a.kv_heads}, a.slots, a.capacity, a.page_size,
                        a.dim, n, a.rot};
  const int64_t heads = (int64_t)a.heads + 2 * a.kv_heads;
  if constexpr (DT != AFA_F64) {
    constexpr int EPC = RowChunk<DT>::EPC;
    if (in_chunks<DT>(a.dim, a.tokens, heads, {a.q, a.k, a.v, a.q_out, a.k_pages, a.v_pages},
                      {a.q_t, a.q_h, a.k_t, a.k_h, a.v_t, a.v_h, a.ps.k_page, a.ps.k_head, a.ps.k_slot, a.ps.v_page,
                       a.ps.v_head, a.ps.v_slot})) {
      bool many;
      const NormGrid g = norm_grid(a.tokens, {a.heads, a.kv_heads, a.kv_heads}, a.dim / EPC, true, HEADS, many);
      return many ? norm_chunks_go<DT, HEADS, false>(rows, g, st) : norm_chunks_go<DT, 1, false>(rows, g, st);
    }
  }
  return norm_rows_go<DT>(rows, a.tokens, heads, st);
}

// Parts of q's and of k's rows: `most` in all, as their heads are, and no more than there are sets of rows.
inline void parts_of(NormParts& p, int64_t most, int64_t q, int64_t k, int64_t per) {
  const int64_t all = q + k, nq = (q + per - 1) / per, nk = (k + per - 1) / per;
  int64_t a = most * q / all;
  a = a < 1 ? 1 : a;
  const int64_t b = most - a < 1 ? 1 : most - a;
  p.parts[0] = (uint32_t)(a < nq ? a : nq);
  p.parts[1] = k == 0 ? 0 : (uint32_t)(b < nk ? b : nk);
}
// With one a CU 32768 tokens of 24 heads of 64 in bf16 take 85 us for 67, with four 66; 5460 tokens 19.7, and 19.3, for 16.5.
inline int64_t most_parts(int cus) { return 2 * (int64_t)cus; }

template <int DT, int HG, bool STREAM>
hipError_t norm_bwd_chunks_go(const NormArgs& a, const NormGrid& g, const NormParts& p, hipStream_t st) {
  const dim3 grid(p.parts[0] + p.parts[1]), block(BWD);
  switch (lanes_of((int)g.chunks)) {
    case 4: hipLaunchKernelGGL((ago_norm_bwd_chunk_kernel<DT, 4, HG, STREAM>), grid, block, 0, st, a, g, p); break;
    case 8: hipLaunchKernelGGL((ago_norm_bwd_chunk_kernel<DT, 8, HG, STREAM>), grid, block, 0, st, a, g, p); break;
    case 16: hipLaunchKernelGGL((ago_norm_bwd_chunk_kernel<DT, 16, HG, STREAM>), grid, block, 0, st, a, g, p); break;
    case 32: hipLaunchKernelGGL((ago_norm_bwd_chunk_kernel<DT, 32, HG, STREAM>), grid, block, 0, st, a, g, p); break;
    default: hipLaunchKernelGGL((ago_norm_bwd_chunk_kernel<DT, 64, HG, STREAM>), grid, block, 0, st, a, g, p); break;
  }
  return hipGetLastError();
}

template <int DT>
hipError_t norm_bwd_go(const NormArgs& a, void* const dscale[2], void* ws, int cus, hipStream_t st) {
  using A = Wide<DT>;
  const int64_t tokens = a.batch * a.seq, heads = (int64_t)a.heads[0] + a.heads[1];
  NormParts p = {};
  p.sums = ws;
  hipError_t e = hipSuccess;
  bool chunks = false;
  if constexpr (DT != AFA_F64) {
    constexpr int EPC = RowChunk<DT>::EPC;
    const auto &x = a.sx, &y = a.sy, &z = a.sg;
    chunks = in_chunks<DT>(a.dim, tokens, heads, {a.x[0], a.y[0], a.g[0], a.x[1], a.y[1], a.g[1]},
                           {x[0][0], x[0][1], x[0][2], x[1][0], x[1][1], x[1][2], y[0][0], y[0][1], y[0][2], y[1][0], y[1][1],
                            y[1][2], z[0][0], z[0][1], z[0][2], z[1][0], z[1][1], z[1][2]});
    if (chunks) {
      bool many;
      constexpr int HG = 2;  // by ones 81 us for 67 (32768 tokens of 24 heads of 64, bf16); by fours as long as by twos past the caches
      const NormGrid g = norm_grid(tokens, {a.heads[0], a.heads[1]}, a.dim / EPC, a.sx[0][1] < a.sx[0][2], HG, many);
      parts_of(p, most_parts(cus), tokens * g.groups[0], tokens * g.groups[1], BWD / lanes_of(a.dim / EPC));
      if (many && past_caches(tokens * heads * a.dim / EPC)) e = norm_bwd_chunks_go<DT, HG, true>(a, g, p, st);
      else e = many ? norm_bwd_chunks_go<DT, HG, false>(a, g, p, st) : norm_bwd_chunks_go<DT, 1, false>(a, g, p, st);
    }
  }
  if (!chunks) {
    parts_of(p, most_parts(cus), tokens * a.heads[0], tokens * a.heads[1], 1);
    hipLaunchKernelGGL((ago_norm_bwd_row_kernel<DT>), dim3(p.parts[0] + p.parts[1]), dim3(64), 0, st, a, p);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((ago_norm_join_kernel<A>), dim3((unsigned)((a.dim + 63) / 64), a.heads[1] > 0 ? 2 : 1), dim3(JOIN), 0, st, p,
                     a.dim, (A*)dscale[0], (A*)dscale[1]);
  return hipGetLastError();
}

}  // namespace

hipError_t norm_rotate_launch(int dtype, const NormArgs& a, hipStream_t st) {
  switch (dtype) {
    case AFA_F32: return norm_go<AFA_F32>(a, st);
    case AFA_BF16: return norm_go<AFA_BF16>(a, st);
    case AFA_F16: return norm_go<AFA_F16>(a, st);
    default: return norm_go<AFA_F64>(a, st);
  }
}

size_t norm_rotate_bwd_workspace(int dtype, int dim, int cus) {
  return (size_t)(most_parts(cus) + 1) * (size_t)dim * (dtype == AFA_F64 ? 8 : 4);
}

hipError_t norm_rotate_bwd_launch(int dtype, const NormArgs& a, void* const dscale[2], void* ws, int cus, hipStream_t st) {
  switch (dtype) {
    case AFA_F32: return norm_bwd_go<AFA_F32>(a, dscale, ws, cus, st);
    case AFA_BF16: return norm_bwd_go<AFA_BF16>(a, dscale, ws, cus, st);
    case AFA_F16: return norm_bwd_go<AFA_F16>(a, dscale, ws, cus, st);
    default: return norm_bwd_go<AFA_F64>(a, dscale, ws, cus, st);
  }
}

hipError_t paged_append_norm_launch(int dtype, const AppendArgs& a, const HeadNorm& n, hipStream_t st) {
  switch (dtype) {
    case AFA_F32: return append_norm_go<AFA_F32>(a, n, st);
    case AFA_BF16: return append_norm_go<AFA_BF16>(a, n, st);
    case AFA_F16: return append_norm_go<AFA_F16>(a, n, st);
    default: return append_norm_go<AFA_F64>(a, n, st);
  }
}

}  // namespace afa
