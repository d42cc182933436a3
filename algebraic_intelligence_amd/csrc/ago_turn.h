// The Cayley rotation of pairs and of 16-byte chunks by positions of several axes, for the kernels that turn rows.
#pragma once

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

// Entry i of the positions; i itself where there are none.
__device__ __forceinline__ int64_t position(const AxisRotation& r, int64_t i) {
  if (r.positions == nullptr) return i;
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

// A 16-byte chunk's table entries and its rotation.
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

  __device__ __forceinline__ void turn_values(float (&v)[R::EPC]) const {
#pragma clang fp contract(off)
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const float x0 = v[2 * p], x1 = v[2 * p + 1];
      v[2 * p] = keep[p] ? x0 : c[p] * x0 - s[p] * x1;
      v[2 * p + 1] = keep[p] ? x1 : s[p] * x0 + c[p] * x1;
    }
  }

  __device__ __forceinline__ u32x4_t turned(u32x4_t w) const {
    float v[R::EPC];
    R::unpack(w, v);
    turn_values(v);
    return R::pack(v);
  }
};

}  // namespace afa
