// Tiles of scores and parts that pass between workgroups, for the kernels over the paged cache on the matrix cores.
#pragma once

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

template <int DT>
__device__ __forceinline__ f32x4_t mma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  if constexpr (DT == AFA_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                  0);
}

// Weights end at 2^-126, the smallest normal number (scores of -27554 and below): the eighth power is cut off there
// before its inverse is formed.  Further down it no longer fits and then the square of the score does not, which
// gives an infinity and a NaN, and the cut takes either.
constexpr float kMostPower = 0x1p126f;

// rho(s)^8 in fp32 with the square root and the reciprocal refined by one Newton step each: the
// hardware's are off by 1 ulp, which three squarings make 8.
__device__ __forceinline__ float rho8_refined(float s) {
  const float a = __builtin_fabsf(s);
  const float t = __builtin_fmaf(a, a, 1.0f);
  const float r = __builtin_amdgcn_rsqf(t);
  const float root = t * r;
  const float rho = __builtin_fmaf(0.5f * r, __builtin_fmaf(-root, root, t), root) + a;
  const float p2 = rho * rho;
  const float p4 = p2 * p2;
  const float p8 = p4 * p4;
  const float cut = __builtin_fminf(p8, kMostPower);
  const float i0 = __builtin_amdgcn_rcpf(cut);
  const float inv = __builtin_fmaf(i0, __builtin_fmaf(-cut, i0, 1.0f), i0);
  return s < 0.0f ? inv : p8;  // a NaN stays one
}

// rho(s)^8 in bf16 and fp16 calls: above kLowScore the branch-free form, which costs half of the other and loses
// nothing above 0, and below it 16 s^2 times the error of the hardware's rsqrt, 2.2e-4 at -8; below kLowScore the
// form without cancellation.  A weight goes by its own score alone, whatever scores a wave forms beside it, of
// keys that the row does not see among them.
constexpr float kLowScore = -8.0f;
__device__ __forceinline__ float rho8_by_score(float s) {
  const bool low = s <= kLowScore;
  const float t = __builtin_fmaf(s, s, 1.0f);
  const float r = __builtin_amdgcn_rsqf(t);
  const float rho = __builtin_fmaf(t, r, low ? __builtin_fabsf(s) : s);
  const float p2 = rho * rho;
  const float p4 = p2 * p2;
  const float p8 = p4 * p4;
  return low ? __builtin_amdgcn_rcpf(__builtin_fminf(p8, kMostPower)) : p8;  // a NaN stays one
}

// Makes values new ones to the compiler, at no cost.  In one side of a branch over both forms of the weights it keeps what
// they share from being formed once for both, and the branch from turning into a select, which would cost every tile both.
template <int N>
__device__ __forceinline__ void apart(float (&w)[N]) {
#pragma unroll
  for (int e = 0; e < N; ++e) asm volatile("" : "+v"(w[e]));
}

// The power of two by which a row's fp16 weights begin.  It is only ever lowered, so it decides how small weights may
// be that have a row to themselves: 2^-120, a score of -16384, is 1 then.  A first weight of about 1 lowers it
// at once, as any start does; its inverse and that of the lowest, 2^-123, are normal numbers.
constexpr float kFirstScale = 0x1p120f;

// Bits of `len` consecutive drafted tokens from index i0 on (negative: cached, seen) that the row sees.
// words: the row's masks, nullptr for a chain whose row is token `self`; n: the request's new tokens.
__device__ __forceinline__ unsigned sees_bits(int i0, int len, int n, int self, const int64_t* words, int W) {
  const unsigned all = (1u << len) - 1;
  if (i0 + len <= 0) return all;
  unsigned bits;
  if (words != nullptr) {
    const int at = max(i0, 0), w = at >> 6, sh = at & 63;
    uint64_t x = 0;
    if (w < W) x = (uint64_t)words[w] >> sh;
    if (sh > 64 - len && w + 1 < W) x |= (uint64_t)words[w + 1] << (64 - sh);
    bits = (unsigned)x & all;
    if (i0 < 0) bits = (bits << -i0) | ((1u << -i0) - 1);
  } else {
    const int c = min(max(self + 1 - i0, 0), len);
    bits = (1u << c) - 1;
  }
  const int live = min(max(n - i0, 0), len);
  return bits & ((1u << live) - 1);
}

// ------------------------------------------------------------------ parts of cut keys
// Parts pass between workgroups by device-scope relaxed stores and loads, which go to where every XCD sees
// them: a part's stores are complete (vmcnt 0) before its count, and the last to count reads after its
// own.  An acquire and release edge would write back and invalidate the whole L2 for each part.
typedef unsigned long long u64;
__device__ __forceinline__ void put1(float* p, float x) {
  __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float get1(const float* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// 16 bytes at byte `at` of a head's parts, of the same scope (sc1).
constexpr int kDeviceScope = 16;
__device__ __forceinline__ void put4(__amdgpu_buffer_rsrc_t parts, uint32_t at, f32x4_t x) {
  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, x), parts, at, 0, kDeviceScope);
}
__device__ __forceinline__ f32x4_t get4(__amdgpu_buffer_rsrc_t parts, uint32_t at) {
  return __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(parts, at, 0, kDeviceScope));
}

// Whether this workgroup is the last of `n` to get here; its stores are complete before it counts.  The last
// one leaves the count at 0.
__device__ __forceinline__ bool arrived(int* count, int n, int* flag) {
  __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  __syncthreads();
  if (threadIdx.x == 0) {
    *flag = atomicAdd(count, 1) == n - 1;
    if (*flag) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  return *flag != 0;
}

}  // namespace afa
