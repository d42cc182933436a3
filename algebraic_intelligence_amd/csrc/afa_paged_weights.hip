// What each token of the cache was given by a step's rows, added up:
//
//   W[r][j] += sum over the step's tokens i of request r that see j, and heads h, of  rho(s_ihj)^8 / d_ih
//
// with d the denominators that the step's attention returned, sink and prefix included.  A token of the step
// itself has no weight yet: its place is set, not added to.
//
// On the matrix cores (bf16, fp16, fp32; head_dim 32, 48, 64, 96, 128, 256; pages of a power of two) a workgroup takes 32
// keys of one request.  S = Q K^T with 16 rows of Q as A and two times 16 keys as B leaves each lane with the scores
// of one key in a group, so that the sum over the rows stays in the lane; K is in registers for all rows of its head, and
// Q comes from the caches.  The four waves share a head's row blocks, or the heads where these are few, and add up in
// LDS.  Where the requests' tiles are too few to fill the device, workgroups share a tile's heads too, and the last one
// of a tile adds their parts in order.  So every sum has one order, which atomics would not give it.
#include <algorithm>
#include <initializer_list>

#include "afa_common.h"
#include "afa_paged.h"
#include "afa_paged_tile.h"

namespace afa {

namespace {

constexpr int KEYS = 256;

template <int DT, typename A>
__device__ __forceinline__ A elem_of(const void* p, int64_t i) {
  if constexpr (DT == AFA_F64) return ((const double*)p)[i];
  else return Elem<DT>::load(p, i);
}

// Any head_dim, type, stride and page size: a key a thread, its rows one after the other.
template <int DT>
__global__ __launch_bounds__(KEYS) void afa_paged_weight_key_kernel(const WeightArgs a, int64_t blocks, int64_t total) {
  using A = typename std::conditional<DT == AFA_F64, double, float>::type;
  const afa_paged_plan& p = a.plan;
  const int D = (int)p.head_dim, H = (int)p.heads, W = (int)(p.max_tree / 64);
  for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
    const int r = (int)(item / blocks);
    const int pos = (int)(item % blocks) * KEYS + (int)threadIdx.x;
    const int start = p.starts[r], n = p.starts[r + 1] - start, c = a.sched.cached[r];
    if (p.status[r] != AFA_PAGED_OK || n <= 0 || pos >= c + n) continue;
    const int page = p.block_tables[r * p.table_width + pos / p.page_size];
    double sum = 0;  // of rows * heads terms, one after the other
    if (page >= 0 && page < p.num_pages) {
      const bool tree = a.masks != nullptr && n <= p.max_tree;
      const int j = pos - c;
      for (int i = j < 0 || tree ? 0 : j; i < n; ++i) {
        if (j >= 0 && tree && !((a.masks[(int64_t)(start + i) * W + j / 64] >> (j & 63)) & 1)) continue;
        for (int h = 0; h < H; ++h) {
          const int64_t t = start + i;
          const A d = ((const A*)a.denom)[t * H + h];
          if (d == 0) continue;  // the row saw no key
          const int64_t q = t * a.q_t + h * a.q_h;
          const int64_t k = page * a.k_page + h / a.group * a.k_head + pos % p.page_size * a.k_slot;
          A s = 0;
          for (int e = 0; e < D; ++e) s += elem_of<DT, A>(a.q, q + e) * elem_of<DT, A>(a.k_pages, k + e);
          if constexpr (DT == AFA_F64) sum += rho8_f64(s * a.scale) / d;
          else sum += (double)(rho8_ref(s * (float)a.scale) / d);
        }
      }
    }
    float* w = a.weights + r * a.row + pos;
    *w = (float)(pos < c ? *w + sum : sum);
  }
}

template <int DT>
hipError_t weight_keys_go(const WeightArgs& a, int cus, hipStream_t st) {
  const int64_t blocks = (a.plan.table_width * a.plan.page_size + KEYS - 1) / KEYS, total = a.plan.requests * blocks;
  const int64_t most = 16 * (int64_t)cus;
  hipLaunchKernelGGL((afa_paged_weight_key_kernel<DT>), dim3((unsigned)(total < most ? total : most)), dim3(KEYS), 0, st, a,
                     blocks, total);
  return hipGetLastError();
}

// ------------------------------------------------------------------ matrix cores
// parts of tiles that share their heads
constexpr int64_t kWeightParts = 4096;
constexpr int WTILE = 32, WAVES = 4, THREADS = 64 * WAVES;
constexpr int SCAN = 4 * THREADS;  // requests whose tiles a workgroup counts at a time

struct WeightFast {
  WeightArgs a;
  float* part;      // (tiles * splits, WTILE)
  int* count;       // of a tile's parts; 0 between calls
  int most;         // parts that there is room for
  int log_page;
};

// Sums of x over the threads before this one; all: over the workgroup.
__device__ __forceinline__ int tiles_before(int x, int* lds, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int s = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(s, o);
    if (lane >= o) s += u;
  }
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  int base = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w == wave) base = all;
    all += lds[w];
  }
  return base + s - x;
}

template <int DT, int D>
__global__ __launch_bounds__(THREADS) void afa_paged_weight_tile_kernel(const WeightFast f) {
  constexpr bool F32 = DT == AFA_F32;
  constexpr int ESZ = F32 ? 4 : 2;
  constexpr int EPC = 16 / ESZ;           // features of a 16-byte chunk
  constexpr int KB = 4 * EPC;             // of a chunk over the four lane groups
  constexpr int KS = (D + KB - 1) / KB;   // chunks of a row a lane
  constexpr bool FULL = D % KB == 0;
  constexpr int NG = WTILE / 16;
  __shared__ int first[SCAN + 1], scan[WAVES], flag;
  __shared__ float red[WAVES][WTILE];
  const WeightArgs& a = f.a;
  const afa_paged_plan& p = a.plan;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int H = (int)p.heads, K = (int)p.kv_heads, G = a.group, W = (int)(p.max_tree / 64), R = (int)p.requests;
  const int lp = f.log_page, in_page = (1 << lp) - 1;
  const float scale = (float)a.scale;
  for (int r0 = 0; r0 < R; r0 += SCAN) {
    // tiles of the requests before each of these
    {
      int n[4], sum = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = r0 + 4 * tid + u;
        n[u] = 0;
        if (r < R && p.status[r] == AFA_PAGED_OK) {
          const int fresh = p.starts[r + 1] - p.starts[r];
          if (fresh > 0) n[u] = (int)((unsigned)(a.sched.cached[r] + fresh + WTILE - 1) / WTILE);
        }
        sum += n[u];
      }
      int all;
      int at = tiles_before(sum, scan, all);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        first[4 * tid + u] = at;
        at += n[u];
      }
      if (tid == THREADS - 1) first[SCAN] = at;
      __syncthreads();
    }
    const int tiles = first[SCAN];
    // heads of a tile over so many workgroups; requests beyond the first SCAN would need counts of their own
    const int splits = R <= SCAN && tiles > 0 ? max(1, min(K, f.most / tiles)) : 1;
    const int64_t items = (int64_t)tiles * splits;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
      const int tile = (int)(item / splits), split = (int)(item - (int64_t)tile * splits);
      // the request: the last whose first tile is not behind this one
      int lo = 0, hi = SCAN;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= tile) lo = mid;
        else hi = mid;
      }
      const int r = r0 + lo, kb = (tile - first[lo]) * WTILE;
      const int start = p.starts[r], n = p.starts[r + 1] - start, c = a.sched.cached[r], keys = c + n, nrows = n * G;
      const bool tree = a.masks != nullptr && n <= p.max_tree;
      // this lane's keys, and where their rows lie
      const char* krow[NG];
      bool lost[NG];
#pragma unroll
      for (int u = 0; u < NG; ++u) {
        const int pos = min(kb + 16 * u + m, keys - 1), page = p.block_tables[(int64_t)r * p.table_width + (pos >> lp)];
        lost[u] = (unsigned)page >= (unsigned)p.num_pages;
        krow[u] = (const char*)a.k_pages +
                  ((lost[u] ? 0 : page) * a.k_page + (int64_t)(pos & in_page) * a.k_slot + EPC * g) * ESZ;
      }
      // chains: row blocks whose last token is before the tile see nothing of it
      const int blocks = (nrows + 15) / 16;
      const int block0 = tree || kb <= c ? 0 : (kb - c) * G / 16;
      // waves that share a head's row blocks
      const int share = blocks - block0 >= WAVES ? WAVES : blocks - block0 >= 2 ? 2 : 1;
      const int heads_at_once = WAVES / share, rsub = wave % share;
      float acc[NG];
#pragma unroll
      for (int u = 0; u < NG; ++u) acc[u] = 0.0f;
      for (int hk = split + splits * (wave / share); hk < K; hk += splits * heads_at_once) {
        u32x4_t kf[NG][KS];
#pragma unroll
        for (int u = 0; u < NG; ++u)
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            kf[u][ks] = FULL || KB * ks + EPC * g < D ? *(const u32x4_t*)(krow[u] + (hk * a.k_head + KB * ks) * ESZ)
                                                      : u32x4_t{0, 0, 0, 0};
        float head[NG];
#pragma unroll
        for (int u = 0; u < NG; ++u) head[u] = 0.0f;
        for (int b = block0 + rsub; b < blocks; b += share) {
          const int row = min(16 * b + m, nrows - 1), token = row / G;
          const char* x = (const char*)a.q +
                          ((int64_t)(start + token) * a.q_t + (hk * G + row - token * G) * a.q_h + EPC * g) * ESZ;
          u32x4_t qf[KS];
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            qf[ks] = FULL || KB * ks + EPC * g < D ? *(const u32x4_t*)(x + KB * ks * ESZ) : u32x4_t{0, 0, 0, 0};
          // over the rows' denominators; rows behind the last have none, nor has one that saw no key
          float over[4];
          int who[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int rr = 16 * b + 4 * g + i, at = min(rr, nrows - 1);
            who[i] = at / G;
            const float d = ((const float*)a.denom)[(int64_t)(start + who[i]) * H + hk * G + (at - who[i] * G)];
            over[i] = rr < nrows && d != 0.0f ? __builtin_amdgcn_rcpf(d) : 0.0f;
          }
          f32x4_t s4[NG];
#pragma unroll
          for (int u = 0; u < NG; ++u) {
            s4[u] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const unsigned y = qf[ks][e], z = kf[u][ks][e];
                  s4[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, y), __builtin_bit_cast(float, z),
                                                               s4[u], 0, 0, 0);
                }
              } else {
                s4[u] = mma16<DT>(qf[ks], kf[u][ks], s4[u]);
              }
            }
          }
          float w[NG][4];
          if constexpr (F32) {
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) w[u][i] = rho8_refined(s4[u][i] * scale);
          } else {
            float least = 0.0f;
#pragma unroll
            for (int u = 0; u < NG; ++u)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                w[u][i] = s4[u][i] * scale;
                least = __builtin_fminf(least, w[u][i]);
              }
            // a score that is no number takes either form
            if (__ballot(!(least > kLowScore)) == 0) {
#pragma unroll
              for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[u][i] = rho8_fast(w[u][i]);
            } else {
#pragma unroll
              for (int u = 0; u < NG; ++u) apart(w[u]);
#pragma unroll
              for (int u = 0; u < NG; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[u][i] = rho8_by_score(w[u][i]);
            }
          }
          // every key of the tile is seen by these rows, which all give something, or each by its own
          const bool some = (over[0] != 0.0f && over[1] != 0.0f) && (over[2] != 0.0f && over[3] != 0.0f);
          const bool whole = kb + WTILE <= (tree ? c : c + 1 + 16 * b / G) && __ballot(!some) == 0;
          if (!whole) {
#pragma unroll
            for (int u = 0; u < NG; ++u) {
              const int pos = kb + 16 * u + m, j = pos - c;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                bool sees = pos < keys && over[i] != 0.0f;
                if (sees && j >= 0)
                  sees = tree ? a.masks[(int64_t)(start + who[i]) * W + (j >> 6)] >> (j & 63) & 1 : j <= who[i];
                w[u][i] = sees ? w[u][i] : 0.0f;
              }
            }
          }
#pragma unroll
          for (int u = 0; u < NG; ++u) {
            float x4 = w[u][0] * over[0];
#pragma unroll
            for (int i = 1; i < 4; ++i) x4 = __builtin_fmaf(w[u][i], over[i], x4);
            head[u] += x4;
          }
        }
#pragma unroll
        for (int u = 0; u < NG; ++u) acc[u] += head[u];
      }
      __syncthreads();  // red is free of the item before
#pragma unroll
      for (int u = 0; u < NG; ++u) {
        float x = lost[u] ? 0.0f : acc[u];
        x += __shfl_xor(x, 16);
        x += __shfl_xor(x, 32);
        if (g == 0) red[wave][16 * u + m] = x;
      }
      __syncthreads();
      const int pos = kb + tid;
      float sum = 0.0f;
      if (tid < WTILE) sum = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
      if (splits > 1) {
        float* part = f.part + (int64_t)tile * splits * WTILE;
        if (tid < WTILE) put1(part + split * WTILE + tid, sum);
        if (!arrived(f.count + tile, splits, &flag)) continue;
        if (tid < WTILE) {
          sum = 0.0f;
          for (int i0 = 0; i0 < splits; i0 += 8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = get1(part + min(i0 + i, splits - 1) * WTILE + tid);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += i0 + i < splits ? y[i] : 0.0f;
          }
        }
      }
      if (tid < WTILE && pos < keys) {
        float* to = a.weights + r * a.row + pos;
        *to = pos < c ? *to + sum : sum;
      }
    }
    __syncthreads();  // first is free
  }
}

template <int DT, int D>
hipError_t weight_tiles_launch(const WeightFast& f, int cus, hipStream_t st) {
  hipLaunchKernelGGL((afa_paged_weight_tile_kernel<DT, D>), dim3((unsigned)(4 * cus)), dim3(THREADS), 0, st, f);
  return hipGetLastError();
}

template <int DT>
hipError_t weight_tiles_go(const WeightFast& f, int cus, hipStream_t st) {
  switch ((int)f.a.plan.head_dim) {
    case 32: return weight_tiles_launch<DT, 32>(f, cus, st);
    case 48: return weight_tiles_launch<DT, 48>(f, cus, st);
    case 64: return weight_tiles_launch<DT, 64>(f, cus, st);
    case 96: return weight_tiles_launch<DT, 96>(f, cus, st);
    case 128: return weight_tiles_launch<DT, 128>(f, cus, st);
    default: return weight_tiles_launch<DT, 256>(f, cus, st);
  }
}

}  // namespace

bool paged_weights_fast(const WeightArgs& a) {
  const int64_t unit = a.plan.dtype == AFA_F32 ? 4 : 8;
  bool fast = paged_fast_supported(a.plan) && (((uintptr_t)a.q | (uintptr_t)a.k_pages) & 15u) == 0;
  for (int64_t v : {a.q_t, a.q_h, a.k_page, a.k_head, a.k_slot}) fast = fast && v % unit == 0;
  return fast;
}

hipError_t paged_weights_launch(const WeightArgs& a, const PagedCut& cut, int cus, void* ws, size_t ws_bytes, hipStream_t st) {
  if (ws != nullptr) {
    WeightFast f;
    f.a = a;
    f.part = (float*)ws;
    f.count = a.sched.count;
    // a tile has two parts at least where it is split
    const int64_t counts = 2 * a.plan.kv_heads * 4 * cut.slots, room = (int64_t)(ws_bytes / (WTILE * 4));
    f.most = (int)std::min<int64_t>(kWeightParts, std::min(counts, room));
    f.log_page = __builtin_ctzll((unsigned long long)a.plan.page_size);
    switch ((int)a.plan.dtype) {
      case AFA_F32: return weight_tiles_go<AFA_F32>(f, cus, st);
      case AFA_BF16: return weight_tiles_go<AFA_BF16>(f, cus, st);
      default: return weight_tiles_go<AFA_F16>(f, cus, st);
    }
  }
  switch ((int)a.plan.dtype) {
    case AFA_F32: return weight_keys_go<AFA_F32>(a, cus, st);
    case AFA_BF16: return weight_keys_go<AFA_BF16>(a, cus, st);
    case AFA_F16: return weight_keys_go<AFA_F16>(a, cus, st);
    default: return weight_keys_go<AFA_F64>(a, cus, st);
  }
}

}  // namespace afa
