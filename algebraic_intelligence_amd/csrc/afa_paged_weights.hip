// What each token of the cache was given by a step's rows, added up:
//
//   W[r][j] += sum over the step's tokens i of request r that see j, and heads h, of  rho(s_ihj)^8 / d_ih
//
// with d the denominators that the step's attention returned, sink and prefix included.  A token of the step
// itself has no weight yet: its place is set, not added to.
//
// On the matrix cores (bf16, fp16, fp32; head_dim 32, 48, 64, 96, 128, 256; pages of a power of two) a workgroup takes 64
// keys of one request (32 where rows are longer than 256 bytes).  S = Q K^T with 16 rows of Q as A and four times 16 keys as
// B leaves each lane with the scores of one key in a group, so that the sum over the rows stays in the lane; K is in registers
// for all rows of its head, and Q comes from the caches.  The four waves share a head's row blocks, or the heads where these are few, and add up in
// LDS.  Where the requests' tiles are too few to fill the device, workgroups share a tile's heads too, and the last one
// of a tile adds their parts in order.  So every sum has one order, which atomics would not give it.
//
// One token of 64 requests over up to 8192, 16 heads on 4 of 128 in bf16: 78 us, K read once at 4.2 TB/s.  Prompts are bound by the
// vector instructions of rho^8 (7 for 64 weights and a square root, which is as long as 4): 8 of 2048 tokens, 12 heads of 64 in bf16,
// take 105 us, and about 70 if the vector units never paused.
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
          sum += (double)(rho8_above_0(s, a.scale) / d);
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
// parts of tiles that share their heads, and the most keys of a tile
constexpr int64_t kWeightParts = 4096;
constexpr int MOST_KEYS = 64;
constexpr int WAVES = 4, THREADS = 64 * WAVES;
constexpr int SCAN = 4 * THREADS;  // requests whose tiles a workgroup counts at a time

struct WeightFast {
  WeightArgs a;
  float* part;      // (tiles * splits, keys of a tile)
  int* count;       // of a tile's parts; 0 between calls
  int most;         // parts that there is room for
  int log_page;
};

// Sums of x over the threads before this one.
__device__ __forceinline__ int tiles_before(int x, int* lds) {
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
#pragma unroll
  for (int w = 0; w < WAVES - 1; ++w)
    if (w < wave) base += lds[w];
  return base + s - x;
}

// Groups of 16 keys of a tile: as many as leave their rows of K room in the registers.
template <int DT, int D>
constexpr int key_groups() {
  return D * (DT == AFA_F32 ? 4 : 2) <= 256 ? 4 : 2;
}

// Workgroups that a CU's registers hold, and as many are launched for each: with a third more, which wait for the first to
// end, 64 requests of one token over up to 8192 take 111 us for 78.
template <int DT, int D>
constexpr int resident() {
  constexpr int bytes = D * (DT == AFA_F32 ? 4 : 2);
  return bytes <= 128 ? 3 : bytes <= 512 ? 2 : 1;
}

template <int DT, int D>
__global__ __launch_bounds__(THREADS, (resident<DT, D>())) void afa_paged_weight_tile_kernel(const WeightFast f) {
  constexpr bool F32 = DT == AFA_F32;
  constexpr int ESZ = F32 ? 4 : 2;
  constexpr int EPC = 16 / ESZ;           // features of a 16-byte chunk
  constexpr int KB = 4 * EPC;             // of a chunk over the four lane groups
  constexpr int KS = (D + KB - 1) / KB;   // chunks of a row a lane
  constexpr bool FULL = D % KB == 0;
  constexpr int NG = key_groups<DT, D>(), TILE = 16 * NG;
  __shared__ int first[SCAN + 1], scan[WAVES], longest[WAVES], flag;
  __shared__ float red[WAVES][TILE];
  const WeightArgs& a = f.a;
  const afa_paged_plan& p = a.plan;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int H = (int)p.heads, K = (int)p.kv_heads, G = a.group, W = (int)(p.max_tree / 64), R = (int)p.requests;
  const int lp = f.log_page, in_page = (1 << lp) - 1;
  // 1 / sqrt(D) where it is a power of two: K carries it without a rounding (in fp16 small numbers would lose digits), which is
  // an instruction less for every weight (8 prompts of 2048 take 111 us for 124)
  constexpr bool CARRIED = DT == AFA_BF16 && (D == 64 || D == 256);
  const float scale = (float)a.scale;
  for (int r0 = 0; r0 < R; r0 += SCAN) {
    // tiles of the requests before each of these
    {
      int n[4], sum = 0, most = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = r0 + 4 * tid + u;
        n[u] = 0;
        if (r < R && p.status[r] == AFA_PAGED_OK) {
          const int fresh = p.starts[r + 1] - p.starts[r];
          if (fresh > 0) n[u] = (int)((unsigned)(a.sched.cached[r] + fresh + TILE - 1) / TILE);
        }
        sum += n[u];
        most = max(most, n[u]);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) most = max(most, __shfl_xor(most, o));
      if (lane == 0) longest[wave] = most;
      int at = tiles_before(sum, scan);
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        first[4 * tid + u] = at;
        at += n[u];
      }
      if (tid == THREADS - 1) first[SCAN] = at;
      __syncthreads();
    }
    const int tiles = __builtin_amdgcn_readfirstlane(first[SCAN]);
    const int coarse = first[SCAN / 64 * lane];
    // heads of a tile over so many workgroups; requests beyond the first SCAN would need counts of their own
    const int splits = R <= SCAN && tiles > 0 ? max(1, min(K, f.most / tiles)) : 1;
    // Long prompts (1024 rows of a key head or more, on average) of about one length go by columns: all requests' first tiles, then
    // their second, for the later tiles of a prompt are seen by fewer rows.  8 of 2048 tokens take 104 us, one after the other 111;
    // 8 of 1024 to 2048 90 and 92; 32 of 512 to 1024, two rows each, 71 and 69; 64 of 256 take 56 either way.
    const int tall = __builtin_amdgcn_readfirstlane(max(max(longest[0], longest[1]), max(longest[2], longest[3])));
    const bool columns = R <= SCAN && (int64_t)p.starts[R] * G >= 1024 * R && 3 * (int64_t)tall * R <= 4 * (int64_t)tiles;
    const int64_t items = (columns ? (int64_t)tall * R : tiles) * splits;
    // there and back, for the same reason: 124 us for 131 without, one after the other
    for (int64_t k = 0, item; (item = k * gridDim.x + (k & 1 ? gridDim.x - 1 - blockIdx.x : blockIdx.x)) < items; ++k) {
      int tile = (int)(item / splits), lo;
      const int split = (int)(item - (int64_t)tile * splits);
      if (columns) {
        const int column = tile / R;
        lo = tile - column * R;
        tile = __builtin_amdgcn_readfirstlane(first[lo]) + column;
        if (tile >= __builtin_amdgcn_readfirstlane(first[lo + 1])) continue;
      } else {
        // the request: the last whose first tile is not behind this one, in two steps of the lanes
        static_assert(SCAN / 64 <= 64, "entries between two coarse ones");
        const int step = SCAN / 64, at0 = (__popcll(__ballot(coarse <= tile)) - 1) * step;
        const int mine = first[at0 + min(lane, step - 1)];
        lo = __builtin_amdgcn_readfirstlane(at0 + __popcll(__ballot(lane < step && mine <= tile)) - 1);
      }
      const int r = r0 + lo, kb = (tile - first[lo]) * TILE;
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
      // what the tile's tokens had, which is needed last
      const int pos = kb + tid;
      float* to = a.weights + r * a.row + pos;
      const float old = tid < TILE && pos < c ? *to : 0.0f;
      // chains: row blocks whose last token is before the tile see nothing of it
      const int blocks = (nrows + 15) / 16;
      const int block0 = tree || kb <= c ? 0 : (int)((int64_t)(kb - c) * G / 16);
      // waves that share a head's row blocks
      const int share = blocks - block0 >= WAVES ? WAVES : blocks - block0 >= 2 ? 2 : 1;
      const int heads_at_once = WAVES / share, rsub = wave % share;
      // a lane's row, 16 * share further on each time: its token and head of the group
      const int row0 = 16 * (block0 + rsub) + m, token0 = row0 / G, in0 = row0 - token0 * G;
      const int more_tokens = 16 * share / G, more_in = 16 * share - more_tokens * G;
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
        if constexpr (CARRIED) {
#pragma unroll
          for (int u = 0; u < NG; ++u)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const unsigned y = kf[u][ks][e];
                kf[u][ks][e] = Elem<DT>::pack(Elem<DT>::lo(y) * scale, Elem<DT>::hi(y) * scale);
              }
        }
        float head[NG];
#pragma unroll
        for (int u = 0; u < NG; ++u) head[u] = 0.0f;
        int token = token0, in = in0;
        u32x4_t next[KS];
        float next_den;
        // the row's features and its denominator; behind the last row that one's
        auto load = [&]() {
          const int t = start + min(token, n - 1), h = hk * G + (token < n ? in : G - 1);
          const char* x = (const char*)a.q + ((int64_t)t * a.q_t + h * a.q_h + EPC * g) * ESZ;
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            next[ks] = FULL || KB * ks + EPC * g < D ? *(const u32x4_t*)(x + KB * ks * ESZ) : u32x4_t{0, 0, 0, 0};
          next_den = ((const float*)a.denom)[(int64_t)t * H + h];
        };
        load();
        for (int b = block0 + rsub; b < blocks; b += share) {
          u32x4_t qf[KS];
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) qf[ks] = next[ks];
          // over the row's denominator; -1 for rows behind the last, which have none, and for one that saw no key.  The hardware
          // makes a subnormal inverse, above 2^126, 0: these take two steps (8 prompts of 2048 take 105.5 us for 104.7, by a
          // branch 107).
          const float den = next_den, step = den > 0x1p126f ? 0x1p-24f : 1.0f;
          const float over_m = token < n && den != 0.0f ? __builtin_amdgcn_rcpf(den * step) * step : -1.0f;
          const int token_m = token;
          token += more_tokens;
          in += more_in;
          if (in >= G) {
            in -= G;
            ++token;
          }
          if (b + share < blocks) load();
          float over[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) over[i] = __shfl(over_m, 4 * g + i);
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
          float w[4 * NG];
#pragma unroll
          for (int e = 0; e < 4 * NG; ++e) w[e] = CARRIED ? s4[e >> 2][e & 3] : s4[e >> 2][e & 3] * scale;
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4 * NG; ++e) w[e] = rho8_refined(w[e]);
          } else {
            float least = 0.0f;
#pragma unroll
            for (int e = 0; e < 4 * NG; ++e) least = __builtin_fminf(least, w[e]);
            // a score that is no number takes either form
            if (__ballot(!(least > kLowScore)) == 0) {
#pragma unroll
              for (int e = 0; e < 4 * NG; ++e) w[e] = rho8_fast(w[e]);
            } else {
              apart(w);
#pragma unroll
              for (int e = 0; e < 4 * NG; ++e) w[e] = rho8_by_score(w[e]);
            }
          }
          // every key of the tile is seen by these rows, which all give something, or each by its own
          const bool whole = kb + TILE <= (tree ? c : c + 1 + 16 * b / G) && __ballot(over_m == -1.0f) == 0;
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int who = __shfl(token_m, 4 * g + i);
              const int64_t* words = tree ? a.masks + (int64_t)(start + min(who, n - 1)) * W : nullptr;
#pragma unroll
              for (int u = 0; u < NG; ++u) {
                const int at = kb + 16 * u + m, j = at - c;
                bool sees = at < keys && over[i] != -1.0f;
                if (sees && j >= 0) sees = tree ? words[j >> 6] >> (j & 63) & 1 : j <= who;
                w[4 * u + i] = sees ? w[4 * u + i] : 0.0f;
              }
            }
          }
#pragma unroll
          for (int u = 0; u < NG; ++u) {
            float x = w[4 * u] * over[0];
#pragma unroll
            for (int i = 1; i < 4; ++i) x = __builtin_fmaf(w[4 * u + i], over[i], x);
            head[u] += x;
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
      float sum = 0.0f;
      if (tid < TILE) sum = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
      if (splits > 1) {
        float* part = f.part + (int64_t)tile * splits * TILE;
        if (tid < TILE) put1(part + split * TILE + tid, sum);
        if (!arrived(f.count + tile, splits, &flag)) continue;
        if (tid < TILE) {
          sum = 0.0f;
          for (int i0 = 0; i0 < splits; i0 += 8) {
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = get1(part + min(i0 + i, splits - 1) * TILE + tid);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += i0 + i < splits ? y[i] : 0.0f;
          }
        }
      }
      if (tid < TILE && pos < keys) *to = old + sum;
    }
    __syncthreads();  // first is free
  }
}

template <int DT, int D>
hipError_t weight_tiles_launch(const WeightFast& f, int cus, hipStream_t st) {
  hipLaunchKernelGGL((afa_paged_weight_tile_kernel<DT, D>), dim3((unsigned)(resident<DT, D>() * cus)), dim3(THREADS), 0, st, f);
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
    const int64_t counts = 2 * a.plan.kv_heads * 4 * cut.slots, room = (int64_t)(ws_bytes / (MOST_KEYS * 4));
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
