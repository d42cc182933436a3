// AFA of a serving step's tokens over the paged cache on the matrix cores (bf16, fp16, fp32; head_dim 32,
// 48, 64, 96, 128, 256; pages of a power of two, 8 tokens or more).
//
//   out_i = sum_j w_ij v_j / (sum_j w_ij + Omega),  w_ij = rho(q_i.k_j / sqrt(D))^8
//
// The few query rows of a request that share a key/value head (its new tokens times the heads of the
// group) meet every cached key once: the bytes of K and V bound the work.  A workgroup takes a slot of the
// plan (afa_paged.h): stretches of 32-key tiles of one head, of one segment after the other.  A wave needs no
// other until a segment's end:
//
//   S^T = K Q^T    A = 16 keys, B = 16 rows; a lane ends with 8 keys' scores of row lane % 16
//   w = rho^8      in place; they are the B operand of
//   O^T += V^T w   A = the feature columns of V, formed in registers
//
// The order of the keys within a tile is free, so K's rows are handed to the lanes such that the 8 scores
// of a lane belong to the 8 consecutive keys that it holds of V (16-bit types: keys 8g..8g+7 for lane
// group g = lane / 16).  Likewise feature d = EPL * row + j is row `row` of product j: a lane reads EPL
// consecutive features of 8 V rows, 16 lanes a whole row, and forms the columns by 4 byte permutes each.
// No cross-lane step is in the loop, and with up to 32 rows no LDS and no barrier: K of the next tile comes
// while a tile's weights are formed, V while the next scores are.  With 64 and 128 rows the four waves have 16
// or 32 rows each and share a ring of tiles in LDS, which direct loads fill up to three tiles ahead: a tile is
// loaded once for all, and the loads in flight cost no registers.
//
// The sums are additive: rows split over waves, and over workgroups where the plan cut the keys, are
// joined by adding numerators and denominators in a fixed order (LDS; fp32 parts that the last workgroup of a
// row block to finish adds up).
//
// Weights are the B operand in two planes of the type (w = hi + lo), so that what is left of their rounding is
// its square.  With few rows the second plane is free, as the matrix cores idle beside the loads; with 128 rows
// it is 16 of a tile's 48 products, and is kept all the same.  The row sums are fp32.  fp16 ends at 65504: there
// a row's weights are scaled by a power of two, lowered when a larger weight comes (kFirstScale).
//
// HBM bound where requests are many or long.  96 requests of one token over up to 4096 cached, 16 heads of 64,
// bf16: 160 us, 5.7 TB/s.  4 requests of 6 tokens over up to 131072, 16 query on 4 key heads of 128, fp16: 119 us,
// 4.7 TB/s, of which the parts take 5.  32 requests of up to 32 drafted tokens over up to 8192, 16 on 4 heads of
// 128, bf16 (128 rows): 94 us, 3.3 TB/s: MFMA and vector instructions one after the other (about 73), and the
// parts (about 10).  40 requests of up to 13 over 3001, 6 heads of 48, fp32: 38 us, 3.8 TB/s, the parts 7.  One token
// over 700, 12 heads of 64: 8 us, a chain of dependent reads (plan, table, keys, parts).
#include <type_traits>

#include "afa_common.h"
#include "afa_paged.h"

namespace afa {

namespace {

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

template <int DT>
__device__ __forceinline__ bool nonfinite(unsigned w) {
  if constexpr (DT == AFA_F32) return (w & 0x7f800000u) == 0x7f800000u;
  constexpr unsigned E = DT == AFA_BF16 ? 0x7f80u : 0x7c00u;
  return (w & E) == E || (w >> 16 & E) == E;
}

struct PagedFast {
  PagedFwdArgs a;
  float* part;                 // (kv_heads, 2 slots, rows, D) numerators
  float *part_den, *part_sum;  // (kv_heads, 2 slots, rows) row sums of the parts, and of their groups
  int64_t slots;
  int log_page, dim;
  uint32_t k_page, k_slot, v_page, v_slot;  // strides in bytes
};

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

// Sums of `n` parts in their order, part i at row base(i): of every row into `sums` (LDS), and of four features at a
// time, handed to put(row, feature, sums).  Up to 24 reads of a thread are in flight: they come from memory
// that all XCDs see, and one workgroup has several hundred KB to read where rows are many.
template <int THREADS, typename B, typename P>
__device__ __forceinline__ void sum_parts(__amdgpu_buffer_rsrc_t parts, const float* den, int n, int rows, int D, float* sums,
                                          const B& base, const P& put) {
  for (int row = threadIdx.x; row < rows; row += THREADS) {
    float x = 0.0f;
    for (int i0 = 0; i0 < n; i0 += 8) {
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = get1(den + base(min(i0 + i, n - 1)) + row);
#pragma unroll
      for (int i = 0; i < 8; ++i) x += i0 + i < n ? y[i] : 0.0f;
    }
    sums[row] = x;
  }
  __syncthreads();
  const int quads = D / 4, all = rows * quads;
  constexpr int U = 3, N = 8;
  for (int e0 = threadIdx.x; e0 < all; e0 += U * THREADS) {
    f32x4_t x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = f32x4_t{0, 0, 0, 0};
    for (int i0 = 0; i0 < n; i0 += N) {
      f32x4_t y[N][U];
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u)
          // past the last part or row: outside the resource, 0
          y[i][u] = get4(parts, i0 + i < n && e0 + u * THREADS < all
                                    ? (uint32_t)(base(i0 + i) * D * 4 + (int64_t)(e0 + u * THREADS) * 16)
                                    : 0xfffffff0u);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] += y[i][u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int e = e0 + u * THREADS, row = e / quads;
      if (e < all) put(row, 4 * (e - row * quads), x[u]);
    }
  }
}

// Parts are summed in groups, these by the last of each, and the groups by the last of them: one
// workgroup reads at most about 2 sqrt(parts).
__device__ __forceinline__ int group_size(int parts) {
  if (parts <= 8) return parts;
  const int s = (int)__builtin_sqrtf((float)parts);
  return s * s < parts ? s + 1 : s;
}

// Four waves of QB row blocks of 16 each: all along the keys, each with tiles of its own (RW = 1), two by two, or
// side by side (RW = 4).  Waves side by side meet the same keys; four of them share a ring of tiles in LDS,
// which direct loads fill ahead of them, two read the tile once each.
constexpr int WAVES = 4, THREADS = 64 * WAVES;

// Tiles of the ring: as many as leave room for the workgroups that the registers hold.
template <int DT, int DP>
constexpr int ring_tiles() {
  constexpr int bytes = 2 * kPagedTile * DP * (DT == AFA_F32 ? 4 : 2);
  return bytes <= 16384 || (DP == 256 && bytes <= 32768) ? 4 : 2;
}

// D features in products of 16 of 64, 128 or 256.
constexpr int padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

template <int DT, int D, int QB, int RW>
__global__ __launch_bounds__(THREADS, D == 256 ? 1 : 2) void afa_paged_tile_kernel(const PagedFast f) {
  constexpr int DP = padded(D);
  constexpr bool FULL = D == DP;
  constexpr int KW = WAVES / RW, NBUF = KW > 1 ? KW / 2 : 1;
  constexpr bool F32 = DT == AFA_F32;
  constexpr int ESZ = F32 ? 4 : 2;
  constexpr int EPL = DP / 16;            // features of V a lane, and products of O
  constexpr int VW = EPL * ESZ / 4;       // their 32-bit words
  constexpr int KB = F32 ? 16 : 32;       // features of a 16-byte chunk over the four lane groups
  constexpr int KS = (D + KB - 1) / KB;   // chunks of a K row a lane
  constexpr int GR = F32 ? 2 : 1;         // groups of 8 keys that a lane reads of K, and of V
  constexpr int ROWS = 16 * QB * RW, LD = DP + 4;
  // the ring, in rows of PITCH bytes whose 16-byte chunks are swizzled by swizzle(row), and the joined rows after it
  constexpr bool SHARED = RW == 4;
  constexpr int NST = SHARED ? ring_tiles<DT, DP>() : 1, PITCH = DP * ESZ, HALF = kPagedTile * PITCH, TILE = 2 * HALF;
  constexpr int NI = HALF / 1024 / WAVES;  // direct loads of a wave for K of a tile, and for V
  constexpr int RED = NBUF * ROWS * LD * 4, RING = SHARED ? NST * TILE : 0;
  __shared__ __attribute__((aligned(1024))) char smem[RED > RING ? RED : RING];
  float (*red)[ROWS][LD] = (float (*)[ROWS][LD])smem;
  __shared__ float red_den[KW][ROWS];
  __shared__ int red_odd[WAVES], flag;
  const PagedFwdArgs& a = f.a;
  const afa_paged_plan& p = a.plan;
  const int tid = threadIdx.x, lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), kw = wave / RW, rw = wave % RW;
  const int H = (int)p.heads, G = a.group, W = (int)(p.max_tree / 64), lp = f.log_page, in_page = (1 << lp) - 1;
  const float scale = (float)a.scale;
  // heads run fastest: with 8 key heads the row blocks of one meet its keys in the same XCD's L2
  const int slot = (int)(blockIdx.x / (unsigned)p.kv_heads), hk = (int)(blockIdx.x - (unsigned)slot * (unsigned)p.kv_heads);
  // a row's four features d.. from its sums
  auto store4 = [&](int64_t at, int d, f32x4_t x, float sum) {
    const float all = sum + (float)a.omega;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = all == 0.0f ? 0.0f : x[i] / all;
    if constexpr (F32) {
      *(f32x4_t*)((float*)a.out + at * D + d) = x;
    } else {
      u32x2_t y = {Elem<DT>::pack(x[0], x[1]), Elem<DT>::pack(x[2], x[3])};
      *(u32x2_t*)((unsigned short*)a.out + at * D + d) = y;
    }
    if (d == 0 && a.denom != nullptr) ((float*)a.denom)[at] = all;
  };

  const bool busy = slot < a.sched.header->slots;
  const PagedSlot begin = a.sched.slot[busy ? slot : 0];
  const int64_t stretch = a.sched.header->stretch;
  int64_t pos = slot * stretch;
  const int64_t stop = busy ? min(pos + stretch, a.sched.header->end) : pos;
  int live = begin.live, block = begin.block, unit = begin.at;
  while (pos < stop) {
    const PagedLive q = a.sched.live[live];
    const int c = q.cached, n = q.fresh, keys = c + n, nrows = n * G, row0 = block * ROWS;
    const bool tree = a.masks != nullptr && n <= p.max_tree;
    const int take = (int)min((int64_t)(q.cost - unit), stop - pos);
    const int tiles = paged_block_tiles(c, n, tree, block, ROWS, G);
    const int tile0 = max(unit - kPagedLead, 0), tile1 = min(unit + take - kPagedLead, tiles);
    // the slots that hold keys of this segment
    const int64_t key0 = pos - unit + kPagedLead;
    const int from_slot = (int)(key0 / stretch), parts = (int)((key0 + tiles - 1) / stretch) - from_slot + 1;
    pos += take;
    unit += take;
    if (unit == q.cost) {
      unit = 0;
      if (++block == q.blocks) {
        block = 0;
        ++live;
      }
    }
    if (tile0 >= tile1) continue;
    const int32_t* table = p.block_tables + (int64_t)q.request * p.table_width;
    const char* k_base = (const char*)a.k_pages + hk * a.ps.k_head * ESZ;
    const char* v_base = (const char*)a.v_pages + hk * a.ps.v_head * ESZ;
    const int per = (tile1 - tile0 + KW - 1) / KW;
    // a wave without rows has no keys
    const bool rows_here = row0 + 16 * rw < nrows, both = QB == 2 && row0 + 16 * (RW + rw) < nrows;
    const int t0 = tile0 + kw * per, t1 = rows_here || SHARED ? min(t0 + per, tile1) : t0;

    // 64 entries of the table, one a lane, from the page of the wave's first tile on
    int entry0 = 0, entry = 0;
    auto load_entries = [&](int t) {
      entry0 = (t * kPagedTile) >> lp;
      entry = table[min(entry0 + lane, (keys - 1) >> lp)];
      if ((unsigned)entry >= (unsigned)p.num_pages) entry = -1;
    };
    // Where a lane's K and V rows of a tile lie: groups of 8 consecutive keys, each within a page.  lost: the
    // V group's page is none of the pool's.
    const char *kp[GR], *vp[GR];
    bool lost[GR], lost_next[GR];
    auto locate = [&](int t) {
      const int kb = t * kPagedTile;
      if (((kb + kPagedTile - 1) >> lp) - entry0 > 63) load_entries(t);
      if (lp >= 5) {  // the tile lies within one page
        const int page = __builtin_amdgcn_readlane(entry, (kb >> lp) - entry0), at = max(page, 0);
        const char* k = k_base + ((uint64_t)(uint32_t)at * f.k_page + (uint32_t)(kb & in_page) * f.k_slot);
        const char* v = v_base + ((uint64_t)(uint32_t)at * f.v_page + (uint32_t)(kb & in_page) * f.v_slot);
#pragma unroll
        for (int u = 0; u < GR; ++u) {
          lost_next[u] = page < 0;
          kp[u] = k + ((F32 ? 16 * u + m : 8 * (m >> 2) + (m & 3)) * f.k_slot + 16 * g);
          vp[u] = v + ((F32 ? 16 * u + 4 * g : 8 * g) * f.v_slot + EPL * ESZ * m);
        }
        return;
      }
#pragma unroll
      for (int u = 0; u < GR; ++u) {
        const int kpos = kb + (F32 ? 16 * u + m : 8 * (m >> 2) + (m & 3)), vpos = kb + (F32 ? 16 * u + 4 * g : 8 * g);
        const int kpage = __shfl(entry, (min(kpos, keys - 1) >> lp) - entry0);
        const int vpage = __shfl(entry, (min(vpos, keys - 1) >> lp) - entry0);
        lost_next[u] = vpage < 0;
        kp[u] = k_base + (uint64_t)(uint32_t)max(kpage, 0) * f.k_page + ((uint32_t)(kpos & in_page) * f.k_slot + 16 * g);
        vp[u] = v_base + (uint64_t)(uint32_t)max(vpage, 0) * f.v_page +
                ((uint32_t)(vpos & in_page) * f.v_slot + EPL * ESZ * m);
      }
    };
    // eight rows that a ds_read_b128 touches at once take eight different chunks of a bank cycle
    auto swizzle = [](int row) { return F32 ? row & 7 : (row & 3) | (row >> 1 & 4); };
    unsigned lost_ring = 0;
    // a wave's share of a tile into the ring: its rows' chunks, lane by lane
    auto stage = [&](int t) {
      const int kb = t * kPagedTile, st = t & (NST - 1);
      if (((kb + kPagedTile - 1) >> lp) - entry0 > 63) load_entries(t);
      char* to = smem + st * TILE;
      if (lp >= 5) {
        const int page = __builtin_amdgcn_readlane(entry, (kb >> lp) - entry0), from = max(page, 0);
        const char* k = k_base + ((uint64_t)(uint32_t)from * f.k_page + (uint32_t)(kb & in_page) * f.k_slot);
        const char* v = v_base + ((uint64_t)(uint32_t)from * f.v_page + (uint32_t)(kb & in_page) * f.v_slot);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int at = (wave * NI + i) * 1024, row = (at + 16 * lane) / PITCH;
          const int chunk = ((at + 16 * lane) % PITCH / 16) ^ swizzle(row);
          if (FULL || chunk * 16 < D * ESZ) {
            lds_dma16(k, row * f.k_slot + 16 * chunk, to + at);
            lds_dma16(v, row * f.v_slot + 16 * chunk, to + HALF + at);
          }
        }
        lost_ring = (lost_ring & ~(3u << 2 * st)) | (page < 0 ? 3u : 0u) << 2 * st;
        return;
      }
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const int at = (wave * NI + i) * 1024, row = (at + 16 * lane) / PITCH;
        const int chunk = ((at + 16 * lane) % PITCH / 16) ^ swizzle(row);
        const int page = max(__shfl(entry, (min(kb + row, keys - 1) >> lp) - entry0), 0);
        const uint32_t in = (uint32_t)((kb + row) & in_page);
        if (FULL || chunk * 16 < D * ESZ) {
          lds_dma16(k_base + (uint64_t)(uint32_t)page * f.k_page + (in * f.k_slot + 16 * chunk), to + at);
          lds_dma16(v_base + (uint64_t)(uint32_t)page * f.v_page + (in * f.v_slot + 16 * chunk), to + HALF + at);
        }
      }
      unsigned gone = 0;
#pragma unroll
      for (int u = 0; u < GR; ++u) {
        const int vpos = kb + (F32 ? 16 * u + 4 * g : 8 * g);
        gone |= (__shfl(entry, (min(vpos, keys - 1) >> lp) - entry0) < 0 ? 1u : 0u) << u;
      }
      lost_ring = (lost_ring & ~(3u << 2 * st)) | gone << 2 * st;
    };
    u32x4_t kf[2][KS];
    unsigned vf[8][VW];
    auto read_k = [&](int st) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int row = F32 ? 16 * u + m : 8 * (m >> 2) + (m & 3) + 4 * u;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          const int chunk = 4 * ks + g;
          kf[u][ks] = *(const u32x4_t*)(smem + st * TILE + row * PITCH + (chunk ^ swizzle(row)) * 16);
          if (!FULL && KB * ks + 16 / ESZ * g >= D) kf[u][ks] = u32x4_t{0, 0, 0, 0};
        }
      }
    };
    auto read_v = [&](int st) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = F32 ? 16 * (i >> 2) + 4 * g + (i & 3) : 8 * g + i;
        const char* r = smem + st * TILE + HALF + row * PITCH;
        if constexpr (VW == 2) {
          const u32x2_t x = *(const u32x2_t*)(r + ((m >> 1) ^ swizzle(row)) * 16 + 8 * (m & 1));
          const bool in = FULL || EPL * m < D;  // nothing is staged behind the row
          vf[i][0] = in ? x[0] : 0;
          vf[i][1] = in ? x[1] : 0;
        } else {
#pragma unroll
          for (int q4 = 0; q4 < VW / 4; ++q4) {
            const u32x4_t x = *(const u32x4_t*)(r + ((VW / 4 * m + q4) ^ swizzle(row)) * 16);
            const bool in = FULL || EPL * m + 16 / ESZ * q4 < D;
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[i][4 * q4 + e] = in ? x[e] : 0;
          }
        }
      }
    };
    auto load_k = [&]() {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const char* r = F32 ? kp[F32 ? u : 0] : kp[0] + 4 * u * f.k_slot;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          kf[u][ks] = FULL || KB * ks + 16 / ESZ * g < D ? *(const u32x4_t*)(r + KB * ks * ESZ) : u32x4_t{0, 0, 0, 0};
      }
    };
    auto load_v = [&]() {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const char* r = F32 ? vp[F32 ? i >> 2 : 0] + (i & 3) * f.v_slot : vp[0] + i * f.v_slot;
        if constexpr (VW == 2) {
          u32x2_t x = {0, 0};
          if (FULL || EPL * m < D) x = *(const u32x2_t*)r;
          vf[i][0] = x[0];
          vf[i][1] = x[1];
        } else {
#pragma unroll
          for (int q4 = 0; q4 < VW / 4; ++q4) {
            u32x4_t x = {0, 0, 0, 0};
            if (FULL || EPL * m + 16 / ESZ * q4 < D) x = *(const u32x4_t*)(r + 16 * q4);
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[i][4 * q4 + e] = x[e];
          }
        }
      }
    };
    if constexpr (SHARED) {
      load_entries(t0);
    } else if (t0 < t1) {
      load_entries(t0);
      locate(t0);
      load_k();
      load_v();
    }

    // the rows of Q: chunk ks of a lane holds features KB ks + (16 / ESZ) g ..
    u32x4_t qf[QB][KS];
    int token[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      const int row = min(row0 + 16 * (b * RW + rw) + m, nrows - 1);
      token[b] = row / G;
      const char* x = (const char*)a.q + ((int64_t)(q.start + token[b]) * a.q_t + (hk * G + row - token[b] * G) * a.q_h) * ESZ;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = KB * ks + 16 / ESZ * g;
        qf[b][ks] = FULL || d < D ? *(const u32x4_t*)(x + d * ESZ) : u32x4_t{0, 0, 0, 0};
      }
    }

    if constexpr (SHARED) {
      // Q is here before the ring's first loads.  The compiler does not count those, so that a wait for Q
      // in the loop would be one for every load of the ring, each time:
      // 105 us for 95 with trees of up to 32 over up to 8192 keys, 80 for 69 with 64 rows over 8192.
#pragma unroll
      for (int b = 0; b < QB; ++b)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[b][ks]));
      __syncthreads();  // smem is free of the segment before
#pragma unroll
      for (int i = 0; i < NST - 1; ++i)
        if (t0 + i < t1) stage(t0 + i);
    }

    f32x4_t acc[QB][EPL];
    float den[QB], sc[QB];
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      den[b] = 0.0f;
      sc[b] = kFirstScale;
#pragma unroll
      for (int j = 0; j < EPL; ++j) acc[b][j] = f32x4_t{0, 0, 0, 0};
    }
    bool any_odd = false;

    // the wave's tiles for its first NB row blocks
    auto meet = [&](auto blocks) {
      constexpr int NB = decltype(blocks)::value;
      for (int t = t0; t < t1; ++t) {
        if constexpr (SHARED) {
          // this wave's loads of tile t are done, those of up to NST - 2 later ones may go on; then every wave's,
          // and every wave has read tile t - 1, whose place the next one takes
          const int later = min(NST - 2, t1 - 1 - t);
          if (later == 2) __builtin_amdgcn_s_waitcnt(vmcnt_only(4 * NI));
          else if (later == 1) __builtin_amdgcn_s_waitcnt(vmcnt_only(2 * NI));
          else __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          if (t + NST - 1 < t1) stage(t + NST - 1);
          if (!rows_here) continue;
          const int st = t & (NST - 1);
#pragma unroll
          for (int u = 0; u < GR; ++u) lost[u] = lost_ring >> (2 * st + u) & 1;
          read_k(st);
          read_v(st);
        } else {
#pragma unroll
          for (int u = 0; u < GR; ++u) lost[u] = lost_next[u];
        }
        const int kb = t * kPagedTile;
        // scores of row m of row block b: element e is key 8 g + e (fp32: 16 (e / 4) + 4 g + e % 4)
        f32x4_t s4[NB][2];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            s4[b][u] = f32x4_t{0, 0, 0, 0};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
              if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const unsigned x = kf[u][ks][e], y = qf[b][ks][e];
                  s4[b][u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y),
                                                                  s4[b][u], 0, 0, 0);
                }
              } else {
                s4[b][u] = mma16<DT>(kf[u][ks], qf[b][ks], s4[b][u]);
              }
            }
          }
        // K of the next tile comes while this one's weights are formed, V while the next one's scores are
        const bool more = t + 1 < t1;
        if constexpr (!SHARED) {
          __builtin_amdgcn_sched_barrier(0);
          if (more) {
            locate(t + 1);
            load_k();
          }
          __builtin_amdgcn_sched_barrier(0);
        }

        // Tiles with drafted keys, keys behind the last or lost pages: rows past the end are cleared, and
        // drafted values that are not finite are taken out of the product, in which a weight of 0 would
        // not hide them; the rows that see them get them at the end.
        bool any_lost = lost[0];
        if constexpr (F32) any_lost = any_lost || lost[GR - 1];
        const bool masked = kb + kPagedTile > c || __ballot(any_lost) != 0;
        if (masked) {
          bool odd = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int pos = kb + (F32 ? 16 * (i >> 2) + 4 * g + (i & 3) : 8 * g + i);
            const bool gone = pos >= keys || lost[F32 ? i >> 2 : 0];
#pragma unroll
            for (int e = 0; e < VW; ++e) {
              unsigned x = gone ? 0u : vf[i][e];
              if (pos >= c && nonfinite<DT>(x)) {
                odd = true;
                if constexpr (F32) {
                  x = 0;
                } else {
                  constexpr unsigned E = DT == AFA_BF16 ? 0x7f80u : 0x7c00u;
                  x &= ((x & E) == E ? 0xffff0000u : ~0u) & ((x >> 16 & E) == E ? 0xffffu : ~0u);
                }
              }
              vf[i][e] = x;
            }
          }
          any_odd = any_odd || __ballot(odd) != 0;
        }

        // Weights, in place of the scores in fp32, as planes otherwise.
        u32x4_t hi[F32 ? 1 : NB], lo[F32 ? 1 : NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          float w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) w[e] = s4[b][e >> 2][e & 3] * scale;
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = rho8_refined(w[e]);
          } else {
            // where no score is low all lanes take the branch-free form, which gives such scores the same bits
            float least = w[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) least = __builtin_fminf(least, w[e]);
            if (__ballot(!(least > kLowScore)) == 0) {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = rho8_fast(w[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] = rho8_by_score(w[e]);
            }
          }
          if (masked) {
            const int64_t* words = tree ? a.masks + (int64_t)(q.start + token[b]) * W : nullptr;
            unsigned sees;
            if constexpr (F32) {
              sees = sees_bits(kb - c + 4 * g, 4, n, token[b], words, W) |
                     sees_bits(kb - c + 16 + 4 * g, 4, n, token[b], words, W) << 4;
              if (lost[0]) sees &= 0xf0;
              if (lost[GR - 1]) sees &= 0x0f;
            } else {
              sees = lost[0] ? 0 : sees_bits(kb - c + 8 * g, 8, n, token[b], words, W);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = sees >> e & 1 ? w[e] : 0.0f;
          }
          den[b] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s4[b][e >> 2][e & 3] = w[e];
          } else {
            if constexpr (DT == AFA_F16) {
              float top = w[0];
#pragma unroll
              for (int e = 1; e < 8; ++e) top = __builtin_fmaxf(top, w[e]);
              if (__ballot(!(top * sc[b] <= 32768.0f)) != 0) {
                // a row's largest weight so far now lies in [16, 32)
                top = __builtin_fmaxf(top, __shfl_xor(top, 16));
                top = __builtin_fmaxf(top, __shfl_xor(top, 32));
                if (top * sc[b] > 32768.0f && top < __builtin_inff()) {
                  const int e = (__builtin_bit_cast(int, top) >> 23) - 127;
                  const float to = __builtin_bit_cast(float, (127 + 4 - e) << 23);
                  const float ratio = to / sc[b];
                  sc[b] = to;
#pragma unroll
                  for (int j = 0; j < EPL; ++j) acc[b][j] *= ratio;
                }
              }
#pragma unroll
              for (int e = 0; e < 8; ++e) w[e] *= sc[b];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const unsigned x = Elem<DT>::pack(w[2 * e], w[2 * e + 1]);
              hi[b][e] = x;
              lo[b][e] = Elem<DT>::pack(w[2 * e] - Elem<DT>::lo(x), w[2 * e + 1] - Elem<DT>::hi(x));
            }
          }
        }

        // a wave with products ready goes before one that forms weights (trees: 94 us for 96)
        if constexpr (SHARED) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int j = 0; j < EPL; ++j) {
          if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const unsigned x = vf[e][j];
              const float v = __builtin_bit_cast(float, x);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                acc[b][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, s4[b][e >> 2][e & 3], acc[b][j], 0, 0, 0);
            }
          } else {
            u32x4_t v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[e] = __builtin_amdgcn_perm(vf[2 * e + 1][j >> 1], vf[2 * e][j >> 1], j & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][j] = mma16<DT>(v, hi[b], acc[b][j]);
#pragma unroll
            for (int b = 0; b < NB; ++b) acc[b][j] = mma16<DT>(v, lo[b], acc[b][j]);
          }
        }
        if constexpr (SHARED) __builtin_amdgcn_s_setprio(0);
        if constexpr (!SHARED) {
          __builtin_amdgcn_sched_barrier(0);
          if (more) load_v();
        }
      }
    };
    if (both) meet(std::integral_constant<int, QB>());
    else meet(std::integral_constant<int, 1>());

    // join the waves along the keys: the first half stores, the second adds to theirs
    __syncthreads();  // red is free of the item before
    if (lane == 0) red_odd[wave] = any_odd;
#pragma unroll
    for (int b = 0; b < QB; ++b) {
      den[b] += __shfl_xor(den[b], 16);
      den[b] += __shfl_xor(den[b], 32);
      if (g == 0) red_den[kw][16 * (b * RW + rw) + m] = den[b];
      if constexpr (DT == AFA_F16) {
        const float by = sc[b];  // a power of two
        const float back = __builtin_bit_cast(float, (254 << 23) - __builtin_bit_cast(int, by));
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[b][j] *= back;
      }
    }
#pragma unroll
    for (int half = 0; half < KW / NBUF; ++half) {
      if (kw / NBUF == half) {
#pragma unroll
        for (int b = 0; b < QB; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < EPL; j += 4) {
              f32x4_t* to = (f32x4_t*)&red[kw % NBUF][16 * (b * RW + rw) + m][EPL * (4 * g + i) + j];
              f32x4_t x = {acc[b][j][i], acc[b][j + 1][i], acc[b][j + 2][i], acc[b][j + 3][i]};
              *to = half ? *to + x : x;
            }
      }
      __syncthreads();
    }
    auto out_row = [&](int row) {
      const int who = (row0 + row) / G;
      return (int64_t)(q.start + who) * H + hk * G + (row0 + row - who * G);
    };
    bool odd = false;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) odd = odd || red_odd[w] != 0;
    const int mine = min(ROWS, nrows - row0), quads = D / 4;
    // part i of this segment: a slot's second where it begins there, else its first
    auto part_of = [&](int i) { return (int64_t)2 * (from_slot + i) + (i == 0); };
    const int64_t head0 = (int64_t)hk * 2 * f.slots * ROWS;
    float *part_den = f.part_den + head0, *part_sum = f.part_sum + head0;
    const __amdgpu_buffer_rsrc_t buffer =
        __builtin_amdgcn_make_buffer_rsrc(f.part + head0 * D, 0, (int)(2 * f.slots * ROWS * D * 4), 0x00020000);
    const int64_t my_part = part_of(slot - from_slot);
    f32x4_t zero = {0, 0, 0, 0};  // NaN where a sum is not finite
    auto hand_on = [&](auto again) {
      for (int e = tid; e < mine * quads; e += THREADS) {
        const int row = e / quads, d = 4 * (e - row * quads);
        f32x4_t x = *(const f32x4_t*)&red[0][row][d];
        float sum = red_den[0][row];
#pragma unroll
        for (int w = 1; w < NBUF; ++w) x += *(const f32x4_t*)&red[w][row][d];
#pragma unroll
        for (int w = 1; w < KW; ++w) sum += red_den[w][row];
        if constexpr (decltype(again)::value) {
          const int who = (row0 + row) / G;
          const int64_t* words = a.masks + (int64_t)(q.start + who) * W;
          f32x4_t y = {0, 0, 0, 0};
          for (int pos = tile0 * kPagedTile; pos < min(tile1 * kPagedTile, keys); ++pos) {
            const bool sees = pos < c || (tree ? words[(pos - c) >> 6] >> ((pos - c) & 63) & 1 : pos - c <= who);
            const int page = table[pos >> lp];
            if (!sees || (unsigned)page >= (unsigned)p.num_pages) continue;
            const char* v = v_base + (uint64_t)(uint32_t)page * f.v_page + (uint32_t)(pos & in_page) * f.v_slot;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float z = Elem<DT>::load(v, d + i);
              if (!(__builtin_fabsf(z) < __builtin_inff())) y[i] += z;
            }
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!(__builtin_fabsf(y[i]) < __builtin_inff())) x[i] = y[i];
        } else if constexpr (!F32) {
#pragma unroll
          for (int i = 0; i < 4; ++i) zero[i] = __builtin_fmaf(x[i], 0.0f, zero[i]);
        }
        if (parts > 1) {
          put4(buffer, (uint32_t)((my_part * ROWS + row) * D + d) * 4, x);
          if (d == 0) put1(part_den + my_part * ROWS + row, sum);
        } else {
          store4(out_row(row), d, x, sum);
        }
      }
    };
    hand_on(std::false_type());
    // A value that is not finite is the sum of every row that sees it, as weights are above 0.  Drafted ones were taken
    // out of the products; a cached one may have become NaN there, since a weight's second plane may be 0 or
    // negative.  Such sums are formed again, from these values alone.
    if (odd || (zero[0] + zero[1]) + (zero[2] + zero[3]) != 0.0f) hand_on(std::true_type());
    if (parts == 1) continue;

    const int size = group_size(parts), groups = (parts + size - 1) / size, g0 = (slot - from_slot) / size * size;
    const int here = min(size, parts - g0);
    int* count = a.sched.count + (int64_t)hk * 4 * f.slots;
    if (!arrived(count + part_of(g0), here, &flag)) continue;
    const int64_t to = part_of(g0) * ROWS;
    sum_parts<THREADS>(buffer, part_den, here, mine, D, red_den[0], [&](int i) { return part_of(g0 + i) * ROWS; },
                       [&](int row, int d, f32x4_t x) {
                         if (groups == 1) {
                           store4(out_row(row), d, x, red_den[0][row]);
                         } else {
                           // over the group's first part, of which this thread alone reads these features
                           put4(buffer, (uint32_t)((to + row) * D + d) * 4, x);
                           if (d == 0) put1(part_sum + to + row, red_den[0][row]);
                         }
                       });
    if (groups == 1 || !arrived(count + 2 * f.slots + part_of(0), groups, &flag)) continue;
    sum_parts<THREADS>(buffer, part_sum, groups, mine, D, red_den[0], [&](int i) { return part_of(i * size) * ROWS; },
                       [&](int row, int d, f32x4_t x) { store4(out_row(row), d, x, red_den[0][row]); });
  }

  // The rows that no segment has: those of requests that were not served, and those behind the last
  // request's where they are asked for.  A lane looks at a token, its wave writes the row.
  const int64_t waves = (int64_t)gridDim.x * WAVES, me = (int64_t)blockIdx.x * WAVES + wave;
  for (int64_t t0 = me; t0 < p.max_tokens; t0 += 64 * waves) {
    const int64_t t = t0 + lane * waves;
    int r = -1;
    bool dead = false;
    if (t < p.max_tokens) {
      r = p.token_request[t];
      dead = r < 0 ? a.zero_tail != 0 : p.status[r] != AFA_PAGED_OK;
    }
    for (u64 left = __ballot(dead); left != 0; left &= left - 1) {
      const int which = __ffsll(left) - 1;
      const int64_t row = (t0 + which * waves) * H;
      const float all = __shfl(r, which) < 0 ? 0.0f : (float)a.omega;
      for (int64_t e = lane; e < (int64_t)H * D; e += 64) Elem<DT>::store(a.out, row * D + e, 0.0f);
      if (a.denom != nullptr)
        for (int h = lane; h < H; h += 64) ((float*)a.denom)[row + h] = all;
    }
  }
}

template <int DT, int D, int QB, int RW>
hipError_t tile_launch(const PagedFast& f, hipStream_t st) {
  hipLaunchKernelGGL((afa_paged_tile_kernel<DT, D, QB, RW>), dim3((unsigned)(f.slots * f.a.plan.kv_heads)), dim3(THREADS), 0,
                     st, f);
  return hipGetLastError();
}

template <int DT, int D>
hipError_t tile_go(const PagedFast& f, int rows, hipStream_t st) {
  constexpr int ROW = D * (DT == AFA_F32 ? 4 : 2);
  if (rows == 16) return tile_launch<DT, D, 1, 1>(f, st);
  // 32 rows: a wave's own where two row blocks fit its registers, else two waves that meet the same keys
  if (rows == 32) return tile_launch<DT, D, ROW <= 128 ? 2 : 1, ROW <= 128 ? 1 : 2>(f, st);
  if (rows == 64) return tile_launch<DT, D, 1, 4>(f, st);
  if constexpr (ROW <= 256) return tile_launch<DT, D, 2, 4>(f, st);
  return hipErrorInvalidValue;  // no plan has more than 64 rows of these
}

template <int DT>
hipError_t fast_go(const PagedFast& f, int rows, hipStream_t st) {
  switch (f.dim) {
    case 32: return tile_go<DT, 32>(f, rows, st);
    case 48: return tile_go<DT, 48>(f, rows, st);
    case 64: return tile_go<DT, 64>(f, rows, st);
    case 96: return tile_go<DT, 96>(f, rows, st);
    case 128: return tile_go<DT, 128>(f, rows, st);
    default: return tile_go<DT, 256>(f, rows, st);
  }
}

}  // namespace

bool paged_fast_supported(const afa_paged_plan& p) {
  const int64_t d = p.head_dim;
  return p.dtype != AFA_F64 && (d == 32 || d == 48 || d == 64 || d == 96 || d == 128 || d == 256) && p.page_size >= 8 &&
         (p.page_size & (p.page_size - 1)) == 0;
}

size_t paged_fast_workspace(const afa_paged_plan& p, const PagedCut& c) {
  return (size_t)(p.kv_heads * 2 * c.slots * c.rows) * (size_t)(p.head_dim + 2) * 4;
}

hipError_t paged_fwd_fast_launch(const PagedFwdArgs& a, const PagedCut& c, void* ws, hipStream_t st) {
  PagedFast f;
  f.a = a;
  f.part = (float*)ws;
  f.part_den = f.part + a.plan.kv_heads * 2 * c.slots * c.rows * a.plan.head_dim;
  f.part_sum = f.part_den + a.plan.kv_heads * 2 * c.slots * c.rows;
  f.slots = c.slots;
  f.dim = (int)a.plan.head_dim;
  const uint32_t esz = a.plan.dtype == AFA_F32 ? 4 : 2;
  f.k_page = (uint32_t)a.ps.k_page * esz;
  f.k_slot = (uint32_t)a.ps.k_slot * esz;
  f.v_page = (uint32_t)a.ps.v_page * esz;
  f.v_slot = (uint32_t)a.ps.v_slot * esz;
  f.log_page = __builtin_ctzll((unsigned long long)a.plan.page_size);
  switch ((int)a.plan.dtype) {
    case AFA_F32: return fast_go<AFA_F32>(f, c.rows, st);
    case AFA_BF16: return fast_go<AFA_BF16>(f, c.rows, st);
    default: return fast_go<AFA_F16>(f, c.rows, st);
  }
}

}  // namespace afa
