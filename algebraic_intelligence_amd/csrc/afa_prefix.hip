// A prefix that all requests share, met once by the rows of all the step's tokens: sum_j w_ij v_j and sum_j w_ij over its
// keys in fp32, for the attention of the requests' own keys to start from.  The sums are additive, so that nothing else
// passes between the two launches.
//
// Up to 64 rows a key head, fp32, and head_dim 256 run on the paged kernel (afa_paged_attend.h, PREFIX).  More rows of bf16
// and fp16 are a product of matrices, which the kernel below is for: four waves of 32 rows each share a ring of four tiles of
// 32 keys in LDS, filled by direct loads three tiles ahead.
//
//   S^T = K Q^T    32 keys x 32 rows; a lane ends with 16 keys' scores of row lane % 32
//   w = rho^8      in place, the B operand of
//   O^T += V^T w   V's columns by transposing LDS reads, in the order of keys that S^T leaves
//
// While a wave forms the weights of a tile, the scores of the next one are on the matrix cores, and the other wave of its
// SIMD has its products there.  Weights enter the product rounded to the type, as in the training forward: vector and matrix
// instructions bound this kernel, and the second plane that the paged kernel keeps would be a third of its products and a
// sixth of its vector instructions.  The rounding is as large as the result's own in bf16, and in fp16 for weights of 2^-18 of the row's
// largest and more.  Smaller ones are off by up to 2^-29 of the largest each: of very many keys far below one that is 2^-11, as the
// result's own rounding, for 2^18 keys, and grows with them.  Row sums are of the weights in fp32.
// The line of a key head's tiles over all row blocks is cut into even stretches, one for each resident workgroup.  What a cut
// leaves of a row block is added up by a launch of its own, which has all of the device for it: the last workgroup of a row block
// alone takes longer (84 us in all for 40 and 7, 256 rows of 4 heads behind 8192), and so does the own keys' launch (16 us more).
//
// 32 requests of up to 32 tokens, 16 heads on 4 of 128 in fp16, behind 30001 tokens: 340 us, 65 of them for the own keys and 12 for the
// parts, so 0.8 PFLOP/s; matrix instructions take 34% of the SIMDs' cycles and vector ones 51%, an eighth of them at once.  The
// paged kernel takes 435 us for the prefix alone.  256 requests of one token behind 8192: 41 us and 10, a third of it parts.
#include "afa_paged_attend.h"

namespace afa {

namespace {

typedef __attribute__((ext_vector_type(4))) short s16x4_t;
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;

template <int DT>
__device__ __forceinline__ f32x16_t mma32(u32x4_t a, u32x4_t b, f32x16_t c) {
  if constexpr (DT == AFA_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0,
                                                   0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

constexpr int WIDE_ROWS = 32 * WAVES, RING = 4;
// kFirstScale's eighth root and logarithm
constexpr float kFirstRoot = 0x1p15f;
constexpr int kFirstPower = 120;

// 2^(p / 8)
__device__ __forceinline__ float eighth_root_of_2(int p) {
  const float half = p & 4 ? 1.41421356f : 1.0f, quarter = p & 2 ? 1.18920712f : 1.0f, eighth = p & 1 ? 1.09050773f : 1.0f;
  return __builtin_bit_cast(float, (127 + (p >> 3)) << 23) * (half * (quarter * eighth));
}

// Parts of a row block that the join adds up; of more, groups are added up first, each by its last workgroup.
constexpr int WIDE_PARTS = 16;
__host__ __device__ inline int wide_group(int parts) { return (parts + WIDE_PARTS - 1) / WIDE_PARTS; }
// The length of a slot's stretch of a key head's line.
__device__ __forceinline__ int64_t wide_stretch(int nrows, int cost, int64_t slots) {
  const int64_t end = (int64_t)((nrows + WIDE_ROWS - 1) / WIDE_ROWS) * cost;
  return max((end + slots - 1) / slots, (int64_t)kPagedMin);
}

template <int DT, int D>
__global__ __launch_bounds__(THREADS, 2) void afa_prefix_wide_kernel(const PagedFast f) {
  constexpr int DP = D <= 64 ? 64 : 128;
  constexpr int CH = DP / 8, CHD = D / 8;          // 16-byte chunks of a row in LDS, and of data
  constexpr int LPT = kPagedTile * CH / THREADS;   // direct loads of a thread for K of a tile, and for V
  constexpr int LOADS = 2 * LPT;
  constexpr int NK = DP / 16, NDB = DP / 32;
  __shared__ __attribute__((aligned(1024))) unsigned short lds_k[RING][kPagedTile * DP], lds_v[RING][kPagedTile * DP];
  __shared__ float sums[WIDE_ROWS];
  __shared__ int flag;
  const PagedFwdArgs& a = f.a;
  const afa_paged_plan& p = a.plan;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, g = lane >> 5, l16 = lane & 15, m16 = lane >> 4 & 1;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int G = a.group, L = a.prefix.len;
  // With y = c s, (c rho(s))^8 = (y + sqrt(y^2 + c^2))^8: a factor of the weights costs nothing where the scores carry its eighth
  // root.  In bf16 q carries 1/8, exactly, so that y is what the products give and c^2 = D / 64; 1/16 where that would be above 1
  // and weights would leave fp32 before the formula's do, by c^8 = 16 for D = 128 (scores from 23000 on).  In fp16, where small
  // numbers would lose digits, y = kappa q.k, and kappa takes the eighth root of the power of two by which a row's weights are
  // scaled too: off by up to 2^-22, which is 2^-19 of a part's weights.
  constexpr bool F16 = DT == AFA_F16;
  constexpr float CARRIED = F16 || D <= 64 ? 0.125f : 0.0625f;
  constexpr float C2 = (float)D * CARRIED * CARRIED;
  constexpr float LOW = kLowScore * 8 * CARRIED *
                        (D == 32 ? 0.70710678f : D == 48 ? 0.8660254f : D == 64 ? 1.0f : D == 96 ? 1.2247449f : 1.4142136f);
  // heads run fastest: with 8 key heads the row blocks of one meet its keys in the same XCD's L2
  const int slot = (int)(blockIdx.x / (unsigned)p.kv_heads), hk = (int)(blockIdx.x - (unsigned)slot * (unsigned)p.kv_heads);
  const char* k_base = (const char*)a.prefix.k + hk * a.prefix.k_head * 2;
  const char* v_base = (const char*)a.prefix.v + hk * a.prefix.v_head * 2;
  const int nrows = p.starts[p.requests] * G, tiles = (L + kPagedTile - 1) / kPagedTile, cost = kPagedLead + tiles;
  const int64_t end = (int64_t)((nrows + WIDE_ROWS - 1) / WIDE_ROWS) * cost;
  const int64_t stretch = wide_stretch(nrows, cost, f.slots);
  int64_t pos = slot * stretch;
  const int64_t stop = min(pos + stretch, end);
  int block = (int)(pos / cost), unit0 = (int)(pos - (int64_t)block * cost);
  const int64_t head0 = (int64_t)hk * 2 * f.slots * WIDE_ROWS;
  float *part_den = f.part_den + head0, *part_sum = f.part_sum + head0;
  const __amdgpu_buffer_rsrc_t buffer =
      __builtin_amdgcn_make_buffer_rsrc(f.part + head0 * D, 0, (int)(2 * f.slots * WIDE_ROWS * D * 4), 0x00020000);

  while (pos < stop) {
    const int row0 = block * WIDE_ROWS, take = (int)min((int64_t)(cost - unit0), stop - pos);
    const int t0 = max(unit0 - kPagedLead, 0), t1 = unit0 + take - kPagedLead;
    // the slots that hold keys of this row block
    const int64_t key0 = pos - unit0 + kPagedLead;
    const int from_slot = (int)(key0 / stretch), parts = (int)((key0 + tiles - 1) / stretch) - from_slot + 1;
    pos += take;
    unit0 += take;
    if (unit0 == cost) {
      unit0 = 0;
      ++block;
    }
    if (t0 >= t1) continue;

    // this lane's row, features 16 kc + 8 g .. of chunk kc
    const int row = min(row0 + 32 * wave + l32, nrows - 1), token = row / G;
    u32x4_t qf[NK];
    {
      const char* x = (const char*)a.q + ((int64_t)token * a.q_t + (hk * G + row - token * G) * a.q_h) * 2;
#pragma unroll
      for (int kc = 0; kc < NK; ++kc)
        qf[kc] = CHD == CH || 2 * kc + g < CHD ? *(const u32x4_t*)(x + (2 * kc + g) * 16) : u32x4_t{0, 0, 0, 0};
    }
    if constexpr (!F16) {
#pragma unroll
      for (int kc = 0; kc < NK; ++kc)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned u = qf[kc][e];
          qf[kc][e] = Elem<DT>::pack(Elem<DT>::lo(u) * CARRIED, Elem<DT>::hi(u) * CARRIED);
        }
    }
    // they are here before the ring's first loads, which the compiler does not count
#pragma unroll
    for (int kc = 0; kc < NK; ++kc) asm volatile("" : "+v"(qf[kc]));
    __syncthreads();  // the ring is free of the row block before

    // Tile t into buffer buf.  What lies behind the prefix's last row, and chunks behind a row's features, is out of the
    // resource's range and comes as zeros.
    auto issue = [&](int t, int buf) {
      const uint32_t rows = (uint32_t)min(L - t * kPagedTile, kPagedTile) - 1;
      const i32x4_t k = raw_buffer_srd(k_base + (uint64_t)(uint32_t)(t * kPagedTile) * f.k_slot, rows * f.k_slot + D * 2);
      const i32x4_t v = raw_buffer_srd(v_base + (uint64_t)(uint32_t)(t * kPagedTile) * f.v_slot, rows * f.v_slot + D * 2);
#pragma unroll
      for (int i = 0; i < LPT; ++i) {
        const int s = tid + THREADS * i, r = s / CH, c = s % CH, ck = c ^ k_key<DP>(r), cv = v_swizzle<DP>(r, c);
        const uint32_t ko = CHD == CH || ck < CHD ? (uint32_t)r * f.k_slot + 16 * ck : 0xfffffff0u;
        const uint32_t vo = CHD == CH || cv < CHD ? (uint32_t)r * f.v_slot + 16 * cv : 0xfffffff0u;
        lds_dma16_buf(k, ko, &lds_k[buf][(THREADS * i + wave * 64) * 8]);
        lds_dma16_buf(v, vo, &lds_v[buf][(THREADS * i + wave * 64) * 8]);
      }
    };
    f32x16_t o[NDB], s_even, s_odd;
    float den = 0.0f;
    int power = kFirstPower;  // fp16: the row's weights are scaled by 2^power; kappa is an eighth of its eighth root, and c2 with it
    float kappa = kFirstRoot * 0.125f, c2 = F16 ? C2 * kFirstRoot * kFirstRoot : C2;
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] = 0.0f;

    auto scores = [&](int buf, f32x16_t& s) {
      u32x4_t kf[NK];
      const unsigned short* at = &lds_k[buf][l32 * DP];
#pragma unroll
      for (int kc = 0; kc < NK; ++kc) kf[kc] = *(const u32x4_t*)(at + (((2 * kc + g) ^ k_key<DP>(l32)) * 8));
#pragma unroll
      for (int e = 0; e < 16; ++e) s[e] = 0.0f;
#pragma unroll
      for (int kc = 0; kc < NK; ++kc) s = mma32<DT>(kf[kc], qf[kc], s);
    };
    // weights of a tile's scores and its products; MASK: keys from L on weigh nothing
    auto meet = [&](int t, int buf, f32x16_t s, auto mask) {
      auto behind = [&](int e) { return t * kPagedTile + (e >> 2) * 8 + 4 * g + (e & 3) >= L; };
      if constexpr (decltype(mask)::value) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[e] = behind(e) ? -__builtin_inff() : s[e];
      }
      u32x4_t vf[NDB][2];
#pragma unroll
      for (int db = 0; db < NDB; ++db)
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int hh = 0; hh < 2; ++hh) {
            const int r = kk * 16 + hh * 8 + 4 * g + (l16 >> 2), col = db * 32 + m16 * 16 + 4 * (l16 & 3);
            const unsigned short* at = &lds_v[buf][r * DP + v_swizzle<DP>(r, col >> 3) * 8 + (col & 7)];
            const u32x2_t w = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)at));
            vf[db][kk][2 * hh] = w[0];
            vf[db][kk][2 * hh + 1] = w[1];
          }
      __builtin_amdgcn_sched_barrier(0);
      float w[16];
      if constexpr (F16) {
        float top = -__builtin_inff();
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          w[e] = s[e] * kappa;
          top = __builtin_fmaxf(top, w[e]);
        }
        // weights end at kMost^8 = 32768: y ends where y + sqrt(y^2 + c2) is kMost
        constexpr float kMost = 3.6680162f;
        if (__ballot(!(top <= __builtin_fmaf(c2, -0.5f / kMost, 0.5f * kMost))) != 0) {
          // A row's largest weight so far now lies in [16, 32), as in the paged kernel: weights below the normal numbers are off
          // by up to 2^-25 / 16 = 2^-29 of it each, and it may grow by 2^10 before the row comes here again.  32 drafts behind 30001
          // tokens take 329 us with it in [1, 2), 337 in [16, 32), 352 in [128, 256) and 361 in [1024, 2048).
          top = __builtin_fmaxf(top, __shfl_xor(top, 32));
          // below 0 without cancellation: a row begins with c2 so large that its scores may lie far down and weigh much
          const float t = __builtin_fmaf(top, top, c2), far = __builtin_fmaf(t, __builtin_amdgcn_rsqf(t), __builtin_fabsf(top));
          const float z = top < 0.0f ? c2 * __builtin_amdgcn_rcpf(far) : far;
          if (z > kMost && z < __builtin_inff()) {
            // z^8 = 2^(8 e) m^8, m in [1, 2): j is its logarithm, rounded down, less 4, which is 11 and more
            const int bits = __builtin_bit_cast(int, z), e8 = 8 * ((bits >> 23) - 127);
            const float m = __builtin_bit_cast(float, (bits & 0x7fffff) | 0x3f800000), m2 = m * m, m4 = m2 * m2, m8 = m4 * m4;
            const int j = e8 + (__builtin_bit_cast(int, m8) >> 23) - 127 - 4;
            const float root = eighth_root_of_2(-j);
            const float ratio = j < 127 ? __builtin_bit_cast(float, (127 - j) << 23) : 0.0f;
            power -= j;
            kappa = 0.125f * eighth_root_of_2(power);
            c2 = 64 * C2 * kappa * kappa;
            den *= ratio;
#pragma unroll
            for (int e = 0; e < 16; ++e) w[e] *= root;
#pragma unroll
            for (int db = 0; db < NDB; ++db) o[db] *= ratio;
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = s[e];
      }
      const float low = F16 ? LOW * 8.0f * kappa : LOW;
      float least = 0.0f;
#pragma unroll
      for (int e = 0; e < 16; ++e) least = __builtin_fminf(least, w[e]);
      // a score that is no number takes either form
      if (__ballot(!(least > low)) == 0) {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float t = __builtin_fmaf(w[e], w[e], c2);
          const float rho = __builtin_fmaf(t, __builtin_amdgcn_rsqf(t), w[e]);
          const float p2 = rho * rho;
          const float p4 = p2 * p2;
          w[e] = p4 * p4;
        }
      } else {
        apart(w);
        // Weights end at 2^-126, as those of the requests' own keys do, while the row's factor leaves that a normal number.  In bf16 it is
        // that of the scaled weights: 2^-122 for heads of 32 and 128, 2^-120 for 96 (scores of -16800 and below).
        constexpr float C8 = C2 * C2 * C2 * C2;
        const float end = F16 ? __builtin_fmaxf(C8 * __builtin_bit_cast(float, max(power + 1, 1) << 23), 0x1p-126f) : 0x1p-126f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          // far below 0 without cancellation, and above 0 to the end: -infinity weighs the least there is too; a NaN stays one
          const float y = w[e], t = __builtin_fmaf(y, y, c2);
          const float far = __builtin_fmaf(t, __builtin_amdgcn_rsqf(t), y <= low ? __builtin_fabsf(y) : y);
          const float rho = y <= low ? c2 * __builtin_amdgcn_rcpf(far) : far;
          const float p2 = rho * rho;
          const float p4 = p2 * p2;
          const float p8 = p4 * p4;
          w[e] = y < -0x1p60f || p8 < end ? end : p8;
        }
      }
      if constexpr (decltype(mask)::value) {
#pragma unroll
        for (int e = 0; e < 16; ++e) w[e] = behind(e) ? 0.0f : w[e];
      }
      float tree[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) tree[e] = w[e] + w[e + 8];
      den += ((tree[0] + tree[4]) + (tree[1] + tree[5])) + ((tree[2] + tree[6]) + (tree[3] + tree[7]));
      u32x4_t wp[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) wp[kk][e] = Elem<DT>::pack(w[kk * 8 + 2 * e], w[kk * 8 + 2 * e + 1]);
      __builtin_amdgcn_sched_barrier(0);
      // a wave with products ready goes before one that forms weights (32 drafts behind 30001: 336 us for 342 in all)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int db = 0; db < NDB; ++db) o[db] = mma32<DT>(vf[db][kk], wp[kk], o[db]);
      __builtin_amdgcn_s_setprio(0);
    };

    const int n = t1 - t0;
#pragma unroll
    for (int i = 0; i < RING - 1; ++i)
      if (i < n) issue(t0 + i, i);
    if (n >= RING - 1) __builtin_amdgcn_s_waitcnt(vmcnt_only(LOADS * (RING - 2)));
    else __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __syncthreads();
    scores(0, s_even);
    // before tile u's weights: this wave's loads of tile u + 1 are done, those of u + 2 may go on; then every wave's, and every
    // wave has read tile u - 1, whose place the next one takes
    auto step = [&](int u, int buf) {
      if (u + 2 < n) __builtin_amdgcn_s_waitcnt(vmcnt_only(LOADS * (RING - 3)));
      else __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      __syncthreads();
      if (u + RING - 1 < n) issue(t0 + u + RING - 1, (buf + RING - 1) & (RING - 1));
    };
    auto more = [&](int u, int buf, const f32x16_t& now, f32x16_t& next) {  // tile u has a next one
      step(u, buf);
      scores((buf + 1) & (RING - 1), next);
      meet(t0 + u, buf, now, std::false_type());
    };
    auto last = [&](int u, int buf, const f32x16_t& now) {
      step(u, buf);
      if (t1 * kPagedTile > L) meet(t0 + u, buf, now, std::true_type());
      else meet(t0 + u, buf, now, std::false_type());
    };
    int u = 0;
    for (; u + 4 < n; u += 4) {
      more(u, 0, s_even, s_odd);
      more(u + 1, 1, s_odd, s_even);
      more(u + 2, 2, s_even, s_odd);
      more(u + 3, 3, s_odd, s_even);
    }
    if (u + 2 < n) {
      more(u, u & 3, s_even, s_odd);
      more(u + 1, (u + 1) & 3, s_odd, s_even);
      u += 2;
    }
    if (u + 1 < n) {
      more(u, u & 3, s_even, s_odd);
      last(u + 1, (u + 1) & 3, s_odd);
    } else {
      last(u, u & 3, s_even);
    }

    den += __shfl_xor(den, 32);
    // the factor is taken back: c^8, and in fp16 the rows' powers of two
    constexpr float C8 = C2 * C2 * C2 * C2;
    float back = 1.0f / C8;
    if constexpr (F16) back *= __builtin_bit_cast(float, min(max(127 - power, 1), 254) << 23);
    den *= back;
    auto part_of = [&](int i) { return (int64_t)2 * (from_slot + i) + (i == 0); };
    const int64_t my_part = part_of(slot - from_slot);
    const int size = wide_group(parts);
    const bool mine = row0 + 32 * wave + l32 < nrows;
    // All of a row block's keys are the sums themselves: their place is the row's.  Only a row block that goes on behind this
    // stretch has a part in it that is the first, so that a slot has room for one of these; where row blocks are more than slots,
    // several lie within a stretch.
    int mine_at = row0 + 32 * wave + l32;
    asm volatile("" : "+v"(mine_at));  // formed again: no register holds it over the keys
    const int mine_token = mine_at / G;
    const int64_t at = (int64_t)mine_token * (int)p.heads + (hk * G + mine_at - mine_token * G);
    float* const to = parts == 1 ? f.shared.top + at * D : f.part + head0 * D + (my_part * WIDE_ROWS + 32 * wave + l32) * D;
    float* const to_den = parts == 1 ? f.shared.bottom + at : part_den + my_part * WIDE_ROWS + 32 * wave + l32;
    float zero = 0.0f;  // NaN where a sum is not finite
#pragma unroll
    for (int db = 0; db < NDB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int d = db * 32 + r4 * 8 + 4 * g;
        f32x4_t x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = o[db][4 * r4 + i] * back;
          zero = __builtin_fmaf(x[i], 0.0f, zero);
        }
        if (!mine || (D < DP && d >= D)) continue;
        // a part that is added up here goes where every XCD sees it
        if (size > 1) put4(buffer, (uint32_t)((my_part * WIDE_ROWS + 32 * wave + l32) * D + d) * 4, x);
        else *(f32x4_t*)(to + d) = x;
      }
    if (mine && g == 0) put1(to_den, den);
    // A value that is not finite is the sum of every row, as weights are above 0.  It may have become NaN in the product, where
    // a weight may be rounded to 0: each feature's sum of such values, the same for all rows, takes its place.  (Where the row
    // sum is not finite either the row is NaN already.)
    if (__syncthreads_or(mine && zero != 0.0f && __builtin_fabsf(den) < __builtin_inff())) {
      float* odd = (float*)&lds_k[0][0];
      for (int d = tid; d < D; d += THREADS) odd[d] = 0.0f;
      __syncthreads();
      for (int64_t e = tid; e < (int64_t)(min(t1 * kPagedTile, L) - t0 * kPagedTile) * CHD; e += THREADS) {
        const int key = (int)(e / CHD), c = (int)(e - (int64_t)key * CHD);
        float x[8];
        RowChunk<DT>::unpack(*(const u32x4_t*)(v_base + (uint64_t)(uint32_t)(t0 * kPagedTile + key) * f.v_slot + 16 * c), x);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(__builtin_fabsf(x[i]) < __builtin_inff())) atomicAdd(&odd[8 * c + i], x[i]);
      }
      __syncthreads();
      if (mine)
        for (int d = 4 * g; d < D; d += 8)
          for (int i = d; i < d + 4; ++i) {
            if (__builtin_fabsf(odd[i]) < __builtin_inff()) continue;
            if (size > 1) put1(to + i, odd[i]);
            else to[i] = odd[i];
          }
    }
    if (size == 1) continue;

    // the last of a group to finish adds its parts up, over the first of them
    const int g0 = (slot - from_slot) / size * size, here = min(size, parts - g0);
    if (!arrived(a.sched.count + (int64_t)hk * 4 * f.slots + part_of(g0), here, &flag)) continue;
    const int64_t sum_at = part_of(g0) * WIDE_ROWS;
    sum_parts<THREADS>(buffer, part_den, here, min(WIDE_ROWS, nrows - row0), D, sums,
                       [&](int i) { return part_of(g0 + i) * WIDE_ROWS; },
                       [&](int r, int d, f32x4_t x) {
                         // of the first part this thread alone reads these features
                         put4(buffer, (uint32_t)((sum_at + r) * D + d) * 4, x);
                         if (d == 0) put1(part_sum + sum_at + r, sums[r]);
                       });
  }
}

// The parts of every row that has several, added up in their order: a thread has four features of a row.
__global__ __launch_bounds__(THREADS) void afa_prefix_join_kernel(const PagedFast f) {
  const afa_paged_plan& p = f.a.plan;
  const int D = f.dim, quads = D / 4, G = f.a.group, H = (int)p.heads;
  const int nrows = p.starts[p.requests] * G, tiles = (f.a.prefix.len + kPagedTile - 1) / kPagedTile, cost = kPagedLead + tiles;
  const int64_t stretch = wide_stretch(nrows, cost, f.slots), all = (int64_t)nrows * (int)p.kv_heads * quads;
  for (int64_t e = (int64_t)blockIdx.x * THREADS + threadIdx.x; e < all; e += (int64_t)gridDim.x * THREADS) {
    // rows of the call one after the other: token, then head
    const int d = 4 * (int)(e % quads), at = (int)(e / quads), token = at / H, hk = (at - token * H) / G;
    const int row = token * G + (at - token * H - hk * G), block = row / WIDE_ROWS, r = row - block * WIDE_ROWS;
    const int64_t key0 = (int64_t)block * cost + kPagedLead, from = key0 / stretch;
    const int parts = (int)((key0 + tiles - 1) / stretch - from) + 1, size = wide_group(parts), n = (parts + size - 1) / size;
    if (parts == 1) continue;  // these are in their places
    const float* den = size > 1 ? f.part_sum : f.part_den;
    // part i of the row block: a slot's second where it begins there, else its first
    auto place = [&](int i) {
      return ((int64_t)hk * 2 * f.slots + 2 * (from + (int64_t)i * size) + (i == 0)) * WIDE_ROWS + r;
    };
    f32x4_t x = {0, 0, 0, 0};
    float sum = 0.0f;
    constexpr int N = 8;
    for (int i0 = 0; i0 < n; i0 += N) {
      f32x4_t y[N];
      float z[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        y[i] = f32x4_t{0, 0, 0, 0};
        z[i] = 0.0f;
        if (i0 + i >= n) continue;
        y[i] = *(const f32x4_t*)(f.part + place(i0 + i) * D + d);
        if (d == 0) z[i] = den[place(i0 + i)];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        x += y[i];
        sum += z[i];
      }
    }
    *(f32x4_t*)(f.shared.top + (int64_t)at * D + d) = x;
    if (d == 0) f.shared.bottom[at] = sum;
  }
}

template <int DT, int D>
hipError_t wide_launch(const PagedFast& f, hipStream_t st) {
  hipLaunchKernelGGL((afa_prefix_wide_kernel<DT, D>), dim3((unsigned)(f.slots * f.a.plan.kv_heads)), dim3(THREADS), 0, st, f);
  return hipGetLastError();
}

template <int DT>
hipError_t wide_go(const PagedFast& f, hipStream_t st) {
  switch (f.dim) {
    case 32: return wide_launch<DT, 32>(f, st);
    case 48: return wide_launch<DT, 48>(f, st);
    case 64: return wide_launch<DT, 64>(f, st);
    case 96: return wide_launch<DT, 96>(f, st);
    default: return wide_launch<DT, 128>(f, st);
  }
}

}  // namespace

PagedCut prefix_cut(const afa_paged_plan& p, int cus) {
  afa_paged_plan all = p;
  all.max_new = p.max_tokens;  // the rows of one key head are those of all tokens
  return paged_cut(all, cus);
}

hipError_t prefix_sums_launch(const PagedFwdArgs& a, const PagedCut& c, const PrefixSums& shared, void* ws, hipStream_t st) {
  const PrefixKeys& x = a.prefix;
  const PagedFast f = paged_fast_args(a, c, PageStrides{0, x.k_head, x.k_key, 0, x.v_head, x.v_key}, shared, ws);
  if (c.rows != WIDE_ROWS || a.plan.dtype == AFA_F32) return fast_launch<true>(f, c.rows, st);
  const hipError_t e = a.plan.dtype == AFA_BF16 ? wide_go<AFA_BF16>(f, st) : wide_go<AFA_F16>(f, st);
  if (e != hipSuccess) return e;
  const int64_t groups = (a.plan.max_tokens * a.plan.heads * (a.plan.head_dim / 4) + THREADS - 1) / THREADS;
  hipLaunchKernelGGL(afa_prefix_join_kernel, dim3((unsigned)(groups < 65536 ? groups : 65536)), dim3(THREADS), 0, st, f);
  return hipGetLastError();
}

}  // namespace afa
