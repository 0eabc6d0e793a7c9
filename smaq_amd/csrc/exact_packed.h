// Attention over a step's own exact tokens: the kernel of smaq_packed_attention,
// instantiated per type (exact_packed_f16.hip, exact_packed_bf16.hip).
//
// 4 D operations per visible pair and head over a few bytes per token: the matrix
// cores bound it, and beside them the power they share with the vector unit (the
// exponentials) and LDS (operand reads): the clock falls from 2.4 to 1.7-1.9 GHz.
// 16384 causal tokens of 32 / 8 heads of 128 bf16 dims take 2.1 ms (1.04 PFLOP/s; a 16384^3
// matrix product reaches 1.58), capped 2.5 ms (0.87), biased 2.36 (0.93).  A tile less
// vector work moves that little: without the exponentials it is 4% shorter, without the
// copies to LDS 15%; eight waves on one copy, with two or three buffers, take 1-4% longer
// than two workgroups of four, tiles of 32 keys 3%.
//
// A unit of work is 32 tokens of one query head; a workgroup's four waves take four
// units of one KV head, heads before tokens, so that they read the same keys (with
// four heads or more on a KV head, exactly the same).  Token blocks are cut from the
// packed rows, not from the documents: rows carry their own visible ranges, many
// short documents share a block, and no block needs to be looked up.  A row sees at
// most two ranges, [lo, hi) and a prefix apart from it.
//
//   S^T[key][q] = K . Q^T      A = K rows from LDS, B = Q in registers
//   softmax per column q       a lane holds half the keys of its column
//   O^T[dim][q] += V^T . P^T   B = P^T straight from the S^T accumulators (the
//                              k-elements of half h are keys 4 h .. 4 h + 3 and
//                              8 + 4 h ..), A = V^T by transposing LDS reads
//
// Tiles of 64 keys (32 at 256 dims) are copied global -> LDS one tile ahead, 16-byte
// units placed by an XOR of the row so that operand reads meet no bank twice.  Small
// grids have two groups of four waves per workgroup (KG = 2), each with every second
// tile; their results are joined in LDS.
//
// Masks.  A tile that every row of a wave sees whole takes no mask.  In others the sums
// of masked scores begin at -inf (a cap, which brings them back, is followed by a mask of
// the weights).  A masked key that is not finite makes NaN of that, a masked value 0 * NaN
// in the second product.  Both show as a result that is not finite: such a workgroup runs
// again with the masked scores set to -inf by selection, and the masked tiles' values that
// are not finite taken out of the product (the other rows keep their bits) and added key
// by key to the rows that see them.
//
// Rounding.  Scores, maxima, sums and outputs are fp32.  The weights are rounded to the
// values' type, as the matrix instruction takes two operands of one type: half a step of
// each weight, of either sign.  Their sum l is of the weights before that.
#pragma once

#include <math.h>

#include <type_traits>

#include "exact_attention.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr int kIntMax = 0x7fffffff;

typedef short s16x4 __attribute__((ext_vector_type(4)));

__device__ const u32x4v kZeroUnit = {0, 0, 0, 0};

// Layout of a tile row of DT dims in LDS: 16-byte unit u of row r sits at u ^ swizzle.
// Keys are read 32 rows x one unit, values 8 rows x 4 units at a time.
template <int DT>
__device__ __forceinline__ int key_swizzle(int r) { return DT == 64 ? (r >> 1) & 7 : r & 15; }
template <int DT>
__device__ __forceinline__ int val_swizzle(int r) { return DT == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3); }

// the last i of the ascending s[0..n) with s[i] <= x, 0 if there is none; by the wave
__device__ __forceinline__ int wave_last(const int* s, int n, int x, int lane) {
  int lo = 0, len = n;
  while (len > 1) {
    const int step = (len + 63) / 64, i = lane * step;
    const unsigned long long at = __ballot(i < len && s[lo + min(i, len - 1)] <= x);
    const int below = (int)__popcll(at);  // signed: none may be
    const int pos = below > 0 ? (below - 1) * step : 0;
    lo += pos;
    len = min(step, len - pos);
  }
  return lo;
}

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, __shfl_xor(v, o, 64));
  return __builtin_amdgcn_readfirstlane(v);
}

template <typename T, int DT, bool FULL, bool CAP, bool ALIBI, int KG>
__global__ __launch_bounds__(KG * kThreads, DT == 64 && KG == 1 ? 3 : 2) void packed_kernel(smaq_packed_params p, ScoreRule rule, int blocks) {
  constexpr int KT = DT == 256 ? 32 : 64;  // keys per tile
  constexpr int KB = KT / 32;              // 32-key blocks
  constexpr int KS = DT / 16;              // k steps of a product over the head dim
  constexpr int DB = DT / 32;              // 32-dim blocks of the output
  constexpr int UPR = DT / 8;              // 16-byte units of a row
  constexpr int RS = DT * 2;               // bytes of a row
  constexpr int TILE = KT * RS;            // bytes of a key or value tile
  constexpr int LOADS = KT * UPR / kThreads;
  // Matrix sections at raised wave priority: 256 dims 1.17 -> 1.12 ms; at up to 128 dims they
  // are better left alone (16384 tokens 2.14 -> 2.11 ms, capped 2.56 -> 2.53, 8192 tokens of
  // 8 / 8 heads 231 -> 214 us).
  constexpr bool PRIO = DT == 256;
  __shared__ __attribute__((aligned(16))) char all_lds[KG * 4 * TILE];  // of each key group two buffers of (keys, values)
  __shared__ int span[4][4];
  __shared__ float joined[KG == 2 ? 4 : 1][2][64];
  const int tid = threadIdx.x % kThreads, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kg = KG == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / kThreads);
  char* lds = all_lds + kg * 4 * TILE;
  const int g = p.n_q_heads / p.n_kv_heads, D = p.head_dim, T_all = (int)p.n_tokens;
  const int h = blockIdx.x % p.n_kv_heads;
  // The last tokens first: with a causal mask they have the most keys.  A grid that the card
  // holds at once puts the i-th workgroup of every 256 on the same CU: every second 256 runs
  // the other way round, so that a CU gets long and short ones.
  const int groups = (blocks * g + 3) / 4;
  int rank = blockIdx.x / p.n_kv_heads;
  if (KG == 1 && gridDim.x <= 256 * (DT == 64 ? 3 : 2) && 256 % p.n_kv_heads == 0) {
    const int per = 256 / p.n_kv_heads, first = rank / per * per;
    if (rank / per & 1) rank = first + min(groups, first + per) - 1 - rank;
  }
  const int unit = 4 * (groups - 1 - rank) + w;
  const int tb = unit / g, hq = h * g + unit % g;
  const int row = 32 * tb + n;

  // ---- queries: column n, dims 16 ks + 8 half ..; a negative scale is taken into them,
  // and a scale of 0 makes them 0
  u32x4v qr[KS];
  {
    const T* src = (const T*)p.q + (int64_t)row * p.q_stride_t + hq * p.q_stride_h;
    const uint32_t flip = p.scale < 0.0f ? 0x80008000u : 0u, keep = p.scale == 0.0f ? 0u : ~0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      qr[ks] = u32x4v{0, 0, 0, 0};
      if (row < T_all && unit < blocks * g && (FULL || 16 * ks + 8 * half < D)) qr[ks] = (*(const u32x4v*)(src + 16 * ks + 8 * half) ^ flip) & keep;
    }
  }
  // ---- the ranges of this lane's row: [lo, hi), and [lo2, hi2) if the prefix is apart;
  // and of the wave: first and last key, the gap no row looks into, the keys all rows see
  int lo = 0, hi = 0, lo2 = 0, hi2 = 0;
  int w_lo = kIntMax, w_hi = 0, w_gap0 = 0, w_gap1 = kIntMax, w_full0 = 0, w_full1 = kIntMax;
  auto see = [&](int t, int s, int e, int prefix, int& a0, int& a1, int& b0, int& b1) {
    a0 = p.window ? max(s, t - p.window + 1) : s;
    a1 = p.causal ? t + 1 : e;
    b0 = b1 = 0;
    const int pre = s + min(max(prefix, 0), e - s);
    if (pre >= a0) {
      a0 = s;
      a1 = max(a1, pre);
    } else if (pre > s) {
      b0 = s;
      b1 = pre;
    }
  };
  if (unit < blocks * g && p.n_docs > 0) {
    const int t0 = 32 * tb, t1 = min(t0 + 31, T_all - 1);
    int d0, d1, v = 0;
    const bool few = p.n_docs < 64;  // the starts of all documents in one register
    if (few) {
      v = p.starts[min(lane, p.n_docs)];
      const unsigned long long at0 = __ballot(lane < p.n_docs && v <= t0), at1 = __ballot(lane < p.n_docs && v <= t1);
      d0 = max((int)__popcll(at0) - 1, 0);
      d1 = max((int)__popcll(at1) - 1, 0);
    } else {
      d0 = wave_last(p.starts, p.n_docs, t0, lane);
      d1 = wave_last(p.starts, p.n_docs, t1, lane);
    }
    if (d0 == d1) {
      // rows of one document: lo, hi, and whether the prefix is apart do not fall from row
      // to row, so the first and last row bound the wave
      const int s = max(few ? __builtin_amdgcn_readlane(v, d0) : p.starts[d0], 0);
      const int e = min(few ? __builtin_amdgcn_readlane(v, d0 + 1) : p.starts[d0 + 1], T_all);
      const int prefix = p.prefix_lens ? p.prefix_lens[d0] : 0;
      const int ra = max(t0, s), rb = min(t1, e - 1);
      if (ra <= rb) {
        int x0, x1, a_lo, a_hi, b_lo, b_hi;
        see(ra, s, e, prefix, a_lo, a_hi, x0, x1);
        see(rb, s, e, prefix, b_lo, b_hi, x0, x1);
        const bool rb_apart = x1 > x0;
        w_lo = rb_apart ? s : a_lo;
        w_hi = b_hi;
        w_gap0 = rb_apart ? x1 : b_lo;
        w_gap1 = a_lo;
        w_full0 = b_lo;
        w_full1 = a_hi;
        if (row >= ra && row <= rb) see(row, s, e, prefix, lo, hi, lo2, hi2);
      }
    } else {
      int d = d0;
      for (int end = d1 + 1; end - d > 1;) {
        const int mid = (d + end) >> 1;
        if (p.starts[mid] <= row) d = mid; else end = mid;
      }
      const int s = max(p.starts[d], 0), e = min(p.starts[d + 1], T_all);
      if (row >= s && row < e) see(row, s, e, p.prefix_lens ? p.prefix_lens[d] : 0, lo, hi, lo2, hi2);
      const bool in = hi > lo, out = hi2 > lo2;
      w_lo = wave_min(in ? (out ? lo2 : lo) : kIntMax);
      w_hi = wave_max(in ? hi : 0);
      w_gap0 = wave_max(out ? hi2 : (in ? lo : 0));
      w_gap1 = wave_min(in ? lo : kIntMax);
      w_full0 = wave_max(in ? lo : 0);
      w_full1 = wave_min(in ? hi : kIntMax);
    }
  }
  const bool live = hi > lo;
  const bool w_apart = __any(hi2 > lo2);
  // of the workgroup; waves of one block have the same (the branch is the workgroup's)
  int k_lo = w_lo, k_hi = w_hi, gap0 = w_gap0, gap1 = w_gap1;
  if ((unit - w) / g != (unit - w + 3) / g) {
    if (lane == 0) {
      span[w][0] = w_lo;
      span[w][1] = w_hi;
      span[w][2] = w_gap0;
      span[w][3] = w_gap1;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      k_lo = min(k_lo, __builtin_amdgcn_readfirstlane(span[x][0]));
      k_hi = max(k_hi, __builtin_amdgcn_readfirstlane(span[x][1]));
      gap0 = max(gap0, __builtin_amdgcn_readfirstlane(span[x][2]));
      gap1 = min(gap1, __builtin_amdgcn_readfirstlane(span[x][3]));
    }
  }

  const float slope = ALIBI ? (live ? p.alibi_slopes[hq] * kLog2eF : 0.0f) : 0.0f;
  // Where no row sees a key behind it the distance needs no absolute value and the bias goes
  // into the product's scaling (16384 tokens 2.46 -> 2.36 ms); its parts stay finite.
  const bool linear = ALIBI && !CAP && p.causal && !p.prefix_lens && __all(fabsf(slope) < 1e25f);

  // ---- tile copies: load i of thread tid fills unit 256 i + tid of the tile, of row
  // i kThreads / UPR + tid / UPR
  constexpr int RPL = kThreads / UPR;  // rows of a load
  const T* kc = (const T*)p.k + h * p.k_stride_h;
  const T* vc = (const T*)p.v + h * p.v_stride_h;
  const int r0 = tid / UPR, u0 = tid % UPR;
  constexpr int PER = RPL < 16 ? 2 : 1;  // loads until the swizzle of a row returns
  static_assert(RPL * PER % 16 == 0, "whole periods");
  uint32_t k_lane[PER];
  for (int i = 0; i < PER; ++i) k_lane[i] = (uint32_t)(2 * r0 * (int)p.k_stride_t) + 16 * (u0 ^ key_swizzle<DT>(i * RPL + r0));
  const uint32_t v_lane = (uint32_t)(2 * r0 * (int)p.v_stride_t) + 16 * (u0 ^ val_swizzle<DT>(r0));
  auto to_lds = [&](const void* src, char* dst) {
    __builtin_amdgcn_global_load_lds(src, (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
  };
  auto copy_tile = [&](int k, int buf) {
    char* kd = lds + buf * 2 * TILE + 1024 * w;
    if (FULL && k + KT <= k_hi) {
      // whole tiles: a base of the wave and a 32-bit offset of the lane (not hoisted as 64
      // bits, which the load does not take as an offset)
      uint32_t ko[PER], vo = v_lane;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        ko[i] = k_lane[i];
        asm volatile("" : "+v"(ko[i]));
      }
      asm volatile("" : "+v"(vo));
      const char *ks = (const char*)(kc + k * p.k_stride_t), *vs = (const char*)(vc + k * p.v_stride_t);
#pragma unroll
      for (int i = 0; i < LOADS; ++i) {
        to_lds(ks + ko[i % PER], kd + 4096 * i);
        to_lds(vs + vo, kd + TILE + 4096 * i);
        ks += 2 * RPL * p.k_stride_t;
        vs += 2 * RPL * p.v_stride_t;
      }
      return;
    }
#pragma unroll 1
    for (int i = 0; i < LOADS; ++i) {
      const int r = i * RPL + r0;
      const int64_t key = min(k + r, k_hi - 1);
      const int uk = u0 ^ key_swizzle<DT>(r), uv = u0 ^ val_swizzle<DT>(r);
      to_lds(FULL || 8 * uk < D ? (const void*)(kc + key * p.k_stride_t + 8 * uk) : (const void*)&kZeroUnit, kd + 4096 * i);
      to_lds(FULL || 8 * uv < D ? (const void*)(vc + key * p.v_stride_t + 8 * uv) : (const void*)&kZeroUnit, kd + TILE + 4096 * i);
    }
  };
  // the tile behind k: the next keys, or past the gap
  auto next_tile = [&](int k) {
    k += KT;
    return k >= gap0 && k + KT <= gap1 && gap1 < k_hi ? gap1 : k;
  };

  // ---- operand addresses within a tile: rows are multiples of RS, so a step along the
  // units of a row is an XOR of the whole address
  const int koff = n * RS + 16 * (half ^ key_swizzle<DT>(n));
  const int vr0 = 4 * half + ((lane & 15) >> 2);
  const int voff = vr0 * RS + 16 * ((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ val_swizzle<DT>(vr0)) + 8 * (lane & 1);

  f32x16v acc[DB];
  float m_ref, m_use, m_thr, l;
  auto run = [&](auto careful_tag) {
    constexpr bool careful = decltype(careful_tag)::value;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = f32x16v{};
    m_ref = m_thr = kNegInf;
    m_use = l = 0.0f;
    // of every KG tiles this wave's group takes the kg-th
    const int k_first = kg == 0 ? k_lo : next_tile(k_lo);
    if (k_lo < k_hi && k_first < k_hi) copy_tile(k_first, 0);
    int buf = 0;
    for (int k = k_lo, k_mine = k_first; k < k_hi; buf ^= 1) {
      // this thread's copies have landed, then everyone's; everyone is done with the
      // other buffer
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_waitcnt(0);
      asm volatile("" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      const int k0 = k_mine;
      k = next_tile(k);
      if (KG == 2) k = next_tile(k);
      k_mine = kg == 0 ? k : next_tile(k);
      if (k_mine < k_hi) copy_tile(k_mine, buf ^ 1);
      if (k0 >= w_hi || k0 + KT <= w_lo || (k0 >= w_gap0 && k0 + KT <= w_gap1)) continue;
      const int kt = buf * 2 * TILE + koff, vt = buf * 2 * TILE + TILE + voff;
      // key of register i of block kb: k0 + 32 kb + 8 (i / 4) + 4 half + i % 4
      const bool full = k0 >= w_full0 && k0 + KT <= w_full1;
      f32x16v s[KB];
      // put(kb, i, whether the row sees the key)
      auto each_seen = [&](auto put) {
        const int a1 = hi - k0 - 4 * half;
        if (!w_apart && k0 >= w_full0) {  // causal and last tiles: cut above only
#pragma unroll
          for (int i = 0; i < 16 * KB; ++i) put(i / 16, i % 16, 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4 < a1);
          return;
        }
        const int a0 = lo - k0 - 4 * half, b0 = lo2 - k0 - 4 * half, b1 = hi2 - k0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16 * KB; ++i) {
          const int key = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4;
          put(i / 16, i % 16, ((key >= a0) & (key < a1)) | ((key >= b0) & (key < b1)));
        }
      };
      auto product = [&](auto masked_tag) {
        if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          if constexpr (!decltype(masked_tag)::value) s[kb] = f32x16v{};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks)
            s[kb] = Mat<T>::mma32(*(const u32x4v*)(lds + (kt ^ (32 * ks)) + kb * 32 * RS), qr[ks], s[kb]);
        }
        if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
      };
      // A masked tile's sums begin at -inf where the key is not seen: code of its own, as
      // masks behind one product cost whole tiles 16 register copies
      if (full) {
        product(std::false_type{});
      } else {
        each_seen([&](int kb, int i, bool seen) { s[kb][i] = seen ? 0.0f : kNegInf; });
        product(std::true_type{});
      }
      auto get = [&](int i) { return s[i / 16][i % 16]; };
      if constexpr (ALIBI) {
        const float gap = (float)(row - k0 - 4 * half);
        auto offset = [](int i) { return (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4); };
        auto put = [&](int i, float x) { s[i / 16][i % 16] = fmaf(-slope, fabsf(gap - offset(i)), x); };
        if constexpr (CAP) {
          each_score<16 * KB>(rule, get, put);
        } else if (linear) {
          const float base = -slope * gap;
#pragma unroll
          for (int i = 0; i < 16 * KB; ++i) s[i / 16][i % 16] = fmaf(get(i), rule.scale, fmaf(slope, offset(i), base));
        } else {
#pragma unroll
          for (int i = 0; i < 16 * KB; ++i) put(i, get(i) * rule.scale);
        }
      }
      // -inf plus a product that is not finite, and -inf behind a cap, are no longer -inf
      if (careful || (CAP && ALIBI))
        if (!full) each_seen([&](int kb, int i, bool seen) { s[kb][i] = seen ? s[kb][i] : kNegInf; });
      float mx = kNegInf, size = 0.0f;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          mx = fmaxf(mx, s[kb][i]);
          if constexpr (CAP && !ALIBI) size = fmaxf(size, fabsf(s[kb][i]));
        }
      // of the wave; masked tiles never, or what is masked (NaN or not) would choose
      const bool near = CAP && !ALIBI && full && __all(size < rule.near);
      if constexpr (CAP && !ALIBI)
        mx = near ? near_score(rule, mx) : rule.wide ? capped_score<true>(rule, mx) : capped_score<false>(rule, mx);
      else if constexpr (!ALIBI)
        mx *= rule.scale;
      if (__any(mx > m_thr)) {
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_ref, mx);
        m_use = m_new == kNegInf ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_ref - m_use);
        l *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= alpha;
        m_ref = m_new;
        m_thr = m_new + kRaise;
      }
      if constexpr (CAP && !ALIBI) {
        if (near) {
#pragma unroll
          for (int i = 0; i < 16 * KB; ++i) s[i / 16][i % 16] = __builtin_amdgcn_exp2f(near_score(rule, get(i), m_use));
        } else {
          each_score<16 * KB>(rule, get, [&](int i, float x) { s[i / 16][i % 16] = __builtin_amdgcn_exp2f(x - m_use); });
        }
      } else {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[kb][i] = __builtin_amdgcn_exp2f(ALIBI ? s[kb][i] - m_use : fmaf(s[kb][i], rule.scale, -m_use));
      }
      if constexpr (CAP && !ALIBI) {  // the cap brings a masked score back to -cap
        if (!full) each_seen([&](int kb, int i, bool seen) { s[kb][i] = seen ? s[kb][i] : 0.0f; });
      }
      uint32_t pk[KB][8];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          l += s[kb][i] + s[kb][i + 1];
          pk[kb][i / 2] = Mat<T>::pack(s[kb][i], s[kb][i + 1]);
        }
      // O^T += V^T P^T, 16 keys c at a time
      auto values = [&](int c, int db) {
        const char* a = lds + (vt ^ (64 * (db & 3))) + (db >> 2) * 256 + 16 * c * RS;
        const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)a);
        const s16x4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(a + 8 * RS));
        const u32x2v xx = __builtin_bit_cast(u32x2v, x), yy = __builtin_bit_cast(u32x2v, y);
        return u32x4v{xx[0], xx[1], yy[0], yy[1]};
      };
      if (!careful || full) {
        if constexpr (PRIO) __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int c = 0; c < KT / 16; ++c) {
          const uint32_t* q = &pk[c >> 1][4 * (c & 1)];
          const u32x4v pt = {q[0], q[1], q[2], q[3]};
#pragma unroll
          for (int db = 0; db < DB; ++db) acc[db] = Mat<T>::mma32(values(c, db), pt, acc[db]);
        }
        if constexpr (PRIO) __builtin_amdgcn_s_setprio(0);
      } else if constexpr (careful) {
#pragma unroll
        for (int c = 0; c < KT / 16; ++c) {
          const uint32_t* q = &pk[c >> 1][4 * (c & 1)];
          const u32x4v pt = {q[0], q[1], q[2], q[3]};
#pragma unroll
          for (int db = 0; db < DB; ++db) {
            const u32x4v v = values(c, db);
            u32x4v bad;
#pragma unroll
            for (int y = 0; y < 4; ++y) bad[y] = not_finite_halves<Mat<T>::kExp>(v[y]);
            acc[db] = Mat<T>::mma32(v & ~bad, pt, acc[db]);
            if (!__any(bad[0] | bad[1] | bad[2] | bad[3])) continue;
            for (int x = 0; x < 16; ++x) {  // k-element x & 7 of half x >> 3 alone
              const int j = x & 7, key = k0 + 16 * c + 4 * (x >> 3) + (j & 3) + 8 * (j >> 2);
              const bool seen = (key >= lo && key < hi) || (key >= lo2 && key < hi2);
              u32x4v only;
#pragma unroll
              for (int y = 0; y < 4; ++y)
                only[y] = half == (x >> 3) && (j >> 1) == y ? (j & 1 ? 0xffff0000u : 0x0000ffffu) : 0u;
              const f32x16v one = Mat<T>::mma32(v & bad & only, pt & only, f32x16v{});
#pragma unroll
              for (int i = 0; i < 16; ++i) acc[db][i] = seen ? acc[db][i] + one[i] : acc[db][i];
            }
          }
        }
      }
    }
  };
  run(std::false_type{});
  float z = l * 0.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) z = fmaf(acc[db][i], 0.0f, z);
  if (__syncthreads_or(live && z != z)) run(std::true_type{});

  // ---- the result, turned in LDS (every wave is done with its tiles) so that it leaves in
  // whole rows
  __syncthreads();
  l += __shfl_xor(l, 32, 64);
  char* turned = all_lds + w * (KG == 1 ? 32 * RS : DB * 4096);
  if constexpr (KG == 2) {
    // the second key group's (m, l, o) into the first's, register by register
    f32x4v* other = (f32x4v*)turned + lane;
    if (kg == 1) {
      joined[w][0][lane] = m_ref;
      joined[w][1][lane] = l;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          other[64 * (4 * db + i / 4)] = f32x4v{acc[db][i], acc[db][i + 1], acc[db][i + 2], acc[db][i + 3]};
    }
    __syncthreads();
    if (kg == 1) return;
    const float m1 = joined[w][0][lane], m = fmaxf(m_ref, m1);
    const float mu = m == kNegInf ? 0.0f : m, a0 = __builtin_amdgcn_exp2f(m_ref - mu), a1 = __builtin_amdgcn_exp2f(m1 - mu);
    l = l * a0 + joined[w][1][lane] * a1;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4v o = other[64 * (4 * db + i / 4)];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[db][i + e] = acc[db][i + e] * a0 + o[e] * a1;
      }
  }
  const float inv = live ? 1.0f / l : 0.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const u32x2v y = {Mat<T>::pack(acc[db][i] * inv, acc[db][i + 1] * inv), Mat<T>::pack(acc[db][i + 2] * inv, acc[db][i + 3] * inv)};
      *(u32x2v*)(turned + n * RS + 16 * ((4 * db + i / 4) ^ (n & (UPR < 16 ? 7 : 15))) + 8 * half) = live ? y : u32x2v{0, 0};
    }
  const unsigned long long rows_live = __ballot(live);
  if (unit >= blocks * g) return;
#pragma unroll
  for (int k = 0; k < 32 * UPR / 64; ++k) {
    const int r = (64 * k + lane) / UPR, u = lane % UPR;
    const u32x4v y = *(const u32x4v*)(turned + r * RS + 16 * (u ^ (r & (UPR < 16 ? 7 : 15))));
    if (32 * tb + r < T_all && (p.zero_rest || ((rows_live >> r) & 1)) && (FULL || 8 * u < D))
      *(u32x4v*)((T*)p.out + (int64_t)(32 * tb + r) * p.out_stride_t + hq * p.out_stride_h + 8 * u) = y;
  }
}

template <typename T, int DT, bool FULL, bool CAP, bool ALIBI>
void launch_packed(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st) {
  // A grid that leaves the card's waves idle, or that is as long as its longest workgroup
  // (two a CU, long documents), gives every unit two groups of waves, which take the key
  // tiles in turn: one prompt of 1500 tokens 43 -> 34 us, 8192 tokens of 8 / 8 heads 214 ->
  // 163; but four prompts of 512 23 -> 32, and 3000 tokens 91 -> 105 us.
  const bool split = (grid <= 256 && p.n_tokens > 256) || (grid <= 512 && p.n_tokens >= 768ll * p.n_docs);
  if (split)
    packed_kernel<T, DT, FULL, CAP, ALIBI, 2><<<grid, 2 * kThreads, 0, st>>>(p, rule, blocks);
  else
    packed_kernel<T, DT, FULL, CAP, ALIBI, 1><<<grid, kThreads, 0, st>>>(p, rule, blocks);
}

template <typename T, int DT, bool FULL>
void launch_packed(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st) {
  if (p.score_cap > 0.0f) {
    if (p.alibi_slopes)
      launch_packed<T, DT, FULL, true, true>(p, rule, grid, blocks, st);
    else
      launch_packed<T, DT, FULL, true, false>(p, rule, grid, blocks, st);
  } else if (p.alibi_slopes) {
    launch_packed<T, DT, FULL, false, true>(p, rule, grid, blocks, st);
  } else {
    launch_packed<T, DT, FULL, false, false>(p, rule, grid, blocks, st);
  }
}

template <typename T, int DT>
void launch_packed(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st) {
  // a whole tile's lane offsets fit 32 bits (else every row is addressed by itself)
  const bool near = p.k_stride_t >= 0 && p.k_stride_t < (1 << 24) && p.v_stride_t >= 0 && p.v_stride_t < (1 << 24);
  if (p.head_dim == DT && near)
    launch_packed<T, DT, true>(p, rule, grid, blocks, st);
  else
    launch_packed<T, DT, false>(p, rule, grid, blocks, st);
}

template <typename T>
void launch_packed(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st) {
  if (p.head_dim <= 64)
    launch_packed<T, 64>(p, rule, grid, blocks, st);
  else if (p.head_dim <= 128)
    launch_packed<T, 128>(p, rule, grid, blocks, st);
  else
    launch_packed<T, 256>(p, rule, grid, blocks, st);
}

}  // namespace
}  // namespace smaq
