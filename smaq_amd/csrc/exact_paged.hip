// Attention of one new token per sequence over a paged exact cache
// (smaq_paged_attention).
//
// A step moves every visible key and value once: at D = 128 a token-head is 512
// bytes and, with g query heads on it, 512 g operations, so HBM bounds it.  The
// kernel streams rows from the pages straight into the registers that the matrix
// instructions read; nothing but the last merge goes through LDS.
//
//   S^T[token][q] = K . Q^T       A = 16 tokens x 32 dims: lane (n, g) loads the 16
//                                 bytes of dims 32 c + 8 g of token n
//   O^T[dim][q] += V^T . P^T      32 tokens a step.  The k-elements of lane group g
//                                 are tokens 4 g .. 4 g + 3 of both 16-token tiles,
//                                 where S^T's registers leave P^T: P needs no move.
//                                 Lane (n, g) loads dims n D/16 .. of its 8 tokens
//                                 (whole rows over the 16 lanes) and turns that 8 x
//                                 D/16 block with v_perm; matrix e holds dims
//                                 n D/16 + e.
//
// A wave has its own running maximum and sum.  Keys of the next step are loaded as
// soon as this step's products have read theirs, values likewise: half of a step's
// 16 KB is in flight at any time.  The four waves of a workgroup take the steps of one
// head in turn, or four heads side by side (HW = 4): rows of four heads lie next to each
// other, and reading them together is kinder to the memory.
//
// 32 sequences of 32768 tokens, 32 / 8 heads of 128 bf16 dims (4.3 GB): 0.72 ms, 6.0 TB/s;
// 256 of 1 to 4096 tokens, capped (1.5 GB): 0.27 ms, 5.5 TB/s, 13 us of it the merge; one of
// 65408 tokens (134 MB): 34 us, 3.9 TB/s, 6 us of it the merge.  A plain read of that size
// reaches 7.2 TB/s, a copy 5.2.  Weights are rounded to the values' type for the second
// product, as the matrix instruction takes two operands of one type; all else is fp32.
//
// All steps of the batch are dealt to the workgroups in equal shares, however long
// each sequence is: a share begins and ends inside sequences, and a row whose steps
// went to several workgroups is joined from their partial results in order by a second
// launch.  Nothing is atomic; the result depends on the lengths and the launch alone.
#include <algorithm>

#include "exact_attention.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxShares = 1024;
constexpr uint32_t kLeastSteps = 2;  // of a share
constexpr int64_t kLongest = 0x7fff0000;  // positions fit an int, those of 32 rounds ahead too

// How the work is dealt.  `shares` 0: workgroup u takes unit u whole and no merge follows.
// Else share i holds the steps [i W / shares, (i + 1) W / shares) of all W, in the order
// sequence, unit, step; a unit that lies in several shares leaves in each a slot of
// slot_rows rows: slot 1 of the share it starts in, slot 0 of the others.
struct PagedPlan {
  int group;      // heads that a workgroup takes side by side
  int units;      // per sequence: head groups x tiles of 16 query rows
  int tiles;      // of one head group
  int slot_rows;  // heads of a group x rows of a tile
  int shares;
  float *m, *l, *o;  // [shares][2][slot_rows], o with head_dim
  uint32_t* base;    // [batch] first step of each sequence; [batch]: W (below 2^31)
};

// W = `all` steps dealt to the shares that have some (kLeastSteps or more each): the first
// `more` hold each + 1, the others each.
struct Deal {
  uint32_t each, more, shares;
  __device__ __forceinline__ Deal(uint32_t all, uint32_t most) {
    shares = max(1u, min(most, all / kLeastSteps));
    each = all / shares;
    more = all - each * shares;
  }
  __device__ __forceinline__ uint32_t start(uint32_t i) const { return i * each + min(i, more); }
  __device__ __forceinline__ uint32_t owner(uint32_t step) const {
    const uint32_t low = more * (each + 1);
    return step < low ? step / (each + 1) : more + (step - low) / max(each, 1u);
  }
};

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }

// the tokens [first, end) that sequence b's query sees
__device__ __forceinline__ void visible(const smaq_paged_params& p, int b, int& first, int& end) {
  const int64_t n = p.seq_lens_wide ? (int64_t)((const long long*)p.seq_lens)[b] : (int64_t)((const int*)p.seq_lens)[b];
  end = (int)max((int64_t)0, min(min(n, (int64_t)p.max_seq_len), min((int64_t)p.max_blocks * p.block_size, kLongest)));
  if (p.num_blocks == 0) end = 0;
  first = p.window && end > p.window ? end - p.window : 0;
}

// steps of `step` tokens of a unit of sequence b; they start on a page's 16 tokens
__device__ __forceinline__ int unit_steps(const smaq_paged_params& p, int b, int step) {
  int first, last;
  visible(p, b, first, last);
  return last > first ? (int)(((int64_t)last - (first & ~15) + step - 1) / step) : 0;
}

template <typename T, int DT, bool FULL, int HW, bool WHOLE>
__global__ __launch_bounds__(kThreads, DT == 256 ? 2 : 3) void paged_kernel(smaq_paged_params p, ScoreRule rule,
                                                                           PagedPlan plan) {
  constexpr int KC = DT / 32;   // k steps of a product over the head dim
  constexpr int VE = DT / 16;   // dims of a lane, matrices of a V step
  constexpr int VW = VE / 2;    // words of a lane's value row
  constexpr int WPH = 4 / HW;   // waves of a head
  constexpr int STEP = 32 * WPH;
  constexpr int OS = DT + 4;
  __shared__ float so[4][16][OS];
  __shared__ float sm[4][16], sl[4][16];
  // at 256 dims the queries stay in LDS: with them in registers the loop spills
  constexpr bool QL = DT == 256;
  static_assert(!QL || HW == 1, "the waves share the queries in LDS");
  __shared__ uint32_t sq[QL ? 16 : 1][DT / 2 + 4];
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = p.n_q_heads / p.n_kv_heads, D = p.head_dim, bs = p.block_size;

  // ---- this workgroup's steps [at, at_end) and the sequence b (first step `base`) of the first
  int b;
  uint32_t base = 0, at = 0, at_end = 1;
  if constexpr (WHOLE) {
    b = blockIdx.x / plan.units;
  } else {
    // every wave sums the sequences' steps, a run of sequences a lane, and finds the run and
    // then the sequence that hold its first step
    auto scan = [&](uint32_t sum) {
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const uint32_t x = __shfl_up(sum, o, 64);
        sum += lane >= o ? x : 0;
      }
      return sum;
    };
    const uint32_t units = plan.units;
    const int run = (p.batch + 63) / 64;
    uint32_t sum = 0;
    for (int i = lane * run, e = min(p.batch, i + run); i < e; ++i) sum += unit_steps(p, i, STEP);
    const uint32_t in = scan(sum);
    const uint32_t all = (uint32_t)__builtin_amdgcn_readlane((int)in, 63) * units;
    const Deal deal(all, plan.shares);
    if (blockIdx.x == 0 && tid == 0) plan.base[p.batch] = all;
    at_end = 0;
    if (blockIdx.x < deal.shares) {
      at = uniform(deal.start(blockIdx.x));
      at_end = uniform(deal.start(blockIdx.x + 1));
    }
    // the lanes whose run ends at or before the first step come first
    const int in_run = min((int)__popcll(__ballot(in * units <= at)), 63);
    b = in_run * run;
    base = (uint32_t)__builtin_amdgcn_readlane((int)(in - sum), in_run) * units;
    for (int left = run; left > 1 && at < at_end; left -= 64) {
      const int i = b + lane;
      const uint32_t mine = lane < left && i < p.batch ? unit_steps(p, i, STEP) : 0;
      const uint32_t upto = scan(mine);
      const int past = (int)__popcll(__ballot(base + upto * units <= at));
      if (past < 64) {
        base += (uint32_t)__builtin_amdgcn_readlane((int)(upto - mine), past) * units;
        b += past;
        break;
      }
      base += (uint32_t)__builtin_amdgcn_readlane((int)upto, 63) * units;
      b += 64;
    }
    // rows that see no token
    for (int i = blockIdx.x; i < p.batch; i += gridDim.x)
      if (unit_steps(p, i, STEP) == 0)
        for (int u = tid; u < p.n_q_heads * (D / 4); u += kThreads)
          *(u32x2v*)((T*)p.out + (int64_t)i * p.out_stride_b + (u / (D / 4)) * p.out_stride_h + 4 * (u % (D / 4))) = u32x2v{0, 0};
    if (at >= at_end) return;
  }
  const uint32_t at_first = at;

  while (at < at_end) {
    int first, last;
    visible(p, b, first, last);
    first = uniform(first);
    last = uniform(last);
    int unit, begin = first & ~15, end = last;
    bool direct = true;
    uint32_t unit0 = 0, stop = at_end;
    if constexpr (WHOLE) {
      unit = blockIdx.x % plan.units;
    } else {
      const uint32_t steps = last > first ? (uint32_t)(last - begin + STEP - 1) / STEP : 0, here = steps * plan.units;
      if (at >= base + here) {
        base += here;
        ++b;
        continue;
      }
      if (at == base && tid == 0) plan.base[b] = base;
      unit = uniform((at - base) / steps);
      unit0 = base + unit * steps;
      stop = min(unit0 + steps, at_end);
      direct = at == unit0 && stop == unit0 + steps;
      end = min(begin + (int)(stop - unit0) * STEP, last);
      begin += (int)(at - unit0) * STEP;
    }

    const int tile = unit % plan.tiles, h0 = unit / plan.tiles * HW, h = HW == 1 ? h0 : h0 + w;
    const int row = 16 * tile + n, hq = h * rows + row;
    const int* table = p.block_table + (int64_t)b * p.max_blocks;
    const T* kc = (const T*)p.k_cache + h * p.k_stride_h;
    const T* vc = (const T*)p.v_cache + h * p.v_stride_h;
    const uint32_t klane = (uint32_t)(2 * n * p.k_stride_t + 16 * g);
    const uint32_t vlane = (uint32_t)(2 * 4 * g * p.v_stride_t + 2 * VE * n);

    auto load_q = [&](int c) {
      u32x4v x = {0, 0, 0, 0};
      if (row < rows && (FULL || 32 * c + 8 * g < D))
        x = *(const u32x4v*)((const T*)p.q + (int64_t)b * p.q_stride_b + hq * p.q_stride_h + 32 * c + 8 * g);
      return x;
    };
    u32x4v qr[QL ? 1 : KC];
    if constexpr (QL) {
#pragma unroll
      for (int c = 0; c < KC; c += 4) *(u32x4v*)&sq[n][16 * (c + w) + 4 * g] = load_q(c + w);
      __syncthreads();
    } else {
#pragma unroll
      for (int c = 0; c < KC; ++c) qr[c] = load_q(c);
    }
    const float slope = p.alibi_slopes && row < rows ? p.alibi_slopes[hq] * kLog2eF : 0.0f;

    // pages of this wave's next 32 steps, two 16-token tiles each, one per lane
    auto load_ids = [&](int t) {
      const int tt = t + STEP * (lane >> 1) + 16 * (lane & 1);
      int id = -1;
      if (tt < end) id = table[(uint32_t)tt / (uint32_t)bs];
      return id >= 0 && id < p.num_blocks ? id : -1;
    };

    f32x4v acc[VE];
#pragma unroll
    for (int e = 0; e < VE; ++e) acc[e] = f32x4v{0.f, 0.f, 0.f, 0.f};
    float m_ref = kNegInf, m_use = 0.0f, m_thr = kNegInf, l = 0.0f;
    bool some = false;

    u32x4v kr[2][KC];
    uint32_t vr[2][4][VW];
    auto load_k = [&](int t, const int* id) {
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t off = (uint32_t)(t + 16 * a) % (uint32_t)bs;
        const char* src = (const char*)(kc + (int64_t)max(id[a], 0) * p.k_stride_block + (int64_t)off * p.k_stride_t);
#pragma unroll
        for (int c = 0; c < KC; ++c) {
          if (FULL || 32 * c + 8 * g < D)
            kr[a][c] = *(const u32x4v*)(src + klane + 64 * c);
          else
            kr[a][c] = u32x4v{0, 0, 0, 0};
        }
      }
    };
    // whether the rows of a step are all there and seen
    auto whole_step = [&](int t, const int* id) { return id[0] >= 0 && id[1] >= 0 && t >= first && t + 32 <= end; };
    // a value that is not seen must not meet its zero weight: it is read as 0
    auto load_v = [&](int t, const int* id) {
      const bool inside = whole_step(t, id);
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        const uint32_t off = (uint32_t)(t + 16 * a) % (uint32_t)bs;
        const char* src = (const char*)(vc + (int64_t)max(id[a], 0) * p.v_stride_block + (int64_t)off * p.v_stride_t);
        auto rows_of = [&](auto seen) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const char* r = src + 2 * j * p.v_stride_t + vlane;
            if constexpr (VW == 2) {
              u32x2v x = {0, 0};
              if (seen(j) && (FULL || VE * n < D)) x = *(const u32x2v*)r;
              vr[a][j][0] = x[0];
              vr[a][j][1] = x[1];
            } else {
#pragma unroll
              for (int c = 0; c < VW / 4; ++c) {
                u32x4v x = {0, 0, 0, 0};
                if (seen(j) && (FULL || VE * n + 8 * c < D)) x = *(const u32x4v*)(r + 16 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) vr[a][j][4 * c + e] = x[e];
              }
            }
          }
        };
        if (inside)
          rows_of([](int) { return true; });
        else
          rows_of([&](int j) {
            const int tok = t + 16 * a + 4 * g + j;
            return id[a] >= 0 && tok >= first && tok < end;
          });
      }
    };

    int t = begin + 32 * (w % WPH);
    int step = 0, ids = -1, id[2], nid[2];
    if (t < end) {
      ids = load_ids(t);
      id[0] = __builtin_amdgcn_readlane(ids, 0);
      id[1] = __builtin_amdgcn_readlane(ids, 1);
      load_k(t, id);
      load_v(t, id);
    }
    for (; t < end; t += STEP) {
      const bool more = t + STEP < end;
      if (more) {
        if (++step == 32) {
          step = 0;
          ids = load_ids(t + STEP);
        }
        nid[0] = __builtin_amdgcn_readlane(ids, 2 * step);
        nid[1] = __builtin_amdgcn_readlane(ids, 2 * step + 1);
      }
      f32x4v s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      if constexpr (QL) asm volatile("" ::: "memory");  // read again each step
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        u32x4v q;
        if constexpr (QL) q = *(const u32x4v*)&sq[n][16 * c + 4 * g]; else q = qr[c];
#pragma unroll
        for (int a = 0; a < 2; ++a) s[a] = Mat<T>::mma16(kr[a][c], q, s[a]);
      }
      if (more) load_k(t + STEP, nid);
      const bool inside = whole_step(t, id);
      float x[2][4], mx = kNegInf;
      const float gap = (float)(last - 1 - t - 4 * g);
      each_score<8>(rule, [&](int i) { return s[i / 4][i % 4]; }, [&](int i, float y) { x[i / 4][i % 4] = y; });
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p.alibi_slopes) x[a][i] = fmaf(-slope, gap - (float)(16 * a + i), x[a][i]);
          if (!inside) {
            const int tok = t + 16 * a + 4 * g + i;
            const bool ok = id[a] >= 0 && tok >= first && tok < end;
            x[a][i] = ok ? x[a][i] : kNegInf;
            some |= ok;
          }
          mx = fmaxf(mx, x[a][i]);
        }
      some |= inside;
      if (__any(mx > m_thr)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_ref, mx);
        m_use = m_new == kNegInf ? 0.0f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_ref - m_use);
        l *= alpha;
#pragma unroll
        for (int e = 0; e < VE; ++e) acc[e] *= alpha;
        m_ref = m_new;
        m_thr = m_new + kRaise;
      }
      u32x4v pt;
#pragma unroll
      for (int a = 0; a < 2; ++a) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = __builtin_amdgcn_exp2f(x[a][i] - m_use);
          l += e[i];
        }
        pt[2 * a] = Mat<T>::pack(e[0], e[1]);
        pt[2 * a + 1] = Mat<T>::pack(e[2], e[3]);
      }
#pragma unroll
      for (int e = 0; e < VW; ++e) {
        u32x4v lo, hi;
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            lo[2 * a + j] = low_halves(vr[a][2 * j][e], vr[a][2 * j + 1][e]);
            hi[2 * a + j] = high_halves(vr[a][2 * j][e], vr[a][2 * j + 1][e]);
          }
        acc[2 * e] = Mat<T>::mma16(lo, pt, acc[2 * e]);
        acc[2 * e + 1] = Mat<T>::mma16(hi, pt, acc[2 * e + 1]);
      }
      if (more) load_v(t + STEP, nid);
      id[0] = nid[0];
      id[1] = nid[1];
    }

    // ---- the waves' (m, l, o).  A wave that saw a NaN score has m = +inf, so that its
    // weight is NaN; one that saw scores of -inf alone has l = NaN and counts only when no
    // wave saw more.
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (l != l)
      m_ref = __builtin_inff();
    else if (m_ref == kNegInf && __any(some))
      l = __builtin_nanf("");
    if (g == 0) {
      sm[w][n] = m_ref;
      sl[w][n] = l;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VE; e += 4)
        *(f32x4v*)&so[w][n][VE * (4 * g + i) + e] = f32x4v{acc[e][i], acc[e + 1][i], acc[e + 2][i], acc[e + 3][i]};
    __syncthreads();
    const int live = min(16, rows - 16 * tile);
    const int64_t slot = 2 * (int64_t)blockIdx.x + (at_first > unit0 ? 0 : 1);
    for (int u = tid; u < HW * live * (DT / 4); u += kThreads) {
      const int hs = u / (live * (DT / 4)), r = u / (DT / 4) % live, d = 4 * (u % (DT / 4));
      if (!FULL && d >= D) continue;
      float m = kNegInf;
#pragma unroll
      for (int x = 0; x < WPH; ++x) m = fmaxf(m, sm[hs * WPH + x][r]);
      f32x4v o = {0.f, 0.f, 0.f, 0.f};
      float sum = 0.0f;
#pragma unroll
      for (int x = 0; x < WPH; ++x) {
        const float mw = sm[hs * WPH + x][r];
        if (mw == kNegInf && m != kNegInf) continue;
        const float a = m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
        sum = fmaf(a, sl[hs * WPH + x][r], sum);
        o += a * *(const f32x4v*)&so[hs * WPH + x][r][d];
      }
      if (direct) {
        const float inv = begin < end && !(m == kNegInf && sum == 0.0f) ? 1.0f / sum : 0.0f;
        T* dst = (T*)p.out + (int64_t)b * p.out_stride_b + ((h0 + hs) * rows + 16 * tile + r) * p.out_stride_h + d;
        *(u32x2v*)dst = u32x2v{Mat<T>::pack(o[0] * inv, o[1] * inv), Mat<T>::pack(o[2] * inv, o[3] * inv)};
      } else {
        const int64_t i = slot * plan.slot_rows + hs * min(16, rows) + r;
        *(f32x4v*)(plan.o + i * D + d) = o;
        if (d == 0) {
          plan.m[i] = m;
          plan.l[i] = sum;
        }
      }
    }
    at = stop;
    if (at < at_end) __syncthreads();  // the next unit writes the same LDS
  }
}

// One row whose steps went to several shares, joined in their order: a workgroup a
// row.  First the partial results' weights into LDS, then thread (x, y) sums dims 4 x of
// every ny-th, and the ny sums are added in order.
template <typename T, int THREADS>
__global__ __launch_bounds__(THREADS) void paged_merge_kernel(smaq_paged_params p, PagedPlan plan) {
  __shared__ float sa[kMaxShares], sl[kMaxShares];
  __shared__ float so[THREADS][4], red[2][THREADS / 64];
  const int tid = threadIdx.x, b = blockIdx.x / p.n_q_heads, hq = blockIdx.x % p.n_q_heads, D = p.head_dim;
  const int steps = unit_steps(p, b, 128 / plan.group);
  if (steps == 0) return;
  const int rows = p.n_q_heads / p.n_kv_heads, h = hq / rows, row = hq % rows;
  const uint32_t all = plan.base[p.batch];
  const uint32_t unit0 = plan.base[b] + (uint32_t)(h / plan.group * plan.tiles + row / 16) * steps;
  const Deal deal(all, plan.shares);
  const uint32_t g0 = deal.owner(unit0), g1 = deal.owner(unit0 + steps - 1);
  if (g0 == g1) return;
  const int live = g1 - g0 + 1, in_slot = h % plan.group * min(16, rows) + row % 16;
  // the i-th: slot 1 of share g0, then slots 0
  auto at = [&](int i) { return (int64_t)(2 * (g0 + i) + (i == 0)) * plan.slot_rows + in_slot; };
  const int nx = D / 4, ny = THREADS / nx, x = tid % nx, y = tid / nx;
  // the first results are on their way before the first wait, the next ones while those
  // are added
  constexpr int AHEAD = 4;
  f32x4v v[2][AHEAD];
  auto fetch = [&](int k0, f32x4v* u) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = y + (k0 + k) * ny;
      u[k] = f32x4v{0.f, 0.f, 0.f, 0.f};
      if (y < ny && i < live) u[k] = *(const f32x4v*)(plan.o + at(i) * D + 4 * x);
    }
  };
  fetch(0, v[0]);
  fetch(AHEAD, v[1]);
  float m = kNegInf, l = 0.0f;
  for (int i = tid; i < live; i += THREADS) {
    sa[i] = plan.m[at(i)];
    sl[i] = plan.l[at(i)];
    m = fmaxf(m, sa[i]);
  }
  m = warp_max(m);
  if (THREADS > 64) {
    if ((tid & 63) == 0) red[0][tid >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) m = fmaxf(m, red[0][i]);
  }
  for (int i = tid; i < live; i += THREADS) {
    const float mi = sa[i];
    const float a = m == kNegInf ? 1.0f : (mi == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(mi - m));
    sa[i] = a;
    if (a != 0.0f) l = fmaf(a, sl[i], l);  // NaN is not 0
  }
  l = warp_sum(l);
  if ((tid & 63) == 0) red[1][tid >> 6] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int i = 0; i < THREADS / 64; ++i) l += red[1][i];
  f32x4v o = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](int k0, const f32x4v* u) {
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int i = y + (k0 + k) * ny;
      if (y >= ny || i >= live || sa[i] == 0.0f) continue;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = fmaf(sa[i], u[k][e], o[e]);
    }
  };
  for (int k0 = 0; k0 * ny < live; k0 += 2 * AHEAD) {
    add(k0, v[0]);
    fetch(k0 + 2 * AHEAD, v[0]);
    add(k0 + AHEAD, v[1]);
    fetch(k0 + 3 * AHEAD, v[1]);
  }
  *(f32x4v*)so[tid] = o;
  __syncthreads();
  if (y != 0) return;
  for (int k = 1; k < ny; ++k) o += *(const f32x4v*)so[x + k * nx];
  const float inv = m == kNegInf && l == 0.0f ? 0.0f : 1.0f / l;
  T* dst = (T*)p.out + (int64_t)b * p.out_stride_b + hq * p.out_stride_h + 4 * x;
  *(u32x2v*)dst = u32x2v{Mat<T>::pack(o[0] * inv, o[1] * inv), Mat<T>::pack(o[2] * inv, o[3] * inv)};
}

int check_paged(const smaq_paged_params* p) {
  SMAQ_REQUIRE(p, "smaq_paged_attention: null parameters");
  SMAQ_REQUIRE(p->batch >= 0 && p->batch <= 65535 && p->n_q_heads > 0 && p->n_kv_heads > 0 &&
                   p->n_q_heads % p->n_kv_heads == 0 && p->n_q_heads <= 1024,
               "smaq_paged_attention: bad shape (%d sequences, %d heads over %d)", p->batch, p->n_q_heads, p->n_kv_heads);
  SMAQ_REQUIRE(p->head_dim > 0 && p->head_dim <= 256 && p->head_dim % 8 == 0,
               "smaq_paged_attention: head_dim %d is not a multiple of 8 up to 256", p->head_dim);
  SMAQ_REQUIRE(p->block_size > 0 && p->block_size % 16 == 0 && p->block_size <= 65536 && p->num_blocks >= 0 &&
                   p->max_blocks >= 0 && p->max_seq_len >= 0,
               "smaq_paged_attention: block_size %d must be a multiple of 16 (num_blocks %d, max_blocks %d, max_seq_len "
               "%lld of 0 or more)", p->block_size, p->num_blocks, p->max_blocks, p->max_seq_len);
  SMAQ_REQUIRE(p->window >= 0 && score_range(p->scale, p->score_cap),
               "smaq_paged_attention: window %d must be 0 or more, score_cap %g 0 or in 1e-30..1e30, scale %g below 1e38",
               p->window, (double)p->score_cap, (double)p->scale);
  if (p->dtype != SMAQ_F16 && p->dtype != SMAQ_BF16) {
    set_error("smaq_paged_attention: unsupported dtype %d", p->dtype);
    return SMAQ_EUNSUPPORTED;
  }
  return SMAQ_OK;
}

PagedPlan make_plan(const smaq_paged_params* p) {
  const int rows = p->n_q_heads / p->n_kv_heads;
  PagedPlan plan{};
  plan.tiles = (rows + 15) / 16;
  const int64_t longest = std::min<int64_t>(std::min<int64_t>(p->max_seq_len, (int64_t)p->max_blocks * p->block_size), kLongest);
  const int64_t span = p->window ? std::min<int64_t>(longest, (int64_t)p->window + 15) : longest;
  const int64_t room = 256 * (p->head_dim <= 64 ? 4 : p->head_dim <= 128 ? 3 : 2);  // workgroups the card holds
  const int64_t heads = (int64_t)p->n_kv_heads * plan.tiles * p->batch;
  // four heads side by side while that leaves every workgroup four steps of 32 tokens (at
  // 256 dims a row is long enough by itself)
  const bool wide = p->head_dim <= 128 && p->n_kv_heads % 4 == 0 && (span + 31) / 32 * (heads / 4) >= 4 * room;
  const int64_t most = wide ? (span + 31) / 32 * (heads / 4) : (span + 127) / 128 * heads;
  // Few units are cut into no more than 64 pieces each beyond one workgroup a CU: one
  // sequence of 65408 tokens runs as long with 256 workgroups as with 768 (26 us), and its
  // merge 6 us instead of 9.
  const int64_t pieces = std::max<int64_t>(256, 64 * (wide ? heads / 4 : heads));
  if (span > 256 && most < (1ll << 31))
    plan.shares = (int)std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(room, pieces), most / kLeastSteps));
  plan.group = wide && plan.shares ? 4 : 1;
  plan.units = p->n_kv_heads / plan.group * plan.tiles;
  plan.slot_rows = plan.group * std::min(16, rows);
  return plan;
}

int64_t plan_bytes(const smaq_paged_params* p, const PagedPlan& plan) {
  if (plan.shares == 0) return 0;
  const int64_t rows = 2 * (int64_t)plan.shares * plan.slot_rows;
  return rows * (p->head_dim + 2) * (int64_t)sizeof(float) + ((int64_t)p->batch + 1) * (int64_t)sizeof(uint32_t);
}

template <typename T, int DT, int HW, bool WHOLE>
void launch_paged(const smaq_paged_params& p, const ScoreRule& rule, const PagedPlan& plan, unsigned blocks, hipStream_t st) {
  if (p.head_dim == DT)
    paged_kernel<T, DT, true, HW, WHOLE><<<blocks, kThreads, 0, st>>>(p, rule, plan);
  else
    paged_kernel<T, DT, false, HW, WHOLE><<<blocks, kThreads, 0, st>>>(p, rule, plan);
}

template <typename T, int DT>
void launch_paged(const smaq_paged_params& p, const ScoreRule& rule, const PagedPlan& plan, unsigned blocks, hipStream_t st) {
  if (plan.shares == 0) return launch_paged<T, DT, 1, true>(p, rule, plan, blocks, st);
  if constexpr (DT <= 128)
    if (plan.group == 4) return launch_paged<T, DT, 4, false>(p, rule, plan, blocks, st);
  launch_paged<T, DT, 1, false>(p, rule, plan, blocks, st);
}

template <typename T>
void launch_paged(const smaq_paged_params& p, const ScoreRule& rule, const PagedPlan& plan, unsigned blocks, hipStream_t st) {
  if (p.head_dim > 128)
    launch_paged<T, 256>(p, rule, plan, blocks, st);
  else if (p.head_dim > 64)
    launch_paged<T, 128>(p, rule, plan, blocks, st);
  else
    launch_paged<T, 64>(p, rule, plan, blocks, st);
  if (plan.shares <= 1) return;
  const unsigned rows = (unsigned)(p.batch * p.n_q_heads);
  if (rows <= 1024)
    paged_merge_kernel<T, 256><<<rows, 256, 0, st>>>(p, plan);
  else
    paged_merge_kernel<T, 64><<<rows, 64, 0, st>>>(p, plan);
}

}  // namespace
}  // namespace smaq

extern "C" long long smaq_paged_workspace_bytes(const smaq_paged_params* p) {
  using namespace smaq;
  if (check_paged(p) != SMAQ_OK) return -1;
  return p->batch ? plan_bytes(p, make_plan(p)) : 0;
}

extern "C" int smaq_paged_attention(const smaq_paged_params* p, void* stream) {
  using namespace smaq;
  const int bad = check_paged(p);
  if (bad != SMAQ_OK) return bad;
  if (p->batch == 0) return SMAQ_OK;
  SMAQ_REQUIRE(p->q && p->out && p->seq_lens && (!p->max_blocks || p->block_table) &&
                   (!p->num_blocks || (p->k_cache && p->v_cache)),
               "smaq_paged_attention: null pointer");
  SMAQ_REQUIRE(rows_on_16(p->q, p->q_stride_b, p->q_stride_h) && rows_on_16(p->out, p->out_stride_b, p->out_stride_h) &&
                   rows_on_16(p->k_cache, p->k_stride_block, p->k_stride_t, p->k_stride_h) &&
                   rows_on_16(p->v_cache, p->v_stride_block, p->v_stride_t, p->v_stride_h),
               "smaq_paged_attention: rows must start on 16 bytes");
  SMAQ_REQUIRE(p->k_stride_t >= 0 && p->v_stride_t >= 0 && p->k_stride_t < (1ll << 26) && p->v_stride_t < (1ll << 26),
               "smaq_paged_attention: a token stride of %lld or %lld elements is not below 2^26", p->k_stride_t,
               p->v_stride_t);
  PagedPlan plan = make_plan(p);
  const int64_t need = plan_bytes(p, plan);
  SMAQ_REQUIRE(need == 0 || (p->workspace && p->workspace_bytes >= need && (uintptr_t)p->workspace % 16 == 0),
               "smaq_paged_attention: a 16-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need,
               p->workspace_bytes);
  if (plan.shares) {
    const int64_t rows = 2 * (int64_t)plan.shares * plan.slot_rows;
    plan.o = (float*)p->workspace;
    plan.m = plan.o + rows * p->head_dim;
    plan.l = plan.m + rows;
    plan.base = (uint32_t*)(plan.l + rows);
  }
  const int64_t blocks = plan.shares ? plan.shares : (int64_t)p->batch * plan.units;
  const ScoreRule rule = score_rule(p->scale, p->score_cap);
  if (p->dtype == SMAQ_F16)
    launch_paged<_Float16>(*p, rule, plan, (unsigned)blocks, (hipStream_t)stream);
  else
    launch_paged<bf16>(*p, rule, plan, (unsigned)blocks, (hipStream_t)stream);
  return launch_status("smaq_paged_attention");
}
