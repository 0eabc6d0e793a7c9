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
// A wave has its own running maximum and sum; four waves take 32-token steps in
// turn, so a workgroup covers 128 tokens a round.  Keys of the next step are
// loaded as soon as this step's products have read theirs, values likewise: half
// of a step's 16 KB is in flight at any time.
#include <algorithm>

#include "exact_attention.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr int kRound = 128;  // tokens of a round of the four waves
constexpr int64_t kLongest = 0x7fff0000;  // positions fit an int, those of 32 rounds ahead too

struct PagedPart {  // partials of [batch * n_q_heads] rows and `splits` splits
  float *m, *l, *o;
  int splits;
  int64_t split_len;
};

// the tokens [first, end) that sequence b's query sees
__device__ __forceinline__ void visible(const smaq_paged_params& p, int b, int& first, int& end) {
  const int64_t n = p.seq_lens_wide ? (int64_t)((const long long*)p.seq_lens)[b] : (int64_t)((const int*)p.seq_lens)[b];
  end = (int)max((int64_t)0, min(min(n, (int64_t)p.max_seq_len), min((int64_t)p.max_blocks * p.block_size, kLongest)));
  if (p.num_blocks == 0) end = 0;
  first = p.window && end > p.window ? end - p.window : 0;
}

template <typename T, int DT, bool FULL>
__global__ __launch_bounds__(kThreads, DT == 256 ? 2 : 3) void paged_kernel(smaq_paged_params p, ScoreRule rule,
                                                                           PagedPart part) {
  constexpr int KC = DT / 32;  // k steps of a product over the head dim
  constexpr int VE = DT / 16;  // dims of a lane, matrices of a V step
  constexpr int VW = VE / 2;   // words of a lane's value row
  constexpr int OS = DT + 4;
  __shared__ float so[4][16][OS];
  __shared__ float sm[4][16], sl[4][16];
  // at 256 dims the queries stay in LDS: with them in registers the loop spills
  constexpr bool QL = DT == 256;
  __shared__ uint32_t sq[QL ? 16 : 1][DT / 2 + 4];
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int rows = p.n_q_heads / p.n_kv_heads, tiles = (rows + 15) / 16;
  int idx = blockIdx.x;
  const int tile = idx % tiles;
  idx /= tiles;
  const int h = idx % p.n_kv_heads;
  idx /= p.n_kv_heads;
  const int split = idx % part.splits, b = idx / part.splits;
  int first, last;
  visible(p, b, first, last);
  const int64_t begin64 = (first & ~15) + split * part.split_len;
  const int begin = (int)min(begin64, (int64_t)last), end = (int)min(begin64 + part.split_len, (int64_t)last);
  const bool direct = part.splits == 1;
  if (begin >= end && !direct) return;  // the merge knows

  const int D = p.head_dim, bs = p.block_size;
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
    const int tt = t + kRound * (lane >> 1) + 16 * (lane & 1);
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
  auto load_v = [&](int t, const int* id) {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      const uint32_t off = (uint32_t)(t + 16 * a) % (uint32_t)bs;
      const char* src = (const char*)(vc + (int64_t)max(id[a], 0) * p.v_stride_block + (int64_t)off * p.v_stride_t);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const char* r = src + 2 * j * p.v_stride_t + vlane;
        if constexpr (VW == 2) {
          u32x2v x = {0, 0};
          if (FULL || VE * n < D) x = *(const u32x2v*)r;
          vr[a][j][0] = x[0];
          vr[a][j][1] = x[1];
        } else {
#pragma unroll
          for (int c = 0; c < VW / 4; ++c) {
            u32x4v x = {0, 0, 0, 0};
            if (FULL || VE * n + 8 * c < D) x = *(const u32x4v*)(r + 16 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) vr[a][j][4 * c + e] = x[e];
          }
        }
      }
    }
  };

  int t = begin + 32 * w;
  int step = 0, ids = -1, id[2], nid[2];
  if (t < end) {
    ids = load_ids(t);
    id[0] = __builtin_amdgcn_readlane(ids, 0);
    id[1] = __builtin_amdgcn_readlane(ids, 1);
    load_k(t, id);
    load_v(t, id);
  }
  for (; t < end; t += kRound) {
    const bool more = t + kRound < end;
    if (more) {
      if (++step == 32) {
        step = 0;
        ids = load_ids(t + kRound);
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
    if (more) load_k(t + kRound, nid);
    const bool whole = id[0] >= 0 && id[1] >= 0 && t >= first && t + 32 <= end;
    float x[2][4], mx = kNegInf;
    const float gap = (float)(last - 1 - t - 4 * g);
    each_score<8>(rule, [&](int i) { return s[i / 4][i % 4]; }, [&](int i, float y) { x[i / 4][i % 4] = y; });
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (p.alibi_slopes) x[a][i] = fmaf(-slope, gap - (float)(16 * a + i), x[a][i]);
        if (!whole) {
          const int tok = t + 16 * a + 4 * g + i;
          const bool ok = id[a] >= 0 && tok >= first && tok < end;
          x[a][i] = ok ? x[a][i] : kNegInf;
          some |= ok;
        }
        mx = fmaxf(mx, x[a][i]);
      }
    some |= whole;
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
    if (!whole) {  // a masked value must not meet a zero weight
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int tok = t + 16 * a + 4 * g + j;
          const bool ok = id[a] >= 0 && tok >= first && tok < end;
#pragma unroll
          for (int e = 0; e < VW; ++e) vr[a][j][e] = ok ? vr[a][j][e] : 0u;
        }
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
    if (more) load_v(t + kRound, nid);
    id[0] = nid[0];
    id[1] = nid[1];
  }

  // the four waves' (m, l, o) into one.  A wave that saw a NaN score has m = +inf, so
  // that its weight is NaN; one that saw scores of -inf alone has l = NaN and counts
  // only when no wave saw more.
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
  for (int u = threadIdx.x; u < live * (DT / 4); u += kThreads) {
    const int r = u / (DT / 4), d = 4 * (u % (DT / 4));
    if (!FULL && d >= D) continue;
    float m = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
    f32x4v o = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.0f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float mw = sm[x][r];
      if (mw == kNegInf && m != kNegInf) continue;
      const float a = m == kNegInf ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
      sum = fmaf(a, sl[x][r], sum);
      o += a * *(const f32x4v*)&so[x][r][d];
    }
    const int hr = h * rows + 16 * tile + r;
    if (direct) {
      const float inv = begin < end && !(m == kNegInf && sum == 0.0f) ? 1.0f / sum : 0.0f;
      T* dst = (T*)p.out + (int64_t)b * p.out_stride_b + hr * p.out_stride_h + d;
      *(u32x2v*)dst = u32x2v{Mat<T>::pack(o[0] * inv, o[1] * inv), Mat<T>::pack(o[2] * inv, o[3] * inv)};
    } else {
      const int64_t i = ((int64_t)b * p.n_q_heads + hr) * part.splits + split;
      *(f32x4v*)(part.o + i * D + d) = o;
      if (d == 0) {
        part.m[i] = m;
        part.l[i] = sum;
      }
    }
  }
}

// The splits of one row joined in their order: a workgroup a row.  First the splits'
// weights into LDS, then thread (x, y) sums dims 4 x of every ny-th split, and the ny
// sums are added in order.
constexpr int kMaxSplits = 3072;

template <typename T>
__global__ __launch_bounds__(kThreads) void paged_merge_kernel(smaq_paged_params p, PagedPart part) {
  __shared__ float sa[kMaxSplits];
  __shared__ float so[kThreads][4], red[kThreads / 64];
  const int tid = threadIdx.x, b = blockIdx.x / p.n_q_heads, hq = blockIdx.x % p.n_q_heads, D = p.head_dim;
  int first, last;
  visible(p, b, first, last);
  const int64_t span = last - (first & ~15);
  const int live = last > first ? (int)((span + part.split_len - 1) / part.split_len) : 0;
  const int64_t i0 = (int64_t)blockIdx.x * part.splits;
  float m = kNegInf;
  for (int s = tid; s < live; s += kThreads) {
    sa[s] = part.m[i0 + s];
    m = fmaxf(m, sa[s]);
  }
  m = warp_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) m = fmaxf(m, red[w]);
  __syncthreads();
  // a split of scores of -inf alone (m = -inf, l = NaN) counts only when all are
  float l = 0.0f;
  for (int s = tid; s < live; s += kThreads) {
    const float ms = sa[s];
    const float a = m == kNegInf ? 1.0f : (ms == kNegInf ? 0.0f : __builtin_amdgcn_exp2f(ms - m));
    sa[s] = a;
    if (a != 0.0f) l = fmaf(a, part.l[i0 + s], l);  // NaN is not 0
  }
  l = warp_sum(l);
  if ((tid & 63) == 0) red[tid >> 6] = l;
  __syncthreads();
  l = 0.0f;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) l += red[w];
  const int nx = D / 4, ny = kThreads / nx, x = tid % nx, y = tid / nx;
  f32x4v o = {0.f, 0.f, 0.f, 0.f};
  if (y < ny) {
    const float* src = part.o + i0 * D + 4 * x;
#pragma unroll 8
    for (int s = y; s < live; s += ny) {
      const float a = sa[s];
      const f32x4v v = *(const f32x4v*)(src + (int64_t)s * D);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = a != 0.0f ? fmaf(a, v[e], o[e]) : o[e];
    }
  }
  *(f32x4v*)so[tid] = o;
  __syncthreads();
  if (y != 0) return;
  for (int k = 1; k < ny; ++k) o += *(const f32x4v*)so[x + k * nx];
  const float inv = live > 0 && !(m == kNegInf && l == 0.0f) ? 1.0f / l : 0.0f;
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
  SMAQ_REQUIRE(p->window >= 0 && p->score_cap >= 0.0f && p->score_cap < 1e30f && p->scale == p->scale,
               "smaq_paged_attention: window %d, score_cap %g and scale %g must be numbers of 0 or more, finite and a "
               "number", p->window, (double)p->score_cap, (double)p->scale);
  if (p->dtype != SMAQ_F16 && p->dtype != SMAQ_BF16) {
    set_error("smaq_paged_attention: unsupported dtype %d", p->dtype);
    return SMAQ_EUNSUPPORTED;
  }
  return SMAQ_OK;
}

// Splits of the longest sequence.  Enough workgroups for four rounds of the card (three
// to a CU), but none of fewer than 256 tokens.
PagedPart plan_splits(const smaq_paged_params* p) {
  const int64_t longest = std::min<int64_t>(std::min<int64_t>(p->max_seq_len, (int64_t)p->max_blocks * p->block_size), kLongest);
  int64_t span = p->window ? std::min<int64_t>(longest, (int64_t)p->window + 15) : longest;
  span = std::max<int64_t>(span, 1);
  const int rows = p->n_q_heads / p->n_kv_heads;
  const int64_t units = (int64_t)p->batch * p->n_kv_heads * ((rows + 15) / 16);
  const int64_t want = kMaxSplits;
  int64_t len = (span * units + want - 1) / want;
  len = std::max<int64_t>((len + kRound - 1) / kRound * kRound, 256);
  PagedPart part{nullptr, nullptr, nullptr, (int)((span + len - 1) / len), len};
  return part;
}

int64_t part_bytes(const smaq_paged_params* p, const PagedPart& part) {
  if (part.splits == 1) return 0;
  return (int64_t)p->batch * p->n_q_heads * part.splits * (p->head_dim + 2) * (int64_t)sizeof(float);
}

template <typename T, int DT>
void launch_paged(const smaq_paged_params& p, const ScoreRule& rule, const PagedPart& part, unsigned blocks, hipStream_t st) {
  if (p.head_dim == DT)
    paged_kernel<T, DT, true><<<blocks, kThreads, 0, st>>>(p, rule, part);
  else
    paged_kernel<T, DT, false><<<blocks, kThreads, 0, st>>>(p, rule, part);
}

template <typename T>
void launch_paged(const smaq_paged_params& p, const ScoreRule& rule, const PagedPart& part, unsigned blocks, hipStream_t st) {
  if (p.head_dim <= 64)
    launch_paged<T, 64>(p, rule, part, blocks, st);
  else if (p.head_dim <= 128)
    launch_paged<T, 128>(p, rule, part, blocks, st);
  else
    launch_paged<T, 256>(p, rule, part, blocks, st);
  if (part.splits > 1) paged_merge_kernel<T><<<(unsigned)(p.batch * p.n_q_heads), kThreads, 0, st>>>(p, part);
}

}  // namespace
}  // namespace smaq

extern "C" long long smaq_paged_workspace_bytes(const smaq_paged_params* p) {
  using namespace smaq;
  if (check_paged(p) != SMAQ_OK) return -1;
  return p->batch ? part_bytes(p, plan_splits(p)) : 0;
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
  PagedPart part = plan_splits(p);
  const int64_t need = part_bytes(p, part);
  SMAQ_REQUIRE(need == 0 || (p->workspace && p->workspace_bytes >= need && (uintptr_t)p->workspace % 16 == 0),
               "smaq_paged_attention: a 16-byte aligned workspace of %lld bytes is needed, got %lld", (long long)need,
               p->workspace_bytes);
  const int64_t rows = (int64_t)p->batch * p->n_q_heads;
  part.o = (float*)p->workspace;
  if (part.splits > 1) {
    part.m = part.o + rows * part.splits * p->head_dim;
    part.l = part.m + rows * part.splits;
  }
  const int tiles = (p->n_q_heads / p->n_kv_heads + 15) / 16;
  const int64_t blocks = (int64_t)p->batch * part.splits * p->n_kv_heads * tiles;
  SMAQ_REQUIRE(blocks <= 0x7fffffffll, "smaq_paged_attention: %lld workgroups are more than one launch takes",
               (long long)blocks);
  const ScoreRule rule = score_rule(p->scale, p->score_cap);
  if (p->dtype == SMAQ_F16)
    launch_paged<_Float16>(*p, rule, part, (unsigned)blocks, (hipStream_t)stream);
  else
    launch_paged<bf16>(*p, rule, part, (unsigned)blocks, (hipStream_t)stream);
  return launch_status("smaq_paged_attention");
}
