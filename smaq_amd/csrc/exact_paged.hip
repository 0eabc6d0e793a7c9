// Attention of one new token per sequence over a paged exact cache
// (smaq_paged_attention).
#include "exact_attention.h"

namespace smaq {
namespace {

// One wave per (sequence, query head).
template <typename T>
__global__ __launch_bounds__(64) void paged_any_kernel(smaq_paged_params p, ScoreRule rule) {
  const int lane = threadIdx.x;
  const int b = blockIdx.x / p.n_q_heads, hq = blockIdx.x % p.n_q_heads;
  const int h = hq / (p.n_q_heads / p.n_kv_heads), D = p.head_dim;
  T* out = (T*)p.out + (int64_t)b * p.out_stride_b + hq * p.out_stride_h;
  int64_t n = p.seq_lens_wide ? ((const long long*)p.seq_lens)[b] : (long long)((const int*)p.seq_lens)[b];
  n = min(n, min((int64_t)p.max_seq_len, (int64_t)p.max_blocks * p.block_size));
  const float slope = p.alibi_slopes ? p.alibi_slopes[hq] * kLog2eF : 0.0f;
  const T* q = (const T*)p.q + (int64_t)b * p.q_stride_b + hq * p.q_stride_h;
  const int* table = p.block_table + (int64_t)b * p.max_blocks;
  float m = -__builtin_inff(), l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
  bool some = false;
  const int64_t first = p.window && n > p.window ? n - p.window : 0;
  for (int64_t j0 = first; j0 < n; j0 += 64) {
    const int64_t j = j0 + lane;
    int blk = j < n ? table[j / p.block_size] : -1;
    const bool seen = blk >= 0 && blk < p.num_blocks;
    const int64_t off = j % p.block_size;
    float x = -__builtin_inff();
    if (seen) {
      const T* k = (const T*)p.k_cache + blk * p.k_stride_block + off * p.k_stride_t + h * p.k_stride_h;
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(Num<T>::to_f(q[d]), Num<T>::to_f(k[d]), dot);
      x = rule_score(rule, dot) - slope * (float)(n - 1 - j);
    }
    const float m_new = fmaxf(m, warp_max(x));
    const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float w = seen ? exp2f(x - m_use) : 0.0f, a = exp2f(m - m_use);
    l = l * a + warp_sum(w);
    m = m_new;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
    const unsigned long long any = __ballot(seen);
    some |= any != 0;
    for (int e = 0; e < 64; ++e) {
      if (!((any >> e) & 1)) continue;
      const float we = __shfl(w, e, 64);
      const T* v = (const T*)p.v_cache + (int64_t)__shfl(blk, e, 64) * p.v_stride_block +
                   ((j0 + e) % p.block_size) * p.v_stride_t + h * p.v_stride_h;
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) o[c] = fmaf(we, Num<T>::to_f(v[lane + 64 * c]), o[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < D) out[lane + 64 * c] = Num<T>::from_f(some ? o[c] / l : 0.0f);
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

}  // namespace
}  // namespace smaq

extern "C" long long smaq_paged_workspace_bytes(const smaq_paged_params* p) {
  return smaq::check_paged(p) == SMAQ_OK ? 0 : -1;
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
  const ScoreRule rule = score_rule(p->scale, p->score_cap);
  const unsigned blocks = (unsigned)(p->batch * p->n_q_heads);
  if (p->dtype == SMAQ_F16)
    paged_any_kernel<_Float16><<<blocks, 64, 0, (hipStream_t)stream>>>(*p, rule);
  else
    paged_any_kernel<bf16><<<blocks, 64, 0, (hipStream_t)stream>>>(*p, rule);
  return launch_status("smaq_paged_attention");
}
