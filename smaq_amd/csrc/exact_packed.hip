// Attention over a step's own exact tokens (smaq_packed_attention).
#include "exact_attention.h"

namespace smaq {
namespace {

constexpr int kWaves = 4;

// One wave per (token, query head).
template <typename T>
__global__ __launch_bounds__(64 * kWaves) void packed_any_kernel(smaq_packed_params p, ScoreRule rule) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (row >= p.n_tokens * p.n_q_heads) return;
  const int64_t t = row / p.n_q_heads;
  const int hq = (int)(row - t * p.n_q_heads), h = hq / (p.n_q_heads / p.n_kv_heads), D = p.head_dim;
  T* out = (T*)p.out + t * p.out_stride_t + hq * p.out_stride_h;
  int lo = 0, hi = p.n_docs;  // the document of token t: the last that starts at or before it
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.starts[mid] <= t) lo = mid; else hi = mid;
  }
  const int64_t s0 = p.n_docs ? max(p.starts[lo], 0) : 0, s1 = p.n_docs ? min((int64_t)p.starts[lo + 1], p.n_tokens) : 0;
  if (t < s0 || t >= s1) {
    if (p.zero_rest)
      for (int d = lane; d < D; d += 64) out[d] = Num<T>::from_f(0.0f);
    return;
  }
  const int64_t i = t - s0, n = s1 - s0;
  const int64_t prefix = p.prefix_lens ? p.prefix_lens[lo] : 0;
  const float slope = p.alibi_slopes ? p.alibi_slopes[hq] * kLog2eF : 0.0f;
  const T* q = (const T*)p.q + t * p.q_stride_t + hq * p.q_stride_h;
  const T* k = (const T*)p.k + s0 * p.k_stride_t + h * p.k_stride_h;
  const T* v = (const T*)p.v + s0 * p.v_stride_t + h * p.v_stride_h;
  float m = -__builtin_inff(), l = 0.0f, o[4] = {0.f, 0.f, 0.f, 0.f};
  for (int64_t j0 = 0; j0 < n; j0 += 64) {
    const int64_t j = j0 + lane;
    const bool seen = j < n && (!p.causal || j <= i || j < prefix) && (!p.window || j > i - p.window || j < prefix);
    float x = -__builtin_inff();
    if (seen) {
      float dot = 0.0f;
      for (int d = 0; d < D; ++d) dot = fmaf(Num<T>::to_f(q[d]), Num<T>::to_f(k[j * p.k_stride_t + d]), dot);
      x = rule_score(rule, dot) - slope * (float)llabs(i - j);
    }
    const float m_new = fmaxf(m, warp_max(x));
    const float m_use = m_new == -__builtin_inff() ? 0.0f : m_new;
    const float w = seen ? exp2f(x - m_use) : 0.0f, a = exp2f(m - m_use);
    l = l * a + warp_sum(w);
    m = m_new;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= a;
    const unsigned long long any = __ballot(seen);
    for (int e = 0; e < 64; ++e) {
      if (!((any >> e) & 1)) continue;
      const float we = __shfl(w, e, 64);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < D) o[c] = fmaf(we, Num<T>::to_f(v[(j0 + e) * p.v_stride_t + lane + 64 * c]), o[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (lane + 64 * c < D) out[lane + 64 * c] = Num<T>::from_f(o[c] / l);
}

}  // namespace
}  // namespace smaq

extern "C" int smaq_packed_attention(const smaq_packed_params* p, void* stream) {
  using namespace smaq;
  SMAQ_REQUIRE(p, "smaq_packed_attention: null parameters");
  SMAQ_REQUIRE(p->n_tokens >= 0 && p->n_tokens <= 0x7fffff00ll && p->n_docs >= 0 && p->n_q_heads > 0 &&
                   p->n_kv_heads > 0 && p->n_q_heads % p->n_kv_heads == 0 && p->n_q_heads <= 65536,
               "smaq_packed_attention: bad shape (%lld tokens, %d documents, %d heads over %d)", p->n_tokens, p->n_docs,
               p->n_q_heads, p->n_kv_heads);
  SMAQ_REQUIRE(p->head_dim > 0 && p->head_dim <= 256 && p->head_dim % 8 == 0,
               "smaq_packed_attention: head_dim %d is not a multiple of 8 up to 256", p->head_dim);
  SMAQ_REQUIRE(p->window >= 0 && p->score_cap >= 0.0f && p->score_cap < 1e30f && p->scale == p->scale,
               "smaq_packed_attention: window %d, score_cap %g and scale %g must be numbers of 0 or more, finite and "
               "a number", p->window, (double)p->score_cap, (double)p->scale);
  if (p->dtype != SMAQ_F16 && p->dtype != SMAQ_BF16) {
    set_error("smaq_packed_attention: unsupported dtype %d", p->dtype);
    return SMAQ_EUNSUPPORTED;
  }
  if (p->n_tokens == 0) return SMAQ_OK;
  SMAQ_REQUIRE(p->q && p->k && p->v && p->out && (!p->n_docs || p->starts), "smaq_packed_attention: null pointer");
  SMAQ_REQUIRE(rows_on_16(p->q, p->q_stride_t, p->q_stride_h) && rows_on_16(p->k, p->k_stride_t, p->k_stride_h) &&
                   rows_on_16(p->v, p->v_stride_t, p->v_stride_h) && rows_on_16(p->out, p->out_stride_t, p->out_stride_h),
               "smaq_packed_attention: rows must start on 16 bytes");
  const ScoreRule rule = score_rule(p->scale, p->score_cap);
  const int64_t rows = p->n_tokens * p->n_q_heads;
  const unsigned blocks = (unsigned)((rows + kWaves - 1) / kWaves);
  if (p->dtype == SMAQ_F16)
    packed_any_kernel<_Float16><<<blocks, 64 * kWaves, 0, (hipStream_t)stream>>>(*p, rule);
  else
    packed_any_kernel<bf16><<<blocks, 64 * kWaves, 0, (hipStream_t)stream>>>(*p, rule);
  return launch_status("smaq_packed_attention");
}
