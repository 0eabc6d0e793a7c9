// Attention over a step's own exact tokens (smaq_packed_attention): the fp16
// kernels of exact_packed.h and the entry point.
#include "exact_packed.h"

namespace smaq {

void launch_packed_bf16(const smaq_packed_params& p, const ScoreRule& rule, unsigned grid, int blocks, hipStream_t st);

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
  SMAQ_REQUIRE(p->window >= 0 && score_range(p->scale, p->score_cap),
               "smaq_packed_attention: window %d must be 0 or more, score_cap %g 0 or in 1e-30..1e30, scale %g below 1e38",
               p->window, (double)p->score_cap, (double)p->scale);
  if (p->dtype != SMAQ_F16 && p->dtype != SMAQ_BF16) {
    set_error("smaq_packed_attention: unsupported dtype %d", p->dtype);
    return SMAQ_EUNSUPPORTED;
  }
  if (p->n_tokens == 0) return SMAQ_OK;
  SMAQ_REQUIRE(p->q && p->k && p->v && p->out && (!p->n_docs || p->starts), "smaq_packed_attention: null pointer");
  SMAQ_REQUIRE(rows_on_16(p->q, p->q_stride_t, p->q_stride_h) && rows_on_16(p->k, p->k_stride_t, p->k_stride_h) &&
                   rows_on_16(p->v, p->v_stride_t, p->v_stride_h) && rows_on_16(p->out, p->out_stride_t, p->out_stride_h),
               "smaq_packed_attention: rows must start on 16 bytes");
  // the kernel gives the scale's sign, and a scale of 0, to the queries
  const ScoreRule rule = score_rule(p->scale == 0.0f ? 1.0f : fabsf(p->scale), p->score_cap);
  const int blocks = (int)((p->n_tokens + 31) / 32), g = p->n_q_heads / p->n_kv_heads;
  const int64_t grid = ((int64_t)blocks * g + 3) / 4 * p->n_kv_heads;
  SMAQ_REQUIRE((int64_t)blocks * g < 0x7ffffff0ll && grid <= 0x7fffffffll,
               "smaq_packed_attention: %lld workgroups are more than one launch takes", (long long)grid);
  if (p->dtype == SMAQ_F16)
    launch_packed<_Float16>(*p, rule, (unsigned)grid, blocks, (hipStream_t)stream);
  else
    launch_packed_bf16(*p, rule, (unsigned)grid, blocks, (hipStream_t)stream);
  return launch_status("smaq_packed_attention");
}
