// Queries and keys as attention reads them: RMS norm of each head and the
// position rotation, one pass over both (smaq_norm_rotary).
//
//   y = x * rsqrt(mean(x^2) + eps) * (w + w0)   (only with a weight)
//   (a, b) of pair i at position p -> (a c - b s, a s + b c),
//   c = gain cos(p f_i), s = gain sin(p f_i);
//   pairs (i, r/2 + i) in the half layout, (2i, 2i + 1) interleaved; dims >= r
//   pass as normed.
//
// Everything between the load and the store is fp32, rounded once.  An angle of
// position 10^6 needs 20 bits before the point, so p f_i / 2 pi is formed in
// fp64 and its whole turns dropped there; what is left, at most half a turn,
// goes to sincospif.
#include <algorithm>

#include "smaq_common.h"

namespace smaq {
namespace {

constexpr int kThreads = 256;
constexpr double kTurn = 0.15915494309189535;  // 1 / (2 pi)

struct RotaryIn {
  const char* x;  // [tokens][heads][D], element strides st, sh
  int64_t st, sh;
  const void* w;  // [D] or NULL
  char* out;      // [tokens][heads][D], dense
  int heads;
};

struct RotaryArgs {
  RotaryIn in[2];
  int64_t tokens;
  int D, r, interleaved;
  const void* pos;
  int pos_wide;
  const double* freqs;  // [r/2]
  float gain;
  int wdtype;
  float eps, w0;
};

__device__ __forceinline__ float weight_at(const RotaryArgs& a, const void* w, int i) {
  switch (a.wdtype) {
    case SMAQ_F32: return ((const float*)w)[i] + a.w0;
    case SMAQ_F16: return Num<_Float16>::to_f(((const _Float16*)w)[i]) + a.w0;
    default: return Num<bf16>::to_f(((const bf16*)w)[i]) + a.w0;
  }
}

__device__ __forceinline__ int64_t position(const RotaryArgs& a, int64_t t) {
  return a.pos_wide ? ((const long long*)a.pos)[t] : (int64_t)((const int*)a.pos)[t];
}

// cos and sin of pair i at position p, times the gain
__device__ __forceinline__ void angle(const RotaryArgs& a, int64_t p, int i, float& c, float& s) {
  const double turns = (double)p * (a.freqs[i] * kTurn);
  const float x = (float)(turns - __builtin_rint(turns));
  sincospif(2.0f * x, &s, &c);
  c *= a.gain;
  s *= a.gain;
}

// One wave per (token, head), one element at a time: every layout and alignment.
template <typename T>
__global__ __launch_bounds__(kThreads) void norm_rotary_any_kernel(RotaryArgs a) {
  const int lane = threadIdx.x & 63;
  const int heads = a.in[0].heads + a.in[1].heads;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6);
  if (row >= a.tokens * heads) return;
  const int64_t t = row / heads;
  int h = (int)(row - t * heads);
  const RotaryIn& in = a.in[h >= a.in[0].heads];
  if (h >= a.in[0].heads) h -= a.in[0].heads;
  const T* x = (const T*)in.x + t * in.st + h * in.sh;
  T* out = (T*)in.out + (t * in.heads + h) * a.D;
  float inv = 1.0f;
  if (in.w) {
    float sum = 0.0f;
    for (int i = lane; i < a.D; i += 64) {
      const float v = Num<T>::to_f(x[i]);
      sum = fmaf(v, v, sum);
    }
    inv = 1.0f / sqrtf(warp_sum(sum) / (float)a.D + a.eps);
  }
  auto normed = [&](int i) {
    const float v = Num<T>::to_f(x[i]);
    return in.w ? v * inv * weight_at(a, in.w, i) : v;
  };
  const int half = a.r / 2;
  const int64_t p = position(a, t);
  for (int i = lane; i < half; i += 64) {
    const int ia = a.interleaved ? 2 * i : i, ib = a.interleaved ? 2 * i + 1 : half + i;
    float c, s;
    angle(a, p, i, c, s);
    const float va = normed(ia), vb = normed(ib);
    out[ia] = Num<T>::from_f(fmaf(va, c, -(vb * s)));
    out[ib] = Num<T>::from_f(fmaf(va, s, vb * c));
  }
  for (int i = a.r + lane; i < a.D; i += 64) out[i] = Num<T>::from_f(normed(i));
}

template <typename T>
int launch_rotary(const RotaryArgs& a, hipStream_t st) {
  const int64_t rows = a.tokens * (a.in[0].heads + a.in[1].heads);
  const int64_t blocks = (rows + kThreads / 64 - 1) / (kThreads / 64);
  SMAQ_REQUIRE(blocks <= 0x7fffffffll, "smaq_norm_rotary: %lld rows are more than one launch takes", (long long)rows);
  norm_rotary_any_kernel<T><<<(unsigned)blocks, kThreads, 0, st>>>(a);
  return launch_status("smaq_norm_rotary");
}

}  // namespace
}  // namespace smaq

extern "C" int smaq_norm_rotary(const smaq_rotary_params* p, void* stream) {
  using namespace smaq;
  SMAQ_REQUIRE(p, "smaq_norm_rotary: null parameters");
  SMAQ_REQUIRE(p->tokens >= 0 && p->n_q_heads >= 0 && p->n_k_heads >= 0 && p->n_q_heads <= 65536 &&
                   p->n_k_heads <= 65536,
               "smaq_norm_rotary: bad shape (%lld tokens, %d and %d heads)", p->tokens, p->n_q_heads, p->n_k_heads);
  SMAQ_REQUIRE(p->head_dim > 0 && p->head_dim <= 1024, "smaq_norm_rotary: head_dim %d is not in 1..1024", p->head_dim);
  SMAQ_REQUIRE(p->rotary_dim >= 0 && p->rotary_dim % 2 == 0 && p->rotary_dim <= p->head_dim,
               "smaq_norm_rotary: rotary_dim %d is not an even number up to head_dim %d", p->rotary_dim, p->head_dim);
  if (p->dtype < SMAQ_F32 || p->dtype > SMAQ_BF16 || p->weight_dtype < SMAQ_F32 || p->weight_dtype > SMAQ_BF16) {
    set_error("smaq_norm_rotary: unsupported dtype %d / %d", p->dtype, p->weight_dtype);
    return SMAQ_EUNSUPPORTED;
  }
  if (p->tokens == 0 || p->n_q_heads + p->n_k_heads == 0) return SMAQ_OK;
  SMAQ_REQUIRE((!p->n_q_heads || (p->q && p->q_out)) && (!p->n_k_heads || (p->k && p->k_out)) &&
                   (!p->rotary_dim || (p->positions && p->freqs)),
               "smaq_norm_rotary: null pointer");
  SMAQ_REQUIRE(p->position_bytes == 4 || p->position_bytes == 8, "smaq_norm_rotary: positions of %d bytes",
               p->position_bytes);
  RotaryArgs a;
  a.in[0] = {(const char*)p->q, p->q_stride_t, p->q_stride_h, p->q_weight, (char*)p->q_out, p->n_q_heads};
  a.in[1] = {(const char*)p->k, p->k_stride_t, p->k_stride_h, p->k_weight, (char*)p->k_out, p->n_k_heads};
  a.tokens = p->tokens;
  a.D = p->head_dim;
  a.r = p->rotary_dim;
  a.interleaved = p->interleaved;
  a.pos = p->positions;
  a.pos_wide = p->position_bytes == 8;
  a.freqs = p->freqs;
  a.gain = p->gain;
  a.wdtype = p->weight_dtype;
  a.eps = p->eps;
  a.w0 = p->weight_offset;
  hipStream_t st = (hipStream_t)stream;
  switch (p->dtype) {
    case SMAQ_F32: return launch_rotary<float>(a, st);
    case SMAQ_F16: return launch_rotary<_Float16>(a, st);
    default: return launch_rotary<bf16>(a, st);
  }
}
