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
#include <type_traits>

#include "exact_attention.h"

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

// One wave per (token, head), one element at a time: every head_dim, layout and alignment.
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

// 16 bytes a load: a lane holds two units of E elements, the two halves of E pairs (half
// layout: units at l E and r/2 + l E; interleaved: neighbours; behind the rotated dims:
// neighbours), so the rotation needs no exchange and the norm one sum over the
// `lanes` of a row.  A workgroup takes `tb` tokens: their sines and cosines are formed
// once into LDS and kept in registers over the heads (queries', then keys'), which
// `slots` rows of lanes per token take in turn; the first kBatch rows are on their way
// before the sines are begun.  HBM bounds it: 16384 tokens of 32 + 8 heads of 128 bf16
// dims move 336 MB in 59 us (5.7 TB/s; a plain copy of that size reaches 5.2), 64 tokens
// take 4.7 us, most of it the chain position -> angle -> LDS.
constexpr int kBatch = 2;

template <typename T, bool IL, bool STREAM>
__global__ __launch_bounds__(kThreads) void norm_rotary_kernel(RotaryArgs a, int lanes, int tb) {
  constexpr int E = 16 / (int)sizeof(T);
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int tid = threadIdx.x, half = a.r / 2;
  float* sw = lds;            // [2][D] weights of queries and keys, offset added
  float* cs = lds + 2 * a.D;  // [tb][2][r/2]
  const int64_t t0 = (int64_t)blockIdx.x * tb;
  const int l = tid & (lanes - 1), row = tid / lanes, slots = kThreads / lanes / tb;
  const int tok = row / slots, slot = row % slots + blockIdx.y * slots, step = slots * gridDim.y;
  const int64_t t = t0 + tok;
  const int nr = a.r / (2 * E), hq = a.in[0].heads, heads = hq + a.in[1].heads;
  const bool turned = l < nr, live = t < a.tokens && 2 * E * l < a.D;
  const int ia = IL || !turned ? 2 * E * l : E * l, ib = IL || !turned ? ia + E : half + E * l;
  const T* xq = (const T*)a.in[0].x + t * a.in[0].st;
  const T* xk = (const T*)a.in[1].x + t * a.in[1].st;
  uint4 raw[kBatch][2];
  auto load = [&](int h0) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = h0 + u * step;
      raw[u][0] = raw[u][1] = uint4{0, 0, 0, 0};
      if (live && h < heads) {
        const T* x = h < hq ? xq + h * a.in[0].sh : xk + (h - hq) * a.in[1].sh;
        raw[u][0] = *(const uint4*)(x + ia);
        raw[u][1] = *(const uint4*)(x + ib);
      }
    }
  };
  load(slot);
#pragma unroll
  for (int side = 0; side < 2; ++side)
    if (a.in[side].w)
      for (int i = tid; i < a.D; i += kThreads) sw[side * a.D + i] = weight_at(a, a.in[side].w, i);
  for (int i = tid; i < tb * half; i += kThreads) {
    const int tt = i / half, pair = i - tt * half;
    if (t0 + tt < a.tokens) angle(a, position(a, t0 + tt), pair, cs[2 * tt * half + pair], cs[(2 * tt + 1) * half + pair]);
  }
  const float inv_d = 1.0f / (float)a.D;
  __syncthreads();
  float c[E], s[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    c[e] = turned ? cs[2 * tok * half + E * l + e] : 1.0f;
    s[e] = turned ? cs[(2 * tok + 1) * half + E * l + e] : 0.0f;
  }
  for (int h0 = slot; h0 < heads; h0 += kBatch * step) {
    if (h0 != slot) load(h0);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = h0 + u * step;
      if (h >= heads) break;
      const int side = h < hq ? 0 : 1;
      float v[2][E];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        const T* r = (const T*)&raw[u][y];
#pragma unroll
        for (int e = 0; e < E; ++e) v[y][e] = Num<T>::to_f(r[e]);
      }
      if (side ? a.in[1].w != nullptr : a.in[0].w != nullptr) {
        float sum = 0.0f;
#pragma unroll
        for (int y = 0; y < 2; ++y)
#pragma unroll
          for (int e = 0; e < E; ++e) sum = fmaf(v[y][e], v[y][e], sum);
        for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float mean = fmaf(sum, inv_d, a.eps);
        // the instruction's one ulp; it does not take numbers below the normal range
        const float inv = mean > 1e-30f ? __builtin_amdgcn_rsqf(mean) : 1.0f / sqrtf(mean);
        const float* w = sw + side * a.D;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          v[0][e] = v[0][e] * inv * (live ? w[ia + e] : 0.0f);
          v[1][e] = v[1][e] * inv * (live ? w[ib + e] : 0.0f);
        }
      }
      if (!live) continue;
      float o[2][E];
      if constexpr (IL) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float p = ((const float*)v)[2 * e], q = ((const float*)v)[2 * e + 1];
          ((float*)o)[2 * e] = turned ? fmaf(p, c[e], -(q * s[e])) : p;
          ((float*)o)[2 * e + 1] = turned ? fmaf(p, s[e], q * c[e]) : q;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float p = v[0][e], q = v[1][e];
          o[0][e] = turned ? fmaf(p, c[e], -(q * s[e])) : p;
          o[1][e] = turned ? fmaf(p, s[e], q * c[e]) : q;
        }
      }
      uint4 res[2];
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        uint32_t* r = (uint32_t*)&res[y];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (sizeof(T) == 4) r[e] = __float_as_uint(o[y][e]);
          else r[e] = Mat<T>::pack(o[y][2 * e], o[y][2 * e + 1]);
        }
      }
      T* out = side ? (T*)a.in[1].out + (t * a.in[1].heads + h - hq) * a.D : (T*)a.in[0].out + (t * hq + h) * a.D;
      if constexpr (STREAM) {
        __builtin_nontemporal_store(*(const u32x4v*)&res[0], (u32x4v*)(out + ia));
        __builtin_nontemporal_store(*(const u32x4v*)&res[1], (u32x4v*)(out + ib));
      } else {
        *(uint4*)(out + ia) = res[0];
        *(uint4*)(out + ib) = res[1];
      }
    }
  }
}

template <typename T>
int launch_rotary(const RotaryArgs& a, hipStream_t st) {
  constexpr int E = 16 / (int)sizeof(T);
  bool wide = a.D % (2 * E) == 0 && a.r % (2 * E) == 0 && a.D <= 64 * 2 * E;
  for (const RotaryIn& in : a.in)
    wide = wide && (!in.heads || ((uintptr_t)in.x % 16 == 0 && (uintptr_t)in.out % 16 == 0 && in.st % E == 0 && in.sh % E == 0));
  if (wide) {
    const int heads = a.in[0].heads + a.in[1].heads;
    int lanes = 1;
    while (lanes * 2 * E < a.D) lanes *= 2;
    // four tokens a workgroup while that leaves four workgroups to a CU; for few tokens the
    // heads of a token are spread over workgroups as well
    int tb = 4;
    while (tb > 1 && (lanes * tb > kThreads || (a.tokens + tb - 1) / tb < 1024)) tb /= 2;
    const int slots = kThreads / lanes / tb;
    const int64_t gx = (a.tokens + tb - 1) / tb;
    const int gy = (int)std::max<int64_t>(1, std::min<int64_t>((heads + slots - 1) / slots, 1024 / gx));
    SMAQ_REQUIRE(gx <= 0x7fffffffll, "smaq_norm_rotary: %lld tokens are more than one launch takes", (long long)a.tokens);
    const size_t lds = ((size_t)tb * a.r + 2 * a.D) * sizeof(float);
    const dim3 grid((unsigned)gx, (unsigned)gy);
    // Results that no cache holds are stored past them: 16384 tokens of 32 + 8 heads 72 -> 59
    // us, with the attention that reads them 196 -> 192; 4096 tokens 18.1 -> 17.1 us, but
    // with their attention 50 -> 53.
    const bool stream = a.tokens * heads * a.D * (int64_t)sizeof(T) > (64ll << 20);
    auto launch = [&](auto il, auto st_past) {
      norm_rotary_kernel<T, decltype(il)::value, decltype(st_past)::value><<<grid, kThreads, lds, st>>>(a, lanes, tb);
    };
    if (a.interleaved)
      stream ? launch(std::true_type{}, std::true_type{}) : launch(std::true_type{}, std::false_type{});
    else
      stream ? launch(std::false_type{}, std::true_type{}) : launch(std::false_type{}, std::false_type{});
    return launch_status("smaq_norm_rotary");
  }
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
