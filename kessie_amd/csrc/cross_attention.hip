// Cross attention for gfx950: each sequence's queries over its own encoder
// states, all of them (no causal order, no window), any state length.
//
//   out[t, h] = sum_j softmax_j(q[t, h] . k[j, h / G] * sm_scale) v[j, h / G]
//
// over the states j of t's sequence that key_mask leaves; no state, zeros.
#include "common.h"

namespace kessie {
namespace cross {
namespace {

constexpr float kNegInf = -__builtin_huge_valf();
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* q;
  int64_t q_ts, q_hs;
  const void* k;
  int64_t k_ts, k_hs;
  const void* v;
  int64_t v_ts, v_hs;
  void* out;
  int64_t o_ts, o_hs;
  const int32_t* q_start;
  const int32_t* kv_start;
  const int32_t* kv_lens;
  const uint8_t* mask;
  int B, max_q, max_kv, Tq, Tkv;
  int Hq, Hkv, G, D;
  float c2;  // sm_scale * log2(e): the softmax is base 2
};

// Sequence b's rows, cut to what exists.
struct Seq {
  int q0, nq, kv0, nkv;
};
__device__ __forceinline__ Seq sequence(const Args& a, int b) {
  Seq s;
  s.q0 = a.q_start[b] - a.q_start[0];
  s.nq = min(a.q_start[b + 1] - a.q_start[b], a.max_q);
  if (s.q0 < 0 || s.q0 >= a.Tq) s.nq = 0;
  s.nq = max(min(s.nq, a.Tq - s.q0), 0);
  s.kv0 = a.kv_start[b];
  s.nkv = min(a.kv_lens[b], a.max_kv);
  if (s.kv0 < 0 || s.kv0 >= a.Tkv) s.nkv = 0;
  s.nkv = max(min(s.nkv, a.Tkv - s.kv0), 0);
  return s;
}

// Any head_dim up to 256, any strides and type: one wave per (query, head),
// the states 64 at a time -- one a lane for the scores, then one head_dim
// element a lane (of up to four) for the sum.
constexpr int kMaxD = 256;
template <typename T>
__global__ __launch_bounds__(64) void cross_generic_kernel(Args a) {
  __shared__ float sq[kMaxD];
  __shared__ float sp[64];
  const int b = blockIdx.x / a.max_q, i = blockIdx.x % a.max_q, h = blockIdx.y, lane = threadIdx.x;
  const Seq s = sequence(a, b);
  if (i >= s.nq) return;
  const T* q = static_cast<const T*>(a.q) + (int64_t)(s.q0 + i) * a.q_ts + (int64_t)h * a.q_hs;
  for (int d = lane; d < a.D; d += 64) sq[d] = to_f32(q[d]) * a.c2;
  __syncthreads();
  const int g = h / a.G;
  const T* k = static_cast<const T*>(a.k) + (int64_t)s.kv0 * a.k_ts + (int64_t)g * a.k_hs;
  const T* v = static_cast<const T*>(a.v) + (int64_t)s.kv0 * a.v_ts + (int64_t)g * a.v_hs;
  float o[kMaxD / 64] = {}, m = kNegInf, l = 0.0f;
  for (int j0 = 0; j0 < s.nkv; j0 += 64) {
    const int j = j0 + lane;
    float y = kNegInf;
    if (j < s.nkv && (a.mask == nullptr || a.mask[s.kv0 + j])) {
      y = 0.0f;
      for (int d = 0; d < a.D; ++d) y = fmaf(sq[d], to_f32(k[(int64_t)j * a.k_ts + d]), y);
    }
    float top = y;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
    const float mn = fmaxf(m, top);
    if (mn == kNegInf) continue;  // (uniform: nothing seen so far)
    const float alpha = exp2f(m - mn), p = exp2f(y - mn);
    m = mn;
    float sum = p;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    l = l * alpha + sum;
    __syncthreads();
    sp[lane] = p;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kMaxD / 64; ++e) {
      const int d = lane + 64 * e;
      if (d >= a.D) break;
      float acc = o[e] * alpha;
      const int n = min(64, s.nkv - j0);
      for (int jj = 0; jj < n; ++jj)
        if (sp[jj] != 0.0f) acc = fmaf(sp[jj], to_f32(v[(int64_t)(j0 + jj) * a.v_ts + d]), acc);
      o[e] = acc;
    }
  }
  T* out = static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_ts + (int64_t)h * a.o_hs;
  const float il = l > 0.0f ? 1.0f / l : 0.0f;
  for (int e = 0; e < kMaxD / 64; ++e)
    if (lane + 64 * e < a.D) out[lane + 64 * e] = from_f32<T>(o[e] * il);
}

template <typename T>
int launch_generic(const Args& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.B * a.max_q;
  KESSIE_REQUIRE(rows <= 0x7fffffff, KESSIE_ERR_UNSUPPORTED, "cross attention: %lld rows exceed one launch", (long long)rows);
  hipLaunchKernelGGL(cross_generic_kernel<T>, dim3((unsigned)rows, a.Hq), dim3(64), 0, s, a);
  return check_launch("cross attention");
}

}  // namespace
}  // namespace cross
}  // namespace kessie

using namespace kessie;
using namespace kessie::cross;

extern "C" size_t kessie_cross_attention_workspace_bytes(int batch, int max_query_len, int num_q_tokens, int num_q_heads,
                                                         int num_kv_heads, int head_dim, int max_kv_len, int dtype) {
  return 0;
}

extern "C" int kessie_cross_attention(const void* q, int64_t q_tok_stride, int64_t q_head_stride, const void* k,
                                      int64_t k_tok_stride, int64_t k_head_stride, const void* v, int64_t v_tok_stride,
                                      int64_t v_head_stride, const int32_t* query_start_loc, const int32_t* kv_start,
                                      const int32_t* kv_lens, const uint8_t* key_mask, void* out, int64_t out_tok_stride,
                                      int64_t out_head_stride, int batch, int max_query_len, int max_kv_len,
                                      int num_q_tokens, int num_kv_tokens, int num_q_heads, int num_kv_heads,
                                      int head_dim, float sm_scale, int dtype, void* workspace, size_t workspace_bytes,
                                      void* stream) {
  clear_error();
  KESSIE_REQUIRE(batch >= 0 && max_query_len >= 0 && max_kv_len >= 0 && num_q_tokens >= 0 && num_kv_tokens >= 0,
                 KESSIE_ERR_INVALID, "cross attention: bad sizes B=%d queries=%d states=%d Tq=%d Tkv=%d", batch,
                 max_query_len, max_kv_len, num_q_tokens, num_kv_tokens);
  KESSIE_REQUIRE(num_kv_heads > 0 && num_q_heads > 0 && num_q_heads % num_kv_heads == 0, KESSIE_ERR_INVALID,
                 "cross attention: %d query heads over %d kv heads", num_q_heads, num_kv_heads);
  KESSIE_REQUIRE(head_dim > 0, KESSIE_ERR_INVALID, "cross attention: head_dim %d", head_dim);
  KESSIE_REQUIRE(head_dim <= kMaxD, KESSIE_ERR_UNSUPPORTED, "cross attention: head_dim %d above %d", head_dim, kMaxD);
  KESSIE_REQUIRE(num_q_heads <= 65535, KESSIE_ERR_UNSUPPORTED, "cross attention: %d heads", num_q_heads);
  KESSIE_REQUIRE(dtype_size(dtype) > 0, KESSIE_ERR_UNSUPPORTED, "cross attention: dtype %d", dtype);
  if (batch == 0 || max_query_len == 0 || num_q_tokens == 0) return KESSIE_OK;
  KESSIE_REQUIRE(q && out && query_start_loc && kv_start && kv_lens && (num_kv_tokens == 0 || (k && v)), KESSIE_ERR_INVALID,
                 "cross attention: null pointer");
  Args a{};
  a.q = q, a.q_ts = q_tok_stride, a.q_hs = q_head_stride;
  a.k = k, a.k_ts = k_tok_stride, a.k_hs = k_head_stride;
  a.v = v, a.v_ts = v_tok_stride, a.v_hs = v_head_stride;
  a.out = out, a.o_ts = out_tok_stride, a.o_hs = out_head_stride;
  a.q_start = query_start_loc, a.kv_start = kv_start, a.kv_lens = kv_lens, a.mask = key_mask;
  a.B = batch, a.max_q = max_query_len, a.max_kv = max_kv_len, a.Tq = num_q_tokens, a.Tkv = num_kv_tokens;
  a.Hq = num_q_heads, a.Hkv = num_kv_heads, a.G = num_q_heads / num_kv_heads, a.D = head_dim;
  a.c2 = sm_scale * kLog2e;
  const hipStream_t s = as_stream(stream);
  switch (dtype) {
    case KESSIE_DTYPE_BF16: return launch_generic<bf16_t>(a, s);
    case KESSIE_DTYPE_F16: return launch_generic<f16_t>(a, s);
    default: return launch_generic<float>(a, s);
  }
}
