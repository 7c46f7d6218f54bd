// Rotary positions with several axes (time, height, width), for gfx950.
//
//   ang_j   = pos[axis(j)][t] * inv_freq[j]          j < R/2, R <= head_dim
//   y1, y2  = x1 cos - x2 sin, x1 sin + x2 cos       (x1, x2) = (x[j], x[j + R/2]) or, adjacent, (x[2j], x[2j+1])
// and elements from R on as they are.  axis(j) comes from the section sizes:
// axis 0's pairs, then axis 1's, ..., or (interleaved) dealt out in turn.
//
// Angles: pos * inv_freq is taken in 64 bits (exact: 31 + 24 bits), in turns,
// and only its fraction is rounded to fp32, so a position of a million costs no
// digits (its fp32 product is off by up to 0.03 rad).  cos and sin are
// evaluated once per (token, pair) into LDS for all heads; the rotation is fp32
// and rounded once.
//
// Three uses of one body: Q and K into tensors (or in place), Q into a tensor
// with K and V into their cache slots, and K in place in its pages by the
// difference of two positions.  Bound: HBM -- each row read and written once,
// with 16-byte loads that are under way while the angles are computed.
#include "common.h"

namespace kessie {
namespace axes {
namespace {

constexpr int kMaxHalf = 128;  // rotary_dim <= 256
constexpr int kMaxAxes = 4;
constexpr int kGridShift = 21;  // workgroups in x before y counts (a launch counts a dimension's threads in 32 bits)

struct Args {
  // Rows of (token, head): x at src + t*s_ts + h*s_hs, written to dst.
  const void* q;
  int64_t q_ts, q_hs;
  void* qo;
  int64_t qo_ts, qo_hs;
  const void* k;
  int64_t k_ts, k_hs;
  void* ko;
  int64_t ko_ts, ko_hs;
  const void* v;  // copied to the pool, never rotated
  int64_t v_ts, v_hs;
  // Paged destination of K (and of V, kv_stride further), by slot or by page list.
  void* pool;
  int64_t page_stride, tok_stride, kv_stride, head_stride;
  const int64_t* slots;
  const int32_t* pages;
  int page_size, num_pages;
  const void* pos;   // [axes][T], rows pos_as apart
  const void* from;  // positions to take away (remap), or nullptr
  int64_t pos_as, from_as;
  int pos64;
  const float* inv;
  uint64_t axis[kMaxHalf / 32];  // two bits a pair
  int T, Hq, Hk, Hv, D, half;
  int page_shift;    // page_size = 1 << page_shift, or -1
  float inv_heads, inv_half;  // 1 / (Hq + Hk + Hv), 1 / half
  float sign;  // -1: rotate back
};

template <typename T>
struct Vec16;
template <>
struct Vec16<bf16_t> {
  static constexpr int N = 8;
  typedef bf16x8 type;
};
template <>
struct Vec16<f16_t> {
  static constexpr int N = 8;
  typedef f16x8 type;
};
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  typedef f32x4 type;
};

__device__ __forceinline__ int axis_of(const Args& a, int j) {
  const uint64_t w = j < 64 ? (j < 32 ? a.axis[0] : a.axis[1]) : (j < 96 ? a.axis[2] : a.axis[3]);
  return (int)(w >> (2 * (j & 31))) & 3;
}

// What token t's pair j turns by, as loaded: without a branch, so that the loads
// are under way together with the rows' (each is 4 bytes; a position of 32 bits
// is loaded twice).
struct Turn {
  int lo, hi, from_lo, from_hi;
  float inv;
};
__device__ __forceinline__ Turn load_turn(const Args& a, int t, int j) {
  const int ax = axis_of(a, j);
  const int width = a.pos64 ? 2 : 1, more = a.pos64 ? 1 : 0;
  const int32_t* p = static_cast<const int32_t*>(a.pos) + (ax * a.pos_as + t) * width;
  const int32_t* f = static_cast<const int32_t*>(a.from ? a.from : a.pos) + (ax * (a.from ? a.from_as : a.pos_as) + t) * width;
  return {p[0], p[more], f[0], f[more], a.inv[j]};
}
// (cos, sin): the turns in 64 bits, their fraction in 32.
__device__ __forceinline__ float2 angle(const Args& a, const Turn& u) {
  auto whole = [&](int lo, int hi) { return (int64_t)(((uint64_t)(uint32_t)(a.pos64 ? hi : lo >> 31) << 32) | (uint32_t)lo); };
  const int64_t p = whole(u.lo, u.hi) - (a.from ? whole(u.from_lo, u.from_hi) : 0);
  const double r = (double)p * (double)u.inv * 0.15915494309189533577;
  float s, c;
  sincospif(2.0f * (float)(r - rint(r)), &s, &c);
  return make_float2(c, s * a.sign);
}

// Element offset of token t's row in the pool, or -1: no slot, or no such page.
__device__ __forceinline__ int64_t pool_row(const Args& a, int t) {
  int64_t page;
  int off;
  if (a.slots) {
    const int64_t slot = a.slots[t];
    if (slot < 0) return -1;
    page = a.page_shift >= 0 ? slot >> a.page_shift : slot / a.page_size;
    off = (int)(slot - page * a.page_size);
  } else {
    const int i = a.page_shift >= 0 ? t >> a.page_shift : t / a.page_size;
    page = a.pages[i];
    off = t - i * a.page_size;
  }
  if (page < 0 || page >= a.num_pages) return -1;
  return page * a.page_stride + off * a.tok_stride;
}

// Where head h of token t (h counts Q's, K's and V's heads) comes from; K in place in the pages: nullptr.
template <typename T>
__device__ __forceinline__ const T* source(const Args& a, int t, int h, bool& rot) {
  rot = true;
  if (h < a.Hq) return static_cast<const T*>(a.q) + t * a.q_ts + h * a.q_hs;
  h -= a.Hq;
  if (h < a.Hk) return a.k ? static_cast<const T*>(a.k) + t * a.k_ts + h * a.k_hs : nullptr;
  rot = false;
  return static_cast<const T*>(a.v) + t * a.v_ts + (h - a.Hk) * a.v_hs;
}
// And where it goes, or nullptr: nowhere.
template <typename T>
__device__ __forceinline__ T* target(const Args& a, int t, int h) {
  if (h < a.Hq) return static_cast<T*>(a.qo) + t * a.qo_ts + h * a.qo_hs;
  h -= a.Hq;
  if (!a.pool) return static_cast<T*>(a.ko) + t * a.ko_ts + h * a.ko_hs;
  const int64_t row = pool_row(a, t);
  if (row < 0) return nullptr;
  return static_cast<T*>(a.pool) + row + (h < a.Hk ? h * a.head_stride : (h - a.Hk) * a.head_stride + a.kv_stride);
}

// 16-byte chunks, two a thread and step: chunk pair i of a row holds both
// halves of N pairs (or, adjacent, two neighbouring chunks), and past the
// rotated part two chunks to copy, so every row is D / 2N steps of the same
// kind.  kTok tokens a workgroup.  kPer fixes D / 2N (0: any), kPages a K that
// is rotated in place in its pages: the index arithmetic before the first load
// is then shifts (with the angles' loads ahead of the rows', 89 -> 77 us at
// 65,536 tokens).
template <typename T, bool kAdjacent, bool kPages, int kPer, int kThreads, int kTok, int kSteps>
__global__ __launch_bounds__(kThreads) void rope_axes_vec(Args a) {
  typedef typename Vec16<T>::type V;
  constexpr int N = Vec16<T>::N;
  __shared__ float2 cs[kTok * kMaxHalf];
  const int half = a.half, R = 2 * half;
  const uint32_t at = ((blockIdx.y << kGridShift) + blockIdx.x) * kTok;
  if (at >= (uint32_t)a.T) return;
  const int t0 = (int)at;
  const int ntok = min(kTok, a.T - t0);
  const int heads = kPages ? a.Hk : a.Hq + a.Hk + a.Hv;
  const int per = kPer > 0 ? kPer : a.D / (2 * N);  // steps a row
  const int stride = kThreads / per;                // rows a round
  const int i = threadIdx.x % per, r0 = threadIdx.x / per;
  const int o1 = kAdjacent ? 2 * i * N : i * N < half ? i * N : i * N + half;
  const int o2 = kAdjacent ? o1 + N : i * N < half ? o1 + half : o1 + (a.D - R) / 2;
  const int rows = r0 < stride ? ntok * heads : 0;
  // This thread's first angle is asked for before the rows: its wait is then not theirs too.
  auto angle_at = [&](int n) {
    const int tt = (int)(((float)n + 0.5f) * a.inv_half);
    return load_turn(a, t0 + tt, n - tt * half);
  };
  const int angles = ntok * half;
  const Turn first = angle_at(min((int)threadIdx.x, angles - 1));
  bool ready = false;
  for (int base = r0;; base += kSteps * stride) {
    V x1[kSteps], x2[kSteps];
    T* dst[kSteps];
    int csi[kSteps];  // this row's angles, or -1: not rotated
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      const int row = base + s * stride;
      dst[s] = nullptr;
      csi[s] = -1;
      if (row < rows) {
        // (exact: row + 1/2 is at least 1/2 from a multiple of heads, and both are small)
        const int tt = kTok == 1 ? 0 : kTok == 2 ? (row >= heads ? 1 : 0) : (int)(((float)row + 0.5f) * a.inv_heads);
        const int h = row - tt * heads;
        const T* src;
        bool rot = true;
        if constexpr (kPages) {
          const int64_t at = pool_row(a, t0 + tt);
          dst[s] = at < 0 || o1 >= R ? nullptr : static_cast<T*>(a.pool) + at + h * a.head_stride;
          src = dst[s];
        } else {
          src = source<T>(a, t0 + tt, h, rot);
          dst[s] = target<T>(a, t0 + tt, h);
          if (src == dst[s] && o1 >= R) dst[s] = nullptr;  // (in place, the rest of the row stays)
        }
        if (rot) csi[s] = tt * half;
        if (src) {
          x1[s] = __builtin_nontemporal_load(reinterpret_cast<const V*>(src + o1));
          x2[s] = __builtin_nontemporal_load(reinterpret_cast<const V*>(src + o2));
        }
      }
    }
    if (!ready) {
      if (threadIdx.x < angles) cs[threadIdx.x] = angle(a, first);
      for (int n = threadIdx.x + kThreads; n < angles; n += kThreads) cs[n] = angle(a, angle_at(n));
      __syncthreads();
      ready = true;
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if (dst[s] == nullptr) continue;
      V y1 = x1[s], y2 = x2[s];
      if (csi[s] >= 0) {
        if constexpr (kAdjacent) {
          // (rotary_dim is a multiple of N: a chunk is rotated whole or not at all)
          auto rotate = [&](V x, int o) {
            if (o >= R) return x;
            V y;
#pragma unroll
            for (int e = 0; e < N; e += 2) {
              const float2 w = cs[csi[s] + ((o + e) >> 1)];
              const float u = to_f32(x[e]), z = to_f32(x[e + 1]);
              y[e] = from_f32<T>(fmaf(u, w.x, -(z * w.y)));
              y[e + 1] = from_f32<T>(fmaf(u, w.y, z * w.x));
            }
            return y;
          };
          y1 = rotate(x1[s], o1);
          y2 = rotate(x2[s], o2);
        } else if (o1 < half) {
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const float2 w = cs[csi[s] + o1 + e];
            const float u = to_f32(x1[s][e]), z = to_f32(x2[s][e]);
            y1[e] = from_f32<T>(fmaf(u, w.x, -(z * w.y)));
            y2[e] = from_f32<T>(fmaf(u, w.y, z * w.x));
          }
        }
      }
      __builtin_nontemporal_store(y1, reinterpret_cast<V*>(dst[s] + o1));
      __builtin_nontemporal_store(y2, reinterpret_cast<V*>(dst[s] + o2));
    }
    if (base - r0 + kSteps * stride >= ntok * heads) break;  // (uniform)
  }
}

// Any head_dim and alignment: one thread a pair, or a copied element pair.
template <typename T, bool kAdjacent>
__global__ __launch_bounds__(256) void rope_axes_scalar(Args a) {
  const int heads = a.Hq + a.Hk + a.Hv;
  const int R = 2 * a.half, per = a.half + (a.D - R);  // pairs, then single elements
  const int64_t total = (int64_t)a.T * heads * per;
  for (int64_t n = (int64_t)blockIdx.x * 256 + threadIdx.x; n < total; n += (int64_t)gridDim.x * 256) {
    const int i = (int)(n % per);
    const int64_t th = n / per;
    const int t = (int)(th / heads), h = (int)(th - (int64_t)t * heads);
    bool rot;
    const T* src = source<T>(a, t, h, rot);
    T* dst = target<T>(a, t, h);
    if (dst == nullptr) continue;
    if (src == nullptr) src = dst;
    if (i >= a.half) {
      const int d = R + i - a.half;
      if (src != dst) dst[d] = src[d];
      continue;
    }
    const int d1 = kAdjacent ? 2 * i : i, d2 = kAdjacent ? 2 * i + 1 : i + a.half;
    if (!rot) {
      dst[d1] = src[d1];
      dst[d2] = src[d2];
      continue;
    }
    const float2 w = angle(a, load_turn(a, t, i));
    const float u = to_f32(src[d1]), z = to_f32(src[d2]);
    dst[d1] = from_f32<T>(fmaf(u, w.x, -(z * w.y)));
    dst[d2] = from_f32<T>(fmaf(u, w.y, z * w.x));
  }
}

template <typename T, bool kAdjacent>
int launch(const Args& a, hipStream_t s) {
  constexpr int N = Vec16<T>::N;
  const int R = 2 * a.half, per = a.D / (2 * N);
  auto fine = [](const void* p, int64_t s1, int64_t s2) { return p == nullptr || (aligned16(p) && s1 % N == 0 && s2 % N == 0); };
  const bool vec = a.D % (2 * N) == 0 && per <= 64 && (kAdjacent ? R % N == 0 : a.half % N == 0 && (a.D - R) % (2 * N) == 0) &&
                   fine(a.q, a.q_ts, a.q_hs) && fine(a.qo, a.qo_ts, a.qo_hs) && fine(a.k, a.k_ts, a.k_hs) &&
                   fine(a.ko, a.ko_ts, a.ko_hs) && fine(a.v, a.v_ts, a.v_hs) && fine(a.pool, a.tok_stride, a.head_stride) &&
                   (a.pool == nullptr || (a.page_stride % N == 0 && a.kv_stride % N == 0));
  const int heads = a.Hq + a.Hk + a.Hv;
  auto tiles = [&](int64_t tok) {
    const int64_t n = div_up((int64_t)a.T, tok), x = n < 1 << kGridShift ? n : 1 << kGridShift;
    return dim3((unsigned)x, (unsigned)div_up(n, x));
  };
  if (!vec) {
    const int64_t items = (int64_t)a.T * heads * (a.half + a.D - R);
    const int64_t grid = (items + 255) / 256;
    hipLaunchKernelGGL((rope_axes_scalar<T, kAdjacent>), dim3((unsigned)(grid < (1 << 20) ? grid : 1 << 20)), dim3(256), 0, s, a);
  } else if (a.k == nullptr && a.Hq == 0) {
    // In place in the pages: a page's 16 tokens a workgroup.  65,536 bf16 tokens of 8 heads x 128 in random interleaved
    // pages (270 MB): 77.0 us, 8 tokens of 512 threads 80.4, 4 of 256 79.4, the tiles of a page on one XCD 77-79; with
    // the pages in order 61-64, so what bounds it is where the pages lie.
    if (per == 8)
      hipLaunchKernelGGL((rope_axes_vec<T, kAdjacent, true, 8, 1024, 16, 1>), tiles(16), dim3(1024), 0, s, a);
    else
      hipLaunchKernelGGL((rope_axes_vec<T, kAdjacent, true, 0, 512, 8, 1>), tiles(8), dim3(512), 0, s, a);
  } else if (per == 8) {
    // 16,411 bf16 tokens, 32 + 8 + 8 heads of 128, K and V to their slots (404 MB): 70.1 us = 5.8 TB/s; 256 threads 72.2.
    hipLaunchKernelGGL((rope_axes_vec<T, kAdjacent, false, 8, 512, 2, 2>), tiles(2), dim3(512), 0, s, a);
  } else if (per == 4) {
    // 9,005 fp16 tokens, 16 + 16 heads of 64 (74 MB): 17.2 us; 4 tokens 18.4, 1 token 17.6.
    hipLaunchKernelGGL((rope_axes_vec<T, kAdjacent, false, 4, 256, 2, 1>), tiles(2), dim3(256), 0, s, a);
  } else {
    hipLaunchKernelGGL((rope_axes_vec<T, kAdjacent, false, 0, 256, 2, 3>), tiles(2), dim3(256), 0, s, a);
  }
  return check_launch("rope axes");
}

// Checks what the three entries share, fills the axis map and launches.
int dispatch(Args& a, const int32_t* sections, int num_axes, int interleaved, int adjacent, int inverse, int rotary_dim,
             int dtype, hipStream_t s) {
  KESSIE_REQUIRE(a.T >= 0 && a.D > 0 && a.Hq >= 0 && a.Hk >= 0, KESSIE_ERR_INVALID, "rope axes: bad sizes T=%d Hq=%d Hkv=%d D=%d",
                 a.T, a.Hq, a.Hk, a.D);
  KESSIE_REQUIRE(rotary_dim > 0 && rotary_dim % 2 == 0 && rotary_dim <= a.D, KESSIE_ERR_INVALID,
                 "rope axes: rotary_dim %d (even, at most head_dim %d)", rotary_dim, a.D);
  a.half = rotary_dim / 2;
  KESSIE_REQUIRE(a.half <= kMaxHalf, KESSIE_ERR_UNSUPPORTED, "rope axes: rotary_dim %d above %d", rotary_dim, 2 * kMaxHalf);
  KESSIE_REQUIRE(sections != nullptr && num_axes >= 1 && num_axes <= kMaxAxes, KESSIE_ERR_INVALID, "rope axes: %d axes (1 to %d)",
                 num_axes, kMaxAxes);
  int64_t sum = 0;
  for (int i = 0; i < num_axes; ++i) {
    KESSIE_REQUIRE(sections[i] >= 0, KESSIE_ERR_INVALID, "rope axes: section %d has %d pairs", i, sections[i]);
    sum += sections[i];
  }
  KESSIE_REQUIRE(sum == a.half, KESSIE_ERR_INVALID, "rope axes: sections hold %lld pairs, rotary_dim %d has %d", (long long)sum,
                 rotary_dim, a.half);
  for (auto& w : a.axis) w = 0;
  int left[kMaxAxes] = {};
  for (int i = 0; i < num_axes; ++i) left[i] = sections[i];
  for (int j = 0, ax = 0; j < a.half; ++j) {
    int use = ax;
    if (interleaved) {
      // Pair j is axis j mod A's until that section is used up, and axis 0's after.
      use = j % num_axes;
      if (j >= num_axes * sections[use]) use = 0;
    } else {
      while (left[ax] == 0) ++ax;
      use = ax;
    }
    KESSIE_REQUIRE(left[use] > 0, KESSIE_ERR_INVALID,
                   "rope axes: interleaved sections must leave the surplus to axis 0 (axis %d gets more pairs than its section)", use);
    --left[use];
    a.axis[j >> 5] |= (uint64_t)use << (2 * (j & 31));
  }
  a.sign = inverse ? -1.0f : 1.0f;
  a.page_shift = a.page_size > 0 && (a.page_size & (a.page_size - 1)) == 0 ? __builtin_ctz((unsigned)a.page_size) : -1;
  a.inv_heads = 1.0f / (float)(a.Hq + a.Hk + a.Hv > 0 ? a.Hq + a.Hk + a.Hv : 1);
  a.inv_half = 1.0f / (float)a.half;
  if (a.T == 0 || a.Hq + a.Hk == 0) return KESSIE_OK;
  KESSIE_REQUIRE(rows_apart(a.T, a.qo_ts, a.Hq, a.qo_hs, a.D) && (a.pool || rows_apart(a.T, a.ko_ts, a.Hk, a.ko_hs, a.D)),
                 KESSIE_ERR_INVALID, "rope axes: rows of an output overlap");
  KESSIE_REQUIRE(a.pos && a.inv, KESSIE_ERR_INVALID, "rope axes: null pointer");
  switch (dtype) {
    case KESSIE_DTYPE_BF16: return adjacent ? launch<bf16_t, true>(a, s) : launch<bf16_t, false>(a, s);
    case KESSIE_DTYPE_F16: return adjacent ? launch<f16_t, true>(a, s) : launch<f16_t, false>(a, s);
    case KESSIE_DTYPE_F32: return adjacent ? launch<float, true>(a, s) : launch<float, false>(a, s);
  }
  set_error(KESSIE_ERR_UNSUPPORTED, "rope axes: dtype %d", dtype);
  return KESSIE_ERR_UNSUPPORTED;
}

}  // namespace
}  // namespace axes
}  // namespace kessie

using namespace kessie;
using namespace kessie::axes;

extern "C" int kessie_rope_axes(const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out,
                                int64_t q_out_tok_stride, int64_t q_out_head_stride, int num_q_heads, const void* k,
                                int64_t k_tok_stride, int64_t k_head_stride, void* k_out, int64_t k_out_tok_stride,
                                int64_t k_out_head_stride, int num_kv_heads, const void* positions,
                                int64_t positions_axis_stride, int positions_64, const float* inv_freq,
                                const int32_t* sections, int num_axes, int interleaved, int adjacent, int inverse,
                                int num_tokens, int head_dim, int rotary_dim, int dtype, void* stream) {
  clear_error();
  Args a{};
  a.q = q, a.q_ts = q_tok_stride, a.q_hs = q_head_stride;
  a.qo = q_out, a.qo_ts = q_out_tok_stride, a.qo_hs = q_out_head_stride;
  a.k = k, a.k_ts = k_tok_stride, a.k_hs = k_head_stride;
  a.ko = k_out, a.ko_ts = k_out_tok_stride, a.ko_hs = k_out_head_stride;
  a.pos = positions, a.pos_as = positions_axis_stride, a.pos64 = positions_64;
  a.inv = inv_freq;
  a.T = num_tokens, a.Hq = q ? num_q_heads : 0, a.Hk = k ? num_kv_heads : 0, a.D = head_dim;
  KESSIE_REQUIRE((q == nullptr) == (q_out == nullptr) && (k == nullptr) == (k_out == nullptr), KESSIE_ERR_INVALID,
                 "rope axes: an input without its output");
  return dispatch(a, sections, num_axes, interleaved, adjacent, inverse, rotary_dim, dtype, as_stream(stream));
}

extern "C" int kessie_rope_axes_cache_write(
    const void* q, int64_t q_tok_stride, int64_t q_head_stride, void* q_out, int64_t q_out_tok_stride,
    int64_t q_out_head_stride, int num_q_heads, const void* k, int64_t k_tok_stride, int64_t k_head_stride, const void* v,
    int64_t v_tok_stride, int64_t v_head_stride, int num_kv_heads, const void* positions, int64_t positions_axis_stride,
    int positions_64, const float* inv_freq, const int32_t* sections, int num_axes, int interleaved, int adjacent,
    void* kv_pool, int64_t page_stride, int64_t tok_stride, int64_t kv_stride, int64_t head_stride,
    const int64_t* slot_mapping, int page_size, int num_pages, int num_tokens, int head_dim, int rotary_dim, int dtype,
    void* stream) {
  clear_error();
  Args a{};
  a.q = q, a.q_ts = q_tok_stride, a.q_hs = q_head_stride;
  a.qo = q_out, a.qo_ts = q_out_tok_stride, a.qo_hs = q_out_head_stride;
  a.k = k, a.k_ts = k_tok_stride, a.k_hs = k_head_stride;
  a.v = v, a.v_ts = v_tok_stride, a.v_hs = v_head_stride;
  a.pool = kv_pool, a.page_stride = page_stride, a.tok_stride = tok_stride, a.kv_stride = kv_stride, a.head_stride = head_stride;
  a.slots = slot_mapping, a.page_size = page_size, a.num_pages = num_pages;
  a.pos = positions, a.pos_as = positions_axis_stride, a.pos64 = positions_64;
  a.inv = inv_freq;
  a.T = num_tokens, a.Hq = q ? num_q_heads : 0, a.Hk = num_kv_heads, a.Hv = num_kv_heads, a.D = head_dim;
  KESSIE_REQUIRE((q == nullptr) == (q_out == nullptr), KESSIE_ERR_INVALID, "rope axes: an input without its output");
  KESSIE_REQUIRE(page_size > 0 && num_pages >= 0 && num_kv_heads > 0, KESSIE_ERR_INVALID, "rope axes: bad sizes P=%d pages=%d Hkv=%d",
                 page_size, num_pages, num_kv_heads);
  KESSIE_REQUIRE(num_tokens <= 0 || (k && v && kv_pool && slot_mapping), KESSIE_ERR_INVALID, "rope axes: null pointer");
  KESSIE_REQUIRE(rows_apart(page_size, tok_stride, num_kv_heads, head_stride, head_dim) && kv_stride > 0, KESSIE_ERR_INVALID,
                 "rope axes: pool strides overlap");
  return dispatch(a, sections, num_axes, interleaved, adjacent, 0, rotary_dim, dtype, as_stream(stream));
}

extern "C" int kessie_rope_remap_axes(void* kv_pool, int64_t page_stride, int64_t tok_stride, int64_t head_stride,
                                      const int32_t* page_list, int num_pages, const void* orig_pos,
                                      int64_t orig_axis_stride, const void* tgt_pos, int64_t tgt_axis_stride,
                                      int positions_64, const float* inv_freq, const int32_t* sections, int num_axes,
                                      int interleaved, int adjacent, int num_tokens, int num_heads, int head_dim,
                                      int rotary_dim, int page_size, int dtype, void* stream) {
  clear_error();
  Args a{};
  a.pos = tgt_pos, a.pos_as = tgt_axis_stride, a.pos64 = positions_64;
  a.from = orig_pos, a.from_as = orig_axis_stride;
  a.inv = inv_freq;
  a.T = num_tokens, a.Hk = num_heads, a.D = head_dim;
  KESSIE_REQUIRE(num_heads > 0, KESSIE_ERR_INVALID, "rope axes: %d heads", num_heads);
  KESSIE_REQUIRE(num_tokens <= 0 || (kv_pool && orig_pos), KESSIE_ERR_INVALID, "rope axes: null pointer");
  if (page_list) {
    KESSIE_REQUIRE(page_size > 0 && num_pages >= 0, KESSIE_ERR_INVALID, "rope axes: page_size=%d num_pages=%d", page_size, num_pages);
    KESSIE_REQUIRE(rows_apart(page_size, tok_stride, num_heads, head_stride, head_dim), KESSIE_ERR_INVALID,
                   "rope axes: pool strides overlap (tok %lld head %lld)", (long long)tok_stride, (long long)head_stride);
    a.pool = kv_pool, a.page_stride = page_stride, a.tok_stride = tok_stride, a.head_stride = head_stride;
    a.pages = page_list, a.page_size = page_size, a.num_pages = num_pages;
  } else {  // dense rows
    a.k = a.ko = kv_pool;
    a.k_ts = a.ko_ts = tok_stride, a.k_hs = a.ko_hs = head_stride;
  }
  return dispatch(a, sections, num_axes, interleaved, adjacent, 0, rotary_dim, dtype, as_stream(stream));
}
