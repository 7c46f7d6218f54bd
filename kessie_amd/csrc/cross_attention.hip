// Cross attention for gfx950: each sequence's queries over its own encoder
// states, all of them (no causal order, no window), any state length.
//
//   out[t, h] = sum_j softmax_j(q[t, h] . k[j, h / G] * sm_scale) v[j, h / G]
//
// over the states j of t's sequence that key_mask leaves; no state, zeros.
//
// A row is a (query, head) pair: the C * G rows of one (sequence, kv head) are
// packed, since they read the same states.  Two kernels share one core, which
// takes 32 rows and 32 states at a time:
//
//   S^T = K Q^T   v_mfma_f32_32x32x16 (fp32: 32x32x2), states x rows: lane l
//                 holds row l % 32 and, in register i, state 8 (i / 4) + 4 (l / 32)
//                 + i % 4, so the softmax of a row is within a lane and its
//                 partner l ^ 32;
//   O^T += V^T P^T  p leaves the softmax as the B operand: over one MFMA's
//                 16 states the order is free, and taking them as each half-wave
//                 holds them (4 of every 8) only asks that V^T comes in that
//                 order too, which the transposing LDS read does (16 lanes read
//                 4 states x 16 elements, each receives 4 states of one element).
//
// K and V go from global memory to LDS without registers (16 bytes a lane,
// 1 KiB an instruction, LDS-destination buffer loads), rows as they lie but for
// their 16-byte chunks, XOR-ed by the row so that both reads spread over all
// banks.  The buffer's record count ends with the sequence's last state, and
// what lies past it arrives as zeros: no NaN from a neighbour's states meets a
// probability of zero.
#include <type_traits>

#include "attn_common.h"

namespace kessie {
namespace cross {
namespace {

using attn::kNegInf;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRsrcWord3 = 0x00020000;  // word 3 of a raw buffer resource (gfx9 family)

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
#define KESSIE_LDS __attribute__((address_space(3)))

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
  // sm_scale * log2(e), at least the smallest normal number (so that -inf stays -inf
  // at a scale of zero); a negative scale flips q instead (flip).
  float c2;
  int flip;
  // Split partials, per row t * Hq + h and split: unnormalised sums [rows][S][D], base-2
  // maxima and sums [rows][S].
  int S;
  float* ws_o;
  float* ws_m;
  float* ws_l;
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

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// 1 KiB from a buffer into LDS at the (uniform) byte address `lds`, lane l's 16
// bytes at +16 l; lanes past the buffer's end write zeros.  Inline assembly: the
// builtin makes the compiler wait for it before any LDS read that follows.  It
// has no output registers; wait_loads is what it is waited for with.
__device__ __forceinline__ void load_to_lds(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
// All but the last n loads done.
template <int n>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory");
}
// This wave's loads landed and its LDS reads done, then everybody's.
__device__ __forceinline__ void wait_loads_and_meet() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *reinterpret_cast<KESSIE_LDS const V*>(at);
}

// x of this lane and of its partner l ^ 32.  (The builtin, given one value for
// both operands, is folded as if both results were that value; s_nop 1: the two
// wait states the swap needs after a VALU write of its operands.)
__device__ __forceinline__ f32x2 both_halves(float x) {
  float a = x, b = x;
  asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(a), "+v"(b));
  return f32x2{a, b};
}
__device__ __forceinline__ float max_halves(float x) {
  const f32x2 y = both_halves(x);
  return fmaxf(y[0], y[1]);
}
__device__ __forceinline__ float sum_halves(float x) {
  const f32x2 y = both_halves(x);
  return y[0] + y[1];
}

template <typename T>
struct Half;  // the 16-bit types
template <>
struct Half<bf16_t> {
  typedef bf16x8 v8;
  typedef bf16x2 v2;
  static constexpr uint32_t kOnes = 0x3f803f80u;
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // acc + the sum of two packed values
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, kOnes), acc, false);
  }
};
template <>
struct Half<f16_t> {
  typedef f16x8 v8;
  typedef f16x2 v2;
  static constexpr uint32_t kOnes = 0x3c003c00u;
  static __device__ __forceinline__ f32x16 mma(v8 a, v8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ float sum2(uint32_t w, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, w), __builtin_bit_cast(v2, kOnes), acc, false);
  }
};
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2){a, b}, typename Half<T>::v2));
}

// What the kernels share: LDS layout, operands, 32 states at a time.
template <typename T, int D>
struct Core {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int RB = D * (int)sizeof(T);  // bytes of a state's row (128, 256 or 512)
  static constexpr int CH = RB / 16;             // chunks of a row
  static constexpr int RPI = 64 / CH;            // rows a load instruction fills
  static constexpr int DB = D / 32;              // 32-element blocks of O
  // The chunk that row r keeps at place c is c ^ swizzle(r).  K is read a chunk a row, 32 rows at a time:
  // 16 rows spread over all 256 bytes of the banks.  V^T: 4 rows x 32 bytes by 16 lanes, twice (fp32: 32 elements of
  // rows r and r + 4).
  static __device__ __forceinline__ int k_swizzle(int r) { return RB == 128 ? (r >> 1) & 7 : r & 15; }
  static __device__ __forceinline__ int v_swizzle(int r) {
    return kF32 ? ((r >> 2) & 1) << 3 : RB == 128 ? ((r >> 1) & 1) << 2 : (r & 3) << 2;
  }

  // Loads: instruction n of a tile fills rows n * RPI ..; this lane's byte offset in the tile's global rows.
  static __device__ __forceinline__ uint32_t k_offset(int n, int lane, int ts_b) {
    const int r = n * RPI + lane / CH;
    return (uint32_t)r * (uint32_t)ts_b + (uint32_t)(((lane % CH) ^ k_swizzle(r)) * 16);
  }
  static __device__ __forceinline__ uint32_t v_offset(int n, int lane, int ts_b) {
    const int r = n * RPI + lane / CH;
    return (uint32_t)r * (uint32_t)ts_b + (uint32_t)(((lane % CH) ^ v_swizzle(r)) * 16);
  }

  // Q of this lane's row as the B operand: 16-bit, step s holds d = 16 s + 8 half ..; fp32, step s
  // d = half * D / 2 + s (the order of d within the product is free).
  static constexpr int QN = kF32 ? D / 8 : D / 16;
  typedef typename std::conditional<kF32, f32x4, typename std::conditional<kF32, bf16x8, typename Half<typename std::conditional<kF32, bf16_t, T>::type>::v8>::type>::type QV;
  static __device__ __forceinline__ int q_elem(int s, int half) { return kF32 ? half * (D / 2) + 4 * s : 16 * s + 8 * half; }

  uint32_t ka[QN];  // LDS offsets of K's operands of a 32-state block
  uint32_t va[DB];  // and of V^T's
  __device__ __forceinline__ void init(int lane) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int s = 0; s < QN; ++s) ka[s] = (uint32_t)(col * RB + (((kF32 ? half * (CH / 2) + s : 2 * s + half) ^ k_swizzle(col)) * 16));
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      if (kF32) {
        va[db] = (uint32_t)(4 * half * RB + (((8 * db + (col >> 2)) ^ v_swizzle(4 * half)) * 16) + 4 * (col & 3));
      } else {
        const int i = lane & 15, r = 4 * half + (i >> 2);  // of rows 16 c + 8 e + r
        va[db] = (uint32_t)(r * RB + (((4 * db + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1)) ^ v_swizzle(r)) * 16) + 8 * (i & 1));
      }
    }
  }
  __device__ __forceinline__ QV k_read(uint32_t base, int s) const { return lds_read<QV>(base + ka[s]); }
  // V^T of states 16 c .. 16 c + 15 of a block, elements 32 db ..
  __device__ __forceinline__ QV v_read(uint32_t base, int c, int db) const {
    const uint32_t at = base + va[db] + (uint32_t)(16 * c * RB);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<KESSIE_LDS s16x4*>(at));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<KESSIE_LDS s16x4*>(at + 8 * RB));
    return __builtin_bit_cast(QV, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  }

  // S^T of the 32 states whose K lies at `base`.
  __device__ __forceinline__ f32x16 scores(uint32_t base, const QV (&q)[QN]) const {
    f32x16 s = f32x16{};
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      const QV k = k_read(base, i);
      if constexpr (kF32) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(k[e], q[i][e], s, 0, 0, 0);
      } else {
        s = Half<T>::mma(k, q[i], s);
      }
    }
    return s;
  }
  // O^T += V^T P^T over the 32 states whose V lies at `base`.  Returns the sum of this lane's p as the product took
  // them (16-bit types: rounded to T, so that the weights that V meets are the ones that the sum normalises).
  __device__ __forceinline__ float add(uint32_t base, const f32x16& p, f32x16 (&o)[DB]) const {
    float sum = 0.0f;
    if constexpr (kF32) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum += p[i];
#pragma unroll
        for (int db = 0; db < DB; ++db)
          o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(lds_read<float>(base + va[db] + (uint32_t)((8 * (i / 4) + i % 4) * RB)), p[i],
                                                       o[db], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[i] = pack2<T>(p[8 * c + 2 * i], p[8 * c + 2 * i + 1]);
          sum = Half<T>::sum2(w[i], sum);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = Half<T>::mma(v_read(base, c, db), __builtin_bit_cast(QV, w), o[db]);
      }
    }
    return sum;
  }
  // Scores of hidden states (bits of `seen` not set: 32 states) become -inf.
  static __device__ __forceinline__ void hide(f32x16& s, uint32_t seen, int half) {
    const uint32_t mine = seen >> (4 * half);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = (mine >> (8 * (i / 4) + i % 4)) & 1 ? s[i] : kNegInf;
  }
  static __device__ __forceinline__ float top(const f32x16& s) {
    float m = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) m = fmaxf(m, s[i]);
    return m;
  }

  // Q of a row (or zeros).
  static __device__ __forceinline__ void load_q(const Args& a, const Seq& s, int row, int g, int half, QV (&q)[QN], bool ok) {
    const int pos = (unsigned)row / (unsigned)a.G, h = g * a.G + row - pos * a.G;
    const T* at = static_cast<const T*>(a.q) + (int64_t)(s.q0 + pos) * a.q_ts + (int64_t)h * a.q_hs;
#pragma unroll
    for (int i = 0; i < QN; ++i) {
      q[i] = QV{};
      if (ok) q[i] = *reinterpret_cast<const QV*>(at + q_elem(i, half));
      if (a.flip) q[i] = -q[i];
    }
  }
};

// The buffer of a tile of `rows` rows (none: every lane past its end).
__device__ __forceinline__ i32x4 tile_rsrc(const char* base, int rows, int ts_b, int row_bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  return i32x4{uniform((int)(uint32_t)b), uniform((int)((b >> 32) & 0xffff)), uniform(rows > 0 ? (rows - 1) * ts_b + row_bytes : 0),
               kRsrcWord3};
}

// Which states of a tile are there and not hidden, one bit each.  With a mask,
// lane i keeps the bits of tile 64 n + i of this wave's tiles and loads the next
// 64 tiles' when they are asked for (in rising order).
template <bool kMask, int KT>
struct Seen {
  const uint8_t* mask;  // of the sequence's first state
  int nkv, first, step;  // this wave's tile t is tile first + t * step of the sequence
  uint64_t mine;
  __device__ __forceinline__ int rows(int t) const { return min(max(nkv - (first + t * step) * KT, 0), KT); }
  __device__ __forceinline__ uint64_t at(int t, int lane) {
    const int n = rows(t);
    const uint64_t there = n >= 64 ? ~0ull : (1ull << n) - 1ull;
    if constexpr (!kMask) return there;
    if ((t & 63) == 0) {
      const int n_own = rows(t + lane);
      const uint8_t* p = mask + (int64_t)(first + (t + lane) * step) * KT;
      const int sh = (int)(reinterpret_cast<uintptr_t>(p) & 3);
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p - sh);
      // (Aligned words that hold a byte of the tile at least.)
      uint64_t lo = 0, hi = 0;
#pragma unroll
      for (int i = 0; i <= KT / 4; ++i) {
        const uint32_t x = 4 * i < n_own + sh && n_own > 0 ? w[i] : 0u;
        const uint32_t y = ((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) >> 7) & 0x01010101u;  // bit 0 of a byte: it is not zero
        const uint64_t nib = (y * 0x10204080u) >> 28;
        if (i < 16) lo |= nib << (4 * i);
        else hi = nib;
      }
      mine = sh ? (lo >> sh) | (hi << (64 - sh)) : lo;
    }
    const int l = t & 63;
    const uint64_t bits = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, l) |
                          (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(mine >> 32), l) << 32;
    return bits & there;
  }
};

// Stores O^T of a row from the accumulators: element 32 db + 8 (i / 4) + 4 half + i % 4 in register i.
template <typename T, int D>
__device__ __forceinline__ void store_row(T* row, const f32x16 (&o)[D / 32], float by, int half) {
  typedef T V __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      V y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = from_f32<T>(o[db][4 * i + e] * by);
      *reinterpret_cast<V*>(row + 32 * db + 8 * i + 4 * half) = y;
    }
}

// Up to 32 rows of a (sequence, kv head): decoding.  Every wave streams tiles
// of its own (wave w of split s takes tiles s * NW + w, + S * NW, ...) through
// two LDS stages of its own, the next tile in flight while one is computed: no
// barrier before the merge.  Bound: HBM.
template <typename T, int D, int KT, int NW, bool kMask, bool kSplit>
__global__ __launch_bounds__(NW * 64) void cross_rows_kernel(Args a) {
  typedef Core<T, D> C;
  constexpr int NB = KT / 32;            // 32-state blocks of a tile
  constexpr int NI = KT / C::RPI;        // load instructions of a K (or V) tile
  constexpr uint32_t kTile = KT * C::RB;  // bytes of a K (or V) tile
  constexpr int kOut = D + 4;            // row stride of the merge
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(KESSIE_LDS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int g = blockIdx.x % a.Hkv, unit = blockIdx.x / a.Hkv;
  const int b = kSplit ? unit / a.S : unit, split = kSplit ? unit - b * a.S : 0;
  const Seq sq = sequence(a, b);
  const int rows = sq.nq * a.G;
  if (rows == 0) return;
  typename C::QV q[C::QN];
  C::load_q(a, sq, min(col, rows - 1), g, half, q, col < rows);

  const int ts_k = (int)a.k_ts * (int)sizeof(T), ts_v = (int)a.v_ts * (int)sizeof(T);
  const char* kbase = static_cast<const char*>(a.k) + ((int64_t)sq.kv0 * a.k_ts + (int64_t)g * a.k_hs) * (int64_t)sizeof(T);
  const char* vbase = static_cast<const char*>(a.v) + ((int64_t)sq.kv0 * a.v_ts + (int64_t)g * a.v_hs) * (int64_t)sizeof(T);
  const int tiles = div_up(sq.nkv, KT), first = split * NW + wave, step = a.S * NW;
  const int n = tiles > first ? (tiles - first + step - 1) / step : 0;
  Seen<kMask, KT> seen{kMask ? a.mask + sq.kv0 : nullptr, sq.nkv, first, step, 0};
  const uint32_t mine = lds0 + (uint32_t)wave * 4 * kTile;  // this wave's stages: K, V, K, V
  C core;
  core.init(lane);

  uint64_t bits[2];
  auto issue = [&](int t, int stage) {
    const uint64_t at = seen.at(t, lane);
    bits[stage] = at;
    const int tile = first + t * step, r = seen.rows(t);
    const i32x4 kr = tile_rsrc(kbase + (int64_t)tile * KT * ts_k, r, ts_k, C::RB);
    const i32x4 vr = tile_rsrc(vbase + (int64_t)tile * KT * ts_v, r, ts_v, C::RB);
    const uint32_t to = mine + (uint32_t)stage * 2 * kTile;
#pragma unroll
    for (int i = 0; i < NI; ++i) load_to_lds(kr, C::k_offset(i, lane, ts_k), uniform(to + 1024u * i));
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t off = C::v_offset(i, lane, ts_v);
      // (A hidden state's V arrives as zeros, whatever it holds.)
      if (kMask && !((at >> (i * C::RPI + lane / C::CH)) & 1)) off = 0xffffff00u;
      load_to_lds(vr, off, uniform(to + kTile + 1024u * i));
    }
  };

  f32x16 o[C::DB];
#pragma unroll
  for (int i = 0; i < C::DB; ++i) o[i] = f32x16{};
  float m = kNegInf, l = 0.0f;
  auto tile = [&](int t, int stage) {
    wait_loads<2 * NI>();
    const uint32_t at = mine + (uint32_t)stage * 2 * kTile;
    f32x16 s[NB];
    float top = kNegInf;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      s[nb] = core.scores(at + (uint32_t)(32 * nb * C::RB), q);
      const uint32_t some = (uint32_t)(bits[stage] >> (32 * nb));
      if (some != 0xffffffffu) C::hide(s[nb], some, half);
      top = fmaxf(top, C::top(s[nb]));
    }
    const float mn = fmaxf(m, max_halves(top) * a.c2);
    const float use = mn == kNegInf ? 0.0f : mn;
    const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int i = 0; i < C::DB; ++i) o[i] *= alpha;
      l *= alpha;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[nb][i] = __builtin_amdgcn_exp2f(fmaf(s[nb][i], a.c2, -use));
      l += core.add(at + kTile + (uint32_t)(32 * nb * C::RB), s[nb], o);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this stage is read
    issue(t + 2, stage);
  };
  if (n > 0) {
    issue(0, 0);
    issue(1, 1);
    for (int t = 0; t < n; t += 2) {
      tile(t, 0);
      if (t + 1 < n) tile(t + 1, 1);
    }
  }
  l = sum_halves(l);

  // The waves' (o, m, l) meet in LDS, in wave order.
  wait_loads_and_meet();
  float* so = reinterpret_cast<float*>(smem);
  float* sm = so + NW * 32 * kOut;
  float* sl = sm + NW * 32;
  if (col < rows) {
    store_row<float, D>(so + (wave * 32 + col) * kOut, o, 1.0f, half);
    if (half == 0) {
      sm[wave * 32 + col] = m;
      sl[wave * 32 + col] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * (D / 4); i += NW * 64) {
    const int r = i / (D / 4), d = 4 * (i % (D / 4));
    float top = sm[r];
#pragma unroll
    for (int w = 1; w < NW; ++w) top = fmaxf(top, sm[w * 32 + r]);
    const float use = top == kNegInf ? 0.0f : top;
    f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float e = __builtin_amdgcn_exp2f(sm[w * 32 + r] - use);
      sum += e * sl[w * 32 + r];
      if (e != 0.0f) y += e * *reinterpret_cast<const f32x4*>(so + (w * 32 + r) * kOut + d);
    }
    const int pos = (unsigned)r / (unsigned)a.G, h = g * a.G + r - pos * a.G;
    if constexpr (kSplit) {
      const int64_t row = ((int64_t)(sq.q0 + pos) * a.Hq + h) * a.S + split;
      *reinterpret_cast<f32x4*>(a.ws_o + row * D + d) = y;
      if (d == 0) {
        a.ws_m[row] = top;
        a.ws_l[row] = sum;
      }
    } else {
      typedef T V __attribute__((ext_vector_type(4)));
      const float il = sum != 0.0f ? 1.0f / sum : 0.0f;
      V z;
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = from_f32<T>(y[e] * il);
      *reinterpret_cast<V*>(static_cast<T*>(a.out) + (int64_t)(sq.q0 + pos) * a.o_ts + (int64_t)h * a.o_hs + d) = z;
    }
  }
}

// max(a, b, c) in one instruction (fmaxf on MFMA results first quiets each
// input).  Inline assembly gets no wait states from the compiler's MFMA hazard
// checks: its uses read scores whose MFMAs lie a whole PV product back, or
// settle() them first.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// 24 wait states after the MFMAs that wrote s (a 32x32 result needs 18).
__device__ __forceinline__ void settle(f32x16& s) { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" : "+v"(s)); }

// Headroom of the lazy rescale, in log2 units: probabilities up to 2^8, as
// exact in either type as any up to 1; the O accumulators move only when a row's
// maximum rises by more.
constexpr float kSlack = 8.0f;

// Prompts: W waves of 32 rows each over tiles of 64 states that the workgroup
// loads together, two stages of K and of V.  Iteration t asks for K of tile t + 2
// and V of tile t + 1 (their stages were read in iteration t - 1), runs the
// softmax of tile t in the shadow of S^T(t + 1), then O^T += V^T P^T(t); one
// barrier.  Each MFMA is issued with its share of the other work and its
// operands two steps ahead, in a fixed order (a scheduling barrier a step).
template <typename T, int D, int W, bool kMask, bool kSplit>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void cross_tile_kernel(Args a) {
  typedef Core<T, D> C;
  typedef typename C::QV QV;
  constexpr int KT = 64;
  constexpr int NI = KT / C::RPI / W;  // load instructions of a wave for a K (or V) tile
  constexpr uint32_t kTile = KT * C::RB;
  constexpr int kRows = W * 32;
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(KESSIE_LDS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int g = blockIdx.x % a.Hkv;
  int rt = blockIdx.x / a.Hkv;
  // x / Hkv numbers the live (sequence, row tile) pairs in order; the grid's surplus ends here.
  int b = -1;
  for (int b0 = 0, before = 0; b0 < a.B; b0 += 64) {
    const int nt = b0 + lane < a.B ? div_up(sequence(a, b0 + lane).nq * a.G, kRows) : 0;
    int inc = nt;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(inc, o, 64);
      if (lane >= o) inc += y;
    }
    const int total = __builtin_amdgcn_readlane(inc, 63);
    if (rt < before + total) {
      const int l = __ffsll((unsigned long long)__ballot(before + inc > rt)) - 1;
      b = uniform(b0 + l);
      rt = uniform(rt - before - __builtin_amdgcn_readlane(inc - nt, l));
      break;
    }
    before += total;
  }
  if (b < 0) return;
  Seq sq = sequence(a, b);
  sq.q0 = uniform(sq.q0), sq.nq = uniform(sq.nq), sq.kv0 = uniform(sq.kv0), sq.nkv = uniform(sq.nkv);
  const int rows = sq.nq * a.G, row = rt * kRows + wave * 32 + col;
  QV q[C::QN];
  C::load_q(a, sq, min(row, rows - 1), g, half, q, row < rows);

  const int ts_k = (int)a.k_ts * (int)sizeof(T), ts_v = (int)a.v_ts * (int)sizeof(T);
  const char* kbase = static_cast<const char*>(a.k) + ((int64_t)sq.kv0 * a.k_ts + (int64_t)g * a.k_hs) * (int64_t)sizeof(T);
  const char* vbase = static_cast<const char*>(a.v) + ((int64_t)sq.kv0 * a.v_ts + (int64_t)g * a.v_hs) * (int64_t)sizeof(T);
  const int split = kSplit ? (int)blockIdx.z : 0, S = kSplit ? a.S : 1;
  const int tiles = div_up(sq.nkv, KT);
  const int n = uniform(tiles > split ? (tiles - split + S - 1) / S : 0);
  Seen<kMask, KT> seen{kMask ? a.mask + sq.kv0 : nullptr, sq.nkv, split, S, 0};
  C core;
  core.init(lane);
  uint32_t ko[NI], vo[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    ko[i] = C::k_offset(wave + W * i, lane, ts_k);
    vo[i] = C::v_offset(wave + W * i, lane, ts_v);
  }
  // Stages: K, K, V, V.
  auto issue_k = [&](int t, int stage) {
    const i32x4 r = tile_rsrc(kbase + (int64_t)(split + t * S) * KT * ts_k, seen.rows(t), ts_k, C::RB);
#pragma unroll
    for (int i = 0; i < NI; ++i) load_to_lds(r, ko[i], uniform(lds0 + stage * kTile + 1024u * (wave + W * i)));
  };
  auto issue_v = [&](int t, int stage, uint64_t bits) {
    const i32x4 r = tile_rsrc(vbase + (int64_t)(split + t * S) * KT * ts_v, seen.rows(t), ts_v, C::RB);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      uint32_t off = vo[i];
      if (kMask && !((bits >> ((wave + W * i) * C::RPI + lane / C::CH)) & 1)) off = 0xffffff00u;
      load_to_lds(r, off, uniform(lds0 + (2 + stage) * kTile + 1024u * (wave + W * i)));
    }
  };

  f32x16 o[C::DB];
#pragma unroll
  for (int i = 0; i < C::DB; ++i) o[i] = f32x16{};
  float m = kNegInf, l = 0.0f;
  const float c2 = a.c2;
  uint64_t now = 0, next = 0;  // states of tiles t and t + 1
  auto iteration = [&](int t, f32x16 (&s)[2], f32x16 (&sn)[2], const int par) {
    issue_k(t + 2, par);
    issue_v(t + 1, par ^ 1, next);
    const uint32_t kn = lds0 + (par ^ 1) * kTile, vn = lds0 + (2 + par) * kTile;
    if (now != ~0ull) {
      C::hide(s[0], (uint32_t)now, half);
      C::hide(s[1], (uint32_t)(now >> 32), half);
    }
    now = next;
    next = seen.at(t + 2, lane);
    float ma = s[0][0], mb = s[1][0];
#pragma unroll
    for (int i = 1; i < 15; i += 2) {
      ma = max3(ma, s[0][i], s[0][i + 1]);
      mb = max3(mb, s[1][i], s[1][i + 1]);
    }
    ma = max3(ma, s[0][15], mb);
    ma = max3(ma, s[1][15], s[1][15]);
    const float top = max_halves(ma) * c2;
    const float mn = top > m + kSlack ? top : m;
    const float use = mn == kNegInf ? 0.0f : mn;
    const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int i = 0; i < C::DB; ++i) o[i] *= alpha;
      l *= alpha;
    }
    m = mn;
    if constexpr (C::kF32) {
      sn[0] = core.scores(kn, q);
      sn[1] = core.scores(kn + 32 * C::RB, q);
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[nb][i] = __builtin_amdgcn_exp2f(fmaf(s[nb][i], c2, -use));
        l += core.add(vn + (uint32_t)(32 * nb * C::RB), s[nb], o);
      }
    } else {
      constexpr int kQ = 2 * C::QN, kPV = 4 * C::DB, kPairs = 16 / kQ;
      u32x4 w[4];  // p as V^T's partner: w[c] of states 16 c ..
      float l0 = 0.0f, l1 = 0.0f;
      auto exp_pair = [&](int j) {
        const int nb = j >> 3, i = 2 * (j & 7);
        const uint32_t x = pack2<T>(__builtin_amdgcn_exp2f(fmaf(s[nb][i], c2, -use)), __builtin_amdgcn_exp2f(fmaf(s[nb][i + 1], c2, -use)));
        w[j >> 2][j & 3] = x;
        if (j & 1) l1 = Half<T>::sum2(x, l1);
        else l0 = Half<T>::sum2(x, l0);
      };
      auto operand = [&](int i) {
        if (i < kQ) return core.k_read(kn + (uint32_t)(32 * (i & 1) * C::RB), i >> 1);
        const int j = i - kQ, c = j / C::DB;
        return core.v_read(vn + (uint32_t)(32 * (c >> 1) * C::RB), c & 1, j % C::DB);
      };
      constexpr int kAhead = 2;
      QV op[kAhead + 1];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) op[i] = operand(i);
#pragma unroll
      for (int i = 0; i < kQ + kPV; ++i) {
        if (i < kQ) {
          sn[i & 1] = Half<T>::mma(op[i % (kAhead + 1)], q[i >> 1], i < 2 ? f32x16{} : sn[i & 1]);
        } else {
          const int j = i - kQ;
          o[j % C::DB] = Half<T>::mma(op[i % (kAhead + 1)], __builtin_bit_cast(QV, w[j / C::DB]), o[j % C::DB]);
        }
        if (i + kAhead < kQ + kPV) op[(i + kAhead) % (kAhead + 1)] = operand(i + kAhead);
        if (i < kQ) {
#pragma unroll
          for (int e = 0; e < kPairs; ++e) exp_pair(i * kPairs + e);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      l += l0 + l1;
    }
    wait_loads_and_meet();
  };
  if (n > 0) {
    now = seen.at(0, lane);
    next = seen.at(1, lane);
    issue_k(0, 0);
    issue_v(0, 0, now);
    issue_k(1, 1);
    wait_loads_and_meet();
    f32x16 sa[2], sb[2];
    sa[0] = core.scores(lds0, q);
    sa[1] = core.scores(lds0 + 32 * C::RB, q);
    settle(sa[0]);
    settle(sa[1]);
    wait_loads_and_meet();  // (iteration 0 loads over tile 0's K)
    for (int t = 0; t < n; t += 2) {
      iteration(t, sa, sb, 0);
      if (t + 1 < n) iteration(t + 1, sb, sa, 1);
    }
  }
  l = sum_halves(l);
  if (row >= rows) return;
  const int pos = (unsigned)row / (unsigned)a.G, h = g * a.G + row - pos * a.G;
  if constexpr (kSplit) {
    const int64_t r = ((int64_t)(sq.q0 + pos) * a.Hq + h) * S + split;
    store_row<float, D>(a.ws_o + r * D, o, 1.0f, half);
    if (half == 0) {
      a.ws_m[r] = m;
      a.ws_l[r] = l;
    }
  } else {
    store_row<T, D>(static_cast<T*>(a.out) + (int64_t)(sq.q0 + pos) * a.o_ts + (int64_t)h * a.o_hs, o, l != 0.0f ? 1.0f / l : 0.0f, half);
  }
}

// Merges the S partials of a row: one wave a (query, head), in split order.
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_combine_kernel(Args a) {
  const int lane = threadIdx.x & 63;
  const int64_t n = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int64_t item = n / a.Hq;
  const int h = (int)(n - item * a.Hq), b = (int)(item / a.max_q), i = (int)(item - (int64_t)b * a.max_q);
  if (b >= a.B) return;
  const Seq s = sequence(a, b);
  if (i >= s.nq) return;
  const int64_t row = ((int64_t)(s.q0 + i) * a.Hq + h) * a.S;
  float top = kNegInf;
  for (int x = lane; x < a.S; x += 64) top = fmaxf(top, a.ws_m[row + x]);
#pragma unroll
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
  const float use = top == kNegInf ? 0.0f : top;
  constexpr int N = D / 64;  // elements of a lane
  float y[N] = {}, sum = 0.0f;
  for (int x = 0; x < a.S; ++x) {
    const float e = __builtin_amdgcn_exp2f(a.ws_m[row + x] - use);
    sum += e * a.ws_l[row + x];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float v = a.ws_o[(row + x) * D + lane * N + k];
      if (e != 0.0f) y[k] += e * v;
    }
  }
  const float il = sum != 0.0f ? 1.0f / sum : 0.0f;
  T* out = static_cast<T*>(a.out) + (int64_t)(s.q0 + i) * a.o_ts + (int64_t)h * a.o_hs + lane * N;
#pragma unroll
  for (int k = 0; k < N; ++k) out[k] = from_f32<T>(y[k] * il);
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
  for (int d = lane; d < a.D; d += 64) sq[d] = to_f32(q[d]) * (a.flip ? -a.c2 : a.c2);
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

// Dynamic LDS past 64 KiB is asked for once per kernel and device.
template <typename F>
int launch_lds(F kernel, const Args& a, dim3 grid, int threads, size_t lds, hipStream_t s) {
  static bool set[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!set[dev]) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
      set_error(KESSIE_ERR_HIP, "cross attention: %zu bytes of LDS unavailable", lds);
      return KESSIE_ERR_HIP;
    }
    set[dev] = true;
  }
  hipLaunchKernelGGL(kernel, grid, dim3(threads), lds, s, a);
  return check_launch("cross attention");
}

// The grid: rows kernel or tile kernel, and the splits of the states.
struct Plan {
  bool few;       // cross_rows_kernel
  int S;
  int64_t tiles;  // workgroups per kv head and split
};
constexpr int kRowsWaves = 4, kTileWaves = 4;
template <typename T, int D>
constexpr int rows_kt() {
  return 32;
}
Plan make_plan(int B, int max_q, int Tq, int Hq, int Hkv, int D, int max_kv, int es) {
  const int G = Hq / Hkv, cus = attn::device_cus();
  Plan p;
  p.few = (int64_t)max_q * G <= 32;
  if (p.few) {
    p.tiles = B;
    const int64_t units = (int64_t)B * Hkv;
    const int waves_tiles = div_up(max_kv, 32 * kRowsWaves);  // tiles of a wave, unsplit
    int64_t S = (2 * cus + units - 1) / units;
    if (S > waves_tiles / 4) S = waves_tiles / 4;
    p.S = S < 1 ? 1 : (int)S;
  } else {
    const int rows = kTileWaves * 32;
    const int64_t by_len = (int64_t)B * (((int64_t)max_q * G + rows - 1) / rows), by_rows = (int64_t)Tq * G / rows + B;
    p.tiles = by_len < by_rows ? by_len : by_rows;
    const int64_t wgs = p.tiles * Hkv;
    int64_t S = 2 * cus / wgs;
    if (S > div_up(max_kv, 64) / 8) S = div_up(max_kv, 64) / 8;
    p.S = S < 1 ? 1 : (int)S;
  }
  return p;
}

template <typename T, int D, bool kMask, bool kSplit>
int launch_fast(const Args& a, const Plan& p, hipStream_t s) {
  typedef Core<T, D> C;
  if (p.few) {
    constexpr int KT = rows_kt<T, D>(), NW = C::RB == 512 ? 2 : kRowsWaves;
    constexpr size_t stages = (size_t)NW * 4 * KT * C::RB, merge = (size_t)NW * 32 * (D + 4 + 2) * 4;
    return launch_lds(cross_rows_kernel<T, D, KT, NW, kMask, kSplit>, a, dim3((unsigned)(p.tiles * a.Hkv * p.S)), NW * 64,
                      stages > merge ? stages : merge, s);
  }
  constexpr int W = kTileWaves;
  return launch_lds(cross_tile_kernel<T, D, W, kMask, kSplit>, a, dim3((unsigned)(p.tiles * a.Hkv), 1, p.S), W * 64, (size_t)4 * 64 * C::RB, s);
}

template <typename T, int D>
int launch_split(const Args& a, const Plan& p, hipStream_t s) {
  if (p.S == 1) return a.mask ? launch_fast<T, D, true, false>(a, p, s) : launch_fast<T, D, false, false>(a, p, s);
  const int st = a.mask ? launch_fast<T, D, true, true>(a, p, s) : launch_fast<T, D, false, true>(a, p, s);
  if (st != KESSIE_OK) return st;
  const int64_t rows = (int64_t)a.B * a.max_q * a.Hq;
  hipLaunchKernelGGL((cross_combine_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a);
  return check_launch("cross attention (combine)");
}

size_t partial_bytes(const Plan& p, int Tq, int Hq, int D) {
  return p.S > 1 ? (size_t)Tq * Hq * p.S * (D + 2) * sizeof(float) : 0;
}

template <typename T>
int launch(Args& a, void* ws, size_t ws_bytes, hipStream_t s) {
  constexpr int N = 16 / (int)sizeof(T);
  const bool fast = (a.D == 64 || a.D == 128) && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out) &&
                    a.q_ts % N == 0 && a.q_hs % N == 0 && a.k_ts % N == 0 && a.k_hs % N == 0 && a.v_ts % N == 0 && a.v_hs % N == 0 &&
                    a.o_ts % N == 0 && a.o_hs % N == 0 &&
                    // (a tile's bytes within a buffer's 31 bits)
                    a.k_ts >= 0 && a.v_ts >= 0 && a.k_ts * (int64_t)sizeof(T) < (1 << 24) && a.v_ts * (int64_t)sizeof(T) < (1 << 24);
  if (!fast) return launch_generic<T>(a, s);
  const Plan p = make_plan(a.B, a.max_q, a.Tq, a.Hq, a.Hkv, a.D, a.max_kv, (int)sizeof(T));
  KESSIE_REQUIRE(p.tiles * a.Hkv * (p.few ? p.S : 1) <= 0x7fffffff && (int64_t)a.B * a.max_q * a.Hq <= (int64_t)4 * 0x7fffffff,
                 KESSIE_ERR_UNSUPPORTED, "cross attention: %d sequences of up to %d queries exceed one launch", a.B, a.max_q);
  const size_t need = partial_bytes(p, a.Tq, a.Hq, a.D);
  KESSIE_REQUIRE(ws_bytes >= need && (need == 0 || (ws && aligned16(ws))), KESSIE_ERR_WORKSPACE,
                 "cross attention: workspace of %zu bytes, %zu needed", ws_bytes, need);
  a.S = p.S;
  if (need) {
    a.ws_o = static_cast<float*>(ws);
    a.ws_m = a.ws_o + (size_t)a.Tq * a.Hq * p.S * a.D;
    a.ws_l = a.ws_m + (size_t)a.Tq * a.Hq * p.S;
  }
  return a.D == 64 ? launch_split<T, 64>(a, p, s) : launch_split<T, 128>(a, p, s);
}

}  // namespace
}  // namespace cross
}  // namespace kessie

using namespace kessie;
using namespace kessie::cross;

extern "C" size_t kessie_cross_attention_workspace_bytes(int batch, int max_query_len, int num_q_tokens, int num_q_heads,
                                                         int num_kv_heads, int head_dim, int max_kv_len, int dtype) {
  if (batch <= 0 || max_query_len <= 0 || num_q_tokens <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || max_kv_len < 0 ||
      (head_dim != 64 && head_dim != 128))
    return 0;
  return partial_bytes(make_plan(batch, max_query_len, num_q_tokens, num_q_heads, num_kv_heads, head_dim, max_kv_len, dtype_size(dtype)),
                       num_q_tokens, num_q_heads, head_dim);
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
  KESSIE_REQUIRE(fabsf(sm_scale) <= 3.402823466e38f, KESSIE_ERR_INVALID, "cross attention: sm_scale is not finite");
  KESSIE_REQUIRE(max_kv_len <= 1 << 30, KESSIE_ERR_UNSUPPORTED, "cross attention: %d states", max_kv_len);
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
  a.c2 = fabsf(sm_scale) * kLog2e;
  if (a.c2 < 1.17549435e-38f) a.c2 = 1.17549435e-38f;
  a.flip = sm_scale < 0.0f;
  const hipStream_t s = as_stream(stream);
  switch (dtype) {
    case KESSIE_DTYPE_BF16: return launch<bf16_t>(a, workspace, workspace_bytes, s);
    case KESSIE_DTYPE_F16: return launch<f16_t>(a, workspace, workspace_bytes, s);
    default: return launch<float>(a, workspace, workspace_bytes, s);
  }
}
