// Cross attention for gfx950: each sequence's queries over its own encoder
// states, all of them (no causal order, no window), any state length.
//
//   out[t, h] = sum_j softmax_j(q[t, h] . k[j, h / G] * sm_scale) v[j, h / G]
//
// over the states j of t's sequence that key_mask leaves; no state, zeros.
//
// A row is a (query, head) pair: the C * G rows of one (sequence, kv head) are
// packed, since they read the same states.  cross_rows_kernel (few rows: HBM or
// latency bound) and cross_tile_kernel (many: MFMA bound) share one core, which
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
  // Work split over the states: `shares` workgroups per kv head wanted, each of at least min_steps steps.  plan: what the
  // main kernel's first workgroup leaves for the merge (each sequence's first step; the tile kernel, the pieces' length).
  // Partials of part_rows rows each: unnormalised sums [rows][D], base-2 maxima and sums.
  int shares, min_steps, part_rows;
  int64_t* plan;
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
// The same for what is read once (non-temporal).
__device__ __forceinline__ void stream_to_lds(i32x4 rsrc, uint32_t voff, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
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
  typedef typename Half<typename std::conditional<kF32, bf16_t, T>::type>::v8 Half8;
  typedef typename std::conditional<kF32, f32x4, Half8>::type QV;
  static __device__ __forceinline__ int q_elem(int s, int half) { return kF32 ? half * (D / 2) + 4 * s : 16 * s + 8 * half; }

  uint32_t ka[QN];  // LDS offsets of K's operands of a 32-state block
  uint32_t va[DB];  // and of V^T's
  __device__ __forceinline__ void init(int lane) {
    const int col = lane & 31, half = lane >> 5;
#pragma unroll
    for (int s = 0; s < QN; ++s)
      ka[s] = (uint32_t)(col * RB + (((kF32 ? half * (CH / 2) + s : 2 * s + half) ^ k_swizzle(col)) * 16));
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
  // kAhead: with fp32's operands read a group ahead, in this order (the compiler's own, with little else to do between,
  // waits for each: 32 x 1 on 1,500, 16 heads of 64, 97 us against 83).
  template <bool kAhead>
  __device__ __forceinline__ float add(uint32_t base, const f32x16& p, f32x16 (&o)[DB]) const {
    float sum = 0.0f;
    if constexpr (kF32 && kAhead) {
      float v[2][4][DB];
      auto read = [&](int g) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int db = 0; db < DB; ++db) v[g & 1][i][db] = lds_read<float>(base + va[db] + (uint32_t)((8 * g + i) * RB));
      };
      read(0);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        if (g < 3) read(g + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sum += p[4 * g + i];
#pragma unroll
          for (int db = 0; db < DB; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[g & 1][i][db], p[4 * g + i], o[db], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else if constexpr (kF32) {
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
  // Scores of hidden states (bits of `seen` not set: 32 states) become -inf: the bit as a word of ones (a signed
  // bit-field read), then a select by it.
  static __device__ __forceinline__ void hide(f32x16& s, uint32_t seen, int half) {
    const int mine = (int)(seen >> (4 * half));
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const uint32_t keep = (uint32_t)((mine << (31 - (8 * (i / 4) + i % 4))) >> 31);
      s[i] = __uint_as_float((__float_as_uint(s[i]) & keep) | (0xff800000u & ~keep));
    }
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
    }
  }
  // A negative sm_scale (after the first tiles are asked for: it waits for q).
  static __device__ __forceinline__ void flip_q(const Args& a, QV (&q)[QN]) {
    if (a.flip) {
#pragma unroll
      for (int i = 0; i < QN; ++i) q[i] = -q[i];
    }
  }
};

// The buffer of a tile of `rows` rows (none: every lane past its end).
__device__ __forceinline__ i32x4 tile_rsrc(const char* base, int rows, int ts_b, int row_bytes) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  return i32x4{uniform((int)(uint32_t)b), uniform((int)((b >> 32) & 0xffff)), uniform(rows > 0 ? (rows - 1) * ts_b + row_bytes : 0),
               kRsrcWord3};
}

// Which states of a tile of cross_rows_kernel are there and not hidden, one bit each.  With a mask,
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

// One stretch of a workgroup's work: steps t .. end - 1 of row tile rt of sequence b.
struct Stretch {
  int b, rt, t, end, steps;  // steps: of the whole row tile
  Seq sq;
};

// The row tiles and steps of sequence s (a sequence without states has one step, which stores its zeros).
__device__ __forceinline__ int row_tiles(const Args& a, const Seq& s, int rows) { return div_up(s.nq * a.G, rows); }
__device__ __forceinline__ int steps_of(const Seq& s, int keys) { return max(div_up(s.nkv, keys), 1); }

__device__ __forceinline__ int64_t uniform64(int64_t x) {
  return (int64_t)(((uint64_t)(uint32_t)uniform((int)((uint64_t)x >> 32)) << 32) | (uint32_t)uniform((int)(uint32_t)x));
}
__device__ __forceinline__ Seq uniform_sequence(const Args& a, int b) {
  Seq s = sequence(a, b);
  s.q0 = uniform(s.q0), s.nq = uniform(s.nq), s.kv0 = uniform(s.kv0), s.nkv = uniform(s.nkv);
  return s;
}

// Shared work.  All (sequence, row tile, step) of a kv head in a row, `all` of
// them, are dealt out evenly: workgroup j of n takes all * j / n .. all * (j +
// 1) / n - 1, so lengths of any mix end together.  A row tile that lies in one
// workgroup is stored by it; of the others each workgroup holds a partial --
// number 1 of the tile it begins, 0 of the one that it goes on with -- and
// cross_combine_kernel merges them in order.
struct Share {
  int64_t all;
  int n;
};
__device__ __forceinline__ Share share_of(const Args& a, int64_t all) {
  const int64_t n = all / a.min_steps;
  return {all, (int)(n < 1 ? 1 : n < a.shares ? n : a.shares)};
}
// The workgroup that takes step x.
__device__ __forceinline__ int owner(const Share& s, int64_t x) {
  const uint64_t v = (uint64_t)((x + 1) * s.n - 1);
  return (v | (uint64_t)s.all) >> 32 ? (int)(v / (uint64_t)s.all) : (int)((uint32_t)v / (uint32_t)s.all);
}

// The partial row of this workgroup's row r: of the tile it begins, or goes on with.
__device__ __forceinline__ int64_t part_row(const Args& a, bool begins, int r) {
  return ((int64_t)blockIdx.x * 2 + begins) * a.part_rows + r;
}

// Walks the stretches of a workgroup.
template <bool kShare>
struct Walk {
  int64_t left;
  Stretch now;

  // False: nothing to do.  x: the workgroup's number among its kv head's.
  __device__ __forceinline__ bool begin(const Args& a, int x, int rows, int keys, int lane) {
    // Without sharing, workgroup x takes the x-th row tile of all; with it, the stretch from its first step.
    int64_t before = 0, at = x, count = 1, all = 0;
    if (kShare) {
      for (int b0 = 0; b0 < a.B; b0 += 64) {
        int64_t w = 0;
        if (b0 + lane < a.B) {
          const Seq s = sequence(a, b0 + lane);
          w = (int64_t)row_tiles(a, s, rows) * steps_of(s, keys);
        }
        int64_t inc = w;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int64_t y = __shfl_up(inc, o, 64);
          if (lane >= o) inc += y;
        }
        if (blockIdx.x == 0 && b0 + lane < a.B && threadIdx.x < 64) a.plan[b0 + lane] = all + inc - w;
        all += __shfl(inc, 63, 64);
      }
      if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[a.B] = all;
      const Share s = share_of(a, all);
      if (x >= s.n) return false;
      at = all * x / s.n;
      count = all * (x + 1) / s.n - at;
    }
    at = uniform64(at);
    left = uniform64(count);
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      int64_t w = 0;
      if (b0 + lane < a.B) {
        const Seq s = sequence(a, b0 + lane);
        w = (int64_t)row_tiles(a, s, rows) * (kShare ? steps_of(s, keys) : 1);
      }
      int64_t inc = w;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int64_t y = __shfl_up(inc, o, 64);
        if (lane >= o) inc += y;
      }
      const int64_t total = __shfl(inc, 63, 64);
      if (at < before + total) {
        const int l = __ffsll((unsigned long long)__ballot(before + inc > at)) - 1;
        const int off = uniform((int)(at - before - __shfl(inc - w, l, 64)));
        now.b = uniform(b0 + l);
        now.sq = uniform_sequence(a, now.b);
        now.steps = steps_of(now.sq, keys);
        now.rt = kShare ? uniform(off / now.steps) : off;
        now.t = kShare ? uniform(off - now.rt * now.steps) : 0;
        cut();
        return true;
      }
      before += total;
    }
    return false;
  }
  __device__ __forceinline__ void cut() {
    now.end = kShare ? (int)min((int64_t)now.steps, now.t + left) : now.steps;
    if (kShare) left -= now.end - now.t;
  }
  // On to the next stretch; false: done.
  __device__ __forceinline__ bool next(const Args& a, int rows, int keys) {
    if (!kShare || left <= 0) return false;
    now.t = 0;
    if (++now.rt >= row_tiles(a, now.sq, rows)) {
      now.rt = 0;
      do {
        now.sq = uniform_sequence(a, ++now.b);
      } while (now.sq.nq == 0);  // (there is one: work is left)
      now.steps = steps_of(now.sq, keys);
    }
    cut();
    return true;
  }
};

// The same value for the compiler's eyes too (loop-carried values would stay in vector registers).
__device__ __forceinline__ Stretch uniform(const Stretch& s) {
  return {uniform(s.b), uniform(s.rt), uniform(s.t), uniform(s.end), uniform(s.steps),
          {uniform(s.sq.q0), uniform(s.sq.nq), uniform(s.sq.kv0), uniform(s.sq.nkv)}};
}

// Pieces of the tile kernel: each row tile of a sequence is cut into
// ceil(steps / limit) stretches of equal length, one workgroup a stretch.
struct Piece {
  int rt, t, end, steps, pieces;
  int first;  // number of the row tile's first piece
  Seq sq;
};
// Lane l's sequence of the 64 from b0 on (none: no rows).
__device__ __forceinline__ Seq lane_sequence(const Args& a, int b0, int lane) {
  return b0 + lane < a.B ? sequence(a, b0 + lane) : Seq{0, 0, 0, 0};
}
// Finds the x-th piece of a kv head, or with kMerge its x-th row tile of several pieces; false: there is none.
// limit < 0: to be found first, the longest stretch: an even share of the work.  One load of the lengths for up to 64
// sequences.
template <bool kMerge>
__device__ __forceinline__ bool find_piece(const Args& a, int x, int rows, int keys, int& limit, int lane, Piece& p) {
  Seq mine = lane_sequence(a, 0, lane);
  if (limit < 0) {
    float work = 0.0f;  // (fp32: every workgroup comes to the same limit, exact or not)
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      if (b0 > 0) mine = lane_sequence(a, b0, lane);
      float w = (float)row_tiles(a, mine, rows) * (float)steps_of(mine, keys);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) w += __shfl_xor(w, o, 64);
      work += w;
    }
    if (a.B > 64) mine = lane_sequence(a, 0, lane);
    // (ceil, and a little more for what the sums were rounded off, 2^-24 each of B / 64 + 10: at most `shares` pieces and
    // one a row tile.)
    limit = uniform(max((int)fminf(ceilf(work / (float)a.shares * (1.0001f + 1.0e-8f * (float)a.B)), 1.0e9f), a.min_steps));
  }
  // Long pieces (more than half the limit: all pieces of tiles that are cut are) are numbered first, so that the short
  // ones fill the end.
  int before = 0;
#pragma unroll 1
  for (int cls = 0; cls < (limit && !kMerge ? 2 : 1); ++cls) {
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      if (a.B > 64) mine = lane_sequence(a, b0, lane);
      const int steps = steps_of(mine, keys), c = limit ? div_up(steps, limit) : 1;
      const bool here = !limit || (2 * div_up(steps, c) > limit) == (cls == 0);
      const int n = here ? row_tiles(a, mine, rows) : 0;
      int inc = n * c;
      [[maybe_unused]] int tiles = c > 1 ? n : 0;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(inc, o, 64);
        if (lane >= o) inc += y;
        if (kMerge) {
          const int z = __shfl_up(tiles, o, 64);
          if (lane >= o) tiles += z;
        }
      }
      const int total = __builtin_amdgcn_readlane(kMerge ? tiles : inc, 63);
      if (x < total) {
        const int l = __ffsll((unsigned long long)__ballot((kMerge ? tiles : inc) > x)) - 1;
        const int off = x - __builtin_amdgcn_readlane(kMerge ? tiles - (c > 1 ? n : 0) : inc - n * c, l);
        p.sq = Seq{__builtin_amdgcn_readlane(mine.q0, l), __builtin_amdgcn_readlane(mine.nq, l), __builtin_amdgcn_readlane(mine.kv0, l),
                   __builtin_amdgcn_readlane(mine.nkv, l)};
        p.steps = steps_of(p.sq, keys);
        p.pieces = __builtin_amdgcn_readlane(c, l);
        p.rt = kMerge ? off : uniform(off / p.pieces);
        p.first = before + __builtin_amdgcn_readlane(inc - n * c, l) + p.rt * p.pieces;
        const int i = kMerge ? 0 : off - p.rt * p.pieces, per = uniform(div_up(p.steps, p.pieces));
        p.t = i * per;
        p.end = min(p.t + per, p.steps);
        return true;
      }
      x -= total;
      before += __builtin_amdgcn_readlane(inc, 63);
    }
  }
  return false;
}

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

// 32 rows of a (sequence, kv head): decoding, and prompts too small to fill the
// device with larger tiles.  A step is NW tiles, one a wave; every wave streams
// its tiles through two LDS stages of its own, the next tile in flight while one
// is computed: no barrier before the merge.
//
// Decoding is bound by HBM.  16 x 1 query over 6,400 to 25,600 states (64 / 8
// heads of 128, bf16, 0.92 GB) 151 us with the combine = 6.1 TB/s, 88 % of what
// this card's best reads reach; 32 x 1 over 1,500 (16 heads of 64, 0.2 GB, every
// sequence and head one workgroup) 37 us = 5.3 TB/s.
template <typename T, int D, int KT, int NW, bool kMask, bool kShare>
__global__ __launch_bounds__(NW * 64) void cross_rows_kernel(Args a) {
  typedef Core<T, D> C;
  constexpr int NB = KT / 32;            // 32-state blocks of a tile
  constexpr int NI = KT / C::RPI;        // load instructions of a K (or V) tile
  constexpr uint32_t kTile = KT * C::RB;  // bytes of a K (or V) tile
  constexpr int kOut = D + 4;            // row stride of the merge
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(KESSIE_LDS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int g = blockIdx.x % a.Hkv;
  const int ts_k = (int)a.k_ts * (int)sizeof(T), ts_v = (int)a.v_ts * (int)sizeof(T);
  Walk<kShare> walk;
  if (!walk.begin(a, blockIdx.x / a.Hkv, 32, NW * KT, lane)) return;
  C core;
  core.init(lane);
  do {
    const Stretch now = uniform(walk.now);
    const Seq sq = now.sq;
    const int row0 = now.rt * 32, rows = min(sq.nq * a.G - row0, 32);
    typename C::QV q[C::QN];
    C::load_q(a, sq, row0 + min(col, rows - 1), g, half, q, col < rows);
    const char* kbase = static_cast<const char*>(a.k) + ((int64_t)sq.kv0 * a.k_ts + (int64_t)g * a.k_hs) * (int64_t)sizeof(T);
    const char* vbase = static_cast<const char*>(a.v) + ((int64_t)sq.kv0 * a.v_ts + (int64_t)g * a.v_hs) * (int64_t)sizeof(T);
    const int nkv = (int)min((int64_t)sq.nkv, (int64_t)now.end * (NW * KT));  // states up to this stretch's end
    const int first = now.t * NW + wave, step = NW;
    const int n = uniform(max(div_up(div_up(nkv, KT) - first, step), 0));
    Seen<kMask, KT> seen{kMask ? a.mask + sq.kv0 : nullptr, nkv, first, step, 0};
    const uint32_t mine = lds0 + (uint32_t)wave * 4 * kTile;  // this wave's stages: K, V, K, V

    uint64_t bits[2];
    auto issue = [&](int t, int stage) {
      const uint64_t at = seen.at(t, lane);
      bits[stage] = at;
      const int tile = first + t * step, r = seen.rows(t);
      const i32x4 kr = tile_rsrc(kbase + (int64_t)tile * KT * ts_k, r, ts_k, C::RB);
      const i32x4 vr = tile_rsrc(vbase + (int64_t)tile * KT * ts_v, r, ts_v, C::RB);
      const uint32_t to = mine + (uint32_t)stage * 2 * kTile;
#pragma unroll
      for (int i = 0; i < NI; ++i) stream_to_lds(kr, C::k_offset(i, lane, ts_k), uniform(to + 1024u * i));
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        uint32_t off = C::v_offset(i, lane, ts_v);
        // (A hidden state's V arrives as zeros, whatever it holds.)
        if (kMask && !((at >> (i * C::RPI + lane / C::CH)) & 1)) off = 0xffffff00u;
        stream_to_lds(vr, off, uniform(to + kTile + 1024u * i));
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
        l += core.template add<true>(at + kTile + (uint32_t)(32 * nb * C::RB), s[nb], o);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this stage is read
      issue(t + 2, stage);
    };
    if (n > 0) {
      issue(0, 0);
      issue(1, 1);
      C::flip_q(a, q);
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
      const int pos = (unsigned)(row0 + r) / (unsigned)a.G, h = g * a.G + row0 + r - pos * a.G;
      if (kShare && !(now.t == 0 && now.end == now.steps)) {
        const int64_t row = part_row(a, now.t == 0, r);
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
    if (kShare) __syncthreads();  // (the next stretch loads over the merge)
  } while (walk.next(a, 32, NW * KT));
}

// max(a, b, c) in one instruction (fmaxf on MFMA results first quiets each
// input).  Inline assembly gets no wait states from the compiler's MFMA hazard
// checks (a 32x32 result needs 18): its use reads scores four MFMAs after the
// last one that wrote them.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Headroom of the lazy rescale, in log2 units: probabilities up to 2^8, as
// exact in either type as any up to 1; the O accumulators move only when a row's
// maximum rises by more.
constexpr float kSlack = 8.0f;

// States of a tile of cross_tile_kernel: 64 KiB of LDS or 32, so that two workgroups of four waves share a CU, and each
// SIMD has one's softmax to run beside the other's MFMAs (fp32, head_dim 128: 2 x 1,000 on 4,000, 8 heads, 267 us
// against 344 with one).
__host__ __device__ constexpr int tile_keys(int row_bytes) { return row_bytes == 512 ? 32 : 64; }

// Prompts: W waves of 32 rows each over tiles of 64 states that the workgroup
// loads together, two stages of K and of V.  Iteration t asks for K of tile t + 2
// and V of tile t + 1 (their stages were read in iteration t - 1), runs the
// softmax of tile t in the shadow of S^T(t + 1), then O^T += V^T P^T(t); one
// barrier.  Each MFMA is issued with its share of the other work and its
// operands two steps ahead, in a fixed order (a scheduling barrier a step).
//
// 4,096 queries over 16,384 states (32 / 8 heads of 128, bf16, 1.1 TFLOP): 916 us
// = 1,200 TFLOP/s, 89 % of a large library product; the MFMA pipes are 63 % busy
// at the 1.64 GHz that power leaves, LDS 32 %, no bank conflicts.  More stages or
// operands read 3 to 8 steps ahead changed nothing: a wave's issue bounds a step
// (its MFMA, operand reads and a share of the softmax, 52 to 65 cycles, beside
// the other wave's), and 64 rows a wave, with nothing beside it, came to 937
// TFLOP/s.  2 x 2,048 over 4,096 (16 heads of 64): 77 us, 890 TFLOP/s,
// where the 32 exp2 of a lane take as long as the MFMAs.
template <typename T, int D, int W, bool kMask, bool kShare>
__global__ __launch_bounds__(W * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void cross_tile_kernel(Args a) {
  typedef Core<T, D> C;
  typedef typename C::QV QV;
  constexpr int KT = tile_keys(C::RB), NB = KT / 32;
  constexpr int NI = KT / C::RPI / W;  // load instructions of a wave for a K (or V) tile
  constexpr uint32_t kTile = KT * C::RB;
  constexpr int kRows = W * 32;
  extern __shared__ __align__(16) unsigned char smem[];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(KESSIE_LDS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = uniform((int)threadIdx.x >> 6), col = lane & 31, half = lane >> 5;
  const int g = blockIdx.x % a.Hkv;
  const int ts_k = (int)a.k_ts * (int)sizeof(T), ts_v = (int)a.v_ts * (int)sizeof(T);
  int limit = kShare ? -1 : 0;
  Piece now;
  const bool some = find_piece<false>(a, blockIdx.x / a.Hkv, kRows, KT, limit, lane, now);
  if (kShare && blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<int32_t*>(a.plan) = limit;
  if (!some) return;
  C core;
  core.init(lane);
  uint32_t ko[NI], vo[NI];
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    ko[i] = C::k_offset(wave + W * i, lane, ts_k);
    vo[i] = C::v_offset(wave + W * i, lane, ts_v);
  }
  const Seq sq = now.sq;
  const int rows = sq.nq * a.G, row = now.rt * kRows + wave * 32 + col;
  QV q[C::QN];
  C::load_q(a, sq, min(row, rows - 1), g, half, q, row < rows);
  const char* kbase = static_cast<const char*>(a.k) + ((int64_t)sq.kv0 * a.k_ts + (int64_t)g * a.k_hs) * (int64_t)sizeof(T);
  const char* vbase = static_cast<const char*>(a.v) + ((int64_t)sq.kv0 * a.v_ts + (int64_t)g * a.v_hs) * (int64_t)sizeof(T);
  const int first = now.t, nkv = (int)min((int64_t)sq.nkv, (int64_t)now.end * KT);
  const int n = uniform(max(div_up(nkv, KT) - first, 0));
  auto rows_of = [&](int t) { return min(max(nkv - (first + t) * KT, 0), KT); };
  // The states of a tile that are there and not hidden, one bit each; the mask's bytes are loaded a tile ahead.
  auto mask_byte = [&](int t) {
    const int j = (first + t) * KT + lane;
    return kMask && j < nkv ? (int)a.mask[(int64_t)sq.kv0 + j] : 0;
  };
  auto seen = [&](int t, int byte) {
    const int n = rows_of(t);
    const uint64_t there = n >= 64 ? ~0ull : (1ull << n) - 1ull;  // (KT == 32: n is 32 at most)
    return kMask ? there & __builtin_amdgcn_ballot_w64(byte != 0) : there;
  };
  // Stages: K, K, V, V.  Tiles are loaded in order: the next one's place is carried along.
  const char* kp = kbase + (int64_t)first * KT * ts_k;
  const char* vp = vbase + (int64_t)first * KT * ts_v;
  auto issue_k = [&](int t, int stage) {
    const i32x4 r = tile_rsrc(kp, rows_of(t), ts_k, C::RB);
    kp += KT * ts_k;
#pragma unroll
    for (int i = 0; i < NI; ++i) load_to_lds(r, ko[i], uniform(lds0 + stage * kTile + 1024u * (wave + W * i)));
  };
  auto issue_v = [&](int t, int stage, uint64_t bits) {
    const i32x4 r = tile_rsrc(vp, rows_of(t), ts_v, C::RB);
    vp += KT * ts_v;
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
  uint64_t bits = 0, bits1 = 0;  // the states of tiles t and t + 1
  int byte = 0;                  // this lane's mask byte of tile t + 2
  float high = 0.0f;             // this lane's largest score of tile t, before any are hidden
  // The maximum with this tile's; returns what is taken from the scores.
  auto rescale = [&](float top) {
    const float mn = top > m + kSlack ? top : m;
    const float alpha = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
    if (__builtin_amdgcn_ballot_w64(alpha != 1.0f) != 0) {
#pragma unroll
      for (int i = 0; i < C::DB; ++i) o[i] *= alpha;
      l *= alpha;
    }
    m = mn;
    return mn == kNegInf ? 0.0f : mn;
  };
  constexpr uint64_t kFull = KT == 64 ? ~0ull : 0xffffffffull;
  auto hide = [&](f32x16 (&s)[NB], uint64_t seen) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) C::hide(s[nb], (uint32_t)(seen >> (32 * nb)), half);
  };
  auto largest = [](const f32x16 (&s)[NB]) { return NB == 1 ? C::top(s[0]) : fmaxf(C::top(s[0]), C::top(s[NB - 1])); };
  auto scores = [&](uint32_t base, f32x16 (&s)[NB]) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) s[nb] = core.scores(base + (uint32_t)(32 * nb * C::RB), q);
  };
  auto iteration = [&](int t, f32x16 (&s)[NB], f32x16 (&sn)[NB], const int par) {  // par = t % 2
    const uint64_t bits2 = seen(t + 2, byte);
    byte = mask_byte(t + 3);
    issue_k(t + 2, par);
    issue_v(t + 1, par ^ 1, bits1);
    const uint32_t kn = lds0 + (par ^ 1) * kTile, vn = lds0 + (2 + par) * kTile;
    if (bits != kFull) {
      hide(s, bits);
      high = largest(s);
    }
    bits = bits1;
    bits1 = bits2;
    const float use = rescale(max_halves(high) * c2);
    if constexpr (C::kF32) {
      if (t + 1 < n) scores(kn, sn);
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[nb][i] = __builtin_amdgcn_exp2f(fmaf(s[nb][i], c2, -use));
        l += core.template add<false>(vn + (uint32_t)(32 * nb * C::RB), s[nb], o);
      }
      high = largest(sn);
    } else {
      // Steps: the MFMAs of S^T(t + 1), then those of PV, each with its operand two steps ahead and its share of the
      // 16 score pairs, which go through three stages in three steps -- scaled; exp2; packed -- so that no stage waits
      // for the one before; a pair is packed before the PV step that takes it.  The last steps take the next tile's
      // largest score.  The sums of the packed pairs come after the last MFMA, in its shadow (947 us -> 916 for 4,096 on
      // 16,384; two fewer instructions a step is what counts).
      constexpr int kQ = 2 * C::QN, kPV = 4 * C::DB, kSpread = kQ + 3 * C::DB - 2;
      constexpr int kMaxAt = kQ + 4, kMaxPer = 16 / (kPV - 4) + (16 % (kPV - 4) != 0);
      static_assert(kQ + 3 * C::DB >= kSpread + 2, "the last pairs are packed in time");
      u32x4 w[4];  // p as V^T's partner: w[c] of states 16 c ..
      float l0 = 0.0f, l1 = 0.0f;
      float hi[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
      auto first_pair = [](int i) { return i < 0 ? 0 : i >= kSpread ? 16 : i * 16 / kSpread; };
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
          // (Holds the MFMA to its step: its result is wanted late, and the compiler moved half of them to the end.)
          if (i >= 2) asm volatile("" : "+v"(sn[i & 1]));
        } else {
          const int j = i - kQ;
          o[j % C::DB] = Half<T>::mma(op[i % (kAhead + 1)], __builtin_bit_cast(QV, w[j / C::DB]), o[j % C::DB]);
        }
        if (i + kAhead < kQ + kPV) op[(i + kAhead) % (kAhead + 1)] = operand(i + kAhead);
#pragma unroll
        for (int j = first_pair(i - 2); j < first_pair(i - 1); ++j) {
          const int nb = j >> 3, e = 2 * (j & 7);
          w[j >> 2][j & 3] = pack2<T>(s[nb][e], s[nb][e + 1]);
        }
#pragma unroll
        for (int j = first_pair(i - 1); j < first_pair(i); ++j) {
          const int nb = j >> 3, e = 2 * (j & 7);
          s[nb][e] = __builtin_amdgcn_exp2f(s[nb][e]);
          s[nb][e + 1] = __builtin_amdgcn_exp2f(s[nb][e + 1]);
        }
#pragma unroll
        for (int j = first_pair(i); j < first_pair(i + 1); ++j) {
          const int nb = j >> 3, e = 2 * (j & 7);
          s[nb][e] = fmaf(s[nb][e], c2, -use);
          s[nb][e + 1] = fmaf(s[nb][e + 1], c2, -use);
        }
#pragma unroll
        for (int j = (i - kMaxAt) * kMaxPer; j < (i - kMaxAt + 1) * kMaxPer && j < 16; ++j)
          if (j >= 0) hi[j & 3] = max3(hi[j & 3], sn[j & 1][j & ~1], sn[j & 1][j | 1]);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2) {
        l0 = Half<T>::sum2(w[j >> 2][j & 3], l0);
        l1 = Half<T>::sum2(w[j >> 2][(j + 1) & 3], l1);
      }
      l += l0 + l1;
      high = fmaxf(max3(hi[0], hi[1], hi[2]), hi[3]);
    }
    wait_loads_and_meet();
  };
  if (n > 0 && now.rt * kRows + wave * 32 >= rows) {
    // A wave without rows only loads its part of the tiles (13 x 21..701 on 640..6,404, 97 us -> 95).
    bits1 = seen(0, mask_byte(0));
    issue_k(0, 0);
    issue_v(0, 0, bits1);
    issue_k(1, 1);
    wait_loads_and_meet();
    wait_loads_and_meet();
    for (int t = 0; t < n; ++t) {
      bits1 = seen(t + 1, mask_byte(t + 1));
      issue_k(t + 2, t & 1);
      issue_v(t + 1, (t + 1) & 1, bits1);
      wait_loads_and_meet();
    }
  } else if (n > 0) {
    bits = seen(0, mask_byte(0));
    bits1 = seen(1, mask_byte(1));
    byte = mask_byte(2);
    issue_k(0, 0);
    issue_v(0, 0, bits);
    issue_k(1, 1);
    C::flip_q(a, q);
    wait_loads_and_meet();
    f32x16 sa[NB], sb[NB];
    scores(lds0, sa);
    high = largest(sa);
    wait_loads_and_meet();  // (iteration 0 loads over tile 0's K)
    for (int t = 0; t < n; t += 2) {
      iteration(t, sa, sb, 0);
      if (t + 1 < n) iteration(t + 1, sb, sa, 1);
    }
  }
  l = sum_halves(l);
  if (row < rows) {
    const int pos = (unsigned)row / (unsigned)a.G, h = g * a.G + row - pos * a.G;
    if (!kShare || now.pieces == 1) {
      T* to = static_cast<T*>(a.out) + (int64_t)(sq.q0 + pos) * a.o_ts + (int64_t)h * a.o_hs;
      store_row<T, D>(to, o, l != 0.0f ? 1.0f / l : 0.0f, half);
    } else {
      const int64_t r = (int64_t)blockIdx.x * a.part_rows + wave * 32 + col;
      store_row<float, D>(a.ws_o + r * D, o, 1.0f, half);
      if (half == 0) {
        a.ws_m[r] = m;
        a.ws_l[r] = l;
      }
    }
  }
}

// Sums n partials of a row, the i-th at row at(i) of the workspace, elements d ..
// d + 3: in order, by maximum and sum (the online form), eight in flight.
template <int D, typename F>
__device__ __forceinline__ f32x4 merge_partials(const Args& a, int n, int d, F at) {
  constexpr int kAhead = 8;
  float top = kNegInf, sum = 0.0f;
  f32x4 y = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i0 = 0; i0 < n; i0 += kAhead) {
    float m[kAhead], l[kAhead];
    f32x4 v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t row = at(min(i0 + i, n - 1));
      m[i] = a.ws_m[row];
      l[i] = a.ws_l[row];
      v[i] = *reinterpret_cast<const f32x4*>(a.ws_o + row * D + d);
    }
    float mn = top;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      if (i0 + i >= n) m[i] = kNegInf, l[i] = 0.0f;
      mn = fmaxf(mn, m[i]);
    }
    const float use = mn == kNegInf ? 0.0f : mn, was = __builtin_amdgcn_exp2f(top - use);
    sum *= was;
    y *= was;
    top = mn;
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const float e = __builtin_amdgcn_exp2f(m[i] - use);
      if (l[i] != 0.0f) {  // (a row of NaN scores has no maximum, but a sum: NaN)
        sum += e * l[i];
        y += e * v[i];
      }
    }
  }
  return y * (sum != 0.0f ? 1.0f / sum : 0.0f);
}
template <typename T>
__device__ __forceinline__ void store4(T* to, f32x4 y) {
  typedef T V __attribute__((ext_vector_type(4)));
  V z;
#pragma unroll
  for (int k = 0; k < 4; ++k) z[k] = from_f32<T>(y[k]);
  *reinterpret_cast<V*>(to) = z;
}

// Merges the pieces of `rows_wg` rows of a row tile that was cut.
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_merge_kernel(Args a, int rows_per, int keys, int rows_wg) {
  constexpr int kLanes = D / 4, kAtOnce = 256 / kLanes;
  const int lane = threadIdx.x & 63, d = 4 * (threadIdx.x % kLanes);
  const int g = blockIdx.x % a.Hkv;
  Piece p;
  int limit = uniform(*reinterpret_cast<const int32_t*>(a.plan));
  if (!find_piece<true>(a, blockIdx.x / a.Hkv, rows_per, keys, limit, lane, p)) return;
  const int rows = min(p.sq.nq * a.G - p.rt * rows_per, rows_per), end = min((int)(blockIdx.y + 1) * rows_wg, rows);
  const int64_t step = (int64_t)a.Hkv * a.part_rows, at = ((int64_t)p.first * a.Hkv + g) * a.part_rows;
  for (int r = blockIdx.y * rows_wg + threadIdx.x / kLanes; r < end; r += kAtOnce) {
    const f32x4 y = merge_partials<D>(a, p.pieces, d, [&](int i) { return at + r + i * step; });
    const int row = p.rt * rows_per + r, pos = (unsigned)row / (unsigned)a.G, h = g * a.G + row - pos * a.G;
    store4(static_cast<T*>(a.out) + (int64_t)(p.sq.q0 + pos) * a.o_ts + (int64_t)h * a.o_hs + d, y);
  }
}

// Merges the partials of rows that several workgroups share, in step order.  One
// wave a query and `heads` of its heads; D / 4 lanes a row, so 64 / (D / 4) heads
// at a time: the look-up of the sequence and its workgroups is shared by them.
template <typename T, int D>
__global__ __launch_bounds__(256) void cross_combine_kernel(Args a, int rows_per, int keys, int heads) {
  constexpr int kLanes = D / 4, kAtOnce = 64 / kLanes;
  const int lane = threadIdx.x & 63, sub = lane / kLanes, d = 4 * (lane % kLanes);
  const int t = uniform((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  if (t >= a.Tq) return;
  // The sequence that row t belongs to: the last that starts at or before it.
  const int q0 = a.q_start[0];
  int b = -1;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const bool le = b0 + lane < a.B && a.q_start[b0 + lane] - q0 <= t;
    const unsigned long long m = __ballot(le);
    if (m == 0) break;
    b = b0 + 63 - __clzll((long long)m);
  }
  b = uniform(b);
  if (b < 0) return;
  const Seq s = uniform_sequence(a, b);
  const int i = t - s.q0;
  if (i < 0 || i >= s.nq) return;
  const Share sh = share_of(a, a.plan[a.B]);
  const int steps = steps_of(s, keys);
  const int64_t before = a.plan[b];
  const int h_end = min(a.Hq, (int)(blockIdx.y + 1) * heads);
  int last = -1, j0 = 0, j1 = 0;
  for (int h0 = blockIdx.y * heads; h0 < h_end; h0 += kAtOnce) {
    const int h = min(h0 + sub, h_end - 1), g = h / a.G, row = i * a.G + h - g * a.G, rt = row / rows_per;
    const int64_t r = row - rt * rows_per;
    if (__builtin_amdgcn_ballot_w64(rt != last) != 0) {  // (a query's heads lie in one row tile, or in two)
      const int64_t x = before + (int64_t)rt * steps;
      j0 = owner(sh, x), j1 = owner(sh, x + steps - 1);
      last = rt;
    }
    if (j0 == j1 || h0 + sub >= h_end) continue;  // stored already
    // Partial of workgroup j: number 1 of the first, 0 of those after it.
    const f32x4 y = merge_partials<D>(a, j1 - j0 + 1, d, [&](int i) {
      return (((int64_t)(j0 + i) * a.Hkv + g) * 2 + (i == 0)) * a.part_rows + r;
    });
    store4(static_cast<T*>(a.out) + (int64_t)t * a.o_ts + (int64_t)h * a.o_hs + d, y);
  }
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
    const float mn = fmaxf(m, top), use = mn == kNegInf ? 0.0f : mn;
    const float alpha = exp2f(m - use), p = exp2f(y - use);
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
  const float il = l != 0.0f ? 1.0f / l : 0.0f;
  for (int e = 0; e < kMaxD / 64; ++e)
    if (lane + 64 * e < a.D) out[lane + 64 * e] = from_f32<T>(o[e] * il);
}

template <typename T>
int launch_generic(const Args& a, hipStream_t s) {
  KESSIE_REQUIRE(!attn::env_int("KESSIE_REQUIRE_MFMA", 0), KESSIE_ERR_UNSUPPORTED,
                 "cross attention: head_dim %d or these strides run on the generic kernel", a.D);
  const int64_t rows = (int64_t)a.B * a.max_q;
  KESSIE_REQUIRE(rows < 1 << 26, KESSIE_ERR_UNSUPPORTED, "cross attention: %lld rows exceed one launch", (long long)rows);
  hipLaunchKernelGGL(cross_generic_kernel<T>, dim3((unsigned)rows, a.Hq), dim3(64), 0, s, a);
  return check_launch("cross attention");
}

// Dynamic LDS past 64 KiB is asked for once per kernel and device.
template <auto kKernel>
int launch_lds(const Args& a, dim3 grid, int threads, size_t lds, hipStream_t s) {
  static bool set[64] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) dev = 0;
  if (!set[dev]) {
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kKernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds) != hipSuccess) {
      set_error(KESSIE_ERR_HIP, "cross attention: %zu bytes of LDS unavailable", lds);
      return KESSIE_ERR_HIP;
    }
    set[dev] = true;
  }
  hipLaunchKernelGGL(kKernel, grid, dim3(threads), lds, s, a);
  return check_launch("cross attention");
}

// The launch: which kernel, and whether the states are split.
struct Plan {
  int waves;        // 0: cross_rows_kernel; 4, 8: cross_tile_kernel
  int shares;       // workgroups wanted per kv head; 0: one a row tile, no partials
  int64_t tiles;    // at least the row tiles of a kv head
  int64_t grid;     // workgroups per kv head
  int min_steps, part_rows;
};
constexpr int kRowsKeys = 32;
// Waves of cross_rows_kernel: 32 KiB of LDS each, 64 at fp32 and head_dim 128.
template <typename T, int D>
constexpr int rows_waves() {
  return Core<T, D>::RB == 512 ? 2 : 4;
}
Plan make_plan(int B, int max_q, int Tq, int Hq, int Hkv, int D, int max_kv, int Tkv, int es) {
  const int G = Hq / Hkv, cus = attn::device_cus(), row_bytes = D * es;
  const int64_t most = (int64_t)max_q * G;  // rows of a sequence
  auto tiles_of = [&](int rows) {
    const int64_t by_len = (int64_t)B * ((most + rows - 1) / rows), by_rows = (int64_t)Tq * G / rows + B;
    return by_len < by_rows ? by_len : by_rows;
  };
  Plan p{};
  int keys, per_cu, gain;
  const int nw = row_bytes == 512 ? 2 : 4, rows_per_cu = 160 * 1024 / (nw * 4 * kRowsKeys * row_bytes);
  // Few rows altogether over few states (at most five tiles a wave; fp32: two or three): the waves of a workgroup share the
  // states of 32 rows and merge them in LDS.  1 x 60 on 600 (bf16, 8 heads of 128) 12.3 us against 15.3 with 128 rows a
  // workgroup, 1 x 300 on 100 (fp32, 8 heads of 128) 16.9 against 22.9; past that it loses: 1 x 60 on 1,000 15.7 against
  // 13.6, 2 x 60 on 180 in fp32 21.5 against 13.9, 4 x 50..101 on 577 (fp32, 12 heads of 64) 21.7 against 20.0.
  const int small_kv = (es == 2 ? 5 : row_bytes == 512 ? 2 : 3) * nw * kRowsKeys;
  const bool small = tiles_of(32) * Hkv <= (int64_t)cus * rows_per_cu && max_kv <= small_kv;
  if (most <= 32 || small) {
    p.tiles = most <= 32 ? B : tiles_of(32);
    p.part_rows = (int)(most < 32 ? most : 32);
    p.min_steps = 2;
    keys = nw * kRowsKeys;
    per_cu = rows_per_cu;
    gain = most <= 32 ? 5 : 1 << 30;
  } else {
    // Eight waves share a tile's load where that still gives every CU a workgroup: 4,096 queries on 16,384 (32 / 8
    // heads of 128) 931 us against 1,015 with four; 8 x 200 on 1,000 (8 heads) 32.2 against 23.9.
    // Shorter sequences fill tiles of 256 rows less well.
    p.waves = es == 2 && tiles_of(256) * Hkv >= cus && (int64_t)Tq * G >= (int64_t)1024 * B ? 8 : 4;
    const int rows = p.waves * 32;
    p.tiles = tiles_of(rows);
    p.part_rows = (int)(most < rows ? most : rows);
    keys = tile_keys(row_bytes);
    // fp32: a step is 3 us of MFMA work, so each may have a workgroup of its own while there are CUs for them: 1 x 60 on
    // 1,000 (8 heads of 64) 14.2 us against 17.2 with two steps each; past that it loses: 2 x 60 on 900 (8 heads of 128)
    // 24.2 against 20.9, 4 x 50..101 on 577 (12 heads of 64) 22.5 against 20.0.
    p.min_steps = es == 2 ? 4 : p.tiles * Hkv * div_up(max_kv, keys) <= cus ? 1 : 2;
    per_cu = p.waves == 8 ? 1 : 2;
    gain = es == 4 ? 4 : 14;
  }
  p.grid = p.tiles;
  // Split where the longest sequence would outlast an even share of the work by more than the merge costs (`gain`
  // steps: 5 us of it in decoding, 10 otherwise).  What an even share is goes by the means that the host knows.
  const int64_t slots = (int64_t)cus * per_cu;
  const double mean = B > 0 && Tkv / B < max_kv ? (double)Tkv / B : max_kv;
  const double tiles = p.waves ? (double)Tq * G / (p.waves * 32) + 0.5 * B : B;
  const double even = (tiles < p.tiles ? tiles : (double)p.tiles) * Hkv * (mean / keys + 0.5) / (double)slots;
  if (div_up(max_kv, keys) - even >= gain) {
    p.shares = (int)((slots + Hkv - 1) / Hkv);
    p.grid = p.waves ? p.shares + p.tiles : p.shares;
  }
  return p;
}

struct Layout {
  size_t plan, rows, bytes;  // bytes of the plan, partial rows, all bytes
};
Layout layout(const Plan& p, int B, int Hkv, int D) {
  Layout l{};
  if (p.shares) {
    l.plan = ((size_t)(B + 1) * 8 + 255) / 256 * 256;
    l.rows = (size_t)p.grid * Hkv * (p.waves ? 1 : 2) * p.part_rows;
    l.bytes = l.plan + l.rows * (D + 2) * sizeof(float);
  }
  return l;
}

template <typename T, int D, bool kMask, bool kShare>
int launch_fast(const Args& a, const Plan& p, hipStream_t s) {
  typedef Core<T, D> C;
  const dim3 grid((unsigned)(p.grid * a.Hkv));
  constexpr size_t tile = (size_t)4 * tile_keys(C::RB) * C::RB;
  if constexpr (!C::kF32) {
    if (p.waves == 8) return launch_lds<cross_tile_kernel<T, D, 8, kMask, kShare>>(a, grid, 512, tile, s);
  }
  if (p.waves) return launch_lds<cross_tile_kernel<T, D, 4, kMask, kShare>>(a, grid, 256, tile, s);
  constexpr int KT = kRowsKeys, NW = rows_waves<T, D>();
  constexpr size_t stages = (size_t)NW * 4 * KT * C::RB, merge = (size_t)NW * 32 * (D + 4 + 2) * 4;
  return launch_lds<cross_rows_kernel<T, D, KT, NW, kMask, kShare>>(a, grid, NW * 64, stages > merge ? stages : merge, s);
}

template <typename T, int D>
int launch_shared(const Args& a, const Plan& p, hipStream_t s) {
  if (!p.shares) return a.mask ? launch_fast<T, D, true, false>(a, p, s) : launch_fast<T, D, false, false>(a, p, s);
  const int st = a.mask ? launch_fast<T, D, true, true>(a, p, s) : launch_fast<T, D, false, true>(a, p, s);
  if (st != KESSIE_OK) return st;
  if (p.waves) {
    // 32 rows a workgroup, fewer where that leaves the device idle (each finds its row tile first).
    const int rows_wg = p.tiles * a.Hkv * div_up(p.part_rows, 32) < 2 * attn::device_cus() ? 1024 / D : 32;
    hipLaunchKernelGGL((cross_merge_kernel<T, D>), dim3((unsigned)(p.tiles * a.Hkv), div_up(p.part_rows, rows_wg)), dim3(256), 0, s, a,
                       p.waves * 32, tile_keys(D * (int)sizeof(T)), rows_wg);
    return check_launch("cross attention (merge)");
  }
  int heads = 256 / D;  // (a wave's at once)
  while (heads < a.Hq && (int64_t)a.Tq * div_up(a.Hq, heads) > 16 * attn::device_cus()) heads *= 2;
  hipLaunchKernelGGL((cross_combine_kernel<T, D>), dim3(div_up(a.Tq, 4), div_up(a.Hq, heads)), dim3(256), 0, s, a, 32,
                     rows_waves<T, D>() * kRowsKeys, heads);
  return check_launch("cross attention (combine)");
}

template <typename T>
int launch(Args& a, void* ws, size_t ws_bytes, hipStream_t s) {
  constexpr int N = 16 / (int)sizeof(T);
  const bool fast = (a.D == 64 || a.D == 128) && aligned16(a.q) && aligned16(a.k) && aligned16(a.v) && aligned16(a.out) &&
                    a.q_ts % N == 0 && a.q_hs % N == 0 && a.k_ts % N == 0 && a.k_hs % N == 0 && a.v_ts % N == 0 && a.v_hs % N == 0 &&
                    a.o_ts % N == 0 && a.o_hs % N == 0 &&
                    // (a tile's bytes within a buffer's 31 bits)
                    a.k_ts >= 0 && a.v_ts >= 0 && a.k_ts * (int64_t)sizeof(T) < (1 << 24) && a.v_ts * (int64_t)sizeof(T) < (1 << 24);
  if (!fast || attn::env_int("KESSIE_FORCE_GENERIC", 0)) return launch_generic<T>(a, s);
  const Plan p = make_plan(a.B, a.max_q, a.Tq, a.Hq, a.Hkv, a.D, a.max_kv, a.Tkv, (int)sizeof(T));
  // (A launch counts its threads in 32 bits, 512 a workgroup at most; the kernels count rows in 31.)
  KESSIE_REQUIRE(p.grid * a.Hkv < 1 << 23 && a.Tq <= 1 << 26 && (int64_t)a.Tq * a.G <= 1 << 30, KESSIE_ERR_UNSUPPORTED,
                 "cross attention: %d sequences, %d queries of %d heads exceed one launch", a.B, a.Tq, a.Hq);
  const Layout l = layout(p, a.B, a.Hkv, a.D);
  KESSIE_REQUIRE(ws_bytes >= l.bytes && (l.bytes == 0 || (ws && aligned16(ws))), KESSIE_ERR_WORKSPACE,
                 "cross attention: workspace of %zu bytes, %zu needed", ws_bytes, l.bytes);
  if (l.bytes) {
    a.shares = p.shares, a.min_steps = p.min_steps, a.part_rows = p.part_rows;
    a.plan = static_cast<int64_t*>(ws);
    a.ws_o = reinterpret_cast<float*>(static_cast<char*>(ws) + l.plan);
    a.ws_m = a.ws_o + l.rows * a.D;
    a.ws_l = a.ws_m + l.rows;
  }
  return a.D == 64 ? launch_shared<T, 64>(a, p, s) : launch_shared<T, 128>(a, p, s);
}

}  // namespace
}  // namespace cross
}  // namespace kessie

using namespace kessie;
using namespace kessie::cross;

extern "C" size_t kessie_cross_attention_workspace_bytes(int batch, int max_query_len, int num_q_tokens, int num_kv_tokens,
                                                         int num_q_heads, int num_kv_heads, int head_dim, int max_kv_len,
                                                         int dtype) {
  if (batch <= 0 || max_query_len <= 0 || num_q_tokens <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads || max_kv_len < 0 ||
      num_kv_tokens < 0 || (head_dim != 64 && head_dim != 128) || dtype_size(dtype) <= 0)
    return 0;
  const Plan p = make_plan(batch, max_query_len, num_q_tokens, num_q_heads, num_kv_heads, head_dim, max_kv_len, num_kv_tokens,
                           dtype_size(dtype));
  return layout(p, batch, num_kv_heads, head_dim).bytes;
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
  KESSIE_REQUIRE(fabsf(sm_scale) * kLog2e <= 3.402823466e38f, KESSIE_ERR_INVALID, "cross attention: sm_scale %g", (double)sm_scale);
  KESSIE_REQUIRE(max_kv_len <= 1 << 30, KESSIE_ERR_UNSUPPORTED, "cross attention: %d states", max_kv_len);
  if (batch == 0 || max_query_len == 0 || num_q_tokens == 0) return KESSIE_OK;
  KESSIE_REQUIRE(q && out && query_start_loc && kv_start && kv_lens && (num_kv_tokens == 0 || (k && v)), KESSIE_ERR_INVALID,
                 "cross attention: null pointer");
  KESSIE_REQUIRE(rows_apart(num_q_tokens, out_tok_stride, num_q_heads, out_head_stride, head_dim), KESSIE_ERR_INVALID,
                 "cross attention: rows of out overlap (strides %lld, %lld)", (long long)out_tok_stride, (long long)out_head_stride);
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
