// The tables of one engine step, built on the device from the requests'
// lengths: query_start_loc, seq_lens, the new pages of the block table, the
// slot and the position of every token row.
//
// Request b holds c = computed[b] tokens and brings n = new[b]; with pages of
// P tokens it needs ceil((c+n)/P) - ceil(c/P) pages more.  Page i of a row is
// the table's own entry below ceil(c/P) and free[before[b] + i - ceil(c/P)]
// from there on, where before[b] is the exclusive prefix sum of the needs.
// Both prefix sums (tokens and pages) are over all requests, and every value
// written follows from them, so one launch does it all: each workgroup scans
// the lengths itself (8 bytes a request out of L2), 1,024 requests at a time,
// until it has passed its own token rows, and looks its rows up by bisection
// in the starts it left in LDS.  No workgroup waits for another; nothing is
// read that another one writes (table entries below ceil(c/P) are read, those
// from there on written).
//
// A new page holds at least one new token, and its first one is at offset 0:
// that token's thread writes the page's table entry, flag and position.  A
// row's pages are so spread over as many threads as it has pages, however long
// the row (a prompt of a million tokens brings 65,536).
//
// Bound: latency -- lengths -> scan -> page id -> slot, two dependent loads: 5.0
// us for 24 requests of one token, 6.0 for 1,024 requests and 24,576 token rows.
#include "common.h"

namespace kessie {
namespace step {
namespace {

constexpr int kThreads = 256;   // token rows of a workgroup, one a thread
constexpr int kPer = 4;         // requests a thread takes per pass of the scan
constexpr int kChunk = kThreads * kPer;
constexpr int kWaves = kThreads / 64;

struct Args {
  int32_t* table;
  int64_t table_stride;
  int width;
  const int32_t* computed;
  const int32_t* fresh;
  const int32_t* delta;       // nullptr: zeros
  const int32_t* free_pages;  // nullptr: none
  const int32_t* free_count;
  int max_free;
  int B, P, T;
  int32_t* start_loc;
  int32_t* seq_lens;
  int64_t* slots;
  int32_t* positions;
  int32_t* taken;
  int8_t* valid;      // nullptr: not wanted
  int32_t* page_pos;  // nullptr: not wanted
  int num_pages;      // entries of valid and page_pos
};

// Sums over the requests so far: 64 bits, so that no lengths overflow them.
struct Sums {
  int64_t tokens, pages;
};
__device__ __forceinline__ Sums operator+(Sums a, Sums b) { return {a.tokens + b.tokens, a.pages + b.pages}; }
__device__ __forceinline__ Sums shfl_up(Sums s, int by) { return {__shfl_up(s.tokens, by, 64), __shfl_up(s.pages, by, 64)}; }

__device__ __forceinline__ int32_t saturate(int64_t x) {
  return x > 0x7fffffff ? 0x7fffffff : x < -0x7fffffff ? -0x7fffffff : (int32_t)x;
}

__global__ __launch_bounds__(kThreads) void step_tables_kernel(Args a) {
  __shared__ int32_t s_start[kChunk];   // first token row of the request (its end's, where it has none)
  __shared__ int32_t s_have[kChunk];    // tokens in the cache
  __shared__ int32_t s_before[kChunk];  // free pages that earlier requests take; -1: not granted
  __shared__ Sums s_wave[kWaves];
  __shared__ int32_t s_max[kWaves];

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int t = blockIdx.x * kThreads + tid;  // this thread's token row (T is below 2^31 - 256: the host's check)
  const int tile_end = min(a.T, (int)(blockIdx.x + 1) * kThreads);
  const int64_t free_n = a.free_pages ? min(max(a.free_count[0], 0), a.max_free) : 0;

  // The pass that holds this workgroup's requests (a workgroup past the last request has none).
  const int last_rows = (int64_t)blockIdx.x * kChunk < a.B ? (int)blockIdx.x : 0;

  Sums carry{0, 0};
  int my_row = -1, my_pos = 0, my_before = -1, my_have = 0;
  int64_t taken = 0;
  for (int b0 = 0; b0 < a.B; b0 += kChunk) {
    // One pass: kPer requests a thread.
    int have[kPer], add[kPer], need[kPer];
    Sums mine{0, 0};
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int b = b0 + tid * kPer + i;
      have[i] = b < a.B ? max(a.computed[b], 0) : 0;
      add[i] = b < a.B ? max(a.fresh[b], 0) : 0;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const uint32_t held = ((uint32_t)have[i] + (uint32_t)a.P - 1u) / (uint32_t)a.P;
      // (have + add is below 2^32, so its page count is exact in 32 bits.)
      const uint32_t sum = (uint32_t)have[i] + (uint32_t)add[i];
      const uint32_t all = sum / (uint32_t)a.P + (sum % (uint32_t)a.P != 0);
      // -1: more than a table row or a position holds.
      need[i] = all <= (uint32_t)a.width && sum <= 0x7fffffffu ? (int)(all - held) : -1;
      mine.tokens += add[i];
      mine.pages += max(need[i], 0);
    }
    Sums inc = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const Sums up = shfl_up(inc, o);
      if (lane >= o) inc = inc + up;
    }
    if (lane == 63) s_wave[wave] = inc;
    __syncthreads();
    Sums at = carry, end = carry;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at = at + s_wave[w];
      end = end + s_wave[w];
    }
    at.tokens += inc.tokens - mine.tokens;
    at.pages += inc.pages - mine.pages;
    const bool own_rows = b0 / kChunk == (int)blockIdx.x;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int s = tid * kPer + i, b = b0 + s;
      const int64_t row_end = at.tokens + add[i];
      // Granted: the row fits its table, its tokens the rows, its pages the free list.
      const bool ok = need[i] >= 0 && row_end <= a.T && (need[i] == 0 || at.pages + need[i] <= free_n);
      s_start[s] = saturate(at.tokens);
      s_have[s] = have[i];
      s_before[s] = ok ? (int32_t)min(at.pages, (int64_t)0x7fffffff) : -1;
      if (ok && need[i] > 0) taken = at.pages + need[i];
      if (own_rows && b < a.B) {
        a.start_loc[b + 1] = saturate(row_end);
        a.seq_lens[b] = ok ? saturate((int64_t)have[i] + add[i]) : have[i];
      }
      at.tokens = row_end;
      at.pages += max(need[i], 0);
    }
    __syncthreads();
    // This thread's token row, if it lies among these requests: the last one that starts at or before it.
    if (t < a.T && t >= carry.tokens && t < end.tokens) {
      int lo = 0, hi = min(kChunk, a.B - b0) - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (s_start[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      my_row = b0 + lo;
      my_have = s_have[lo];
      my_pos = saturate((int64_t)my_have + (t - s_start[lo]));
      my_before = s_before[lo];
    }
    carry = end;
    // Done: past this workgroup's token rows and requests.  (The first one goes on to the end, for `taken`.)
    if (blockIdx.x != 0 && b0 / kChunk >= last_rows && carry.tokens >= tile_end) break;
    __syncthreads();  // (before the next pass writes the arrays that this one's rows were looked up in)
  }

  if (t < a.T) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (my_row >= 0) {
      pos = saturate((int64_t)my_pos + (a.delta ? a.delta[my_row] : 0));
      if (my_before >= 0) {
        const int i = my_pos / a.P, off = my_pos - i * a.P;
        const int held = (int)(((uint32_t)my_have + (uint32_t)a.P - 1u) / (uint32_t)a.P);
        int32_t* entry = a.table + (int64_t)my_row * a.table_stride + i;
        int32_t page;
        if (i < held) {
          page = *entry;
        } else {
          page = a.free_pages[(int64_t)my_before + (i - held)];
          if (off == 0) {
            *entry = page;
            if (page >= 0 && page < a.num_pages) {
              if (a.valid) a.valid[page] = 1;
              if (a.page_pos) a.page_pos[page] = pos;
            }
          }
        }
        slot = page >= 0 ? (int64_t)page * a.P + off : -1;
      }
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
  if (blockIdx.x == 0) {
    // The granted needs are a prefix of all needs: the largest sum is their total.
    int32_t m = saturate(taken);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
    __syncthreads();
    if (lane == 0) s_max[wave] = m;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWaves; ++w) m = max(m, s_max[w]);
      a.taken[0] = m;
      a.start_loc[0] = 0;
    }
  }
}

}  // namespace
}  // namespace step
}  // namespace kessie

using namespace kessie;
using namespace kessie::step;

extern "C" int kessie_step_tables(int32_t* block_table, int64_t table_stride, int table_width,
                                  const int32_t* computed_lens, const int32_t* new_lens,
                                  const int32_t* position_delta, const int32_t* free_pages,
                                  const int32_t* free_count, int max_free, int batch, int page_size,
                                  int num_token_rows, int32_t* query_start_loc, int32_t* seq_lens,
                                  int64_t* slot_mapping, int32_t* positions, int32_t* taken, int8_t* page_valid,
                                  int32_t* page_positions, int num_pages, void* stream) {
  clear_error();
  KESSIE_REQUIRE(batch >= 0 && page_size > 0 && table_width >= 0 && max_free >= 0 && num_pages >= 0, KESSIE_ERR_INVALID,
                 "step tables: bad sizes B=%d P=%d W=%d free=%d pages=%d", batch, page_size, table_width, max_free,
                 num_pages);
  KESSIE_REQUIRE(num_token_rows >= 0 && num_token_rows < 0x7fffff00, KESSIE_ERR_INVALID, "step tables: %d token rows",
                 num_token_rows);
  KESSIE_REQUIRE(batch <= 1 << 30, KESSIE_ERR_UNSUPPORTED, "step tables: %d requests", batch);
  KESSIE_REQUIRE(query_start_loc && taken, KESSIE_ERR_INVALID, "step tables: null pointer");
  KESSIE_REQUIRE(batch == 0 || (computed_lens && new_lens && seq_lens && (block_table || table_width == 0)),
                 KESSIE_ERR_INVALID, "step tables: null pointer");
  KESSIE_REQUIRE(num_token_rows == 0 || (slot_mapping && positions), KESSIE_ERR_INVALID, "step tables: null pointer");
  KESSIE_REQUIRE(max_free == 0 || (free_pages && free_count), KESSIE_ERR_INVALID,
                 "step tables: a free list needs its pages and its count");
  KESSIE_REQUIRE(table_stride >= table_width, KESSIE_ERR_INVALID, "step tables: table rows overlap (stride %lld, width %d)",
                 (long long)table_stride, table_width);
  // Every workgroup reads the lengths while others write the tables: none of these may lie over another.
  struct Range {
    const void* at;
    int64_t bytes;
  };
  const int64_t B = batch, T = num_token_rows, W = batch ? (B - 1) * table_stride + table_width : 0;
  const Range in[] = {{computed_lens, 4 * B}, {new_lens, 4 * B}, {position_delta, 4 * B}, {free_pages, 4 * (int64_t)max_free},
                      {max_free ? free_count : nullptr, 4}};
  const Range out[] = {{query_start_loc, 4 * B + 4}, {seq_lens, 4 * B}, {slot_mapping, 8 * T}, {positions, 4 * T}, {taken, 4},
                       {block_table, 4 * W}, {page_valid, num_pages}, {page_positions, 4 * (int64_t)num_pages}};
  constexpr int kOut = sizeof(out) / sizeof(out[0]);
  auto over = [](const Range& x, const Range& y) {
    const char *p = static_cast<const char*>(x.at), *q = static_cast<const char*>(y.at);
    return p && q && x.bytes > 0 && y.bytes > 0 && p < q + y.bytes && q < p + x.bytes;
  };
  for (int i = 0; i < kOut; ++i) {
    for (const Range& x : in)
      KESSIE_REQUIRE(!over(x, out[i]), KESSIE_ERR_INVALID, "step tables: an input lies over an output");
    for (int j = 0; j < i; ++j)
      KESSIE_REQUIRE(!over(out[j], out[i]), KESSIE_ERR_INVALID, "step tables: two outputs lie over each other");
  }
  Args a{block_table, table_stride, table_width, computed_lens, new_lens, position_delta,
         max_free ? free_pages : nullptr, free_count, max_free, batch, page_size, num_token_rows, query_start_loc,
         seq_lens, slot_mapping, positions, taken, page_valid, page_positions, num_pages};
  const int rows = div_up(num_token_rows, kThreads), reqs = div_up(batch, kChunk);
  const int grid = rows > reqs ? rows : reqs;
  hipLaunchKernelGGL(step_tables_kernel, dim3(grid > 0 ? grid : 1), dim3(kThreads), 0, as_stream(stream), a);
  return check_launch("step tables");
}
