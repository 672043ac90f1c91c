// What the attention kernels share: their parameters, the numbering of their
// units of work, and which keys a query sees.
#pragma once

#include <math.h>

#include "kv_cache.cuh"

namespace mcpu {
namespace attn {

static __device__ int g_attn_error = 0;  // one per source file; attn_read_error reads them all

constexpr unsigned kFull = 0xFFFFFFFFu;

enum Kind { kSame = 0, kE4M3 = 1, kInt8 = 2 };

struct Params {
  const void* q;
  long long q_tok, q_head;
  void* out;
  long long o_tok, o_head;
  float* lse;  // [tokens, heads] or NULL
  mcpuKvCache c;
  const int* table;
  long long table_stride;
  int table_width, block_log2;  // block_log2 < 0: not a power of two
  const int* seq_lens;
  const int* cu;
  const long long* mask;  // [tokens, words] or NULL
  long long mask_stride;
  int mask_words;
  int batch, tokens, kv_heads, group;
  int most;  // new tokens of a request
  float scale_log2;
  int rows_log2, keys_log2;  // rows and keys of a unit
  int item_cost;             // what beginning and ending a row tile costs, in key tiles
  int bf16;                  // type of query and out: bf16, else fp16
  float* part_o;             // [grid][2][rows][D]
  float* part_ml;            // [grid][2][rows][2]
  int4* joins;               // [grid]: of the row tile that begins in a block and goes on behind it: its parts (0: there
                             // is none), its request's first token and new tokens, its item
};

// ---------------------------------------------------------------- schedule
struct Request {
  int first, n, len;  // first token, new tokens, length; len = 0: nothing to do
};

__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.first = p.cu[b];
  const int end = p.cu[b + 1];
  r.n = end - r.first;
  r.len = p.seq_lens[b];
  const bool fits = r.first >= 0 && r.n >= 0 && end <= p.tokens;
  const long long room = static_cast<long long>(p.table_width) * p.c.block_size;
  const bool words = p.mask == nullptr || r.n <= 64 * p.mask_words;
  if (!fits || r.len < r.n || r.len > room || !words || r.n > p.most) {
    atomicOr(&g_attn_error, 1);
    if (!fits) r.first = 0, r.n = 0;
    r.len = 0;
  }
  if (r.n == 0) r.len = 0;
  return r;
}

__device__ __forceinline__ int key_tiles(const Params& p, const Request& r) {
  return (r.len + (1 << p.keys_log2) - 1) >> p.keys_log2;
}
__device__ __forceinline__ int row_tiles(const Params& p, const Request& r) {
  return (r.n * p.group + (1 << p.rows_log2) - 1) >> p.rows_log2;
}
// A row tile counts as its key tiles and, in front of them, item_cost more: a
// block that gets many short row tiles does not end after the others.
__device__ __forceinline__ int units(const Params& p, const Request& r) {
  return r.len == 0 ? 0 : p.kv_heads * row_tiles(p, r) * (key_tiles(p, r) + p.item_cost);
}

// Block-wide: total units, then the request that holds `unit` (a function of
// the total) and the units before it.  red: NT / 32 + 2 ints.
template <int NT, typename F>
__device__ __forceinline__ void locate(const Params& p, F&& unit_of, int* red, int& total, int& unit, int& b,
                                       int& before) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int own = tid < p.batch ? units(p, request(p, tid)) : 0;
  int mine = own;
  for (int i = tid + NT; i < p.batch; i += NT) mine += units(p, request(p, i));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(kFull, mine, o);
  if (lane == 0) red[warp] = mine;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) total += red[w];
  unit = unit_of(total);
  int* found = red + NT / 32;
  if (tid == 0) found[0] = p.batch, found[1] = total;
  __syncthreads();
  int base = 0;
  for (int i0 = 0; i0 < p.batch; i0 += NT) {
    const int i = i0 + tid;
    const int u = i0 == 0 ? own : i < p.batch ? units(p, request(p, i)) : 0;
    int incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) red[warp] = incl;
    __syncthreads();
    int off = base;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
      off += w < warp ? red[w] : 0;
      base += red[w];
    }
    const int from = off + incl - u;
    if (unit >= from && unit < from + u) found[0] = i, found[1] = from;
    __syncthreads();
    if (base > unit) break;
  }
  b = found[0];
  before = found[1];
}

// Units a block takes: an equal share of all, down to one (two and four at least cost a single request 0.6 and 1.9 us).
__device__ __forceinline__ int share_of(int total, int grid) { return max((total + grid - 1) / grid, 1); }

// A block's run of units as pieces: key tiles tile0 .. tile0 + nt - 1 of one
// row tile (item: key / value head and row tile of request b).
struct Pieces {
  int b, item, items, tiles;
  Request r;
  int tile0, nt;
  int begin;  // unit the item begins with
  int v, left;  // where the next piece begins in the item, units left

  __device__ __forceinline__ void open(const Params& p) {
    r = request(p, b);
    tiles = key_tiles(p, r);
    items = r.len == 0 ? 0 : p.kv_heads * row_tiles(p, r);
  }
  __device__ __forceinline__ bool start(const Params& p, int b0, int before, int unit, int count) {
    b = b0;
    open(p);
    const int offset = unit - before, span = tiles + p.item_cost;
    item = offset / span;
    v = offset - item * span;
    begin = unit - v;
    left = count;
    return take(p);
  }
  // The next piece with keys; false: no more.
  __device__ __forceinline__ bool next(const Params& p) { return take(p); }

 private:
  __device__ __forceinline__ bool take(const Params& p) {
    while (left > 0) {
      const int span = tiles + p.item_cost;
      if (v == span) {
        v = 0;
        begin += span;
        if (++item == items) {
          item = 0;
          do ++b, open(p);  // units are left, so a request with some follows
          while (items == 0);
        }
        continue;
      }
      const int count = min(span - v, left);
      tile0 = max(v - p.item_cost, 0);
      nt = max(v + count - p.item_cost, 0) - tile0;
      v += count;
      left -= count;
      if (nt > 0) return true;
    }
    return false;
  }
};

// Parts an item is in: from the block of its first key tile to that of its last.
__device__ __forceinline__ int parts_of(const Params& p, const Pieces& pc, int share) {
  const int first = pc.begin + p.item_cost;
  return (first + pc.tiles - 1) / share - first / share + 1;
}

// Requests without work (no keys, or refused) still have outputs: a warp each.
template <int NT>
__device__ __forceinline__ void clear_idle_requests(const Params& p, int D) {
  const int lane = threadIdx.x & 31;
  for (int b = blockIdx.x * (NT / 32) + (threadIdx.x >> 5); b < p.batch; b += gridDim.x * (NT / 32)) {
    const Request r = request(p, b);
    if (r.len != 0 || r.n == 0) continue;
    const int heads = p.kv_heads * p.group;
    for (int i = 0; i < r.n * heads; ++i) {
      const int t = r.first + i / heads, h = i % heads;
      uint16_t* o = static_cast<uint16_t*>(p.out) + t * p.o_tok + h * p.o_head;  // zero in either type
      for (int d = lane; d < D; d += 32) o[d] = 0;
      if (p.lse && lane == 0) p.lse[static_cast<long long>(t) * heads + h] = -INFINITY;
    }
  }
}

// The keys key0 .. key0 + 31 that query i (token t of request r) sees, a bit
// each: the length, and the mask words or the order of the new tokens.
__device__ __forceinline__ uint32_t seen32(const Params& p, const Request& r, int t, int i, int key0) {
  const int left = r.len - key0;
  uint32_t seen = left >= 32 ? kFull : left <= 0 ? 0u : (1u << left) - 1;
  const int d0 = key0 - (r.len - r.n);
  if (d0 + 32 <= 0) return seen;
  if (p.mask == nullptr) {
    const int n = i - d0 + 1;
    return seen & (n >= 32 ? kFull : n <= 0 ? 0u : (1u << n) - 1);
  }
  const long long* words = p.mask + t * p.mask_stride;
  if (d0 < 0) return seen & (static_cast<uint32_t>(words[0]) << -d0 | ((1u << -d0) - 1));
  const int w = d0 >> 6, off = d0 & 63;
  if (w >= p.mask_words) return 0;  // behind the last new token
  uint32_t bits = static_cast<uint32_t>(static_cast<unsigned long long>(words[w]) >> off);
  if (off > 32 && w + 1 < p.mask_words) bits |= static_cast<uint32_t>(words[w + 1] << (64 - off));
  return seen & bits;
}

// Whether some of a request's rows may not see some of its new tokens: without
// a mask a single one sees itself, with one it need not.
__device__ __forceinline__ bool some_unseen(const Params& p, const Request& r) { return r.n > 1 || p.mask != nullptr; }

// ---------------------------------------------------------------- arithmetic
__device__ __forceinline__ float exp2_fast(float x) {  // ex2.approx: 2^-22 relative, 0 for -inf
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Probabilities that are multiplied as fp16 are held times 2^15 (times 2^7 where
// the maximum they refer to may be 2^8 too low), which is taken off the sums at
// the end: those down to 2^-29 (2^-21) of the largest keep fp16's precision,
// and what lies below is off by at most 2^-40 (2^-32) of it.  Held as they are,
// those below 2^-25 were gone from the outputs though not from the sum that
// these are divided by.
//
// Products of probabilities and value scales, w_j = p_j s_j, are multiplied as
// fp16, relative to a reference of each row: w_j 2^lift.  The lift brings the
// largest product so far of the keys the row sees to 2^7 .. 2^8; it falls, with
// the sums scaled down, when a product would pass 2^15, and rises with the
// row's maximum, whose growth makes the earlier products smaller.  So only what
// lies below 2^-21 of the largest product is held with fewer bits than fp16
// has, at most 2^-32 of it off, however far apart the scales are and whatever
// those of unseen keys are.  (From 2^10 the lift falls more often: 145 us
// instead of 137 for the small trees of tree_attention_tc.cu.)  A reference
// taken from the scales alone, the largest of a step, lost whole outputs beside
// one key of a large scale and no probability.  Lifts, and the maxima they go
// with, are whole numbers, so that sums are scaled by powers of two.
constexpr float kLift = 100.0f;    // the highest; where no product above 0 has been seen
constexpr float kRoom = 32768.0f;  // of 65504
__device__ __forceinline__ float exp2_whole(float e) {  // -126 .. 127
  return __int_as_float((static_cast<int>(e) + 127) << 23);
}
__device__ __forceinline__ float lift_for(float w) {
  return fminf(kLift, 7.0f - static_cast<float>(static_cast<int>(__float_as_uint(w) >> 23) - 127));
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (BF16) {
    return pack_bf16x2(lo, hi);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
// Two 8-bit values (bytes B0, B1 of w) as a pair of fp16.
template <int KIND, int B0, int B1>
__device__ __forceinline__ uint32_t widen(uint32_t w) {  // int8: w already biased by 128
  uint32_t h2;
  if constexpr (KIND == kE4M3) {
    const uint32_t two = (B0 == 0 && B1 == 1) ? w : (B0 == 2 && B1 == 3) ? w >> 16 : __byte_perm(w, 0, B0 | B1 << 4);
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(two)));
  } else {
    // 0x6400 + u is 1024 + u in fp16; u = value + 128
    const uint32_t u = __byte_perm(w, 0x64646464u, B0 | 4 << 4 | B1 << 8 | 4 << 12);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    h2 = *reinterpret_cast<const uint32_t*>(&v);
  }
  return h2;
}
// A fragment's finite values (others 0), and ones where a value adds +inf (or
// NaN) and where one adds -inf (or NaN).
template <bool BF16>
__device__ __forceinline__ void split_finite(uint32_t b, uint32_t& clean, uint32_t& plus, uint32_t& minus) {
  constexpr uint32_t kExp = BF16 ? 0x7F807F80u : 0x7C007C00u, kOne = BF16 ? 0x3F803F80u : 0x3C003C00u;
  constexpr uint32_t kFrac = BF16 ? 0x007F007Fu : 0x03FF03FFu;
  const uint32_t wild = __vcmpeq2(b & kExp, kExp);
  const uint32_t nan = wild & ~__vcmpeq2(b & kFrac, 0u);
  const uint32_t neg = __vcmpeq2(b & 0x80008000u, 0x80008000u);
  clean = b & ~wild;
  plus = wild & (~neg | nan) & kOne;
  minus = wild & (neg | nan) & kOne;
}

// cp.async of 16 or 4 bytes, zeros where not valid.
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// The kernel on the tensor-memory path (tree_attention_tc.cu): many rows a key.
// Sets the tile sizes and the grid; the caller launches the joining kernel.
orError_t launch_tc(Params& p, int D, long long rows, cudaStream_t st, int sms, int* grid);
orError_t tc_read_error(int* flag, bool reset);

}  // namespace attn
}  // namespace mcpu
