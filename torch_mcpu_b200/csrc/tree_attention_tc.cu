// Tree attention where many rows share a key: both products on the
// tensor-memory path (tcgen05), 128 rows and 128 keys at a time.
//
// Bound by the tensor pipe and the exponentials: a tile of 128 x 128 scores
// costs 512 cycles of products at D = 128 and 1024 cycles of exponentials (16
// per cycle and SM), which is why two independent streams of tiles share an
// SM: while one stream's scores are turned into probabilities, the other's
// products run.  With up to 128 rows per key / value head the streams are the
// even and the odd key tiles of the same rows (joined at the end of a run);
// with more, two row tiles against every key tile, which also halves the
// traffic of keys and values.
//
// One block per SM, 13 warps:
//   warps 0-3, 4-7  softmax of stream 0 and 1: a thread owns a row (its
//                   tensor-memory lane), reads the scores, keeps the running
//                   maximum and sum, writes the probabilities over the scores
//                   as 16-bit values, the left operand of the second product
//   warps 8-11      loaders: pages to shared memory by 16-byte asynchronous
//                   copies into the 128-byte-swizzled layout; 8-bit caches go
//                   through a raw ring and are widened to fp16
//   warp 12         one thread issues the products
// Tensor memory: scores of the two streams (2 x 128 columns), outputs (2 x D).
//
// The output is scaled down only when a row's maximum grew by more than 2^8
// since the reference was set; until then probabilities up to 256 are summed,
// which fp16 and bf16 hold and fp32 sums take without loss.
#include <algorithm>
#include <type_traits>

#include "sm100.cuh"
#include "tree_attention.cuh"

namespace mcpu {
namespace attn {
namespace tc {

using namespace sm100;

constexpr int kSoftWarps = 8, kLoadWarps = 4;
constexpr int kWarpsTc = kSoftWarps + kLoadWarps + 1;
constexpr int kThreadsTc = 32 * kWarpsTc;
constexpr int kTile = 128;        // rows and keys of a tile
constexpr int kTmemCols = 512;
constexpr int kScaleRing = 8;     // key tiles whose scales are kept
constexpr float kGrow = 8.0f;     // log2 of the growth of a maximum that is tolerated

template <int KIND_, bool BF16_, int D_, bool TOKEN_>
struct Cfg {
  static constexpr int KIND = KIND_, D = D_;
  static constexpr bool BF16 = BF16_;    // type of the products; 8-bit caches: fp16
  static constexpr bool TOKEN = TOKEN_;  // a scale for every token and head
  static constexpr bool kSmall = KIND != kSame;
  static constexpr int kSlots = kSmall ? 3 : 4;  // key or value tiles in shared memory
  static constexpr int kSlot = kTile * D * 2;
  static constexpr int kBlock = kTile * 128;     // 64 dimensions of a tile
  static constexpr int kRaw = kSmall ? kTile * D : 0;
  static constexpr int kWild = KIND == kInt8 ? 0 : kTile * 32;  // two bits per value, in values that are not finite
  // shared memory, from a 1024-byte boundary
  static constexpr int kOffWild = kSlots * kSlot;
  static constexpr int kOffRowWild = kOffWild + kSlots * kWild;
  static constexpr int kOffScale = kOffRowWild + (KIND == kInt8 ? 0 : 2 * kTile * 32);
  static constexpr int kOffMl = kOffScale + (TOKEN ? kScaleRing * (2 * kTile * 4 + 16) : 0);
  static constexpr int kOffBars = kOffMl + 2 * kTile * 8;
  static constexpr int kOffQ = (kOffBars + 512 + 1023) / 1024 * 1024;
  static constexpr int raw_depth(int nq) { return !kSmall ? 0 : nq == 1 ? 4 : 2; }
  static constexpr int smem(int nq) { return kOffQ + nq * kSlot + raw_depth(nq) * kRaw + 1024; }
};

struct Bars {
  uint64_t kv_full[4], kv_empty[4], q_full, s_full[2], p_full[2], o_done[2], both, drain;
  uint32_t tmem;
  int abort;
  int wild[4][kLoadWarps];
};
static_assert(sizeof(Bars) <= 512, "barriers overflow their place");

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
      "r"(accumulate ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
      "r"(accumulate ? 1 : 0)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Bounded wait: a barrier that has not completed after two seconds is a fault
// of this kernel; every role then leaves and the error flag is set.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort) {
  if (mbar_try_wait(bar, parity)) return true;
  unsigned long long begin = 0, now;
  for (uint32_t i = 0;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 63u) != 63u) continue;
    if (*abort) return false;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (begin == 0) begin = now;
    if (now - begin > 2000000000ull || i > (1u << 28)) {
      *abort = 1;
      return false;
    }
  }
}

// Values stored as rows of 128 bytes (64 dimensions) with the 128-byte swizzle,
// one row per key, as the right operand keys x dimensions with dimensions
// contiguous: 8-key groups 1024 bytes apart (stride byte offset), the next 64
// dimensions 128 keys further (leading byte offset).
__device__ __forceinline__ uint64_t desc_values(uint32_t addr) {
  uint64_t d = smem_desc_k128(addr) & ~(0x3FFFull << 16);
  return d | static_cast<uint64_t>((kTile * 128) >> 4) << 16;
}
// Instruction descriptor: fp32 sums, 16-bit operands, 128 x N, left operand
// (and right, unless values) with the summed index contiguous.
__device__ __forceinline__ constexpr uint32_t idesc(bool bf16, int N, bool values) {
  return (1u << 4) | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (values ? 1u << 16 : 0u) |
         static_cast<uint32_t>(N >> 3) << 17 | static_cast<uint32_t>(kTile >> 4) << 24;
}

// Byte offset of 16-byte chunk c (8 dimensions) of a row of a tile.
__device__ __forceinline__ uint32_t place16(int row, int c) {
  return (c >> 3) * (kTile * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4);
}

// ---------------------------------------------------------------- runs of key tiles
// A block's units as pieces: a run of key tiles of one item.
struct Pieces {
  Walk w;
  int left;   // units behind the current piece
  int tile0, nt;
  __device__ __forceinline__ void start(const Params& p, int b0, int offset, int count) {
    w.seek(p, b0, offset);
    left = count;
    take();
  }
  __device__ __forceinline__ void take() {
    tile0 = w.tile;
    nt = min(w.tiles - w.tile, left);
    left -= nt;
  }
  __device__ __forceinline__ bool next(const Params& p) {  // false: no more
    if (left <= 0) return false;
    w.skip(p, nt);
    take();
    return true;
  }
};

// The order in which a piece's key and value tiles are loaded, which is the
// order the products take them: lead key tiles, then a value tile and the next
// key tile in turn.
__device__ __forceinline__ void order(int s, int nt, int lead, bool& is_v, int& tile) {
  const int first = min(lead, nt), pairs = nt - first;
  const int t = s - first;
  if (t < 0) {
    is_v = false, tile = s;
  } else if (t < 2 * pairs) {
    is_v = (t & 1) == 0, tile = (t >> 1) + (is_v ? 0 : lead);
  } else {
    is_v = true, tile = t - pairs;
  }
}

// ---------------------------------------------------------------- loaders
template <typename C>
struct Loader {
  const Params& p;
  Bars* bars;
  uint32_t base;   // shared memory, 1024-byte aligned
  uint8_t* mem;
  uint32_t raw;
  int nq, depth, lw, lane;
  volatile int* abort;

  // where the lane's row (32 lw + lane) of a tile lies
  __device__ __forceinline__ bool row_at(const Pieces& pc, int tile, long long& block, int& slot) const {
    const int key = (pc.tile0 + tile) * kTile + 32 * lw + lane;
    block = 0, slot = 0;
    if (key >= pc.w.r.len) return false;
    const int page = p.block_log2 >= 0 ? key >> p.block_log2 : key / p.c.block_size;
    slot = key - page * p.c.block_size;
    block = kv::checked_block(p.table[pc.w.b * p.table_stride + page], p.c.num_blocks, &g_attn_error);
    return true;
  }

  // Starts the copies of one tile; count = tiles of this block before it, t = key tiles before its own.
  __device__ __forceinline__ bool issue(const Pieces& pc, bool is_v, int tile, uint32_t count, uint32_t t) const {
    long long block;
    int slot;
    const bool valid = row_at(pc, tile, block, slot);
    const unsigned rows_valid = __ballot_sync(kFull, valid);
    const int h = pc.w.item / row_tiles(p, pc.w.r);
    const int64_t* st = is_v ? p.c.value_stride : p.c.key_stride;
    constexpr int kSize = C::kSmall ? 1 : 2;
    const unsigned long long off = static_cast<unsigned long long>((block * st[0] + slot * st[1]) * kSize);
    const uint8_t* from = static_cast<const uint8_t*>(is_v ? p.c.value : p.c.key) + h * st[2] * kSize;
    if constexpr (C::TOKEN) {
      const int64_t* ss = is_v ? p.c.v_scale_stride : p.c.k_scale_stride;
      const float* src = (is_v ? p.c.v_scale : p.c.k_scale) + block * ss[0] + slot * ss[1] + h * ss[2];
      cp_async4(base + C::kOffScale + (((t & (kScaleRing - 1)) * 2 + is_v) * kTile + 32 * lw + lane) * 4, src, valid);
    }
    uint32_t dst;
    if constexpr (C::kSmall) {
      dst = raw + (count % depth) * C::kRaw;
    } else {
      const uint32_t s = count % C::kSlots;
      if (!wait(&bars->kv_empty[s], ((count / C::kSlots) & 1) ^ 1, abort)) return false;
      dst = base + s * C::kSlot;
    }
    constexpr int kChunks = C::D * kSize / 16, kRows = 32 / kChunks;
    const int c = lane % kChunks;
#pragma unroll
    for (int i = 0; i < 32 / kRows; ++i) {
      const int row = i * kRows + lane / kChunks;
      const unsigned long long o = __shfl_sync(kFull, off, row);
      const uint32_t at = C::kSmall ? ((32 * lw + row) * kChunks + c) * 16 : place16(32 * lw + row, c);
      cp_async16(dst + at, from + o + c * 16, (rows_valid >> row) & 1);
    }
    return true;
  }

  // The copies have landed: widen, look for values that are not finite, hand the tile over.
  __device__ __forceinline__ bool finish(const Pieces& pc, bool is_v, int tile, uint32_t count, uint32_t t) const {
    const uint32_t s = count % C::kSlots;
    uint8_t* slot = mem + s * C::kSlot;
    constexpr int kSize = C::kSmall ? 1 : 2;
    constexpr int kChunks = C::D * kSize / 16, kRows = 32 / kChunks;
    const int c = lane % kChunks;
    // new tokens in this tile that some of the request's rows may not see
    const bool tail = C::KIND != kInt8 && is_v && pc.w.r.n > 1 &&
                      (pc.tile0 + tile + 1) * kTile > pc.w.r.len - pc.w.r.n;
    bool wild = false;
    uint8_t* bits = mem + C::kOffWild + s * C::kWild;
    if constexpr (C::kSmall) {
      if (!wait(&bars->kv_empty[s], ((count / C::kSlots) & 1) ^ 1, abort)) return false;
      const uint8_t* from = mem + (raw - base) + (count % depth) * C::kRaw;
#pragma unroll
      for (int i = 0; i < 32 / kRows; ++i) {
        const int row = 32 * lw + i * kRows + lane / kChunks;
        const uint4 u = *reinterpret_cast<const uint4*>(from + (row * kChunks + c) * 16);
        uint32_t w[4] = {u.x, u.y, u.z, u.w}, o[8];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (C::KIND == kInt8) w[x] ^= 0x80808080u;
          o[2 * x] = widen<C::KIND, 0, 1>(w[x]);
          o[2 * x + 1] = widen<C::KIND, 2, 3>(w[x]);
        }
        if (tail) {
#pragma unroll
          for (int hlf = 0; hlf < 2; ++hlf) wild |= clean(bits, row, 2 * c + hlf, &o[4 * hlf]);
        }
        *reinterpret_cast<uint4*>(slot + place16(row, 2 * c)) = make_uint4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<uint4*>(slot + place16(row, 2 * c + 1)) = make_uint4(o[4], o[5], o[6], o[7]);
      }
    } else if (tail) {
      for (int i = 0; i < 32 / kRows; ++i) {
        const int row = 32 * lw + i * kRows + lane / kChunks;
        uint4* at = reinterpret_cast<uint4*>(slot + place16(row, c));
        const uint4 u = *at;
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if (clean(bits, row, c, w)) {
          wild = true;
          *at = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    if (tail) {
      const bool any = __any_sync(kFull, wild);
      if (lane == 0) bars->wild[s][lw] = any;
    }
    if constexpr (C::TOKEN) {
      if (is_v) {  // the tile's largest finite scale of values, one number per warp
        const float* sc = reinterpret_cast<const float*>(mem + C::kOffScale) + ((t & (kScaleRing - 1)) * 2 + 1) * kTile;
        const float mine = sc[32 * lw + lane];
        unsigned top = __float_as_uint(mine > 0.0f && mine < 1e30f ? mine : 0.0f);
        top = __reduce_max_sync(kFull, top);
        if (lane == 0)
          reinterpret_cast<uint32_t*>(mem + C::kOffScale + kScaleRing * 2 * kTile * 4)[(t & (kScaleRing - 1)) * 4 + lw] = top;
      }
    }
    fence_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->kv_full[s]);
    return true;
  }

  // 8 values of a row: those that are not finite become 0 and are noted.
  static __device__ __forceinline__ bool clean(uint8_t* bits, int row, int chunk, uint32_t* w) {
    uint32_t plus = 0, minus = 0, any = 0;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      uint32_t cl, pl, mi;
      split_finite<C::BF16>(w[x], cl, pl, mi);
      any |= pl | mi;
      w[x] = cl;
      plus |= ((pl & 0xFFFFu ? 1u : 0u) | (pl >> 16 ? 2u : 0u)) << (2 * x);
      minus |= ((mi & 0xFFFFu ? 1u : 0u) | (mi >> 16 ? 2u : 0u)) << (2 * x);
    }
    bits[row * 32 + chunk] = static_cast<uint8_t>(plus);
    bits[row * 32 + 16 + chunk] = static_cast<uint8_t>(minus);
    return any != 0;
  }

  template <int LAG>
  __device__ __forceinline__ void run(int b0, int offset, int count) {
    const int lead = nq == 1 ? 2 : 1;
    Pieces a, f;  // tiles being started, tiles being handed over
    a.start(p, b0, offset, count);
    f.start(p, b0, offset, count);
    int as = 0, fs = 0;
    uint32_t ac = 0, fc = 0, at = 0, ft = 0;  // tiles so far, key tiles before the piece
    bool more = true;
    while (true) {
      if (more) {
        bool is_v;
        int tile;
        order(as, a.nt, lead, is_v, tile);
        if (!issue(a, is_v, tile, ac, at + tile)) break;
        ++ac;
        if (++as == 2 * a.nt) {
          as = 0;
          at += a.nt;
          more = a.next(p);
        }
      }
      cp_commit();  // empty groups behind the last tile keep the count
      if (static_cast<int>(ac - fc) > LAG || !more) {
        if (more)
          cp_wait<LAG>();
        else
          cp_wait<0>();
        bool is_v;
        int tile;
        order(fs, f.nt, lead, is_v, tile);
        if (!finish(f, is_v, tile, fc, ft + tile)) break;
        ++fc;
        if (++fs == 2 * f.nt) {
          fs = 0;
          ft += f.nt;
          if (!f.next(p)) break;
        }
      }
    }
    cp_wait<0>();
  }
};

// ---------------------------------------------------------------- main kernel
__device__ __forceinline__ unsigned long long pair(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpair(unsigned long long v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// One thread's row of the softmax.
template <typename C>
struct Soft {
  const Params& p;
  Bars* bars;
  uint8_t* mem;
  uint32_t tmem_s, tmem_o;  // this warp's lanes of the stream's scores and outputs
  volatile int* abort;
  float m, l, vref, qscale;  // reference maximum and sum; reference scale of the values
  bool wild;

  // The row of queries into shared memory: chunks [c0, c1) of 8 dimensions.
  // bf16 queries of an 8-bit cache become fp16 after a power of two brings the
  // row's largest value to [1, 2): exact for all that count beside it.
  __device__ __forceinline__ void load_q(uint8_t* q_tile, int row, const void* src, bool ok, int c0, int c1) {
    const float scale = p.scale_log2;
    qscale = fabsf(scale);
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;  // the sign goes onto the queries: maxima stay maxima
    const uint4* from = static_cast<const uint4*>(src);
    float down = 1.0f;
    const bool convert = C::kSmall && p.bf16;
    if (convert && ok) {
      float top = 0.0f;
      for (int c = 0; c < C::D / 8; ++c) {
        const uint4 u = from[c];
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xFFFF0000u))));
      }
      const uint32_t ex = min(max(__float_as_uint(top) & 0x7F800000u, 0x0A000000u), 0x75000000u);
      down = __uint_as_float(0x7F000000u - ex);
      qscale *= __uint_as_float(ex);
    }
    for (int c = c0; c < c1; ++c) {
      uint4 u = make_uint4(0u, 0u, 0u, 0u);
      if (ok) u = from[c];
      uint32_t w[4] = {u.x, u.y, u.z, u.w};
      if (convert) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          w[x] = pack2<false>(__uint_as_float(w[x] << 16) * down, __uint_as_float(w[x] & 0xFFFF0000u) * down);
      }
      *reinterpret_cast<uint4*>(q_tile + place16(row, c)) = make_uint4(w[0] ^ flip, w[1] ^ flip, w[2] ^ flip, w[3] ^ flip);
    }
  }

  __device__ __forceinline__ void begin() {
    m = -INFINITY, l = 0.0f, vref = 0.0f;
    wild = false;
  }

  // Scores of one key tile to probabilities.  tail: some keys are not seen (a bit each in seen).
  template <bool TAIL>
  __device__ __forceinline__ void tile(const uint32_t (&seen)[4], const float* ks, const float* vs, float vmax, bool first) {
    float top = -INFINITY;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t s[32];
      tmem_ld32(tmem_s + 32 * c, s);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        float v[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) v[x] = __uint_as_float(s[i + x]);
        if constexpr (C::TOKEN) {
          const float4 k = *reinterpret_cast<const float4*>(ks + 32 * c + i);
          const float2 a = unpair(mul2(pair(v[0], v[1]), pair(k.x, k.y))), b = unpair(mul2(pair(v[2], v[3]), pair(k.z, k.w)));
          v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          if (TAIL && !((seen[c] >> (i + x)) & 1)) v[x] = -INFINITY;
          top = fmaxf(top, v[x]);
        }
      }
    }
    top *= qscale;
    // the reference moves when the maximum left it by more than 2^kGrow
    float alpha = 1.0f;
    if (top > m + kGrow || m == -INFINITY) {
      alpha = m == -INFINITY ? 1.0f : exp2_fast(m - top);
      m = fmaxf(top, m);
    }
    l *= alpha;
    if constexpr (C::TOKEN) {
      if (vmax > 64.0f * vref) {
        const float to = __uint_as_float(max(__float_as_uint(vmax) & 0x7F800000u, 0x0A000000u));
        alpha *= vref == 0.0f ? 1.0f : vref / to;  // nothing but zeros so far
        vref = to;
      }
    }
    if (!first && __any_sync(kFull, alpha != 1.0f)) {
#pragma unroll
      for (int c = 0; c < C::D / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tmem_o + 32 * c, o);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
        tmem_st32(tmem_o + 32 * c, o);
      }
    }
    const float sub = m == -INFINITY ? 0.0f : m;
    const unsigned long long q2 = pair(qscale, qscale), m2 = pair(-sub, -sub);
    const float inv = C::TOKEN ? __uint_as_float(0x7F000000u - __float_as_uint(vref)) : 1.0f;
    unsigned long long sum0 = pair(0.0f, 0.0f), sum1 = sum0;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t s[32], out[16];
      tmem_ld32(tmem_s + 32 * c, s);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        unsigned long long a = pair(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
        unsigned long long b = pair(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
        if constexpr (C::TOKEN) {
          const float4 k = *reinterpret_cast<const float4*>(ks + 32 * c + i);
          a = mul2(a, pair(k.x, k.y)), b = mul2(b, pair(k.z, k.w));
        }
        const float2 ea = unpair(fma2(a, q2, m2)), eb = unpair(fma2(b, q2, m2));
        float e[4] = {ea.x, ea.y, eb.x, eb.y};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          e[x] = exp2_fast(e[x]);
          if (TAIL && !((seen[c] >> (i + x)) & 1)) e[x] = 0.0f;
        }
        a = pair(e[0], e[1]), b = pair(e[2], e[3]);
        sum0 = add2(sum0, a), sum1 = add2(sum1, b);
        if constexpr (C::TOKEN) {
          const float4 v = *reinterpret_cast<const float4*>(vs + 32 * c + i);
          const unsigned long long i2 = pair(inv, inv);
          a = mul2(a, mul2(pair(v.x, v.y), i2)), b = mul2(b, mul2(pair(v.z, v.w), i2));
          const float2 fa = unpair(a), fb = unpair(b);
          e[0] = fa.x, e[1] = fa.y, e[2] = fb.x, e[3] = fb.y;
          if (TAIL) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (!((seen[c] >> (i + x)) & 1)) e[x] = 0.0f;  // an unseen scale may be anything
          }
        }
        out[i / 2] = pack2<C::BF16>(e[0], e[1]);
        out[i / 2 + 1] = pack2<C::BF16>(e[2], e[3]);
      }
      tmem_st16(tmem_s + 16 * c, out);
    }
    const float2 sa = unpair(add2(sum0, sum1));
    l += sa.x + sa.y;
  }

  // Values that are not finite, of new tokens this row sees: noted for its output.
  __device__ __forceinline__ void note_wild(const uint32_t (&seen)[4], int slot, int row) {
    uint32_t* mine = reinterpret_cast<uint32_t*>(mem + C::kOffRowWild) + row * 8;
    if (!wild) {
      wild = true;
      for (int x = 0; x < 8; ++x) mine[x] = 0;
    }
    for (int j = 0; j < kTile; ++j) {
      if (!((seen[j >> 5] >> (j & 31)) & 1)) continue;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(mem + C::kOffWild + slot * C::kWild + j * 32);
      for (int x = 0; x < 8; ++x)
        if ((x & 3) < C::D / 32) mine[x] |= bits[x];
    }
  }
};

template <typename C>
__global__ void __launch_bounds__(kThreadsTc, 1) attend_tc_kernel(const __grid_constant__ Params p, int nq) {
  constexpr int D = C::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* mem = smem_raw + ((1024 - (raw_addr & 1023)) & 1023);
  const uint32_t base = smem_u32(mem);
  Bars* bars = reinterpret_cast<Bars*>(mem + C::kOffBars);
  __shared__ int red[kWarpsTc + 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &bars->abort;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (p.bf16)
    clear_idle_requests<__nv_bfloat16, kThreadsTc>(p, D);
  else
    clear_idle_requests<__half, kThreadsTc>(p, D);

  int total, unit, b0, before, share = 0;
  locate<kThreadsTc>(
      p,
      [&](int tot) {
        share = share_of(p, tot, gridDim.x);
        return static_cast<int>(min(static_cast<long long>(blockIdx.x) * share, 2147483647ll));
      },
      red, total, unit, b0, before);
  if (unit >= total) return;
  const int count = min(share, total - unit), offset = unit - before;

  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars->kv_full[i], kLoadWarps);
      mbar_init(&bars->kv_empty[i], 1);
    }
    mbar_init(&bars->q_full, kSoftWarps);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars->s_full[i], 1);
      mbar_init(&bars->p_full[i], kSoftWarps / 2);
      mbar_init(&bars->o_done[i], 1);
    }
    mbar_init(&bars->both, kSoftWarps);
    mbar_init(&bars->drain, 1);
    bars->abort = 0;
    fence_barrier_init();
  }
  if (warp == kWarpsTc - 1) {
    tmem_alloc(&bars->tmem, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const uint32_t q_addr = base + C::kOffQ;

  if (warp >= kSoftWarps && warp < kSoftWarps + kLoadWarps) {
    // ------------------------------------------------ loaders
    Loader<C> ld{p, bars, base, mem, q_addr + nq * C::kSlot, nq, C::raw_depth(nq), warp - kSoftWarps, lane, abort};
    if constexpr (!C::kSmall) {
      ld.template run<2>(b0, offset, count);
    } else if (nq == 1) {
      ld.template run<3>(b0, offset, count);
    } else {
      ld.template run<1>(b0, offset, count);
    }
  } else if (warp == kWarpsTc - 1 && lane == 0) {
    // ------------------------------------------------ products
    Pieces pc;
    pc.start(p, b0, offset, count);
    const int lead = nq == 1 ? 2 : 1;
    uint32_t kv = 0, piece = 0, pp[2] = {0, 0};  // tiles taken, pieces, probabilities taken
    auto scores = [&](int x, uint32_t s) {        // S_x = Q_x K^T
      const uint32_t q = q_addr + (nq == 1 ? 0 : x) * C::kSlot, k = base + s * C::kSlot;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint32_t o = (kk >> 2) * C::kBlock + (kk & 3) * 32;
        mma_ss(tmem + x * kTile, smem_desc_k128(q + o), smem_desc_k128(k + o), idesc(C::BF16, kTile, false), kk > 0);
      }
      umma_commit(&bars->s_full[x]);
    };
    auto outputs = [&](int x, uint32_t s, bool accumulate) {  // O_x += P_x V
      const uint32_t v = base + s * C::kSlot;
#pragma unroll
      for (int kk = 0; kk < kTile / 16; ++kk)
        mma_ts(tmem + 2 * kTile + x * D, tmem + x * kTile + kk * 8, desc_values(v + kk * 2048), idesc(C::BF16, D, true),
               accumulate || kk > 0);
    };
    auto take = [&](uint32_t n) { return wait(&bars->kv_full[n % C::kSlots], (n / C::kSlots) & 1, abort); };
    bool ok = true;
    do {
      const int nt = pc.nt;
      ok = wait(&bars->q_full, piece & 1, abort);
      ++piece;
      if (!ok) break;
      for (int j = 0; j < min(lead, nt) && ok; ++j) {
        ok = take(kv);
        if (!ok) break;
        tc_fence_after();
        if (nq == 1) {
          scores(j, kv % C::kSlots);
        } else {
          scores(0, kv % C::kSlots);
          scores(1, kv % C::kSlots);
        }
        umma_commit(&bars->kv_empty[kv % C::kSlots]);
        ++kv;
      }
      for (int j = 0; j < nt && ok; ++j) {
        const uint32_t v = kv++;
        const bool more = j + lead < nt;
        const uint32_t k = more ? kv++ : 0;
        ok = take(v);
        for (int y = 0; y < nq && ok; ++y) {
          const int x = nq == 1 ? j & 1 : y;
          ok = wait(&bars->p_full[x], pp[x] & 1, abort);
          ++pp[x];
          if (!ok) break;
          tc_fence_after();
          outputs(x, v % C::kSlots, nq == 1 ? j > 1 : j > 0);
          if (nq == 1 ? j + 2 >= nt : j + 1 == nt) umma_commit(&bars->o_done[x]);
          if (y == nq - 1) umma_commit(&bars->kv_empty[v % C::kSlots]);
          if (more) {
            if (y == 0) ok = take(k);
            if (!ok) break;
            tc_fence_after();
            scores(x, k % C::kSlots);
            if (y == nq - 1) umma_commit(&bars->kv_empty[k % C::kSlots]);
          }
        }
      }
    } while (ok && pc.next(p));
    // every product issued has ended before the block gives its memory back
    umma_commit(&bars->drain);
    for (uint32_t n = 0; n < (1u << 22) && !mbar_try_wait(&bars->drain, 0); ++n) {
    }
  } else if (warp < kSoftWarps) {
    // ------------------------------------------------ softmax and output
    const int x = warp >> 2, wrow = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    Soft<C> so{p, bars, mem, tmem + lanes + x * kTile, tmem + lanes + 2 * kTile + x * D, abort};
    float2* ml = reinterpret_cast<float2*>(mem + C::kOffMl);
    const float* scales = reinterpret_cast<const float*>(mem + C::kOffScale);
    const float* vtop = scales + kScaleRing * 2 * kTile;
    uint32_t kv = 0, t0 = 0, sp = 0, op[2] = {0, 0}, meets = 0;
    auto meet = [&]() {  // the two streams' warps
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->both);
      return wait(&bars->both, meets++ & 1, abort);
    };
    const int lead = nq == 1 ? 2 : 1;
    Pieces pc;
    pc.start(p, b0, offset, count);
    bool ok = true;
    do {
      const Request r = pc.w.r;
      const int rts = row_tiles(p, r);
      const int h = pc.w.item / rts, rt = pc.w.item - h * rts;
      const int row = (rt << p.rows_log2) + (nq == 1 ? 0 : x * kTile) + wrow;
      const int rows = r.n * p.group;
      const bool row_ok = row < rows;
      const bool warp_ok = row - lane < rows;
      const int qi = row / p.group, head = h * p.group + row - qi * p.group, t = r.first + qi;
      so.begin();
      {
        const int half = D / 16;  // with one row tile the two warps of a row share the copy
        const uint8_t* src = static_cast<const uint8_t*>(p.q) + (t * p.q_tok + head * p.q_head) * 2;
        so.load_q(mem + C::kOffQ + (nq == 1 ? 0 : x) * C::kSlot, wrow, src, row_ok, nq == 1 ? x * half : 0,
                  nq == 1 ? x * half + half : D / 8);
        if constexpr (C::kSmall && !C::TOKEN) so.qscale *= p.c.k_scale[h * p.c.k_scale_stride[2]];
        fence_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->q_full);
      }
      bool first = true;
      for (int j = nq == 1 ? x : 0; j < pc.nt && ok; j += nq == 1 ? 2 : 1) {
        ok = wait(&bars->s_full[x], sp & 1, abort);
        ++sp;
        if (!ok) break;
        tc_fence_after();
        if (warp_ok) {
          const int key0 = (pc.tile0 + j) * kTile;
          const bool tail = key0 + kTile > r.len - r.n;
          const float *ks = nullptr, *vs = nullptr;
          float vmax = 0.0f;
          uint32_t seen[4] = {kFull, kFull, kFull, kFull};
          int slot = 0;
          if (C::TOKEN || (C::KIND != kInt8 && tail && r.n > 1)) {
            // the value tile's scales and notes are needed: its place in the order of loads
            const uint32_t n = kv + (j + lead < pc.nt ? lead + 2 * j : min(lead, pc.nt) + max(pc.nt - lead, 0) + j);
            slot = n % C::kSlots;
            ok = wait(&bars->kv_full[slot], (n / C::kSlots) & 1, abort);
            if (!ok) break;
            if constexpr (C::TOKEN) {
              const int ring = (t0 + j) & (kScaleRing - 1);
              ks = scales + ring * 2 * kTile, vs = ks + kTile;
              const float4 v4 = *reinterpret_cast<const float4*>(vtop + 4 * ring);
              vmax = fmaxf(fmaxf(v4.x, v4.y), fmaxf(v4.z, v4.w));
            }
          }
          if (tail) {
#pragma unroll
            for (int c = 0; c < 4; ++c) seen[c] = row_ok ? seen32(p, r, t, qi, key0 + 32 * c) : kFull;
            if (C::KIND != kInt8 && r.n > 1) {
              const int* w = bars->wild[slot];
              if (w[0] | w[1] | w[2] | w[3]) so.note_wild(seen, slot, x * kTile + wrow);
            }
            so.template tile<true>(seen, ks, vs, vmax, first);
          } else {
            so.template tile<false>(seen, ks, vs, vmax, first);
          }
          first = false;
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[x]);
      }
      if (!ok) break;

      // ---- end of the run: outputs, or partial sums where the item goes on in another block
      const bool whole = pc.tile0 == 0 && pc.nt == pc.w.tiles;
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + (pc.tile0 == 0 ? 1 : 0)) << p.rows_log2;
      const bool two = nq == 1 && pc.nt > 1;  // both streams hold sums of these rows
      const int streams = nq == 1 ? (two ? 2 : 1) : 0;
      if (nq == 1) {
        for (int y = 0; y < streams && ok; ++y) ok = wait(&bars->o_done[y], op[y]++ & 1, abort);
      } else {
        ok = wait(&bars->o_done[x], op[x]++ & 1, abort);
      }
      if (!ok) break;
      tc_fence_after();
      float f0, f1 = 0.0f, m = so.m, l = so.l;
      int c0 = 0, c1 = D / 32;
      uint32_t o0 = so.tmem_o, o1 = so.tmem_o;
      bool wild = so.wild;
      const float vscale = C::kSmall ? (C::TOKEN ? so.vref : p.c.v_scale[h * p.c.v_scale_stride[2]]) : 1.0f;
      f0 = vscale;
      if (nq == 1) {
        // each stream's warps write half of the dimensions, joining both streams' sums
        ml[x * kTile + wrow] = make_float2(so.m, so.l);
        float* vr = reinterpret_cast<float*>(mem + C::kOffQ);  // every score is done: the queries' place is free
        if (C::TOKEN) vr[x * kTile + wrow] = so.vref;
        if (C::KIND != kInt8) reinterpret_cast<int*>(vr)[2 * kTile + x * kTile + wrow] = so.wild;
        ok = meet();
        if (!ok) break;
        const float2 a = ml[wrow], b = two ? ml[kTile + wrow] : make_float2(-INFINITY, 0.0f);
        m = fmaxf(a.x, b.x);
        const float wa = a.x == -INFINITY ? 1.0f : exp2_fast(a.x - m), wb = b.x == -INFINITY ? 1.0f : exp2_fast(b.x - m);
        l = a.y * wa + b.y * wb;
        const float va = C::TOKEN ? vr[wrow] : vscale, vb = C::TOKEN ? (two ? vr[kTile + wrow] : 0.0f) : vscale;
        f0 = wa * va, f1 = wb * vb;
        if (C::KIND != kInt8) {
          const int* wl = reinterpret_cast<const int*>(vr) + 2 * kTile;
          wild = wl[wrow] || (two && wl[kTile + wrow]);
        }
        o0 = tmem + lanes + 2 * kTile, o1 = o0 + D;
        c0 = x * (D / 64), c1 = c0 + D / 64;
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        f0 *= inv, f1 *= inv;
      }
      const int at_row = (nq == 1 ? 0 : x * kTile) + wrow;
      if (warp_ok) {
        for (int c = c0; c < c1; ++c) {
          uint32_t a[32], b[32];
          tmem_ld32(o0 + 32 * c, a);
          if (two) tmem_ld32(o1 + 32 * c, b);
          tmem_ld_wait();
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] = __uint_as_float(a[i]) * f0;
            if (two) v[i] += __uint_as_float(b[i]) * f1;
          }
          if (C::KIND != kInt8 && wild) {
            const uint32_t* bits = reinterpret_cast<const uint32_t*>(mem + C::kOffRowWild);
            uint32_t plus = 0, minus = 0;
            for (int y = nq == 1 ? 0 : x; y < (nq == 1 ? 2 : x + 1); ++y) {
              const bool noted = nq == 1 ? reinterpret_cast<const int*>(mem + C::kOffQ)[2 * kTile + y * kTile + wrow] != 0 : true;
              if (!noted || (y == 1 && nq == 1 && !two)) continue;
              plus |= bits[(y * kTile + wrow) * 8 + c];
              minus |= bits[(y * kTile + wrow) * 8 + 4 + c];
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if ((plus >> i) & 1) v[i] += INFINITY;
              if ((minus >> i) & 1) v[i] -= INFINITY;
            }
          }
          if (!row_ok) continue;
          if (!whole) {
            float4* to = reinterpret_cast<float4*>(p.part_o + (part + at_row) * D + 32 * c);
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
          } else {
            uint4* to = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p.out) + (t * p.o_tok + head * p.o_head) * 2 + 64 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int y = 0; y < 4; ++y)
                w[y] = p.bf16 ? pack2<true>(v[8 * i + 2 * y], v[8 * i + 2 * y + 1]) : pack2<false>(v[8 * i + 2 * y], v[8 * i + 2 * y + 1]);
              to[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
        if (row_ok && (nq == 2 || x == 0)) {
          if (!whole) {
            p.part_ml[(part + at_row) * 2] = m;
            p.part_ml[(part + at_row) * 2 + 1] = l;
          } else if (p.lse) {
            p.lse[static_cast<long long>(t) * p.kv_heads * p.group + head] =
                l == 0.0f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
          }
        }
      }
      if (nq == 1) {  // notes are read before queries replace them
        ok = meet();
        if (!ok) break;
      }
      kv += 2 * pc.nt;
      t0 += pc.nt;
    } while (pc.next(p));
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort) atomicOr(&g_attn_error, 2);
  if (warp == kWarpsTc - 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename C>
orError_t launch(Params& p, int nq, cudaStream_t st, int sms) {
  const void* fn = reinterpret_cast<const void*>(&attend_tc_kernel<C>);
  MCPU_CUDA_TRY(ensure_dynamic_smem(fn, C::smem(nq)), "tree_attention");
  attend_tc_kernel<C><<<sms, kThreadsTc, C::smem(nq), st>>>(p, nq);
  return from_cuda(cudaGetLastError(), "tree_attention launch");
}

template <int D>
orError_t pick(Params& p, int nq, cudaStream_t st, int sms) {
  const bool token = p.c.scale_mode == MCPU_KV_SCALE_TOKEN;
  switch (p.c.dtype) {
    case MCPU_FLOAT8_E4M3:
      return token ? launch<Cfg<kE4M3, false, D, true>>(p, nq, st, sms) : launch<Cfg<kE4M3, false, D, false>>(p, nq, st, sms);
    case MCPU_INT8:
      return token ? launch<Cfg<kInt8, false, D, true>>(p, nq, st, sms) : launch<Cfg<kInt8, false, D, false>>(p, nq, st, sms);
    case MCPU_BFLOAT16:
      return launch<Cfg<kSame, true, D, false>>(p, nq, st, sms);
    default:
      return launch<Cfg<kSame, false, D, false>>(p, nq, st, sms);
  }
}

}  // namespace tc

orError_t launch_tc(Params& p, int D, long long rows, cudaStream_t st, int sms, int* grid) {
  const int nq = rows <= tc::kTile ? 1 : 2;
  p.rows_log2 = nq == 1 ? 7 : 8;
  p.keys_log2 = 7;
  p.min_share = 1;
  *grid = sms;
  return D == 64 ? tc::pick<64>(p, nq, st, sms) : tc::pick<128>(p, nq, st, sms);
}

orError_t tc_read_error(int* flag, bool reset) {
  int z = 0;
  MCPU_CUDA_TRY(cudaMemcpyFromSymbol(flag, g_attn_error, sizeof(int)), "mcpu_device_error");
  if (reset) MCPU_CUDA_TRY(cudaMemcpyToSymbol(g_attn_error, &z, sizeof(int)), "mcpu_device_error");
  return orSuccess;
}

}  // namespace attn
}  // namespace mcpu
