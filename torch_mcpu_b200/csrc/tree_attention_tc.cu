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
// One block per SM, groups of four warps:
//   2 groups  softmax of stream 0 and 1: a thread owns a row (its
//             tensor-memory lane), reads the scores, keeps the running maximum
//             and sum, writes the probabilities over the scores as 16-bit
//             values, the left operand of the second product
//   1         loaders.  16-bit caches: pages to shared memory by 16-byte
//             asynchronous copies into the 128-byte-swizzled layout.  8-bit
//             ones: rows of a raw ring widened to fp16
//   1         its first warp issues the products; with 8-bit caches two more
//             fetch the rows of keys and of values, with their scales
// Tensor memory: scores of the two streams (2 x 128 columns), outputs (2 x D).
//
// The output is scaled down only when a row's maximum grew by more than 2^8
// since the reference was set; until then probabilities up to 256 are summed,
// which fp16 and bf16 hold and fp32 sums take without loss.
//
// Measured: 16 requests of up to 8192 tokens with trees of 61, 64 / 8 heads of
// 128, bf16 (133 GFLOP) 211 us, 632 TFLOP/s, in a burst, and 245 us, 545
// TFLOP/s, in seconds of calls, when the power cap holds the SM clock at 1.7 GHz
// instead of 1.96; 6 requests of up to 32768 with
// trees of 13, 32 / 8 heads, fp16 over int8 (279 MB) 137 us, 2.0 TB/s.  The
// tensor pipe is 36 % and the exponentials' 31 % busy: each stream's chain
// (scores, softmax, product) is what a pair of tiles waits for, about 3500
// cycles against 2048 of exponentials, and a piece's beginning and end cost as
// much as four tiles.  With 8 bits the widening of the rows adds to it.
// Tried and slower: sixteen softmax warps (234 us), softmax loops unrolled over
// the whole row (308 us, the code outgrew the instruction cache), part of the
// exponentials by polynomial (equal), bulk copies of 128-byte rows (34 cycles
// each to issue).
#include <algorithm>
#include <type_traits>

#include "sm100.cuh"
#include "tree_attention.cuh"

namespace mcpu {
namespace attn {
namespace tc {

using namespace sm100;

constexpr int kSoftWarps = 8;
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
  static constexpr float kBias = TOKEN || BF16 ? 0.0f : 7.0f;  // probabilities are held times 2^kBias
  static constexpr int kLoadWarps = 4;
  static constexpr int kRowsPerWarp = kTile / kLoadWarps;
  static constexpr int kWarps = kSoftWarps + kLoadWarps + 4;
  static constexpr int kThreads = 32 * kWarps;
  // registers: what the block is launched with (a multiple of 8 that fits), then each group's own share of it
  static constexpr int kRegs = 128, kSoftRegs = 144, kLoadRegs = 96, kIssueRegs = 128;
  static_assert(kSoftWarps * kSoftRegs + kLoadWarps * kLoadRegs + 4 * kIssueRegs <= kWarps * kRegs, "more than launched with");
  static constexpr int kSlots = kSmall ? 3 : 4;  // key or value tiles in shared memory
  static constexpr int kSlot = kTile * D * 2;
  static constexpr int kBlock = kTile * 128;     // 64 dimensions of a tile
  static constexpr int kRaw = kSmall ? kTile * D : 0;
  static constexpr int kWild = KIND == kInt8 ? 0 : kTile * 32;  // two bits per value, in values that are not finite
  // shared memory, from a 1024-byte boundary
  static constexpr int kOffWild = kSlots * kSlot;
  static constexpr int kOffRowWild = kOffWild + kSlots * kWild;
  static constexpr int kOffScale = kOffRowWild + (KIND == kInt8 ? 0 : 2 * kTile * 32);
  static constexpr int kOffMl = kOffScale + (TOKEN ? kScaleRing * 2 * kTile * 4 : 0);
  static constexpr int kOffBars = kOffMl + 2 * kTile * 16;
  static constexpr int kOffQ = (kOffBars + 768 + 1023) / 1024 * 1024;
  static constexpr int raw_depth(int nq) { return !kSmall ? 0 : nq == 1 ? 4 : 2; }
  static constexpr int q_bytes(int nq) { return nq * kSlot < 32768 ? 32768 : nq * kSlot; }  // 4 KB a warp for the outputs
  static constexpr int smem(int nq) { return kOffQ + q_bytes(nq) + raw_depth(nq) * kRaw + 1024; }
};

struct Bars {
  uint64_t kv_full[4], kv_empty[4], raw_full[4], raw_empty[4], sc_full[kScaleRing], q_full, s_full[2], p_full[2], o_done[2], both, drain;
  uint32_t tmem;
  int abort;
  int wild[4][8];
};
static_assert(sizeof(Bars) <= 768, "barriers overflow their place");

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The upper half of the operands' descriptors: 8-row groups 1024 bytes apart,
// version 1, 128-byte swizzle.  The lower half is the address / 16, and for
// values the distance of the next 64 dimensions.
constexpr uint32_t kDescHigh = (1024u >> 4) | 1u << 14 | 2u << 29;

__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
      "r"(accumulate), "r"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Whether the phase has completed, without waiting.
__device__ __forceinline__ bool mbar_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
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

// Lower half of the descriptor of values: rows of 128 bytes (64 dimensions),
// one per key, as the right operand keys x dimensions with the dimensions
// contiguous: 8-key groups 1024 bytes apart (stride byte offset), the next 64
// dimensions 128 keys further (leading byte offset).
constexpr uint32_t kValuesLead = static_cast<uint32_t>((kTile * 128) >> 4) << 16;
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

// ---------------------------------------------------------------- loads
// A block's run: where its units begin, and how many they are.
struct Run {
  int b0, before, unit, count;
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
// A row of a tile in the pages, found one tile ahead: the block table's
// latency passes under the previous tile's work.
struct Place {
  int id, slot;
  bool valid;
};
__device__ __forceinline__ Place look(const Params& p, const Pieces& pc, int tile, int row) {
  Place at{0, 0, false};
  const int key = (pc.tile0 + tile) * kTile + row;
  if (key < pc.r.len) {
    const int page = p.block_log2 >= 0 ? key >> p.block_log2 : key / p.c.block_size;
    at.slot = key - page * p.c.block_size;
    at.id = p.table[pc.b * p.table_stride + page];
    at.valid = true;
  }
  return at;
}

// 8 values of a row: those that are not finite become 0 and are noted.
template <bool BF16>
__device__ __forceinline__ bool clean(uint8_t* bits, int row, int chunk, uint32_t* w) {
  uint32_t plus = 0, minus = 0, any = 0;
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    uint32_t cl, pl, mi;
    split_finite<BF16>(w[x], cl, pl, mi);
    any |= pl | mi;
    w[x] = cl;
    plus |= ((pl & 0xFFFFu ? 1u : 0u) | (pl >> 16 ? 2u : 0u)) << (2 * x);
    minus |= ((mi & 0xFFFFu ? 1u : 0u) | (mi >> 16 ? 2u : 0u)) << (2 * x);
  }
  bits[row * 32 + chunk] = static_cast<uint8_t>(plus);
  bits[row * 32 + 16 + chunk] = static_cast<uint8_t>(minus);
  return any != 0;
}

template <typename C>
struct Loader {
  const Params& p;
  Bars* bars;
  uint32_t base;   // shared memory, 1024-byte aligned
  uint8_t* mem;
  uint32_t raw;
  int nq, depth, lw, lane;
  volatile int* abort;

  // Value tiles with new tokens that some of the request's rows may not see: a lane looks through the values it wrote.
  __device__ __forceinline__ void clean_tail(const Pieces& pc, int tile, uint32_t s) const {
    if (C::KIND == kInt8 || !some_unseen(p, pc.r) || (pc.tile0 + tile + 1) * kTile <= pc.r.len - pc.r.n) return;
    constexpr int kChunks = C::D * (C::kSmall ? 1 : 2) / 16, kRows = 32 / kChunks, kSteps = C::kRowsPerWarp / kRows;
    constexpr uint32_t kExp = C::BF16 ? 0x7F807F80u : 0x7C007C00u;
    const int c = lane % kChunks, row0 = C::kRowsPerWarp * lw + lane / kChunks;
    const uint8_t* slot = mem + s * C::kSlot;
    uint32_t any = 0;
#pragma unroll 4
    for (int i = 0; i < kSteps; ++i)
#pragma unroll
      for (int y = 0; y < (C::kSmall ? 2 : 1); ++y) {
        const uint4 u = *reinterpret_cast<const uint4*>(slot + place16(row0 + i * kRows, C::kSmall ? 2 * c + y : c));
        any |= __vcmpeq2(u.x & kExp, kExp) | __vcmpeq2(u.y & kExp, kExp) | __vcmpeq2(u.z & kExp, kExp) | __vcmpeq2(u.w & kExp, kExp);
      }
    const bool wild = __any_sync(kFull, any != 0);
    if (lane == 0) bars->wild[s][lw] = wild;
    if (!wild) return;  // the notes of these rows are not read
    for (int i = 0; i < kSteps; ++i)
      for (int y = 0; y < (C::kSmall ? 2 : 1); ++y) {
        const int row = row0 + i * kRows, c2 = C::kSmall ? 2 * c + y : c;
        uint4* at = reinterpret_cast<uint4*>(mem + s * C::kSlot + place16(row, c2));
        const uint4 u = *at;
        uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if (clean<C::BF16>(mem + C::kOffWild + s * C::kWild, row, c2, w)) *at = make_uint4(w[0], w[1], w[2], w[3]);
      }
  }
  __device__ __forceinline__ void hand_over(uint32_t s) const {
    fence_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&bars->kv_full[s]);
  }

  // ---- 16-bit caches: asynchronous copies straight into the tiles.  A tile is started when its place is free, else the
  // oldest one under way is waited for and handed over.
  __device__ __forceinline__ void copy(const Pieces& pc, const Place& at, bool is_v, uint32_t dst) const {
    const unsigned rows_valid = __ballot_sync(kFull, at.valid);
    const int h = pc.item / row_tiles(p, pc.r);
    const uint32_t off = offset16(at, is_v ? p.c.value_stride : p.c.key_stride);
    constexpr int kChunks = C::D * 2 / 16, kRows = 32 / kChunks;
    const int c = lane % kChunks;
    const uint4* from = static_cast<const uint4*>(is_v ? p.c.value : p.c.key) +
                        (h * (is_v ? p.c.value_stride[2] : p.c.key_stride[2]) / 8 + c);
    // shuffles first: copies and shuffles keep their order, and in turn each copy would wait for its shuffle
    constexpr int kSteps = C::kRowsPerWarp / kRows;
    uint32_t o[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) o[i] = __shfl_sync(kFull, off, i * kRows + lane / kChunks);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int row = i * kRows + lane / kChunks;
      cp_async16(dst + place16(C::kRowsPerWarp * lw + row, c), from + o[i], (rows_valid >> row) & 1);
    }
  }
  // A row's place in 16-byte units: 32 bits reach 64 GB, which the entry point makes sure of.
  __device__ __forceinline__ uint32_t offset16(const Place& at, const int64_t* st) const {
    constexpr int kPer = C::kSmall ? 16 : 8;
    const int block = static_cast<int>(kv::checked_block(at.id, p.c.num_blocks, &g_attn_error));
    return static_cast<uint32_t>(block) * static_cast<uint32_t>(st[0] / kPer) +
           static_cast<uint32_t>(at.slot) * static_cast<uint32_t>(st[1] / kPer);
  }
  __device__ __forceinline__ void run_copies(const Run& run) {
    const int lead = nq == 1 ? 2 : 1, row = C::kRowsPerWarp * lw + lane;
    Pieces a, f, k;  // tiles being started, being handed over, being looked up (two ahead)
    a.start(p, run.b0, run.before, run.unit, run.count);
    f = a, k = a;
    int as = 0, fs = 0, ks = 0;
    uint32_t ac = 0, fc = 0;
    bool more = true, known = true;
    auto look_up = [&]() {
      Place at{0, 0, false};
      if (!known) return at;
      bool v;
      int tile;
      order(ks, k.nt, lead, v, tile);
      at = look(p, k, tile, row);
      if (++ks == 2 * k.nt) {
        ks = 0;
        known = k.next(p);
      }
      return at;
    };
    Place here = look_up(), then = look_up();
    while (true) {
      const uint32_t pending = ac - fc;
      if (more && pending < C::kSlots) {
        uint64_t* bar = &bars->kv_empty[ac % C::kSlots];
        const uint32_t parity = ((ac / C::kSlots) & 1) ^ 1;
        bool free = __all_sync(kFull, mbar_test(bar, parity));
        if (!free && pending == 0) {
          if (!wait(bar, parity, abort)) break;
          free = true;
        }
        if (free) {
          bool is_v;
          int tile;
          order(as, a.nt, lead, is_v, tile);
          copy(a, here, is_v, base + (ac % C::kSlots) * C::kSlot);
          cp_commit();
          here = then;
          then = look_up();
          ++ac;
          if (++as == 2 * a.nt) {
            as = 0;
            more = a.next(p);
          }
          continue;
        }
      }
      if (pending == 0) break;
      switch (pending) {
        case 1: cp_wait<0>(); break;
        case 2: cp_wait<1>(); break;
        case 3: cp_wait<2>(); break;
        default: cp_wait<3>(); break;
      }
      bool fv;
      int ftile;
      order(fs, f.nt, lead, fv, ftile);
      if (fv) clean_tail(f, ftile, fc % C::kSlots);
      hand_over(fc % C::kSlots);
      ++fc;
      if (++fs == 2 * f.nt) {
        fs = 0;
        if (!f.next(p)) break;
      }
    }
    cp_wait<0>();
  }

  // ---- 8-bit caches, fetching: one warp takes the key tiles, one the value tiles.
  __device__ __forceinline__ void run_fetch(bool values, const Run& run) {
    const int lead = nq == 1 ? 2 : 1;
    const int64_t* st = values ? p.c.value_stride : p.c.key_stride;
    const int64_t* ss = values ? p.c.v_scale_stride : p.c.k_scale_stride;
    Pieces pc;
    pc.start(p, run.b0, run.before, run.unit, run.count);
    uint32_t n0 = 0, t0 = 0;  // tiles and key tiles before the piece
    bool ok = true;
    do {
      const int nt = pc.nt, first = min(lead, nt);
      const int h = pc.item / row_tiles(p, pc.r);
      constexpr int kChunks = C::D / 16, kRows = 32 / kChunks;  // rows a copy of the whole warp takes
      const int c = lane % kChunks;
      const uint4* from = static_cast<const uint4*>(values ? p.c.value : p.c.key) + (h * st[2] / 16 + c);
      const float* scales = (values ? p.c.v_scale : p.c.k_scale) + h * ss[2];
      Place next[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) next[i] = look(p, pc, 0, 32 * i + lane);
      for (int j = 0; j < nt && ok; ++j) {
        Place now[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          now[i] = next[i];
          if (j + 1 < nt) next[i] = look(p, pc, j + 1, 32 * i + lane);
        }
        // its number in the order of loads
        const uint32_t n = n0 + (values ? (j + lead < nt ? lead + 2 * j : nt + j) : (j < first ? j : 2 * j - lead + 1));
        const uint32_t r = n & (depth - 1);
        ok = wait(&bars->raw_empty[r], ((n / depth) & 1) ^ 1, abort);
        if (!ok) break;
        const uint32_t dst = raw + r * C::kRaw;
        const uint32_t sc = base + C::kOffScale + ((((t0 + j) & (kScaleRing - 1)) * 2 + values) * kTile + lane) * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned valid = __ballot_sync(kFull, now[i].valid);
          const uint32_t off = offset16(now[i], st);
          uint32_t o[32 / kRows];
#pragma unroll
          for (int k = 0; k < 32 / kRows; ++k) o[k] = __shfl_sync(kFull, off, k * kRows + lane / kChunks);
#pragma unroll
          for (int k = 0; k < 32 / kRows; ++k) {
            const int row = k * kRows + lane / kChunks;
            cp_async16(dst + ((32 * i + row) * kChunks + c) * 16, from + o[k], (valid >> row) & 1);
          }
          if constexpr (C::TOKEN) {
            const long long block = kv::checked_block(now[i].id, p.c.num_blocks, &g_attn_error);
            cp_async4(sc + 128 * i, scales + block * ss[0] + now[i].slot * ss[1], now[i].valid);
          }
        }
        if (C::TOKEN && values) cp_arrive(&bars->sc_full[(t0 + j) & (kScaleRing - 1)]);
        cp_arrive(&bars->raw_full[r]);
      }
      n0 += 2 * nt;
      t0 += nt;
    } while (ok && pc.next(p));
    cp_wait<0>();
  }
  // Arrives when this lane's copies so far have landed.
  static __device__ __forceinline__ void cp_arrive(uint64_t* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  }

  // ---- 8-bit caches, widening: raw rows to fp16 in the swizzled tiles.
  __device__ __forceinline__ void run_widen(const Run& run) {
    const int lead = nq == 1 ? 2 : 1;
    constexpr int kChunks = C::D / 16, kRows = 32 / kChunks, kSteps = C::kRowsPerWarp / kRows;
    const int c = lane % kChunks, row0 = C::kRowsPerWarp * lw + lane / kChunks;
    Pieces pc;
    pc.start(p, run.b0, run.before, run.unit, run.count);
    uint32_t n = 0;
    bool ok = true;
    do {
      for (int st = 0; st < 2 * pc.nt && ok; ++st, ++n) {
        bool is_v;
        int tile;
        order(st, pc.nt, lead, is_v, tile);
        const uint32_t r = n & (depth - 1), s = n % C::kSlots;
        ok = wait(&bars->raw_full[r], (n / depth) & 1, abort);
        if (!ok) break;
        const uint8_t* from = mem + (raw - base) + r * C::kRaw + (row0 * kChunks + c) * 16;
        uint4 u[kSteps];
#pragma unroll
        for (int i = 0; i < kSteps; ++i) u[i] = *reinterpret_cast<const uint4*>(from + i * kRows * kChunks * 16);
        ok = wait(&bars->kv_empty[s], ((n / C::kSlots) & 1) ^ 1, abort);
        if (!ok) break;
        uint8_t* slot = mem + s * C::kSlot;
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
          const int row = row0 + i * kRows;
          uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w}, o[8];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            if (C::KIND == kInt8) w[x] ^= 0x80808080u;
            o[2 * x] = widen<C::KIND, 0, 1>(w[x]);
            o[2 * x + 1] = widen<C::KIND, 2, 3>(w[x]);
          }
          // the lanes of the second 64 dimensions store their halves the other way round: all banks at once
          const bool late = C::D == 128 && c >= kChunks / 2;
          const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
          *reinterpret_cast<uint4*>(slot + place16(row, 2 * c + late)) = late ? hi : lo;
          *reinterpret_cast<uint4*>(slot + place16(row, 2 * c + !late)) = late ? lo : hi;
        }
        if (is_v) clean_tail(pc, tile, s);
        hand_over(s);
        if (lane == 0) mbar_arrive(&bars->raw_empty[r]);
      }
    } while (ok && pc.next(p));
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
  float m, l, lift, qscale;  // reference maximum and sum; lift of the products with the values' scales
  bool wild;

  // Chunks [c0, c1) of 8 dimensions of a row of queries into shared memory.  bf16 queries of an 8-bit cache become fp16 after a power of two brings the row's
  // largest value to [1, 2): exact for all that count beside it.
  __device__ __forceinline__ void load_q(uint8_t* q_tile, int row, const void* src, bool ok, int c0, int c1) {
    const float scale = p.scale_log2;
    qscale = fabsf(scale);
    uint4 q[C::D / 8];
#pragma unroll
    for (int c = 0; c < C::D / 8; ++c) q[c] = ok ? static_cast<const uint4*>(src)[c] : make_uint4(0u, 0u, 0u, 0u);
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;  // the sign goes onto the queries: maxima stay maxima
    if (C::kSmall && p.bf16) {
      float top = 0.0f;
#pragma unroll
      for (int c = 0; c < C::D / 8; ++c) {
        const uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[x] << 16)), fabsf(__uint_as_float(w[x] & 0xFFFF0000u))));
      }
      const uint32_t ex = min(max(__float_as_uint(top) & 0x7F800000u, 0x0A000000u), 0x75000000u);
      const float down = __uint_as_float(0x7F000000u - ex);
      qscale *= __uint_as_float(ex);
#pragma unroll
      for (int c = 0; c < C::D / 8; ++c) {
        uint32_t w[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
        for (int x = 0; x < 4; ++x)
          w[x] = pack2<false>(__uint_as_float(w[x] << 16) * down, __uint_as_float(w[x] & 0xFFFF0000u) * down);
        q[c] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
#pragma unroll
    for (int c = 0; c < C::D / 8; ++c)
      if (c >= c0 && c < c1)
        *reinterpret_cast<uint4*>(q_tile + place16(row, c)) =
            make_uint4(q[c].x ^ flip, q[c].y ^ flip, q[c].z ^ flip, q[c].w ^ flip);
  }

  __device__ __forceinline__ void begin() {
    m = -INFINITY, l = 0.0f, lift = kLift;
    wild = false;
  }

  // Scores 32 c .. 32 c + 31 times the keys' own scales, unseen ones -inf.
  template <bool TAIL>
  static __device__ __forceinline__ void scaled(uint32_t (&s)[32], const float* ks, uint32_t seen) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if constexpr (C::TOKEN) {
        const float4 k = *reinterpret_cast<const float4*>(ks + i);
        const float2 a = unpair(mul2(pair(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), pair(k.x, k.y)));
        const float2 b = unpair(mul2(pair(__uint_as_float(s[i + 2]), __uint_as_float(s[i + 3])), pair(k.z, k.w)));
        s[i] = __float_as_uint(a.x), s[i + 1] = __float_as_uint(a.y);
        s[i + 2] = __float_as_uint(b.x), s[i + 3] = __float_as_uint(b.y);
      }
      if (TAIL) {
#pragma unroll
        for (int x = 0; x < 4; ++x)
          if (!((seen >> (i + x)) & 1)) s[i + x] = 0xFF800000u;
      }
    }
  }
  static __device__ __forceinline__ uint32_t pick(const uint32_t (&w)[4], int c) {
    return c < 2 ? (c == 0 ? w[0] : w[1]) : (c == 2 ? w[2] : w[3]);
  }
  static __device__ __forceinline__ float top_of(const uint32_t (&s)[32], float top) {
    float t0 = top, t1 = __uint_as_float(s[1]);
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      t0 = fmaxf(fmaxf(t0, __uint_as_float(s[i])), __uint_as_float(s[i + 2]));
      t1 = fmaxf(fmaxf(t1, __uint_as_float(s[i + 1])), __uint_as_float(s[i + 3]));
    }
    return fmaxf(t0, t1);
  }

  // The row's output sums times `by`.
  __device__ __forceinline__ void scale_outputs(float by) const {
#pragma unroll 1
    for (int c = 0; c < C::D / 16; ++c) {
      uint32_t o[16];
      tmem_ld16(tmem_o + 16 * c, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
      tmem_st16(tmem_o + 16 * c, o);
    }
  }
  // What the first chunks of 32 scores have become, times `by`.
  __device__ __forceinline__ void scale_written(int chunks, float by) const {
    tmem_st_wait();
#pragma unroll 1
    for (int c = 0; c < chunks; ++c) {
      uint32_t o[16];
      tmem_ld16(tmem_s + 16 * c, o);
      tmem_ld_wait();
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&o[i]));
        o[i] = pack2<false>(f.x * by, f.y * by);
      }
      tmem_st16(tmem_s + 16 * c, o);
    }
  }

  // Scores of one key tile to probabilities.  TAIL: some keys are not seen (a bit each in seen).
  template <bool TAIL>
  __device__ __forceinline__ void tile(const uint32_t (&seen)[4], const float* ks, const float* vs, bool first) {
    // The row is read twice, 32 scores at a time, in rolled loops: reading it is cheap, while the code of a whole row
    // unrolled, beside that of the other roles, overran the instruction cache (full trees 308 us; 64 at a time 224 us, 32
    // 220 us; half of the exponentials by a polynomial on the multiply-add pipe 234 us).
    float top = -INFINITY;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      uint32_t s[32];
      tmem_ld32(tmem_s + 32 * c, s);
      tmem_ld_wait();
      scaled<TAIL>(s, ks + 32 * c, TAIL ? pick(seen, c) : kFull);
      top = top_of(s, top);
    }
    top *= qscale;
    // the reference moves when the maximum left it by more than 2^kGrow
    float alpha = 1.0f, by = 1.0f;  // of the sum, of the outputs
    if (top > m + kGrow || m == -INFINITY) {
      const float now = fmaxf(C::TOKEN ? ceilf(top) : top, m);
      if (m != -INFINITY) {
        alpha = exp2_fast(m - now);
        if constexpr (C::TOKEN) {
          lift += now - m;
          if (lift > kLift) by = exp2_fast(kLift - lift), lift = kLift;
        }
      }
      m = now;
    }
    l *= alpha;
    if constexpr (!C::TOKEN) by = alpha;
    if (!first && __any_sync(kFull, by != 1.0f)) scale_outputs(by);
    const float sub = m == -INFINITY ? 0.0f : m - C::kBias;
    const unsigned long long q2 = pair(qscale, qscale), m2 = pair(-sub, -sub);
    float up = C::TOKEN ? exp2_whole(lift) : 1.0f;
    unsigned long long sum0 = pair(0.0f, 0.0f), sum1 = sum0;
#pragma unroll 1
    for (int c = 0; c < 4; ++c) {
      const uint32_t sees = TAIL ? pick(seen, c) : kFull;
      const unsigned long long u2 = pair(up, up);
      unsigned long long part0 = pair(0.0f, 0.0f), part1 = part0;  // sums of the chunk, with scales
      float w[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      uint32_t v[32], out[16];
      tmem_ld32(tmem_s + 32 * c, v);
      tmem_ld_wait();
      scaled<TAIL>(v, ks + 32 * c, sees);
#pragma unroll
      for (int i = 0; i < 32; i += 4) {
        const float2 xa = unpair(fma2(pair(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), q2, m2));
        const float2 xb = unpair(fma2(pair(__uint_as_float(v[i + 2]), __uint_as_float(v[i + 3])), q2, m2));
        float e[4] = {exp2_fast(xa.x), exp2_fast(xa.y), exp2_fast(xb.x), exp2_fast(xb.y)};
        if (TAIL) {
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (!((sees >> (i + x)) & 1)) e[x] = 0.0f;  // a scale of 0 makes -inf NaN
        }
        unsigned long long a = pair(e[0], e[1]), b = pair(e[2], e[3]);
        if constexpr (C::TOKEN)
          part0 = add2(part0, a), part1 = add2(part1, b);
        else
          sum0 = add2(sum0, a), sum1 = add2(sum1, b);
        if constexpr (C::TOKEN) {
          const float4 vv = *reinterpret_cast<const float4*>(vs + 32 * c + i);
          a = mul2(a, pair(vv.x, vv.y)), b = mul2(b, pair(vv.z, vv.w));
          float2 fa = unpair(a), fb = unpair(b);
          if (TAIL) {  // an unseen scale may be anything
            if (!((sees >> i) & 1)) fa.x = 0.0f;
            if (!((sees >> (i + 1)) & 1)) fa.y = 0.0f;
            if (!((sees >> (i + 2)) & 1)) fb.x = 0.0f;
            if (!((sees >> (i + 3)) & 1)) fb.y = 0.0f;
          }
          w[i / 4 % 2] = fmaxf(fmaxf(w[i / 4 % 2], fa.x), fa.y), w[2 + i / 4 % 2] = fmaxf(fmaxf(w[2 + i / 4 % 2], fb.x), fb.y);
          fa = unpair(mul2(pair(fa.x, fa.y), u2)), fb = unpair(mul2(pair(fb.x, fb.y), u2));
          e[0] = fa.x, e[1] = fa.y, e[2] = fb.x, e[3] = fb.y;
        }
        out[i / 2] = pack2<C::BF16>(e[0], e[1]);
        out[i / 2 + 1] = pack2<C::BF16>(e[2], e[3]);
      }
      if constexpr (C::TOKEN) {
        const float wtop = fmaxf(fmaxf(w[0], w[1]), fmaxf(w[2], w[3]));
        if (__any_sync(kFull, wtop * up > kRoom)) {
          // rare: the lift falls for these scores, which are still there, for what was written of the tile, and for the
          // outputs; in all rows at once, where it would fall soon
          const float to = lift_for(wtop);
          if (__any_sync(kFull, to < lift)) {  // an infinite scale lowers the lift once, to its least
            const float by = to < lift ? exp2_fast(to - lift) : 1.0f;
            lift = fminf(lift, to);
            up = exp2_whole(lift);
            scale_written(c, by);
            if (!first) scale_outputs(by);
            --c;
            continue;
          }
        }
        sum0 = add2(sum0, part0), sum1 = add2(sum1, part1);
      }
      // over the scores 16 c .. 16 c + 15, which have been read
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
      if (!((seen[j >> 5] >> (j & 31)) & 1) || !bars->wild[slot][j / C::kRowsPerWarp]) continue;
      const uint32_t* bits = reinterpret_cast<const uint32_t*>(mem + C::kOffWild + slot * C::kWild + j * 32);
      for (int x = 0; x < 8; ++x)
        if ((x & 3) < C::D / 32) mine[x] |= bits[x];
    }
  }
};

// A warp's staged lines (PARTS x 16 bytes of each of its 32 rows, parts exclusive-ored with the row) to the rows' places.
template <int PARTS>
__device__ __forceinline__ void put_lines(const uint8_t* stage, uint8_t* mine, unsigned rows_ok, int lane) {
  constexpr int kPer = 32 / PARTS;  // rows a store of the whole warp takes
  __syncwarp();
  const int part = lane % PARTS;
  uint4 u[PARTS];
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int row = i * kPer + lane / PARTS;
    u[i] = *reinterpret_cast<const uint4*>(stage + row * 128 + ((part ^ (row & 7)) << 4));
  }
#pragma unroll
  for (int i = 0; i < PARTS; ++i) {
    const int row = i * kPer + lane / PARTS;
    uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(kFull, reinterpret_cast<unsigned long long>(mine), row));
    if ((rows_ok >> row) & 1) *reinterpret_cast<uint4*>(to + part * 16) = u[i];
  }
  __syncwarp();
}

template <typename C>
__global__ void __launch_bounds__(C::kThreads, 1) attend_tc_kernel(const __grid_constant__ Params p, int nq) {
  constexpr int D = C::D;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* mem = smem_raw + ((1024 - (raw_addr & 1023)) & 1023);
  const uint32_t base = smem_u32(mem);
  Bars* bars = reinterpret_cast<Bars*>(mem + C::kOffBars);
  __shared__ int red[C::kWarps + 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  volatile int* abort = &bars->abort;

  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (tid == 0) {
    for (int i = 0; i < 4; ++i) {
      mbar_init(&bars->kv_full[i], C::kLoadWarps);
      mbar_init(&bars->kv_empty[i], 1);
      mbar_init(&bars->raw_full[i], 32);
      mbar_init(&bars->raw_empty[i], C::kLoadWarps);
    }
    for (int i = 0; i < kScaleRing; ++i) mbar_init(&bars->sc_full[i], 32);
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
  if (warp == C::kWarps - 4) {
    tmem_alloc(&bars->tmem, kTmemCols);
    tmem_relinquish();
  }
  int total, unit, b0, before, share = 0;
  locate<C::kThreads>(
      p,
      [&](int tot) {
        share = share_of(tot, gridDim.x);
        return static_cast<int>(min(static_cast<long long>(blockIdx.x) * share, 2147483647ll));
      },
      red, total, unit, b0, before);
  const Run run = {b0, before, unit, min(share, total - unit)};

  clear_idle_requests<C::kThreads>(p, D);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = bars->tmem;
  const uint32_t q_addr = base + C::kOffQ;

  Loader<C> ld{p, bars, base, mem, q_addr + C::q_bytes(nq), nq, C::raw_depth(nq), warp - kSoftWarps, lane, abort};
  bool busy = unit < total;
  if (busy) {  // a run may lie in front of its item's first key
    Pieces any;
    busy = any.start(p, run.b0, run.before, run.unit, run.count);
  }
  if (!busy) {
    if (tid == 0) p.joins[blockIdx.x] = make_int4(0, 0, 0, 0);
  } else if (warp >= kSoftWarps && warp < kSoftWarps + C::kLoadWarps) {
    // ------------------------------------------------ loaders
    regs_down<C::kLoadRegs>();
    if constexpr (C::kSmall)
      ld.run_widen(run);
    else
      ld.run_copies(run);
  } else if (warp >= kSoftWarps + C::kLoadWarps) {
    // ------------------------------------------------ products
    if (warp == C::kWarps - 4) {
      // the whole warp walks the tiles, one lane issues: addresses stay in uniform registers
      const bool leader = elect_one();
      Pieces pc;
      pc.start(p, run.b0, run.before, run.unit, run.count);
      const int lead = nq == 1 ? 2 : 1;
      uint32_t kv = 0, piece = 0, pp0 = 0, pp1 = 0;  // tiles taken, pieces, probabilities taken
      const uint32_t q16 = q_addr >> 4, kv16 = base >> 4;
      auto scores = [&](int x, uint32_t s) {  // S_x = Q_x K^T
        const uint32_t q = q16 + (nq == 1 ? 0 : x) * (C::kSlot >> 4), k = kv16 + s * (C::kSlot >> 4);
        const uint32_t d = tmem + x * kTile;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint32_t o = ((kk >> 2) * C::kBlock + (kk & 3) * 32) >> 4;
            mma_ss(d, q + o, k + o, idesc(C::BF16, kTile, false), kk > 0);
          }
          umma_commit(&bars->s_full[x]);
        }
      };
      auto outputs = [&](int x, uint32_t s, bool accumulate) {  // O_x += P_x V
        const uint32_t v = (kv16 + s * (C::kSlot >> 4)) | kValuesLead;
        const uint32_t d = tmem + 2 * kTile + x * D, a = tmem + x * kTile;
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < kTile / 16; ++kk)
            mma_ts(d, a + kk * 8, v + kk * (2048 >> 4), idesc(C::BF16, D, true), accumulate || kk > 0);
        }
      };
      auto give = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
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
          give(&bars->kv_empty[kv % C::kSlots]);
          ++kv;
        }
        for (int j = 0; j < nt && ok; ++j) {
          const uint32_t v = kv++;
          const bool more = j + lead < nt;
          const uint32_t k = more ? kv++ : 0;
          ok = take(v);
          for (int y = 0; y < nq && ok; ++y) {
            const int x = nq == 1 ? j & 1 : y;
            ok = wait(&bars->p_full[x], (x ? pp1 : pp0) & 1, abort);
            x ? ++pp1 : ++pp0;
            if (!ok) break;
            tc_fence_after();
            outputs(x, v % C::kSlots, nq == 1 ? j > 1 : j > 0);
            if (nq == 1 ? j + 2 >= nt : j + 1 == nt) give(&bars->o_done[x]);
            if (y == nq - 1) give(&bars->kv_empty[v % C::kSlots]);
            if (more) {
              if (y == 0) ok = take(k);
              if (!ok) break;
              tc_fence_after();
              scores(x, k % C::kSlots);
              if (y == nq - 1) give(&bars->kv_empty[k % C::kSlots]);
            }
          }
        }
      } while (ok && pc.next(p));
      // every product issued has ended before the block gives its memory back
      give(&bars->drain);
      for (uint32_t n = 0; n < (1u << 22) && !mbar_try_wait(&bars->drain, 0); ++n) {
      }
    } else if (C::kSmall && warp < C::kWarps - 1) {
      ld.run_fetch(warp == C::kWarps - 2, run);
    }
  } else if (warp < kSoftWarps) {
    // ------------------------------------------------ softmax and output
    regs_up<C::kSoftRegs>();
    const int x = warp >> 2, wrow = (warp & 3) * 32 + lane;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    Soft<C> so{p, bars, mem, tmem + lanes + x * kTile, tmem + lanes + 2 * kTile + x * D, abort};
    float4* ml = reinterpret_cast<float4*>(mem + C::kOffMl);  // a row's maximum, sum, 2^-lift, note
    const float* scales = reinterpret_cast<const float*>(mem + C::kOffScale);
    uint32_t kv = 0, t0 = 0, sp = 0, op0 = 0, op1 = 0, meets = 0;
    auto meet = [&]() {  // the two streams' warps
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars->both);
      return wait(&bars->both, meets++ & 1, abort);
    };
    const int lead = nq == 1 ? 2 : 1;
    Pieces pc;
    pc.start(p, run.b0, run.before, run.unit, run.count);
    // the thread's row of a piece, and its queries
    struct Row {
      int h, qi, head, t;
      bool ok, warp_ok;
      const uint8_t* q;
    };
    auto row_of = [&](const Pieces& at) {
      const int rts = row_tiles(p, at.r), rows = at.r.n * p.group;
      Row o;
      o.h = at.item / rts;
      const int row = ((at.item - o.h * rts) << p.rows_log2) + (nq == 1 ? 0 : x * kTile) + wrow;
      o.ok = row < rows;
      o.warp_ok = row - lane < rows;
      o.qi = row / p.group;
      o.head = o.h * p.group + row - o.qi * p.group;
      o.t = at.r.first + o.qi;
      o.q = static_cast<const uint8_t*>(p.q) + (o.t * p.q_tok + o.head * p.q_head) * 2;
      return o;
    };
    bool ok = true, more = true;
    int4 join = make_int4(0, 0, 0, 0);
    Row me = row_of(pc);
    do {
      const Request r = pc.r;
      const int h = me.h, qi = me.qi, head = me.head, t = me.t;
      const bool row_ok = me.ok, warp_ok = me.warp_ok;
      so.begin();
      {
        const int half = D / 16;  // with one row tile the two warps of a row share the copy
        so.load_q(mem + C::kOffQ + (nq == 1 ? 0 : x) * C::kSlot, wrow, me.q, row_ok, nq == 1 ? x * half : 0,
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
          uint32_t seen[4] = {kFull, kFull, kFull, kFull};
          int slot = 0;
          if constexpr (C::TOKEN) {
            const int ring = (t0 + j) & (kScaleRing - 1);
            ok = wait(&bars->sc_full[ring], ((t0 + j) / kScaleRing) & 1, abort);
            if (!ok) break;
            ks = scales + ring * 2 * kTile, vs = ks + kTile;
          }
          if (C::KIND != kInt8 && tail && some_unseen(p, r)) {
            // the value tile's notes are needed: its place in the order of loads
            const uint32_t n = kv + (j + lead < pc.nt ? lead + 2 * j : pc.nt + j);
            slot = n % C::kSlots;
            ok = wait(&bars->kv_full[slot], (n / C::kSlots) & 1, abort);
            if (!ok) break;
          }
          if (tail) {
#pragma unroll
            for (int c = 0; c < 4; ++c) seen[c] = row_ok ? seen32(p, r, t, qi, key0 + 32 * c) : kFull;
            if (C::KIND != kInt8 && some_unseen(p, r)) {
              int any = 0;
#pragma unroll
              for (int i = 0; i < C::kLoadWarps; ++i) any |= bars->wild[slot][i];
              if (any) so.note_wild(seen, slot, x * kTile + wrow);
            }
          }
          if (tail)
            so.template tile<true>(seen, ks, vs, first);
          else
            so.template tile<false>(seen, ks, vs, first);
          first = false;
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars->p_full[x]);
      }
      if (!ok) break;

      // ---- end of the run: outputs, or partial sums where the item goes on in another block
      const bool whole = pc.tile0 == 0 && pc.nt == pc.tiles;
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + (pc.tile0 == 0 ? 1 : 0)) << p.rows_log2;
      const bool two = nq == 1 && pc.nt > 1;  // both streams hold sums of these rows
      if (tid == 0 && !whole && pc.tile0 == 0)
        join = make_int4(parts_of(p, pc, share), pc.r.first, pc.r.n, pc.item);
      kv += 2 * pc.nt;
      t0 += pc.nt;
      more = pc.next(p);
      if (more) {
        me = row_of(pc);
        if (me.ok) {  // the next queries come to L2 while these outputs go out
#pragma unroll
          for (int i = 0; i < D * 2; i += 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(me.q + i));
        }
      }
      if (nq == 1) {
        ok = wait(&bars->o_done[0], op0++ & 1, abort);
        if (two && ok) ok = wait(&bars->o_done[1], op1++ & 1, abort);
      } else {
        ok = wait(&bars->o_done[x], op0++ & 1, abort);
      }
      if (!ok) break;
      tc_fence_after();
      so.l *= exp2_whole(-C::kBias);
      float f0, f1 = 0.0f, m = so.m, l = so.l;
      int c0 = 0, c1 = D / 32;
      uint32_t o0 = so.tmem_o, o1 = so.tmem_o;
      bool noted0 = so.wild, noted1 = false;
      const float vscale = C::TOKEN    ? exp2_whole(-so.lift)
                           : C::kSmall ? p.c.v_scale[h * p.c.v_scale_stride[2]] * exp2_whole(-C::kBias)
                                       : exp2_whole(-C::kBias);
      f0 = vscale;
      if (nq == 1) {
        // each stream's warps write half of the dimensions, joining both streams' sums
        ml[x * kTile + wrow] = make_float4(so.m, so.l, C::TOKEN ? vscale : 0.0f, so.wild ? 1.0f : 0.0f);
        ok = meet();
        if (!ok) break;
        const float4 a = ml[wrow], b = two ? ml[kTile + wrow] : make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
        m = fmaxf(a.x, b.x);
        const float wa = a.x == -INFINITY ? 1.0f : exp2_fast(a.x - m), wb = b.x == -INFINITY ? 1.0f : exp2_fast(b.x - m);
        l = a.y * wa + b.y * wb;
        f0 = wa * (C::TOKEN ? a.z : vscale), f1 = wb * (C::TOKEN ? b.z : vscale);
        noted0 = a.w != 0.0f, noted1 = b.w != 0.0f;
        o0 = tmem + lanes + 2 * kTile, o1 = o0 + D;
        c0 = x * (D / 64), c1 = c0 + D / 64;
      }
      if (whole) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        f0 *= inv, f1 *= inv;
      }
      const int at_row = (nq == 1 ? 0 : x * kTile) + wrow;
      if (warp_ok) {
        // Rows go out through the queries' place (every score is done): 128 bytes of each of the warp's rows at a time,
        // so that a store fills whole lines
        uint8_t* stage = mem + C::kOffQ + (nq == 1 ? 0 : x) * C::kSlot + (nq == 1 ? warp : warp & 3) * 4096;
        uint8_t* mine = whole ? static_cast<uint8_t*>(p.out) + (t * p.o_tok + head * p.o_head) * 2
                              : reinterpret_cast<uint8_t*>(p.part_o + (part + at_row) * D);
        const unsigned rows_ok = __ballot_sync(kFull, row_ok);
        const uint32_t* bits = reinterpret_cast<const uint32_t*>(mem + C::kOffRowWild);
        uint8_t* line = stage + lane * 128;
        auto take = [&](int c, float (&v)[16]) {  // dimensions 16 c .. 16 c + 15 of the thread's row
          uint32_t a[16], b[16];
          tmem_ld16(o0 + 16 * c, a);
          if (two) tmem_ld16(o1 + 16 * c, b);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            v[i] = __uint_as_float(a[i]) * f0;
            if (two) v[i] += __uint_as_float(b[i]) * f1;
          }
          if (C::KIND != kInt8 && (noted0 || noted1)) {
            uint32_t plus = 0, minus = 0;
            const uint32_t* n0 = bits + ((nq == 1 ? 0 : x * kTile) + wrow) * 8 + (c >> 1);
            if (noted0) plus |= n0[0], minus |= n0[4];
            if (noted1) plus |= n0[kTile * 8], minus |= n0[kTile * 8 + 4];
            plus >>= 16 * (c & 1), minus >>= 16 * (c & 1);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              if ((plus >> i) & 1) v[i] += INFINITY;
              if ((minus >> i) & 1) v[i] -= INFINITY;
            }
          }
        };
        // a line is 64 dimensions of 16 bits or 32 sums (half a line of outputs where a stream's warps write 32 dimensions)
        const int steps = whole ? min(4, 2 * (c1 - c0)) : 2;
#pragma unroll 1
        for (int c = 2 * c0; c < 2 * c1; c += steps) {
#pragma unroll 1
          for (int y = 0; y < steps; ++y) {
            float v[16];
            take(c + y, v);
            if (whole) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int z = 0; z < 4; ++z)
                  w[z] = p.bf16 ? pack2<true>(v[8 * i + 2 * z], v[8 * i + 2 * z + 1]) : pack2<false>(v[8 * i + 2 * z], v[8 * i + 2 * z + 1]);
                *reinterpret_cast<uint4*>(line + (((2 * y + i) ^ (lane & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4*>(line + (((4 * y + i) ^ (lane & 7)) << 4)) =
                    make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
            }
          }
          uint8_t* to = mine + c * (whole ? 32 : 64);
          if (whole && steps == 2)
            put_lines<4>(stage, to, rows_ok, lane);
          else
            put_lines<8>(stage, to, rows_ok, lane);
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
    } while (more);
    if (tid == 0) p.joins[blockIdx.x] = join;
  }

  tc_fence_before();
  __syncthreads();
  if (tid == 0 && *abort) atomicOr(&g_attn_error, 2);
  if (warp == C::kWarps - 4) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename C>
orError_t launch(Params& p, int nq, cudaStream_t st, int sms) {
  const void* fn = reinterpret_cast<const void*>(&attend_tc_kernel<C>);
  MCPU_CUDA_TRY(ensure_dynamic_smem(fn, C::smem(nq)), "tree_attention");
  attend_tc_kernel<C><<<sms, C::kThreads, C::smem(nq), st>>>(p, nq);
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
  p.item_cost = 4;  // measured: 0 340 us, 4 216 us, 10 228 us for full trees of all lengths
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
