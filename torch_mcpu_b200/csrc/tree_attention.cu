// Attention over the paged key / value cache for the tokens of a decoding
// step: one token per request, a chain, or a tree of drafted tokens whose
// keys and values are already in the cache behind the request's context.
//
// Mathematics.  Request b has length L (its n new tokens included) and
// context C = L - n.  Its query i sees key j where j < C, or where bit j - C
// of the query's mask words is set (without a mask: j - C <= i).  Per query
// head: s_j = scale * q.k_j, o = sum p_j v_j / sum p_j, p_j = 2^(s_j log2 e -
// m), computed in one pass over the keys with the running maximum m and sum
// kept in fp32; a query that sees nothing (or only scores of -inf) gives
// zeros and lse = -inf.
//
// Bound by HBM while few rows share a key: the rows of one key / value head
// are the request's queries times the query heads that share it.
//
// Work split.  The unit is one tile of TN keys against one tile of MT rows of
// a (request, key / value head).  Units are numbered request by request, and
// each of a fixed grid of blocks takes an equal contiguous run of them, found
// from the lengths on the device: any mix of lengths fills the GPU evenly, and
// a captured graph stays balanced when the lengths change.  A row tile whose
// keys lie in several blocks leaves partial sums in a workspace (at most two
// per block), which a second kernel, launched ahead and waiting on the first
// (programmatic dependent launch), joins in key order: results do not depend
// on timing.
//
// 8-bit caches are multiplied as fp16, which holds e4m3 and int8 values
// exactly: the scales of the keys go onto the scores, those of the values onto
// the probabilities, relative to a reference of each row (kLift).
//
// Which kernel.  Rows that share a key / value head = queries of the longest
// request x query heads per key / value head.  Up to 8 and up to 16 rows: the
// kernels of this file, which read each key once at the cost of one matrix
// instruction a 16-key tile; the 8-row one is the faster where it applies (100
// requests of up to 6000 tokens, 32 / 8 heads of 128: e4m3 148 us against 161,
// int8 151 against 163, bf16 217 against 228).  More rows: tensor memory,
// tree_attention_tc.cu, whose 128-row tile costs the same however many rows
// of it are used, but which is the only one that keeps up with more than 16.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "tree_attention.cuh"

namespace mcpu {
namespace attn {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kRows = 16;  // rows of a tile: a matrix instruction's
constexpr int kJoinThreads = 128;  // 16 rows a block

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <bool BF16>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Values that are not finite, in drafted tokens that some rows do not see: a
// product with a probability of 0 would make them NaN in those rows too.  A
// fragment is split into its finite values (others 0) and two indicators, of
// values that add +inf (or NaN) and of values that add -inf (or NaN); products
// with the rows' view of the keys tell which outputs they reach.
template <bool BF16>
__device__ __forceinline__ void mma_seen(float (&acc)[4], const uint32_t (&p)[4], const uint32_t (&seen)[4], uint32_t b0,
                                         uint32_t b1) {
  uint32_t c0, c1, p0, p1, m0, m1;
  split_finite<BF16>(b0, c0, p0, m0);
  split_finite<BF16>(b1, c1, p1, m1);
  mma<BF16>(acc, p, c0, c1);
  float up[4] = {0.f, 0.f, 0.f, 0.f}, down[4] = {0.f, 0.f, 0.f, 0.f};
  mma<BF16>(up, seen, p0, p1);
  mma<BF16>(down, seen, m0, m1);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (up[x] > 0.0f) acc[x] += INFINITY;
    if (down[x] > 0.0f) acc[x] -= INFINITY;
  }
}

// An 8 x 8 matrix of 16-bit values, transposed across the warp.
__device__ __forceinline__ uint32_t turned(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// mma_seen with the values as the left operand.
template <bool BF16>
__device__ __forceinline__ void mma_seen_values(float (&acc)[4], const uint32_t (&v)[4], const uint32_t (&p)[2],
                                                const uint32_t (&seen)[2]) {
  uint32_t c[4], plus[4], minus[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) split_finite<BF16>(v[x], c[x], plus[x], minus[x]);
  mma<BF16>(acc, c, p[0], p[1]);
  float up[4] = {0.f, 0.f, 0.f, 0.f}, down[4] = {0.f, 0.f, 0.f, 0.f};
  mma<BF16>(up, plus, seen[0], seen[1]);
  mma<BF16>(down, minus, seen[0], seen[1]);
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    if (up[x] > 0.0f) acc[x] += INFINITY;
    if (down[x] > 0.0f) acc[x] -= INFINITY;
  }
}

// ---------------------------------------------------------------- main kernel
template <typename T, int KIND_, int D_, int STAGES_, int ROWS_>
struct Cfg {
  static constexpr int KIND = KIND_, D = D_, STAGES = STAGES_, ROWS = ROWS_;
  static constexpr bool kSmall = KIND != kSame;
  static constexpr bool kBf16 = !kSmall && std::is_same<T, __nv_bfloat16>::value;  // type of the products
  static constexpr float kBias = kSmall || kBf16 ? 0.0f : 15.0f;                   // probabilities are held times 2^kBias
  static constexpr int kRow = D * (kSmall ? 1 : 2);                                // bytes of a key row
  static constexpr int kChunks = kRow / 16;
  static constexpr int KW = kSmall ? 32 : 16;                                      // keys of a warp's step
  static constexpr int TN = kWarps * KW;                                           // keys of a unit
  static constexpr int kHalf = KW * kRow;                                          // keys, or values, of a step
  static constexpr int kStage = 2 * kHalf + (kSmall ? 2 * KW * 4 : 0);
  static constexpr int kScratch = kWarps * ROWS * (ROWS == 8 ? 36 : 32) * 4;  // joining the warps' sums, 32 dimensions a turn
  static constexpr int kSmem = kWarps * STAGES * kStage + kScratch + kWarps * ROWS * 16;
};

// Byte offset of 16-byte chunk c of a row: rows shifted against one another so
// that the 8 rows a matrix load touches lie in different banks.
template <typename C>
__device__ __forceinline__ uint32_t place(int row, int c) {
  if constexpr (C::kChunks >= 8)
    return row * C::kRow + ((c ^ (row & 7)) << 4);
  else
    return row * C::kRow + ((c ^ ((row >> 1) & 3)) << 4);
}

// A lane's key of a warp's step in the pages, found one step ahead of its copy.
struct Place {
  int id, slot;
  bool valid;
};
template <typename C>
__device__ __forceinline__ Place look(const Params& p, const Pieces& w, int tile, int warp, int lane) {
  Place at{0, 0, false};
  const int key = (w.tile0 + tile) * C::TN + warp * C::KW + lane;
  if (lane < C::KW && key < w.r.len) {
    const int page = p.block_log2 >= 0 ? key >> p.block_log2 : key / p.c.block_size;
    at.slot = key - page * p.c.block_size;
    at.id = p.table[w.b * p.table_stride + page];
    at.valid = true;
  }
  return at;
}

// Starts a warp's copies of its keys and values of a unit.
template <typename C>
__device__ __forceinline__ void copy_step(const Params& p, const Pieces& w, const Place& at, uint32_t stage, int lane) {
  constexpr int kPer = C::kSmall ? 16 : 8;  // values in 16 bytes
  constexpr int kAtOnce = 32 / C::kChunks;  // rows a copy of the whole warp takes
  const int h = w.item;                     // up to 16 rows: items are key / value heads
  const int block = static_cast<int>(kv::checked_block(at.id, p.c.num_blocks, &g_attn_error));
  // places in 16-byte units: 32 bits reach 64 GB, which the entry point makes sure of
  const uint32_t ko = static_cast<uint32_t>(block) * static_cast<uint32_t>(p.c.key_stride[0] / kPer) +
                      static_cast<uint32_t>(at.slot) * static_cast<uint32_t>(p.c.key_stride[1] / kPer);
  const uint32_t vo = static_cast<uint32_t>(block) * static_cast<uint32_t>(p.c.value_stride[0] / kPer) +
                      static_cast<uint32_t>(at.slot) * static_cast<uint32_t>(p.c.value_stride[1] / kPer);
  const unsigned valid = __ballot_sync(kFull, at.valid);
  const int c = lane % C::kChunks, r0 = lane / C::kChunks;
  const uint4* kb = static_cast<const uint4*>(p.c.key) + (h * p.c.key_stride[2] / kPer + c);
  const uint4* vb = static_cast<const uint4*>(p.c.value) + (h * p.c.value_stride[2] / kPer + c);
  // shuffles first: copies and shuffles keep their order, and in turn each copy would wait for its shuffle
  constexpr int kSteps = C::KW / kAtOnce;
  uint32_t k[kSteps], v[kSteps];
#pragma unroll
  for (int i = 0; i < kSteps; ++i) k[i] = __shfl_sync(kFull, ko, i * kAtOnce + r0), v[i] = __shfl_sync(kFull, vo, i * kAtOnce + r0);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int row = i * kAtOnce + r0;
    const bool in = (valid >> row) & 1;
    cp_async16(stage + place<C>(row, c), kb + k[i], in);
    cp_async16(stage + C::kHalf + place<C>(row, c), vb + v[i], in);
  }
  if constexpr (C::kSmall) {
    const long long b = block, sl = at.slot;
    cp_async4(stage + 2 * C::kHalf + 4 * lane,
              p.c.k_scale + b * p.c.k_scale_stride[0] + sl * p.c.k_scale_stride[1] + h * p.c.k_scale_stride[2], at.valid);
    cp_async4(stage + 2 * C::kHalf + 4 * (C::KW + lane),
              p.c.v_scale + b * p.c.v_scale_stride[0] + sl * p.c.v_scale_stride[1] + h * p.c.v_scale_stride[2], at.valid);
  }
}

// Whether any of a warp's value rows holds an infinity or a NaN.
template <typename C>
__device__ __forceinline__ bool any_wild(const uint8_t* values) {
  uint32_t wild = 0;
  const uint4* v = reinterpret_cast<const uint4*>(values);  // rows are whole, their order is no matter
#pragma unroll 4
  for (int i = threadIdx.x & 31; i < C::KW * C::kChunks; i += 32) {
    const uint4 u = v[i];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if constexpr (C::KIND == kE4M3)
        wild |= ((w[x] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
      else if constexpr (C::kBf16)
        wild |= __vcmpeq2(w[x] & 0x7F807F80u, 0x7F807F80u);
      else
        wild |= __vcmpeq2(w[x] & 0x7C007C00u, 0x7C007C00u);
    }
  }
  return __any_sync(kFull, wild != 0);
}

// A row's maximum m moves to top: its sum l, the lift that goes with it, and
// by what its output sums are scaled.  With scales (SMALL) those keep to their
// reference, 2^(m - lift), and the lift rises with m up to its limit.
template <bool SMALL>
__device__ __forceinline__ float grow(float top, float& m, float& l, float& lift) {
  const float now = fmaxf(m, SMALL ? ceilf(top) : top);
  const float alpha = now == -INFINITY ? 1.0f : exp2_fast(m - now);
  float by = alpha;
  if constexpr (SMALL) {
    by = 1.0f;
    if (now > m) {
      lift += now - m;
      if (lift > kLift) by = exp2_fast(kLift - lift), lift = kLift;
    }
  }
  l *= alpha;
  m = now;
  return by;
}
// The lift falls where the products' largest, w, would pass the room: by what
// the output sums are scaled.  An infinite scale lowers it once, to its least.
__device__ __forceinline__ float lower(float w, float& lift, float& up) {
  const float to = lift_for(w);
  if (!(w * up > kRoom) || to >= lift) return 1.0f;
  const float by = exp2_fast(to - lift);
  lift = to;
  up = exp2_whole(to);
  return by;
}

// Up to 16 rows.  Each warp runs through its own keys of a block's units with
// copies of its own (a step is 16 keys, or 32 of 8 bits), so nothing in the loop waits for another warp;
// the warps are joined at the end of a piece.  Bound by the chain of
// instructions a warp works through per step (widening 8-bit values, softmax)
// with two blocks of four warps on an SM: 224 registers and two blocks beat
// 168 and three (264 us against 276; 128 requests of all lengths up to 8192, 32 / 8 heads
// of 128, e4m3), two stages equal three, and one block-wide pipeline with
// barriers took 580.
template <typename T, typename C>
__global__ void __maxnreg__(224) attend_kernel(const __grid_constant__ Params p) {
  constexpr int D = C::D, KW = C::KW, KIND = C::KIND;
  constexpr int kNT = KW / 8;   // 8-key tiles of the scores
  constexpr int kDT = D / 8;    // 8-dimension tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int red[kWarps + 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, j4 = lane & 3;
  uint8_t* mine = smem + warp * (C::STAGES * C::kStage);  // the warp's own stages
  const uint32_t stages = smem_u32(mine);
  float* scratch = reinterpret_cast<float*>(smem + kWarps * C::STAGES * C::kStage);
  float4* warp_ml = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(scratch) + C::kScratch);

  // the joining kernel may start; it waits for this one to end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  int total, unit, b0, before;
  int share = 0;
  locate<kThreads>(
      p,
      [&](int tot) {
        share = share_of(tot, gridDim.x);
        return static_cast<int>(min(static_cast<long long>(blockIdx.x) * share, 2147483647ll));
      },
      red, total, unit, b0, before);
  clear_idle_requests<kThreads>(p, D);
  int4 join = make_int4(0, 0, 0, 0);
  Pieces pc, ahead;  // the piece worked on, the one copied
  const bool busy = unit < total && pc.start(p, b0, before, unit, min(share, total - unit));
  if (!busy) {
    if (tid == 0) p.joins[blockIdx.x] = join;
    return;
  }

  // every warp walks the units by itself: its copies, its steps, no barrier until an item ends
  ahead = pc;
  int ahead_tile = 0;
  bool more = true;
  Place next = look<C>(p, ahead, 0, warp, lane);
  auto load = [&](int s) {
    if (more) {
      const Place at = next;
      copy_step<C>(p, ahead, at, stages + s * C::kStage, lane);
      if (++ahead_tile == ahead.nt) {
        ahead_tile = 0;
        more = ahead.next(p);
      }
      if (more) next = look<C>(p, ahead, ahead_tile, warp, lane);
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) load(s);

  uint4* qs = reinterpret_cast<uint4*>(scratch);  // the queries' fragments, the same for every warp
  float qscale[2];
  float acc[kDT][4];
  float m[2], l[2], lift[2];
  int tok[2], qi[2], head[2];
  bool row_ok[2];
  int stage = 0;

  do {
   for (int tile = 0; tile < pc.nt; ++tile) {
    cp_wait<C::STAGES - 2>();
    __syncwarp();
    {
      int s = stage + C::STAGES - 1;
      if (s >= C::STAGES) s -= C::STAGES;
      load(s);
    }

    if (tile == 0) {
      uint32_t qf[D / 16][4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = g + 8 * e;
        row_ok[e] = row < pc.r.n * p.group;
        qi[e] = row / p.group;
        head[e] = pc.item * p.group + row - qi[e] * p.group;
        tok[e] = pc.r.first + qi[e];
        m[e] = -INFINITY;
        l[e] = 0.0f;
        lift[e] = kLift;
        qscale[e] = p.scale_log2;
        const T* q = static_cast<const T*>(p.q) + tok[e] * p.q_tok + head[e] * p.q_head;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t lo = 0, hi = 0;
          if (row_ok[e]) {
            if constexpr (C::kSmall) {  // dimensions 4j..4j+3, the order the 8-bit keys come in
              const uint2 q4 = *reinterpret_cast<const uint2*>(q + kk * 16 + 4 * j4);
              lo = q4.x, hi = q4.y;
            } else {
              lo = *reinterpret_cast<const uint32_t*>(q + kk * 16 + 2 * j4);
              hi = *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8 + 2 * j4);
            }
          }
          qf[kk][e] = lo;
          qf[kk][2 + e] = hi;
        }
        if constexpr (C::kSmall && std::is_same<T, __nv_bfloat16>::value) {
          // bf16 queries as fp16: scaled by a power of two to a maximum in [1, 2), which is exact for all values
          // that count beside the row's largest
          float top = 0.0f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t v = qf[kk][2 * x + e];
              top = fmaxf(top, fmaxf(fabsf(__uint_as_float(v << 16)), fabsf(__uint_as_float(v & 0xFFFF0000u))));
            }
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
          const uint32_t ex = min(max(__float_as_uint(top) & 0x7F800000u, 0x0A000000u), 0x75000000u);
          const float down = __uint_as_float(0x7F000000u - ex);
          qscale[e] *= __uint_as_float(ex);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              const uint32_t v = qf[kk][2 * x + e];
              qf[kk][2 * x + e] =
                  pack2<false>(__uint_as_float(v << 16) * down, __uint_as_float(v & 0xFFFF0000u) * down);
            }
        }
      }
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
        if (kk % kWarps == warp) qs[kk * 32 + lane] = make_uint4(qf[kk][0], qf[kk][1], qf[kk][2], qf[kk][3]);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kDT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][x] = 0.0f;
    }

    // ---- scores of the 16 rows and the warp's KW keys
    const uint32_t ks = stages + stage * C::kStage, vs = ks + C::kHalf;
    const float* scale_k = reinterpret_cast<const float*>(mine + stage * C::kStage + 2 * C::kHalf);
    const float* scale_v = scale_k + KW;
    float s[kNT][4];
#pragma unroll
    for (int i = 0; i < kNT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[i][x] = 0.0f;
    const int mi = lane >> 3, mr = lane & 7;
    if constexpr (!C::kSmall) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const uint4 q4 = qs[kk * 32 + lane];
        const uint32_t qf[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
        for (int n = 0; n < kNT; n += 2) {
          uint32_t b[4];
          ldsm4(b, ks + place<C>(n * 8 + (mi >> 1) * 8 + mr, kk * 2 + (mi & 1)));
          mma<C::kBf16>(s[n], qf, b[0], b[1]);
          mma<C::kBf16>(s[n + 1], qf, b[2], b[3]);
        }
      }
    } else {
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2) {
        const uint4 qa = qs[kk * 32 + lane], qb = qs[(kk + 1) * 32 + lane];
        const uint32_t qf[2][4] = {{qa.x, qa.y, qa.z, qa.w}, {qb.x, qb.y, qb.z, qb.w}};
#pragma unroll
        for (int n = 0; n < kNT; n += 2) {
          uint32_t b[4];
          ldsm4(b, ks + place<C>(n * 8 + (mi >> 1) * 8 + mr, kk + (mi & 1)));
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t w = KIND == kInt8 ? b[x] ^ 0x80808080u : b[x];
            mma<false>(s[n + (x >> 1)], qf[x & 1], widen<KIND, 0, 1>(w), widen<KIND, 2, 3>(w));
          }
        }
      }
    }

    // ---- scale, mask, running maximum
    const int key0 = (pc.tile0 + tile) * C::TN + warp * KW;
    const bool tail = key0 + KW > pc.r.len - pc.r.n;
    uint32_t view[2] = {kFull, kFull};  // the keys a row sees
    if (tail) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
        view[e] = seen32(p, pc.r, row_ok[e] ? tok[e] : pc.r.first, row_ok[e] ? qi[e] : 0, key0) >> (2 * j4);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      float2 sk = make_float2(1.0f, 1.0f);
      if constexpr (C::kSmall) sk = *reinterpret_cast<const float2*>(scale_k + n * 8 + 2 * j4);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[n][x] *= qscale[x >> 1] * ((x & 1) ? sk.y : sk.x);
        if (tail && !((view[x >> 1] >> (8 * n + (x & 1))) & 1)) s[n][x] = -INFINITY;
        top[x >> 1] = fmaxf(top[x >> 1], s[n][x]);
      }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(kFull, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(kFull, top[e], 2));
    }
    if (__any_sync(kFull, top[0] > m[0] || top[1] > m[1])) {
      float by[2];  // of the sums
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        by[e] = grow<C::kSmall>(top[e], m[e], l[e], lift[e]);
      }
      if (!C::kSmall || __any_sync(kFull, by[0] != 1.0f || by[1] != 1.0f)) {
#pragma unroll
        for (int i = 0; i < kDT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][x] *= by[x >> 1];
      }
    }
    const float sub[2] = {m[0] == -INFINITY ? 0.0f : m[0] - C::kBias, m[1] == -INFINITY ? 0.0f : m[1] - C::kBias};
    float wtop[2] = {0.0f, 0.0f};  // products with the values' scales
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[n][x] = exp2_fast(s[n][x] - sub[x >> 1]);
        l[x >> 1] += s[n][x];
      }
      if constexpr (C::kSmall) {
        const float2 sv = *reinterpret_cast<const float2*>(scale_v + n * 8 + 2 * j4);
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          s[n][x] = s[n][x] == 0.0f && tail ? 0.0f : s[n][x] * ((x & 1) ? sv.y : sv.x);
          wtop[x >> 1] = fmaxf(wtop[x >> 1], s[n][x]);
        }
      }
    }
    float up[2] = {1.0f, 1.0f};
    if constexpr (C::kSmall) {
      up[0] = exp2_whole(lift[0]), up[1] = exp2_whole(lift[1]);
      if (__any_sync(kFull, wtop[0] * up[0] > kRoom || wtop[1] * up[1] > kRoom)) {
        float by[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          wtop[e] = fmaxf(wtop[e], __shfl_xor_sync(kFull, wtop[e], 1));
          wtop[e] = fmaxf(wtop[e], __shfl_xor_sync(kFull, wtop[e], 2));
          by[e] = lower(wtop[e], lift[e], up[e]);
        }
#pragma unroll
        for (int i = 0; i < kDT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][x] *= by[x >> 1];
      }
    }
    uint32_t pf[kNT / 2][4];
#pragma unroll
    for (int n = 0; n < kNT; ++n) {
      pf[n >> 1][(n & 1) * 2] = pack2<C::kBf16>(s[n][0] * up[0], s[n][1] * up[0]);
      pf[n >> 1][(n & 1) * 2 + 1] = pack2<C::kBf16>(s[n][2] * up[1], s[n][3] * up[1]);
    }

    // ---- probabilities times values
    if (KIND != kInt8 && tail && some_unseen(p, pc.r) && any_wild<C>(mine + stage * C::kStage + C::kHalf)) {
#pragma unroll
      for (int kk = 0; kk < kNT / 2; ++kk) {
        const int row = kk * 16 + (mi & 1) * 8 + mr;
        uint32_t ones[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t two = view[x & 1] >> (16 * kk + 8 * (x >> 1));
          ones[x] = ((two & 1u) | (two & 2u) << 15) * (C::kBf16 ? 0x3F80u : 0x3C00u);
        }
        if constexpr (!C::kSmall) {
#pragma unroll
          for (int n = 0; n < kDT; n += 2) {
            uint32_t b[4];
            ldsm4t(b, vs + place<C>(row, n + (mi >> 1)));
            mma_seen<C::kBf16>(acc[n], pf[kk], ones, b[0], b[1]);
            mma_seen<C::kBf16>(acc[n + 1], pf[kk], ones, b[2], b[3]);
          }
        } else {
#pragma unroll
          for (int n = 0; n < D / 16; n += 2) {
            uint32_t b[4];
            ldsm4t(b, vs + place<C>(row, n + (mi >> 1)));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              mma_seen<false>(acc[2 * (n + x)], pf[kk], ones, widen<KIND, 0, 2>(b[2 * x]), widen<KIND, 0, 2>(b[2 * x + 1]));
              mma_seen<false>(acc[2 * (n + x) + 1], pf[kk], ones, widen<KIND, 1, 3>(b[2 * x]), widen<KIND, 1, 3>(b[2 * x + 1]));
            }
          }
        }
      }
    } else
#pragma unroll
    for (int kk = 0; kk < kNT / 2; ++kk) {
      const int row = kk * 16 + (mi & 1) * 8 + mr;
      if constexpr (!C::kSmall) {
#pragma unroll
        for (int n = 0; n < kDT; n += 2) {
          uint32_t b[4];
          ldsm4t(b, vs + place<C>(row, n + (mi >> 1)));
          mma<C::kBf16>(acc[n], pf[kk], b[0], b[1]);
          mma<C::kBf16>(acc[n + 1], pf[kk], b[2], b[3]);
        }
      } else {
        // 16 dimensions of a chunk: even ones in one output tile, odd ones in the next
#pragma unroll
        for (int n = 0; n < D / 16; n += 2) {
          uint32_t b[4];
          ldsm4t(b, vs + place<C>(row, n + (mi >> 1)));
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (KIND == kInt8) b[x] ^= 0x80808080u;
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mma<false>(acc[2 * (n + x)], pf[kk], widen<KIND, 0, 2>(b[2 * x]), widen<KIND, 0, 2>(b[2 * x + 1]));
            mma<false>(acc[2 * (n + x) + 1], pf[kk], widen<KIND, 1, 3>(b[2 * x]), widen<KIND, 1, 3>(b[2 * x + 1]));
          }
        }
      }
    }
    __syncwarp();  // the stage is read before the next copies into it
    if (++stage == C::STAGES) stage = 0;
   }

    // ---- end of the piece: join the warps, write
    {
      const bool whole = pc.nt == pc.tiles;
      const int slot = pc.tile0 == 0 ? 1 : 0;
      if (!whole && pc.tile0 == 0) join = make_int4(parts_of(p, pc, share), pc.r.first, pc.r.n, pc.item);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(kFull, l[e], 1);
        l[e] += __shfl_xor_sync(kFull, l[e], 2);
        l[e] *= exp2_whole(-C::kBias);
        if (j4 == 0) warp_ml[warp * kRows + g + 8 * e] = make_float4(m[e], l[e], 0.0f, 0.0f);
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, warp_ml[w * kRows + g + 8 * e].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 o = warp_ml[w * kRows + g + 8 * e];
          ll += o.x == -INFINITY ? o.y : exp2_fast(o.x - mm) * o.y;
        }
        f[e] = m[e] == -INFINITY ? 1.0f : exp2_fast(m[e] - mm);
        m[e] = mm;
        l[e] = ll;
        f[e] *= C::kSmall ? exp2_whole(-lift[e]) : exp2_whole(-C::kBias);
        if (whole) f[e] = ll == 0.0f ? 0.0f : f[e] / ll;
      }
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + slot) * kRows;
      if (warp == 0 && j4 == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = g + 8 * e;
          if (!whole) {
            p.part_ml[(part + row) * 2] = m[e];
            p.part_ml[(part + row) * 2 + 1] = l[e];
          } else if (row_ok[e] && p.lse) {
            p.lse[static_cast<long long>(tok[e]) * p.kv_heads * p.group + head[e]] =
                l[e] == 0.0f ? -INFINITY : (m[e] + log2f(l[e])) * 0.69314718055994531f;
          }
        }
      }
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += 32) {
        if (d0 > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float* to = scratch + (warp * kRows + g + 8 * e) * 32 + i * 8;
            const float(&x)[4] = acc[d0 / 8 + i];
            const float(&y)[4] = acc[d0 / 8 + i + 1];
            if constexpr (C::kSmall) {
              *reinterpret_cast<float4*>(to + 4 * j4) =
                  make_float4(x[2 * e] * f[e], y[2 * e] * f[e], x[2 * e + 1] * f[e], y[2 * e + 1] * f[e]);
            } else {
              *reinterpret_cast<float2*>(to + 2 * j4) = make_float2(x[2 * e] * f[e], x[2 * e + 1] * f[e]);
              *reinterpret_cast<float2*>(to + 8 + 2 * j4) = make_float2(y[2 * e] * f[e], y[2 * e + 1] * f[e]);
            }
          }
        }
        __syncthreads();
        const int row = tid >> 3, d = (tid & 7) * 4;  // 4 dimensions of a row each
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(scratch + (w * kRows + row) * 32 + d);
          sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        if (!whole) {
          *reinterpret_cast<float4*>(p.part_o + (part + row) * D + d0 + d) = sum;
        } else if (row < pc.r.n * p.group) {
          const int i2 = row / p.group;
          T* o = static_cast<T*>(p.out) + (pc.r.first + i2) * p.o_tok + (pc.item * p.group + row - i2 * p.group) * p.o_head;
          constexpr bool kOutBf16 = std::is_same<T, __nv_bfloat16>::value;
          *reinterpret_cast<uint2*>(o + d0 + d) = make_uint2(pack2<kOutBf16>(sum.x, sum.y), pack2<kOutBf16>(sum.z, sum.w));
        }
      }
      __syncthreads();
    }
  } while (pc.next(p));
  cp_wait<0>();
  if (tid == 0) p.joins[blockIdx.x] = join;
}

// The same for up to 8 rows, which is what a single token mostly has, with the
// operands the other way round: 16 keys (or dimensions) against 8 rows, so that
// no half of a matrix instruction, and no half of the exponentials, is spent on
// rows that are not there.  Fewer sums per thread leave room for three blocks on
// an SM (with two: 267 us; with three: 258; 128 requests of all lengths up to
// 8192, 32 / 8 heads of 128, e4m3 with a scale per token, 1.26 GB: 4.9 TB/s).
// Issue slots are 50 % used, DRAM 60 %: what is left is the latency of each
// warp's chain.  A single request of some hundred tokens takes 12 us, 5 of them
// the joining kernel.
template <typename T, typename C>
__global__ void __launch_bounds__(kThreads, 3) attend8_kernel(const __grid_constant__ Params p) {
  constexpr int D = C::D, KW = C::KW, KIND = C::KIND;
  constexpr int kMT = KW / 16;  // 16-key tiles of the scores
  constexpr int kDT = D / 16;   // 16-dimension tiles of the output
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int red[kWarps + 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, j4 = lane & 3;
  uint8_t* mine = smem + warp * (C::STAGES * C::kStage);  // the warp's own stages
  const uint32_t stages = smem_u32(mine);
  float* scratch = reinterpret_cast<float*>(smem + kWarps * C::STAGES * C::kStage);
  float4* warp_ml = reinterpret_cast<float4*>(reinterpret_cast<uint8_t*>(scratch) + C::kScratch);

  // the joining kernel may start; it waits for this one to end before it reads
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  int total, unit, b0, before;
  int share = 0;
  locate<kThreads>(
      p,
      [&](int tot) {
        share = share_of(tot, gridDim.x);
        return static_cast<int>(min(static_cast<long long>(blockIdx.x) * share, 2147483647ll));
      },
      red, total, unit, b0, before);
  clear_idle_requests<kThreads>(p, D);
  int4 join = make_int4(0, 0, 0, 0);
  Pieces pc, ahead;  // the piece worked on, the one copied
  const bool busy = unit < total && pc.start(p, b0, before, unit, min(share, total - unit));
  if (!busy) {
    if (tid == 0) p.joins[blockIdx.x] = join;
    return;
  }

  // every warp walks the units by itself: its copies, its steps, no barrier until an item ends
  ahead = pc;
  int ahead_tile = 0;
  bool more = true;
  Place next = look<C>(p, ahead, 0, warp, lane);
  auto load = [&](int s) {
    if (more) {
      const Place at = next;
      copy_step<C>(p, ahead, at, stages + s * C::kStage, lane);
      if (++ahead_tile == ahead.nt) {
        ahead_tile = 0;
        more = ahead.next(p);
      }
      if (more) next = look<C>(p, ahead, ahead_tile, warp, lane);
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < C::STAGES - 1; ++s) load(s);

  uint32_t qf[D / 16][2];  // the queries, right operand of the first product
  float qscale[2];         // of the thread's two rows, 2 j and 2 j + 1
  float acc[kDT][4];
  float m[2], l[2], lift[2];
  int tok[2], qi[2], head[2];
  bool row_ok[2];
  int stage = 0;

  do {
   for (int tile = 0; tile < pc.nt; ++tile) {
    cp_wait<C::STAGES - 2>();
    __syncwarp();
    {
      int s = stage + C::STAGES - 1;
      if (s >= C::STAGES) s -= C::STAGES;
      load(s);
    }

    if (tile == 0) {
      const int rows = pc.r.n * p.group;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = 2 * j4 + e;
        row_ok[e] = row < rows;
        qi[e] = row / p.group;
        head[e] = pc.item * p.group + row - qi[e] * p.group;
        tok[e] = pc.r.first + qi[e];
        m[e] = -INFINITY;
        l[e] = 0.0f;
        lift[e] = kLift;
      }
      float mine_scale = p.scale_log2;
      {
        const int i = g / p.group;
        const bool ok = g < rows;
        const T* q = static_cast<const T*>(p.q) + (pc.r.first + i) * p.q_tok + (pc.item * p.group + g - i * p.group) * p.q_head;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          qf[kk][0] = qf[kk][1] = 0;
          if (ok) {
            if constexpr (C::kSmall) {  // dimensions 4j..4j+3, the order the 8-bit keys come in
              const uint2 q4 = *reinterpret_cast<const uint2*>(q + kk * 16 + 4 * j4);
              qf[kk][0] = q4.x, qf[kk][1] = q4.y;
            } else {
              qf[kk][0] = *reinterpret_cast<const uint32_t*>(q + kk * 16 + 2 * j4);
              qf[kk][1] = *reinterpret_cast<const uint32_t*>(q + kk * 16 + 8 + 2 * j4);
            }
          }
        }
        if constexpr (C::kSmall && std::is_same<T, __nv_bfloat16>::value) {
          // bf16 queries as fp16: scaled by a power of two to a maximum in [1, 2), which is exact for all values
          // that count beside the row's largest
          float top = 0.0f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              top = fmaxf(top, fmaxf(fabsf(__uint_as_float(qf[kk][x] << 16)), fabsf(__uint_as_float(qf[kk][x] & 0xFFFF0000u))));
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 1));
          top = fmaxf(top, __shfl_xor_sync(kFull, top, 2));
          const uint32_t ex = min(max(__float_as_uint(top) & 0x7F800000u, 0x0A000000u), 0x75000000u);
          const float down = __uint_as_float(0x7F000000u - ex);
          mine_scale *= __uint_as_float(ex);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int x = 0; x < 2; ++x)
              qf[kk][x] = pack2<false>(__uint_as_float(qf[kk][x] << 16) * down, __uint_as_float(qf[kk][x] & 0xFFFF0000u) * down);
        }
      }
      // the scale of row g lies with lanes 4 g ..; this thread's results are of rows 2 j and 2 j + 1
      qscale[0] = __shfl_sync(kFull, mine_scale, 8 * j4);
      qscale[1] = __shfl_sync(kFull, mine_scale, 8 * j4 + 4);
#pragma unroll
      for (int i = 0; i < kDT; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[i][x] = 0.0f;
    }

    // ---- scores of the warp's KW keys (g and g + 8 of each tile of 16) and the rows 2 j, 2 j + 1
    const uint32_t ks = stages + stage * C::kStage, vs = ks + C::kHalf;
    const float* scale_k = reinterpret_cast<const float*>(mine + stage * C::kStage + 2 * C::kHalf);
    const float* scale_v = scale_k + KW;
    float s[kMT][4];
#pragma unroll
    for (int i = 0; i < kMT; ++i)
#pragma unroll
      for (int x = 0; x < 4; ++x) s[i][x] = 0.0f;
    const int mi = lane >> 3, mr = lane & 7;
    if constexpr (!C::kSmall) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int t = 0; t < kMT; ++t) {
          uint32_t a[4];  // keys 0-7, 8-15 of dimensions 0-7, then of 8-15
          ldsm4(a, ks + place<C>(t * 16 + (mi & 1) * 8 + mr, kk * 2 + (mi >> 1)));
          mma<C::kBf16>(s[t], a, qf[kk][0], qf[kk][1]);
        }
    } else {
#pragma unroll
      for (int kk = 0; kk < D / 16; kk += 2)
#pragma unroll
        for (int t = 0; t < kMT; ++t) {
          uint32_t b[4];  // keys 0-7, 8-15 of 16 dimensions, then of the next 16
          ldsm4(b, ks + place<C>(t * 16 + (mi & 1) * 8 + mr, kk + (mi >> 1)));
#pragma unroll
          for (int x = 0; x < 4; ++x)
            if (KIND == kInt8) b[x] ^= 0x80808080u;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t a[4] = {widen<KIND, 0, 1>(b[2 * y]), widen<KIND, 0, 1>(b[2 * y + 1]), widen<KIND, 2, 3>(b[2 * y]),
                                   widen<KIND, 2, 3>(b[2 * y + 1])};
            mma<false>(s[t], a, qf[kk + y][0], qf[kk + y][1]);
          }
        }
    }

    // ---- scale, mask, running maximum: element x of tile t is key 16 t + g + 8 (x >> 1), row 2 j + (x & 1)
    const int key0 = (pc.tile0 + tile) * C::TN + warp * KW;
    const bool tail = key0 + KW > pc.r.len - pc.r.n;
    uint32_t view[2] = {kFull, kFull};  // the keys a row sees
    if (tail) {
#pragma unroll
      for (int e = 0; e < 2; ++e) view[e] = seen32(p, pc.r, row_ok[e] ? tok[e] : pc.r.first, row_ok[e] ? qi[e] : 0, key0);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int t = 0; t < kMT; ++t) {
      float sk[2] = {1.0f, 1.0f};
      if constexpr (C::kSmall) {
#pragma unroll
        for (int y = 0; y < 2; ++y) sk[y] = scale_k[t * 16 + g + 8 * y];
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[t][x] *= qscale[x & 1] * sk[x >> 1];
        if (tail && !((view[x & 1] >> (16 * t + g + 8 * (x >> 1))) & 1)) s[t][x] = -INFINITY;
        top[x & 1] = fmaxf(top[x & 1], s[t][x]);
      }
    }
    // over the keys: lanes of one j
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(kFull, top[0], o));
      top[1] = fmaxf(top[1], __shfl_xor_sync(kFull, top[1], o));
    }
    if (__any_sync(kFull, top[0] > m[0] || top[1] > m[1])) {
      float by[2];  // of the sums
#pragma unroll
      for (int e = 0; e < 2; ++e) by[e] = grow<C::kSmall>(top[e], m[e], l[e], lift[e]);
      if (!C::kSmall || __any_sync(kFull, by[0] != 1.0f || by[1] != 1.0f)) {
#pragma unroll
        for (int i = 0; i < kDT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][x] *= by[x & 1];
      }
    }
    const float sub[2] = {m[0] == -INFINITY ? 0.0f : m[0] - C::kBias, m[1] == -INFINITY ? 0.0f : m[1] - C::kBias};
    float wtop[2] = {0.0f, 0.0f};  // products with the values' scales
#pragma unroll
    for (int t = 0; t < kMT; ++t)
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float sv = 1.0f;
        if constexpr (C::kSmall) sv = scale_v[t * 16 + g + 8 * y];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          float& w = s[t][2 * y + x];
          w = exp2_fast(w - sub[x]);
          l[x] += w;
          if constexpr (C::kSmall) {
            w = w == 0.0f && tail ? 0.0f : w * sv;
            wtop[x] = fmaxf(wtop[x], w);
          }
        }
      }
    float up[2] = {1.0f, 1.0f};
    if constexpr (C::kSmall) {
      up[0] = exp2_whole(lift[0]), up[1] = exp2_whole(lift[1]);
      if (__any_sync(kFull, wtop[0] * up[0] > kRoom || wtop[1] * up[1] > kRoom)) {
        float by[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) wtop[e] = fmaxf(wtop[e], __shfl_xor_sync(kFull, wtop[e], o));
          by[e] = lower(wtop[e], lift[e], up[e]);
        }
#pragma unroll
        for (int i = 0; i < kDT; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) acc[i][x] *= by[x & 1];
      }
    }
    // probabilities, keys x rows, turned into the right operand (rows x keys) 8 x 8 at a time
    uint32_t pf[kMT][2];
#pragma unroll
    for (int t = 0; t < kMT; ++t)
#pragma unroll
      for (int y = 0; y < 2; ++y) pf[t][y] = turned(pack2<C::kBf16>(s[t][2 * y] * up[0], s[t][2 * y + 1] * up[1]));

    // ---- values (16 dimensions x 16 keys) times probabilities
    auto products = [&](auto some_wild) {
      uint32_t ones[kMT][2];
      if constexpr (some_wild.value) {
#pragma unroll
        for (int t = 0; t < kMT; ++t)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int key = 16 * t + g + 8 * y;
            ones[t][y] = turned((((view[0] >> key) & 1u) | ((view[1] >> key) & 1u) << 16) * (C::kBf16 ? 0x3F80u : 0x3C00u));
          }
      }
#pragma unroll
      for (int t = 0; t < kMT; ++t)
#pragma unroll
        for (int d = 0; d < kDT; d += C::kSmall ? 2 : 1) {
          uint32_t a[2][4];
          if constexpr (!C::kSmall) {  // keys 0-7 of dimensions 0-7, 8-15, then keys 8-15
            ldsm4t(a[0], vs + place<C>(t * 16 + (mi >> 1) * 8 + mr, 2 * d + (mi & 1)));
          } else {
            uint32_t b[4];  // keys 0-7, 8-15 of 16 dimensions, then of the next 16: even dimensions first, odd ones behind
            ldsm4t(b, vs + place<C>(t * 16 + (mi & 1) * 8 + mr, d + (mi >> 1)));
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t lo = KIND == kInt8 ? b[2 * y] ^ 0x80808080u : b[2 * y];
              const uint32_t hi = KIND == kInt8 ? b[2 * y + 1] ^ 0x80808080u : b[2 * y + 1];
              a[y][0] = widen<KIND, 0, 2>(lo), a[y][1] = widen<KIND, 1, 3>(lo);
              a[y][2] = widen<KIND, 0, 2>(hi), a[y][3] = widen<KIND, 1, 3>(hi);
            }
          }
#pragma unroll
          for (int y = 0; y < (C::kSmall ? 2 : 1); ++y) {
            if constexpr (some_wild.value)
              mma_seen_values<C::kBf16>(acc[d + y], a[y], pf[t], ones[t]);
            else
              mma<C::kBf16>(acc[d + y], a[y], pf[t][0], pf[t][1]);
          }
        }
    };
    // one branch for all products: the rare ones stay out of the way of the instruction fetch
    if (KIND != kInt8 && tail && some_unseen(p, pc.r) && any_wild<C>(mine + stage * C::kStage + C::kHalf))
      products(std::true_type());
    else
      products(std::false_type());
    __syncwarp();  // the stage is read before the next copies into it
    if (++stage == C::STAGES) stage = 0;
   }

    // ---- end of the piece: join the warps, write
    {
      const bool whole = pc.nt == pc.tiles;
      const int slot = pc.tile0 == 0 ? 1 : 0;
      if (!whole && pc.tile0 == 0) join = make_int4(parts_of(p, pc, share), pc.r.first, pc.r.n, pc.item);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[e] += __shfl_xor_sync(kFull, l[e], o);
        l[e] *= exp2_whole(-C::kBias);
        if (g == 0) warp_ml[warp * 8 + 2 * j4 + e] = make_float4(m[e], l[e], 0.0f, 0.0f);
      }
      __syncthreads();
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float mm = -INFINITY, ll = 0.0f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mm = fmaxf(mm, warp_ml[w * 8 + 2 * j4 + e].x);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 o = warp_ml[w * 8 + 2 * j4 + e];
          ll += o.x == -INFINITY ? o.y : exp2_fast(o.x - mm) * o.y;
        }
        f[e] = m[e] == -INFINITY ? 1.0f : exp2_fast(m[e] - mm);
        m[e] = mm;
        l[e] = ll;
        f[e] *= C::kSmall ? exp2_whole(-lift[e]) : exp2_whole(-C::kBias);
        if (whole) f[e] = ll == 0.0f ? 0.0f : f[e] / ll;
      }
      const long long part = (static_cast<long long>(blockIdx.x) * 2 + slot) * 8;
      if (warp == 0 && g == 0) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int row = 2 * j4 + e;
          if (!whole) {
            p.part_ml[(part + row) * 2] = m[e];
            p.part_ml[(part + row) * 2 + 1] = l[e];
          } else if (row_ok[e] && p.lse) {
            p.lse[static_cast<long long>(tok[e]) * p.kv_heads * p.group + head[e]] =
                l[e] == 0.0f ? -INFINITY : (m[e] + log2f(l[e])) * 0.69314718055994531f;
          }
        }
      }
#pragma unroll
      for (int d0 = 0; d0 < D; d0 += 32) {
        if (d0 > 0) __syncthreads();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float(&x)[4] = acc[d0 / 16 + i];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float* to = scratch + (warp * 8 + 2 * j4 + e) * 36 + i * 16;  // 36: rows apart in the banks
            if constexpr (C::kSmall) {
              *reinterpret_cast<float2*>(to + 2 * g) = make_float2(x[e] * f[e], x[2 + e] * f[e]);
            } else {
              to[g] = x[e] * f[e];
              to[g + 8] = x[2 + e] * f[e];
            }
          }
        }
        __syncthreads();
        const int row = tid >> 3, d = (tid & 7) * 4;  // 4 dimensions of a row each
        if (row >= 8) continue;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(scratch + (w * 8 + row) * 36 + d);
          sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        if (!whole) {
          *reinterpret_cast<float4*>(p.part_o + (part + row) * D + d0 + d) = sum;
        } else if (row < pc.r.n * p.group) {
          const int i2 = row / p.group;
          T* o = static_cast<T*>(p.out) + (pc.r.first + i2) * p.o_tok + (pc.item * p.group + row - i2 * p.group) * p.o_head;
          constexpr bool kOutBf16 = std::is_same<T, __nv_bfloat16>::value;
          *reinterpret_cast<uint2*>(o + d0 + d) = make_uint2(pack2<kOutBf16>(sum.x, sum.y), pack2<kOutBf16>(sum.z, sum.w));
        }
      }
      __syncthreads();
    }
  } while (pc.next(p));
  cp_wait<0>();
  if (tid == 0) p.joins[blockIdx.x] = join;
}

// ---------------------------------------------------------------- joining kernel
// Block c joins the one row tile that begins in the main kernel's block c and
// goes on behind it: its parts lie in slot 1 of c and slot 0 of the next
// blocks.  A block takes 16 of its rows, four to a warp; where there are fewer
// rows, several warps share the parts of four and join theirs at the end, so
// that a long sequence with few rows is not a chain of loads.  Bound by latency
// (the wait on the main kernel, then two dependent loads): about 5 us.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads, 8) join_kernel(const __grid_constant__ Params p) {
  constexpr int kJoinWarps = kJoinThreads / 32;
  __shared__ float4 sums[kJoinWarps][4][D / 4];
  __shared__ float2 sums_ml[kJoinWarps][4];
  const int c = blockIdx.x, rows = 1 << p.rows_log2;
  // every block waits, also those with nothing to join: what follows on the
  // stream must not overtake the main kernel
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 join = p.joins[c];
  const int parts = join.x, item = join.w;
  if (parts == 0) return;
  const Request r = {join.y, join.z, 0};
  const int rts = row_tiles(p, r);
  const int h = item / rts, rt = item - h * rts;
  const int first = rt * rows + blockIdx.y * (kJoinThreads / 8), left = min(rows - static_cast<int>(blockIdx.y) * (kJoinThreads / 8), r.n * p.group - first);
  if (left <= 0) return;
  int groups = 1;  // of four rows, a power of two up to the block's warps
  while (groups * 4 < left && groups < kJoinWarps) groups *= 2;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int mine = warp % groups, k0 = warp / groups, step = kJoinWarps / groups;
  // D / 4 lanes hold a row, 4 dimensions each; loads of four rows and two parts at a time overlap
  constexpr int kLanes = D / 4, kPerWarp = 32 / kLanes, kAtOnce = 4 / kPerWarp;
  const int d = lane % kLanes, row0 = mine * 4 + lane / kLanes;
  float m[kAtOnce], l[kAtOnce];
  float4 o[kAtOnce];
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) m[i] = -INFINITY, l[i] = 0.0f, o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [](float& m0, float& l0, float4& o0, float2 ml, const float4& v) {
    const float now = fmaxf(m0, ml.x);
    const float a = m0 == -INFINITY ? 1.0f : exp2_fast(m0 - now);  // nothing yet: sums of 0 (or NaN)
    const float w = ml.x == -INFINITY ? 1.0f : exp2_fast(ml.x - now);
    l0 = l0 * a + ml.y * w;
    o0.x = o0.x * a + v.x * w, o0.y = o0.y * a + v.y * w, o0.z = o0.z * a + v.z * w, o0.w = o0.w * a + v.w * w;
    m0 = now;
  };
  for (int k = k0; k < parts; k += 2 * step) {
    float2 ml[2][kAtOnce];
    float4 v[2][kAtOnce];
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int kk = k + y * step, row = row0 + i * kPerWarp;
        const bool in = row < left && kk < parts;
        const long long at = ((static_cast<long long>(c) + kk) * 2 + (kk == 0 ? 1 : 0)) * rows + blockIdx.y * (kJoinThreads / 8) + row;
        ml[y][i] = in ? *reinterpret_cast<const float2*>(p.part_ml + at * 2) : make_float2(-INFINITY, 0.0f);
        v[y][i] = in ? reinterpret_cast<const float4*>(p.part_o + at * D)[d] : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
    for (int y = 0; y < 2; ++y)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) add(m[i], l[i], o[i], ml[y][i], v[y][i]);
  }
  if (step > 1) {  // the warps that shared the rows, in the order of the first parts they took
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      sums[warp][lane / kLanes + i * kPerWarp][d] = o[i];
      if (d == 0) sums_ml[warp][lane / kLanes + i * kPerWarp] = make_float2(m[i], l[i]);
    }
    __syncthreads();
    if (k0 > 0) return;
    for (int w = 1; w < step; ++w)
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int y = lane / kLanes + i * kPerWarp;
        add(m[i], l[i], o[i], sums_ml[mine + w * groups][y], sums[mine + w * groups][y][d]);
      }
  }
#pragma unroll
  for (int i = 0; i < kAtOnce; ++i) {
    if (row0 + i * kPerWarp >= left) break;
    const int rr = first + row0 + i * kPerWarp;
    const float f = l[i] == 0.0f ? 0.0f : 1.0f / l[i];
    const int q = rr / p.group, head = h * p.group + rr - q * p.group;
    const long long t = r.first + q;
    T* out = static_cast<T*>(p.out) + t * p.o_tok + head * p.o_head + 4 * d;
    constexpr bool kOutBf16 = std::is_same<T, __nv_bfloat16>::value;
    *reinterpret_cast<uint2*>(out) =
        make_uint2(pack2<kOutBf16>(o[i].x * f, o[i].y * f), pack2<kOutBf16>(o[i].z * f, o[i].w * f));
    if (p.lse && d == 0)
      p.lse[t * p.kv_heads * p.group + head] = l[i] == 0.0f ? -INFINITY : (m[i] + log2f(l[i])) * 0.69314718055994531f;
  }
}

// ---------------------------------------------------------------- host side
struct Device {
  int sms;
};

orError_t device(Device* d) {
  int dev = 0;
  MCPU_CUDA_TRY(cudaGetDevice(&dev), "tree_attention");
  MCPU_CUDA_TRY(cudaDeviceGetAttribute(&d->sms, cudaDevAttrMultiProcessorCount, dev), "tree_attention");
  return orSuccess;
}

constexpr int kMaxResident = 4;  // blocks per SM the workspace is sized for

// Rows of partial sums a call may leave: two parts for every block.
unsigned long long part_rows(int sms, long long rows) {
  if (rows <= kRows) return 2ull * kMaxResident * sms * kRows;
  return 2ull * sms * (rows <= 128 ? 128 : 256);
}

template <typename T, typename C>
orError_t launch(Params& p, cudaStream_t st, int sms, int* grid) {
  void (*kernel)(Params);
  if constexpr (C::ROWS == 8)
    kernel = &attend8_kernel<T, C>;
  else
    kernel = &attend_kernel<T, C>;
  const void* fn = reinterpret_cast<const void*>(kernel);
  MCPU_CUDA_TRY(ensure_dynamic_smem(fn, C::kSmem), "tree_attention");
  static std::atomic<int> known{0};  // blocks per SM: a property of the kernel, asked once
  int resident = known.load(std::memory_order_relaxed);
  if (resident == 0) {
    MCPU_CUDA_TRY(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&resident, kernel, kThreads, C::kSmem),
                  "tree_attention");
    resident = std::max(1, std::min(resident, kMaxResident));
    known.store(resident, std::memory_order_relaxed);
  }
  *grid = resident * sms;
  p.rows_log2 = C::ROWS == 8 ? 3 : 4;
  p.keys_log2 = C::TN == 64 ? 6 : 7;
  p.item_cost = 2;  // measured: 0 293 us, 2 276 us, 5 275 us for a decoding batch of all lengths
  kernel<<<*grid, kThreads, C::kSmem, st>>>(p);
  return from_cuda(cudaGetLastError(), "tree_attention launch");
}

template <typename T, int D, int ROWS>
orError_t launch_few(Params& p, int dtype, cudaStream_t st, int sms, int* grid) {
  constexpr int kStages = 2;
  if (p.c.dtype == dtype) return launch<T, Cfg<T, kSame, D, kStages, ROWS>>(p, st, sms, grid);
  if (p.c.dtype == MCPU_INT8) return launch<T, Cfg<T, kInt8, D, kStages, ROWS>>(p, st, sms, grid);
  return launch<T, Cfg<T, kE4M3, D, kStages, ROWS>>(p, st, sms, grid);
}

template <typename T, int D>
orError_t run(Params& p, int dtype, long long rows, void* ws, cudaStream_t st, int sms) {
  p.part_o = static_cast<float*>(ws);
  p.part_ml = p.part_o + part_rows(sms, rows) * D;
  p.joins = reinterpret_cast<int4*>(p.part_ml + part_rows(sms, rows) * 2);
  int grid = 0;
  const orError_t e = rows <= 8      ? launch_few<T, D, 8>(p, dtype, st, sms, &grid)
                       : rows <= kRows ? launch_few<T, D, kRows>(p, dtype, st, sms, &grid)
                                       : launch_tc(p, D, rows, st, sms, &grid);
  if (e != orSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, std::max(1, (1 << p.rows_log2) / (kJoinThreads / 8)));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return from_cuda(cudaLaunchKernelEx(&cfg, join_kernel<T, D>, p), "tree_attention join launch");
}

}  // namespace attn

orError_t attn_read_error(int* flag, bool reset) {
  int z = 0;
  int tc = 0;
  const orError_t e = attn::tc_read_error(&tc, reset);
  if (e != orSuccess) return e;
  MCPU_CUDA_TRY(cudaMemcpyFromSymbol(flag, attn::g_attn_error, sizeof(int)), "mcpu_device_error");
  if (reset) MCPU_CUDA_TRY(cudaMemcpyToSymbol(attn::g_attn_error, &z, sizeof(int)), "mcpu_device_error");
  *flag |= tc;
  return orSuccess;
}

}  // namespace mcpu

using namespace mcpu;

extern "C" orError_t mcpu_tree_attention_workspace_bytes(int64_t max_query_len, int num_heads, int num_kv_heads,
                                                         int head_size, uint64_t* bytes) {
  const char* op = "tree_attention";
  MCPU_ARG_CHECK(bytes != nullptr, "%s: bytes is NULL", op);
  MCPU_ARG_CHECK(num_kv_heads > 0 && num_heads > 0 && num_heads % num_kv_heads == 0,
                 "%s: num_heads (%d) must be a multiple of num_kv_heads (%d)", op, num_heads, num_kv_heads);
  MCPU_ARG_CHECK(head_size == 64 || head_size == 128, "%s: head_size %d is not 64 or 128", op, head_size);
  MCPU_ARG_CHECK(max_query_len > 0 && max_query_len <= MCPU_TREE_MAX_QUERIES, "%s: max_query_len must be in 1..%d", op,
                 MCPU_TREE_MAX_QUERIES);
  attn::Device d{};
  if (attn::device(&d) != orSuccess) d.sms = 148;
  *bytes = attn::part_rows(d.sms, max_query_len * (num_heads / num_kv_heads)) * (head_size + 2) * 4 +
           16ull * attn::kMaxResident * d.sms;
  return orSuccess;
}

extern "C" orError_t mcpu_tree_attention(
    const void* query, int64_t query_token_stride, int64_t query_head_stride, int64_t num_tokens, int num_heads,
    void* out, int64_t out_token_stride, int64_t out_head_stride, float* lse, int dtype, const mcpuKvCache* cache,
    const int32_t* block_table, int64_t table_stride, int64_t table_width, int64_t batch, const int32_t* seq_lens,
    const int32_t* cu_query_lens, int64_t max_query_len, const int64_t* tree_mask, int64_t mask_stride,
    int64_t mask_words, float scale, void* workspace, uint64_t workspace_bytes, orStream_t stream) {
  const char* op = "tree_attention";
  orError_t e = kv::check_cache(cache, dtype, op);
  if (e != orSuccess) return e;
  const int D = cache->head_size, kv = cache->kv_heads;
  uint64_t need = 0;
  MCPU_ARG_CHECK(num_tokens >= 0 && num_tokens < (1LL << 31) && batch >= 0 && batch < (1LL << 30) && table_width >= 0 &&
                     table_width < (1LL << 31) && table_stride >= table_width,
                 "%s: bad sizes", op);
  if (num_tokens == 0 || batch == 0) return orSuccess;
  e = mcpu_tree_attention_workspace_bytes(max_query_len, num_heads, kv, D, &need);
  if (e != orSuccess) return e;
  MCPU_ARG_CHECK(cache->num_blocks > 0, "%s: the cache has no blocks", op);
  MCPU_ARG_CHECK(query && out && block_table && seq_lens && cu_query_lens && workspace, "%s: NULL pointer", op);
  MCPU_ARG_CHECK(workspace_bytes >= need, "%s: workspace holds %llu bytes, %llu needed", op,
                 static_cast<unsigned long long>(workspace_bytes), static_cast<unsigned long long>(need));
  MCPU_ARG_CHECK(((reinterpret_cast<uintptr_t>(query) | reinterpret_cast<uintptr_t>(out) |
                   reinterpret_cast<uintptr_t>(workspace)) & 15) == 0 &&
                     (query_token_stride | query_head_stride | out_token_stride | out_head_stride) % 8 == 0,
                 "%s: query, out and workspace must be 16-byte aligned, with strides of whole 16 bytes", op);
  MCPU_ARG_CHECK(tree_mask == nullptr || (mask_words > 0 && mask_words <= (1 << 20) && mask_stride >= mask_words &&
                                          64 * mask_words >= max_query_len),
                 "%s: tree_mask has %lld words of 64 tokens, max_query_len is %lld", op,
                 static_cast<long long>(mask_words), static_cast<long long>(max_query_len));
  for (int i = 0; i < 2; ++i) {  // places in 16-byte units are 32-bit
    const int64_t* st = i == 0 ? cache->key_stride : cache->value_stride;
    const double span = (static_cast<double>(cache->num_blocks - 1) * st[0] + static_cast<double>(cache->block_size - 1) * st[1]) *
                        (cache->dtype == dtype ? 2 : 1);
    MCPU_ARG_CHECK(span < 64.0 * 1073741824.0, "%s: a cache tensor spans at most 64 GB", op);
  }
  // unit numbers are 32-bit: the longest requests the table can hold, with tiles of 64 keys and 16 rows
  const double room = static_cast<double>(table_width) * cache->block_size;
  const double rows = static_cast<double>(max_query_len) * (num_heads / kv);
  MCPU_ARG_CHECK(room < 2147483000.0 && batch * kv * (rows / 16 + 1) * (room / 64 + 9) < 2147483000.0,
                 "%s: batch, heads and block_table are too large for one call", op);
  attn::Device d{};
  e = attn::device(&d);
  if (e != orSuccess) return e;
  attn::Params p{};
  p.q = query, p.q_tok = query_token_stride, p.q_head = query_head_stride;
  p.out = out, p.o_tok = out_token_stride, p.o_head = out_head_stride;
  p.lse = lse;
  p.c = *cache;
  p.table = block_table, p.table_stride = table_stride, p.table_width = static_cast<int>(table_width);
  p.block_log2 = -1;
  for (int i = 0; i < 31; ++i)
    if (cache->block_size == (1 << i)) p.block_log2 = i;
  p.seq_lens = seq_lens, p.cu = cu_query_lens;
  p.mask = reinterpret_cast<const long long*>(tree_mask), p.mask_stride = mask_stride;
  p.mask_words = static_cast<int>(std::min<int64_t>(mask_words, 1 << 20));
  p.batch = static_cast<int>(batch), p.tokens = static_cast<int>(num_tokens);
  p.kv_heads = kv, p.group = num_heads / kv, p.most = static_cast<int>(max_query_len);
  p.scale_log2 = scale * 1.4426950408889634f;
  const long long rows_max = max_query_len * p.group;
  cudaStream_t st = as_cuda(stream);
  p.bf16 = dtype == MCPU_BFLOAT16;
  if (dtype == MCPU_FLOAT16)
    return D == 64 ? attn::run<__half, 64>(p, dtype, rows_max, workspace, st, d.sms)
                   : attn::run<__half, 128>(p, dtype, rows_max, workspace, st, d.sms);
  return D == 64 ? attn::run<__nv_bfloat16, 64>(p, dtype, rows_max, workspace, st, d.sms)
                 : attn::run<__nv_bfloat16, 128>(p, dtype, rows_max, workspace, st, d.sms);
}
