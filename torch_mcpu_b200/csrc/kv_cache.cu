// Rotary positions and the paged key / value cache of the serving path:
//   rotary_embedding           x' = rotation of x by its position's angles, in
//                              place, query and key in one launch
//   reshape_and_cache          key and value rows into their slots of the
//                              cache, quantised to 8 bits as they are written
//   rotary_reshape_and_cache   both in one launch: query rotated in place,
//                              rotated key and value written to the cache
//   gather_cache               the tokens of each sequence read back from
//                              their pages into contiguous rows, dequantised
//
// Mathematics.  A pair (a, b) of a head with angle t becomes
// (a cos t - b sin t, b cos t + a sin t); the pair is (x[i], x[i + R/2]) in
// the half layout, (x[2i], x[2i+1]) in the interleaved one, for the first R
// dimensions.  Quantised rows hold q = rn(x / s) with one fp32 scale s per row
// (token, head): s = rn(max|x| / 448) for e4m3, rn(max|x| / 127) for int8, or
// a scale given per head or for the whole cache.
//
// Results of 8 and 16 bits are the 64-bit values rounded once.  A quantised
// value that lands on the wrong side of a rounding border is a whole 8-bit step
// off, and a key that is rounded the wrong way before it is quantised moves its
// row's scale and with it the whole row; so the fast fp32 results are used only
// where they lie further from a border than their error bound, and the others
// are computed again in 64 bits and rounded once (through an odd fp32, which
// lies on no border of the shorter types): of the rotated values about 2^-13 in
// bf16 and 2^-10 in fp16; of the quantised ones 2^-16 in e4m3, with all below
// 2^-6 of the scale (zeros among them), and 2^-13.6 in int8.  Rotated fp32
// tensors, which no cache holds, stay in fp32: fma(a, c, -rn(b s)), off by at
// most 2^-24 (|b s| + |result|); in 64 bits they took 164 us instead of 118
// (16111 tokens x 40 heads of 128).
//
// Bound by HBM: one read and one write per value.  A thread owns 16 values of
// a row (both halves of 8 pairs), loaded and stored 8 at a time, and keeps its
// 8 cosines and sines in registers over the heads of a token; a row is held by
// D/16 lanes, so its maximum is three shuffles at D = 128.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "kv_cache.cuh"

namespace mcpu {
namespace kv {

__device__ int g_kv_error = 0;

constexpr int kThreads = 128;
constexpr unsigned kFull = 0xFFFFFFFFu;

enum Cache { kNoCache = 0, kSame = 1, kE4M3 = 2, kInt8 = 3 };

struct Rows {
  const void* in;  // [tokens, heads, D]
  long long tok_stride, head_stride;
};

struct Params {
  long long tokens;
  int q_heads, kv_heads, D, R, neox;
  int turn_log2, lanes_log2;  // lanes of a row: where only its rotated part counts, and of a whole row
  int turn_blocks;            // blockIdx.y below it: rows that are rotated in place; from it on: rows for the cache
  int turn_rows, cache_rows;  // rows of a token that a block takes
  Rows q, k, v;  // q (and k without a cache) is written in place
  const long long* positions;
  const float* table;  // [max_position, R]: R/2 cosines, R/2 sines
  long long max_position;
  const long long* slots;
  mcpuKvCache c;
};

// ---------------------------------------------------------------- conversions
template <typename T>
__device__ __forceinline__ float up(T v);
template <>
__device__ __forceinline__ float up<float>(float v) { return v; }
template <>
__device__ __forceinline__ float up<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float up<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T down(float v);
template <>
__device__ __forceinline__ float down<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half down<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 down<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// 64 bits to fp32, inexact values to the neighbour whose last bit is set: a
// second rounding to a type with two bits less or fewer is then the rounding
// of the 64-bit value.
__device__ __forceinline__ float to_odd(double v) {
  float f = __double2float_rz(v);
  if (static_cast<double>(f) != v && f == f) f = __uint_as_float(__float_as_uint(f) | 1u);
  return f;
}

// a*c - b*s rounded once to T (as its fp32 value), in 64 bits; out of line: the
// common path keeps its registers.
template <typename T>
__device__ __noinline__ float rotate_exact(float a, float c, float b, float s) {
  const double bs = static_cast<double>(b) * static_cast<double>(s);
  return up<T>(down<T>(to_odd(static_cast<double>(a) * static_cast<double>(c) - bs)));
}

// Distance of r to the border between two neighbours of T that its bits lie
// next to: the dropped bits replaced by 100..0.
template <typename T>
__device__ __forceinline__ float to_border(float r) {
  constexpr uint32_t kDropped = std::is_same<T, __nv_bfloat16>::value ? 0xFFFFu : 0x1FFFu;
  return fabsf(r - __uint_as_float((__float_as_uint(r) & ~kDropped) | ((kDropped + 1) >> 1)));
}

// One pair in fp32, and how far its results lie from a border of T beyond
// their error (<= 0: the rounding is not sure).  amp: 2^-23 times the largest
// |cos|, |sin|; the error of a result is at most 2^-24 (|b s| + |result|) <=
// amp (|a| + |b|).
template <typename T>
struct Pair {
  float a, b, da, db, e;
  __device__ __forceinline__ Pair(float x, float y, float c, float s, float amp) {
    a = __fmaf_rn(x, c, -__fmul_rn(y, s));
    b = __fmaf_rn(y, c, __fmul_rn(x, s));
    if constexpr (sizeof(T) == 2) {
      e = __fmaf_rn(fabsf(x) + fabsf(y), amp, 1e-35f);  // 1e-35: products that lost bits to underflow
      da = to_border<T>(a), db = to_border<T>(b);
      if constexpr (std::is_same<T, __half>::value) {  // subnormal results have their borders elsewhere
        if (fabsf(a) < 6.2e-5f) da = 0.0f;
        if (fabsf(b) < 6.2e-5f) db = 0.0f;
      }
    }
  }
  __device__ __forceinline__ bool unsure() const { return sizeof(T) == 2 && (da <= e || db <= e); }
};
// Whether any of four pairs is unsure: a chain of comparisons into one
// predicate, which the compiler does not make of the plain expression.
template <typename T>
__device__ __forceinline__ uint32_t any_unsure(const Pair<T>& p0, const Pair<T>& p1, const Pair<T>& p2, const Pair<T>& p3) {
  if constexpr (sizeof(T) == 4) return 0;
  uint32_t r;
  asm("{\n\t.reg .pred p;\n\t"
      "setp.le.f32 p, %1, %3;\n\tsetp.le.or.f32 p, %2, %3, p;\n\t"
      "setp.le.or.f32 p, %4, %6, p;\n\tsetp.le.or.f32 p, %5, %6, p;\n\t"
      "setp.le.or.f32 p, %7, %9, p;\n\tsetp.le.or.f32 p, %8, %9, p;\n\t"
      "setp.le.or.f32 p, %10, %12, p;\n\tsetp.le.or.f32 p, %11, %12, p;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r)
      : "f"(p0.da), "f"(p0.db), "f"(p0.e), "f"(p1.da), "f"(p1.db), "f"(p1.e), "f"(p2.da), "f"(p2.db), "f"(p2.e), "f"(p3.da),
        "f"(p3.db), "f"(p3.e));
  return r;
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// rn(m / top) for a row's maximum.  One multiplication, then the remainder
// (exact in a fused multiply-add) corrects it; out of range: a division.
__device__ __forceinline__ float scale_of(float m, float top, float inv_top) {
  const float q = m * inv_top;
  const float r = __fmaf_rn(__fmaf_rn(-q, top, m), inv_top, q);
  return m > 1e-30f && m < 1e30f ? r : __fdiv_rn(m, top);
}

// rn(x / s) in 64 bits, as the fp32 value that converts to it.
template <int KIND>
__device__ __noinline__ float quotient_exact(float x, float s) {
  if (s == 0.0f) return 0.0f;  // a row of zeros
  if (!(fabsf(x) <= 3.4028235e38f) || !(s <= 3.4028235e38f)) {  // infinities, NaN: as the division has it
    const float t = x / s;
    return KIND == kInt8 ? fminf(fmaxf(t == t ? t : 0.0f, -127.0f), 127.0f) : t;
  }
  const double y = static_cast<double>(x) / static_cast<double>(s);
  if (KIND == kInt8) return static_cast<float>(rint(fmin(fmax(y, -127.0), 127.0)));
  return to_odd(fmin(fmax(y, -448.0), 448.0));
}

// x * inv (inv = 1 / s within an ulp, so x / s within 4) and whether its
// rounding to the 8-bit type is not sure.
template <int KIND>
__device__ __forceinline__ bool quotient(float x, float inv, float& t) {
  t = x * inv;
  if constexpr (KIND == kE4M3) {
    // above 2^-6 e4m3 keeps 3 bits of the fraction: 20 bits of fp32 are dropped; below it is subnormal
    return ((__float_as_uint(t) + 0x80000u + 8u) & 0xFFFFFu) <= 16u || !(fabsf(t) >= 0.015625f);
  } else {
    const float q = rintf(t);
    const bool near = !(fabsf(t - q) < 0.49996f);  // NaN and infinity too
    t = fminf(fmaxf(q, -127.0f), 127.0f);
    return near;
  }
}

// 8 values -> 8 bytes, each rounded once.  plain: s is far from underflow.
template <int KIND>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float s, float inv, bool plain) {
  float t[8];
  bool near = !plain;
#pragma unroll
  for (int i = 0; i < 8; ++i) near |= quotient<KIND>(x[i], inv, t[i]);
  if (near) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float again;
      if (!plain || quotient<KIND>(x[i], inv, again)) t[i] = quotient_exact<KIND>(x[i], s);
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if constexpr (KIND == kE4M3) {
      uint16_t lo, hi;  // the first source goes to the upper byte; saturates, NaN stays NaN
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(t[4 * h + 1]), "f"(t[4 * h]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(t[4 * h + 3]), "f"(t[4 * h + 2]));
      w[h] = static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
    } else {
      // whole numbers: adding 1.5 * 2^23 leaves them in the low bits
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(t[4 * h + i] + 12582912.0f);
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}

// ---------------------------------------------------------------- 8 values at a time
// As loaded: so that a thread's next loads are under way while it works.
template <typename T, bool VEC>
struct Raw8 {
  static constexpr int kWords = VEC ? sizeof(T) / 2 : 1;  // 16 bytes each
  uint4 w[kWords];
  T e[VEC ? 1 : 8];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float (&x)[8]) const {
    const T* t = VEC ? reinterpret_cast<const T*>(w) : e;
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = up<T>(t[i]);
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = up<T>(p[i]);
  } else if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = up<T>(t[i]);
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {  // x already rounded to T
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = down<T>(x[i]);
  } else if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 u;
    T* t = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = down<T>(x[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// The 8 pairs of a thread's 16 values, rotated and rounded to T: in the half
// layout x0[i] with x1[i], in the interleaved one neighbours.
template <typename T>
__device__ __forceinline__ void rotate16(float (&x0)[8], float (&x1)[8], const float (&cs)[8], const float (&sn)[8],
                                         float amp, bool neox) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {  // four pairs at a time
    float a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float(&y)[8] = h ? x1 : x0;
      a[i] = neox ? x0[4 * h + i] : y[2 * i];
      b[i] = neox ? x1[4 * h + i] : y[2 * i + 1];
    }
    const float *c = cs + 4 * h, *s = sn + 4 * h;
    const Pair<T> p0(a[0], b[0], c[0], s[0], amp), p1(a[1], b[1], c[1], s[1], amp);
    const Pair<T> p2(a[2], b[2], c[2], s[2], amp), p3(a[3], b[3], c[3], s[3], amp);
    float ra[4] = {p0.a, p1.a, p2.a, p3.a}, rb[4] = {p0.b, p1.b, p2.b, p3.b};
    if (any_unsure<T>(p0, p1, p2, p3)) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!Pair<T>(a[i], b[i], c[i], s[i], amp).unsure()) continue;
        ra[i] = rotate_exact<T>(a[i], c[i], b[i], s[i]);
        rb[i] = rotate_exact<T>(b[i], c[i], a[i], -s[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float(&y)[8] = h ? x1 : x0;
      (neox ? x0[4 * h + i] : y[2 * i]) = ra[i];
      (neox ? x1[4 * h + i] : y[2 * i + 1]) = rb[i];
    }
  }
}

// One block walks tokens; its threads are split into groups of lanes, one row
// (head) each.  gridDim.y: blocks for the rows that are rotated in place (only
// the rotated part of a row has lanes), then blocks for the cache's rows.
// Bound by issue slots (55 to 64 % used) and the latency of a row's loads, of
// which the next row's are started before this one's work: 16111 tokens x 128
// heads, 64 dimensions rotated in bf16, 123 us (4.3 TB/s of 6.5 copied); 16383
// tokens, 32 + 8 heads rotated and written as e4m3, 82 us (2.9 TB/s).  Eight
// blocks of 64 registers beat more rows at once (168 to 212 us for the first)
// and loads ahead across tokens (167 us).
template <typename T, int CACHE, bool ROPE, bool VEC>
__global__ void __launch_bounds__(kThreads, 8) rows_kernel(const __grid_constant__ Params p) {
  const bool turning = ROPE && static_cast<int>(blockIdx.y) < p.turn_blocks;
  const int lanes_log2 = turning ? p.turn_log2 : p.lanes_log2;
  const int lanes = 1 << lanes_log2, groups = kThreads >> lanes_log2;
  const int g = threadIdx.x & (lanes - 1), slot_in_block = threadIdx.x >> lanes_log2;
  const bool active = g < (turning ? p.R : p.D) / 16;
  const bool turns = ROPE && g < p.R / 16;
  // where this thread's 16 values lie in a row
  int at0 = 16 * g, at1 = 16 * g + 8;
  if (ROPE && p.neox && turns) at0 = 8 * g, at1 = 8 * g + p.R / 2;
  const int rows = turning ? p.q_heads + (CACHE == kNoCache ? p.kv_heads : 0) : 2 * p.kv_heads;
  const int row0 = turning ? blockIdx.y * p.turn_rows : (blockIdx.y - p.turn_blocks) * p.cache_rows;
  const int row1 = min(rows, row0 + (turning ? p.turn_rows : p.cache_rows));
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    float cs[8], sn[8], amp = 0.0f;
    bool rope_ok = true;
    if constexpr (ROPE) {
      const long long pos = p.positions[t];
      rope_ok = pos >= 0 && pos < p.max_position;
      if (!rope_ok && threadIdx.x == 0) atomicOr(&g_kv_error, 1);
      if (turns && rope_ok) {
        const float* row = p.table + pos * p.R + 8 * g;
        load8<float, true>(row, cs);
        load8<float, true>(row + p.R / 2, sn);
#pragma unroll
        for (int i = 0; i < 8; ++i) amp = fmaxf(amp, fmaxf(fabsf(cs[i]), fabsf(sn[i])));
        amp *= 1.1920929e-7f;
      }
    }
    if (turning) {
      if (!rope_ok || !active) continue;
      auto row_at = [&](int r) {
        const Rows& src = r < p.q_heads ? p.q : p.k;
        return reinterpret_cast<T*>(const_cast<void*>(src.in)) + t * src.tok_stride +
               (r < p.q_heads ? r : r - p.q_heads) * src.head_stride;
      };
      int r = row0 + slot_in_block;
      if (r >= row1) continue;
      T* x = row_at(r);
      Raw8<T, VEC> in0, in1;
      in0.load(x + at0);
      in1.load(x + at1);
      while (true) {  // the next row's loads are under way while this one is rotated
        float x0[8], x1[8];
        in0.get(x0);
        in1.get(x1);
        T* to = x;
        const bool more = (r += groups) < row1;
        if (more) {
          x = row_at(r);
          in0.load(x + at0);
          in1.load(x + at1);
        }
        if (p.neox)
          rotate16<T>(x0, x1, cs, sn, amp, true);
        else
          rotate16<T>(x0, x1, cs, sn, amp, false);
        store8<T, VEC>(to + at0, x0);
        store8<T, VEC>(to + at1, x1);
        if (!more) break;
      }
      continue;
    }
    if constexpr (CACHE != kNoCache) {
      const long long at = p.slots[t];
      if (at < 0 || !rope_ok) continue;  // negative: a padded token, nothing is written
      const long long block = at / p.c.block_size, inside = at - block * p.c.block_size;
      if (block >= p.c.num_blocks) {
        if (threadIdx.x == 0) atomicOr(&g_kv_error, 1);
        continue;
      }
      Raw8<T, VEC> in0, in1;
      auto fetch = [&](int r) {
        if (r >= row1 || !active) return;
        const Rows& src = r < p.kv_heads ? p.k : p.v;
        const T* in = static_cast<const T*>(src.in) + t * src.tok_stride + (r < p.kv_heads ? r : r - p.kv_heads) * src.head_stride;
        in0.load(in + at0);
        in1.load(in + at1);
      };
      fetch(row0 + slot_in_block);
      for (int base = row0; base < row1; base += groups) {  // every lane takes every turn: the maxima are shuffled
        const int r = base + slot_in_block;
        const bool is_k = r < p.kv_heads;
        const bool here = r < row1 && active;
        const int h = is_k ? r : r - p.kv_heads;
        const int64_t* st = is_k ? p.c.key_stride : p.c.value_stride;
        const long long to = block * st[0] + inside * st[1] + h * st[2];
        float x0[8], x1[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x0[i] = x1[i] = 0.0f;
        if (here) {
          in0.get(x0);
          in1.get(x1);
          fetch(r + groups);
          if (ROPE && turns && is_k) {
            if (p.neox)
              rotate16<T>(x0, x1, cs, sn, amp, true);
            else
              rotate16<T>(x0, x1, cs, sn, amp, false);
#pragma unroll
            for (int i = 0; i < 8; ++i) x0[i] = up<T>(down<T>(x0[i])), x1[i] = up<T>(down<T>(x1[i]));
          }
        }
        if constexpr (CACHE == kSame) {
          if (here) {
            T* out = static_cast<T*>(is_k ? p.c.key : p.c.value) + to;
            store8<T, true>(out + at0, x0);
            store8<T, true>(out + at1, x1);
          }
        } else {
          const int64_t* ss = is_k ? p.c.k_scale_stride : p.c.v_scale_stride;
          float* scale = (is_k ? p.c.k_scale : p.c.v_scale) + block * ss[0] + inside * ss[1] + h * ss[2];
          float s = 1.0f;
          if (p.c.scale_mode == MCPU_KV_SCALE_TOKEN) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max_nan(m, max_nan(fabsf(x0[i]), fabsf(x1[i])));
            for (int o = lanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFull, m, o));
            s = CACHE == kE4M3 ? scale_of(m, 448.0f, 1.0f / 448.0f) : scale_of(m, 127.0f, 1.0f / 127.0f);
            if (here && g == 0) *scale = s;
          } else if (here) {
            s = *scale;
          }
          if (here) {
            float inv;
            asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(s));
            const bool plain = s > 1e-30f && s < 1e30f;
            uint8_t* out = static_cast<uint8_t*>(is_k ? p.c.key : p.c.value) + to;
            *reinterpret_cast<uint2*>(out + at0) = quantise8<CACHE>(x0, s, inv, plain);
            *reinterpret_cast<uint2*>(out + at1) = quantise8<CACHE>(x1, s, inv, plain);
          }
        }
      }
    }
  }
}

// Rotation for head parts the row kernel does not take (R not a multiple of
// 16): one pair per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads) pairs_kernel(const __grid_constant__ Params p) {
  const int half = p.R / 2;
  const int heads = p.q_heads + p.kv_heads;
  const long long n = static_cast<long long>(heads) * half;
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    const long long pos = p.positions[t];
    if (pos < 0 || pos >= p.max_position) {
      if (threadIdx.x == 0) atomicOr(&g_kv_error, 1);
      continue;
    }
    for (long long i = threadIdx.x + static_cast<long long>(blockIdx.y) * kThreads; i < n;
         i += static_cast<long long>(gridDim.y) * kThreads) {
      const int r = static_cast<int>(i / half), d = static_cast<int>(i - static_cast<long long>(r) * half);
      const Rows& src = r < p.q_heads ? p.q : p.k;
      T* x = reinterpret_cast<T*>(const_cast<void*>(src.in)) + t * src.tok_stride +
             (r < p.q_heads ? r : r - p.q_heads) * src.head_stride;
      T* pa = x + (p.neox ? d : 2 * d);
      T* pb = x + (p.neox ? d + half : 2 * d + 1);
      const float a = up<T>(*pa), b = up<T>(*pb);
      const float c = p.table[pos * p.R + d], s = p.table[pos * p.R + half + d];
      const Pair<T> r2(a, b, c, s, 1.1920929e-7f * fmaxf(fabsf(c), fabsf(s)));
      const bool again = r2.unsure();
      *pa = down<T>(again ? rotate_exact<T>(a, c, b, s) : r2.a);
      *pb = down<T>(again ? rotate_exact<T>(b, c, a, -s) : r2.b);
    }
  }
}

// ---------------------------------------------------------------- read-back
struct GatherParams {
  mcpuKvCache c;
  const int* block_table;
  long long table_stride;
  int table_width, batch;
  const int* cu;
  const int* starts;  // or NULL
  long long tokens;
  void* key_out;
  void* value_out;
};

// q * s cut off to fp32, the last bit set where that lost something, so that
// the rounding to T is that of the product (rounded to fp32 first, one in some
// 10^5 lies on a border of T and goes the wrong way); two at a time.  s in
// 2^-100 .. 2^100: what was lost is an fp32 value.
__device__ __forceinline__ void products_to_odd(float& lo, float& hi, float s) {
  unsigned long long q, p, r, s2, n2;
  asm("mov.b64 %0, {%1, %2};" : "=l"(q) : "f"(lo), "f"(hi));
  asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
  asm("mov.b64 %0, {%1, %1};" : "=l"(n2) : "f"(-s));
  asm("mul.rz.f32x2 %0, %1, %2;" : "=l"(p) : "l"(q), "l"(s2));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(n2), "l"(p));
  float r0, r1;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(p));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r0), "=f"(r1) : "l"(r));
  if (r0 != 0.0f) lo = __uint_as_float(__float_as_uint(lo) | 1u);
  if (r1 != 0.0f) hi = __uint_as_float(__float_as_uint(hi) | 1u);
}

// Dequantises 16 values held in 16 bytes to two 16-byte vectors of T.
template <typename T, int KIND>
__device__ __forceinline__ void dequantise16(const uint4& q, float s, uint4* out) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t two = w[i >> 1] >> (16 * (i & 1));
    float lo, hi;
    if constexpr (KIND == kE4M3) {
      uint32_t h2;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"(static_cast<uint16_t>(two)));
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h2));
      lo = f.x, hi = f.y;
    } else {
      // byte + 128 as the low bits of 2^23: whole numbers without a conversion
      const uint32_t biased = two ^ 0x8080u;
      lo = __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7650)) - 8388736.0f;
      hi = __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7651)) - 8388736.0f;
    }
    products_to_odd(lo, hi, s);
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      o[i] = pack_bf16x2(lo, hi);
    } else {
      const __half2 h = __floats2half2_rn(lo, hi);
      o[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}
// The same for any s, one value at a time in 64 bits.
template <typename T, int KIND>
__device__ __noinline__ void dequantise16_exact(const uint8_t* q, float s, T* out) {
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    float x;
    if constexpr (KIND == kE4M3)
      x = __half2float(__half(__nv_cvt_fp8_to_halfraw(q[i], __NV_E4M3)));
    else
      x = static_cast<float>(static_cast<int8_t>(q[i]));
    out[i] = down<T>(to_odd(static_cast<double>(x) * static_cast<double>(s)));
  }
}

// One warp per token: finds its sequence (32-way search of the offsets, one
// step up to 32 sequences), looks its page up once, and moves all heads' key
// and value, 16 values per lane and step.  Bound by HBM: 698 MB, mostly bf16
// written, in 130 us (5.4 TB/s of 6.5 copied; 124 with products rounded twice;
// 133 with products one at a time, 160 with a branch each for keys and values).
template <typename T, int KIND>
__global__ void __launch_bounds__(256) gather_kernel(const __grid_constant__ GatherParams p) {
  const long long t = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t >= p.tokens) return;
  // b = number of sequences that end at or before t
  int lo = 0, n = p.batch;
  while (n > 0) {
    const int step = (n + 31) >> 5;
    const int i = min(lo + (lane + 1) * step, lo + n);  // sequences before i
    const bool past = (lane * step < n) && p.cu[i] <= t;
    const int c = __popc(__ballot_sync(kFull, past));
    const int skip = min(c * step, n);
    if (step == 1) {
      lo += skip;
      break;
    }
    lo += skip;
    n = min(n - skip, step - 1);
  }
  if (lo >= p.batch) return;  // rows behind the last sequence stay as they are
  const long long pos = t - p.cu[lo] + (p.starts ? p.starts[lo] : 0);
  const long long page = pos / p.c.block_size;
  if (t < p.cu[lo] || pos < 0 || page >= p.table_width) {
    if (lane == 0) atomicOr(&g_kv_error, 1);
    return;
  }
  const int id = p.block_table[lo * p.table_stride + page];
  if (id < 0 || id >= p.c.num_blocks) {
    if (lane == 0) atomicOr(&g_kv_error, 1);
    return;
  }
  const int inside = static_cast<int>(pos - page * p.c.block_size);
  const int per_row = p.c.head_size / 16, chunks = p.c.kv_heads * per_row;
  const long long out_at = t * p.c.kv_heads * p.c.head_size;
  constexpr int kSize = KIND == kSame ? 2 : 1;
  const uint8_t* kin = static_cast<const uint8_t*>(p.c.key) +
                       (id * p.c.key_stride[0] + inside * p.c.key_stride[1]) * kSize;
  const uint8_t* vin = static_cast<const uint8_t*>(p.c.value) +
                       (id * p.c.value_stride[0] + inside * p.c.value_stride[1]) * kSize;
  const float* ks = KIND == kSame ? nullptr : p.c.k_scale + id * p.c.k_scale_stride[0] + inside * p.c.k_scale_stride[1];
  const float* vs = KIND == kSame ? nullptr : p.c.v_scale + id * p.c.v_scale_stride[0] + inside * p.c.v_scale_stride[1];
  T* kout = static_cast<T*>(p.key_out) + out_at;
  T* vout = static_cast<T*>(p.value_out) + out_at;
#pragma unroll 2
  for (int c = lane; c < chunks; c += 32) {
    const int h = c / per_row, d = (c - h * per_row) * 16;
    const uint4* ksrc = reinterpret_cast<const uint4*>(kin + (h * p.c.key_stride[2] + d) * kSize);
    const uint4* vsrc = reinterpret_cast<const uint4*>(vin + (h * p.c.value_stride[2] + d) * kSize);
    uint4* kd = reinterpret_cast<uint4*>(kout + 16ll * c);
    uint4* vd = reinterpret_cast<uint4*>(vout + 16ll * c);
    if constexpr (KIND == kSame) {
      const uint4 a = ksrc[0], b = ksrc[1], e = vsrc[0], f = vsrc[1];
      kd[0] = a, kd[1] = b, vd[0] = e, vd[1] = f;
    } else {
      const uint4 a = *ksrc, e = *vsrc;
      const float sk = ks[h * p.c.k_scale_stride[2]], sv = vs[h * p.c.v_scale_stride[2]];
      if (fminf(sk, sv) >= 7.9e-31f && fmaxf(sk, sv) <= 1.2e30f) {
        dequantise16<T, KIND>(a, sk, kd);
        dequantise16<T, KIND>(e, sv, vd);
      } else {
        dequantise16_exact<T, KIND>(reinterpret_cast<const uint8_t*>(ksrc), sk, reinterpret_cast<T*>(kd));
        dequantise16_exact<T, KIND>(reinterpret_cast<const uint8_t*>(vsrc), sv, reinterpret_cast<T*>(vd));
      }
    }
  }
}

// ---------------------------------------------------------------- host side
int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 148;
  return n;
}

bool aligned(const Rows& r, int elem) {
  const int per = 16 / elem;
  return (reinterpret_cast<uintptr_t>(r.in) & 15) == 0 && r.tok_stride % per == 0 && r.head_stride % per == 0;
}

template <typename T, int CACHE, bool ROPE>
orError_t launch_rows(Params& p, cudaStream_t st, const char* what) {
  auto log2_lanes = [](int values) {
    int n = 0;
    while ((16 << n) < values) ++n;
    return n;
  };
  p.lanes_log2 = log2_lanes(p.D);
  p.turn_log2 = log2_lanes(p.R);
  // Few tokens: a block takes one turn of its threads, so that a token's rows are in flight together; many: a block keeps a
  // token's cosines for as many rows as still leave blocks enough.
  const long long fill = 8LL * sm_count();
  auto split = [&](int rows, int groups, int& per) {
    long long parts = (rows + groups - 1) / groups;
    if (p.tokens * parts > fill) parts = std::max<long long>(1, fill / p.tokens);
    per = static_cast<int>((rows + parts - 1) / parts);
    per = (per + groups - 1) / groups * groups;
    return (rows + per - 1) / per;
  };
  const int turn = !ROPE ? 0 : p.q_heads + (CACHE == kNoCache ? p.kv_heads : 0);
  p.turn_blocks = turn ? split(turn, kThreads >> p.turn_log2, p.turn_rows) : 0;
  const int cache_blocks = CACHE == kNoCache ? 0 : split(2 * p.kv_heads, kThreads >> p.lanes_log2, p.cache_rows);
  const dim3 grid(static_cast<unsigned>(std::min<long long>(p.tokens, fill)), static_cast<unsigned>(p.turn_blocks + cache_blocks));
  const int elem = sizeof(T);
  bool vec = aligned(p.k, elem);
  if (ROPE) vec = vec && aligned(p.q, elem);
  if (CACHE != kNoCache) vec = vec && aligned(p.v, elem);
  if (vec)
    rows_kernel<T, CACHE, ROPE, true><<<grid, kThreads, 0, st>>>(p);
  else
    rows_kernel<T, CACHE, ROPE, false><<<grid, kThreads, 0, st>>>(p);
  return from_cuda(cudaGetLastError(), what);
}

template <typename T, bool ROPE>
orError_t launch_cache(Params& p, int dtype, cudaStream_t st, const char* what) {
  if (p.c.dtype == dtype) return launch_rows<T, kSame, ROPE>(p, st, what);
  if (p.c.dtype == MCPU_INT8) return launch_rows<T, kInt8, ROPE>(p, st, what);
  return launch_rows<T, kE4M3, ROPE>(p, st, what);
}

orError_t check_rotary(const int64_t* positions, int64_t tokens, const float* table, int64_t max_position, int R,
                       const char* op) {
  MCPU_ARG_CHECK(R > 0 && R % 2 == 0, "%s: rotary_dim %d must be even and positive", op, R);
  MCPU_ARG_CHECK(max_position > 0, "%s: cos_sin_cache is empty", op);
  MCPU_ARG_CHECK(positions && table, "%s: NULL pointer", op);
  MCPU_ARG_CHECK((reinterpret_cast<uintptr_t>(table) & 15) == 0, "%s: cos_sin_cache must be 16-byte aligned", op);
  return orSuccess;
}

}  // namespace kv

orError_t kv_read_error(int* flag, bool reset) {
  int z = 0;
  MCPU_CUDA_TRY(cudaMemcpyFromSymbol(flag, kv::g_kv_error, sizeof(int)), "mcpu_device_error");
  if (reset) MCPU_CUDA_TRY(cudaMemcpyToSymbol(kv::g_kv_error, &z, sizeof(int)), "mcpu_device_error");
  return orSuccess;
}

}  // namespace mcpu

using namespace mcpu;

extern "C" orError_t mcpu_rotary_embedding(const int64_t* positions, int64_t num_tokens, void* query, int num_heads,
                                           int64_t query_token_stride, int64_t query_head_stride, void* key,
                                           int num_kv_heads, int64_t key_token_stride, int64_t key_head_stride,
                                           int rotary_dim, const float* cos_sin_cache, int64_t max_position,
                                           int is_neox, int dtype, orStream_t stream) {
  const char* op = "rotary_embedding";
  MCPU_ARG_CHECK(dtype == MCPU_FLOAT32 || dtype == MCPU_BFLOAT16 || dtype == MCPU_FLOAT16,
                 "%s: float32, bfloat16 or float16 tensors expected", op);
  MCPU_ARG_CHECK(num_tokens >= 0 && num_tokens < (1LL << 31) && num_heads >= 0 && num_kv_heads >= 0,
                 "%s: bad sizes", op);
  if (num_tokens == 0 || num_heads + num_kv_heads == 0) return orSuccess;
  MCPU_ARG_CHECK((num_heads == 0 || query) && (num_kv_heads == 0 || key), "%s: NULL pointer", op);
  orError_t e = kv::check_rotary(positions, num_tokens, cos_sin_cache, max_position, rotary_dim, op);
  if (e != orSuccess) return e;
  kv::Params p{};
  p.tokens = num_tokens;
  p.q_heads = num_heads, p.kv_heads = num_kv_heads;
  p.D = p.R = rotary_dim;  // the rest of the head is not touched
  p.neox = is_neox != 0;
  p.q = {query, query_token_stride, query_head_stride};
  p.k = {key, key_token_stride, key_head_stride};
  p.positions = reinterpret_cast<const long long*>(positions);
  p.table = cos_sin_cache;
  p.max_position = max_position;
  cudaStream_t st = as_cuda(stream);
  if (rotary_dim % 16 != 0 || rotary_dim > 512) {
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(num_tokens, 1 << 16)), num_tokens < 1024 ? 4 : 1);
    if (dtype == MCPU_FLOAT32)
      kv::pairs_kernel<float><<<grid, kv::kThreads, 0, st>>>(p);
    else if (dtype == MCPU_FLOAT16)
      kv::pairs_kernel<__half><<<grid, kv::kThreads, 0, st>>>(p);
    else
      kv::pairs_kernel<__nv_bfloat16><<<grid, kv::kThreads, 0, st>>>(p);
    return from_cuda(cudaGetLastError(), "rotary_embedding launch");
  }
  if (dtype == MCPU_FLOAT32) return kv::launch_rows<float, kv::kNoCache, true>(p, st, "rotary_embedding launch");
  if (dtype == MCPU_FLOAT16) return kv::launch_rows<__half, kv::kNoCache, true>(p, st, "rotary_embedding launch");
  return kv::launch_rows<__nv_bfloat16, kv::kNoCache, true>(p, st, "rotary_embedding launch");
}

extern "C" orError_t mcpu_rotary_reshape_and_cache(
    const int64_t* positions, int64_t num_tokens, void* query, int num_heads, int64_t query_token_stride,
    int64_t query_head_stride, const void* key, int64_t key_token_stride, int64_t key_head_stride, const void* value,
    int64_t value_token_stride, int64_t value_head_stride, int rotary_dim, const float* cos_sin_cache,
    int64_t max_position, int is_neox, int dtype, const int64_t* slot_mapping, const mcpuKvCache* cache,
    orStream_t stream) {
  const char* op = rotary_dim ? "rotary_reshape_and_cache" : "reshape_and_cache";
  orError_t e = kv::check_cache(cache, dtype, op);
  if (e != orSuccess) return e;
  MCPU_ARG_CHECK(num_tokens >= 0 && num_tokens < (1LL << 31) && num_heads >= 0, "%s: bad sizes", op);
  if (num_tokens == 0) return orSuccess;
  MCPU_ARG_CHECK(key && value && slot_mapping && (num_heads == 0 || query), "%s: NULL pointer", op);
  kv::Params p{};
  if (rotary_dim) {
    e = kv::check_rotary(positions, num_tokens, cos_sin_cache, max_position, rotary_dim, op);
    if (e != orSuccess) return e;
    MCPU_ARG_CHECK(rotary_dim % 16 == 0 && rotary_dim <= cache->head_size,
                   "%s: rotary_dim %d must be a multiple of 16, at most head_size", op, rotary_dim);
  }
  p.tokens = num_tokens;
  p.q_heads = num_heads, p.kv_heads = cache->kv_heads;
  p.D = cache->head_size, p.R = rotary_dim;
  p.neox = is_neox != 0;
  p.q = {query, query_token_stride, query_head_stride};
  p.k = {key, key_token_stride, key_head_stride};
  p.v = {value, value_token_stride, value_head_stride};
  p.positions = reinterpret_cast<const long long*>(positions);
  p.table = cos_sin_cache;
  p.max_position = max_position;
  p.slots = reinterpret_cast<const long long*>(slot_mapping);
  p.c = *cache;
  cudaStream_t st = as_cuda(stream);
  if (rotary_dim)
    return dtype == MCPU_FLOAT16 ? kv::launch_cache<__half, true>(p, dtype, st, "rotary_reshape_and_cache launch")
                                 : kv::launch_cache<__nv_bfloat16, true>(p, dtype, st, "rotary_reshape_and_cache launch");
  return dtype == MCPU_FLOAT16 ? kv::launch_cache<__half, false>(p, dtype, st, "reshape_and_cache launch")
                               : kv::launch_cache<__nv_bfloat16, false>(p, dtype, st, "reshape_and_cache launch");
}

extern "C" orError_t mcpu_gather_cache(const mcpuKvCache* cache, const int32_t* block_table, int64_t table_stride,
                                       int64_t table_width, int64_t batch, const int32_t* cu_seq_lens,
                                       const int32_t* seq_starts, void* key_out, void* value_out, int64_t num_tokens,
                                       int dtype, orStream_t stream) {
  const char* op = "gather_cache";
  orError_t e = kv::check_cache(cache, dtype, op);
  if (e != orSuccess) return e;
  MCPU_ARG_CHECK(num_tokens >= 0 && num_tokens < (1LL << 31) && batch >= 0 && batch < (1LL << 30) && table_width >= 0 &&
                     table_width < (1LL << 31) && table_stride >= table_width,
                 "%s: bad sizes", op);
  if (num_tokens == 0 || batch == 0) return orSuccess;
  MCPU_ARG_CHECK(block_table && cu_seq_lens && key_out && value_out, "%s: NULL pointer", op);
  MCPU_ARG_CHECK(((reinterpret_cast<uintptr_t>(key_out) | reinterpret_cast<uintptr_t>(value_out)) & 15) == 0,
                 "%s: outputs must be 16-byte aligned", op);
  kv::GatherParams p{};
  p.c = *cache;
  p.block_table = block_table;
  p.table_stride = table_stride;
  p.table_width = static_cast<int>(table_width);
  p.batch = static_cast<int>(batch);
  p.cu = cu_seq_lens;
  p.starts = seq_starts;
  p.tokens = num_tokens;
  p.key_out = key_out;
  p.value_out = value_out;
  const unsigned grid = static_cast<unsigned>((num_tokens + 7) / 8);
  cudaStream_t st = as_cuda(stream);
  const bool half = dtype == MCPU_FLOAT16;
  if (cache->dtype == dtype)
    kv::gather_kernel<__half, kv::kSame><<<grid, 256, 0, st>>>(p);  // bits are copied: either 16-bit type
  else if (cache->dtype == MCPU_INT8 && half)
    kv::gather_kernel<__half, kv::kInt8><<<grid, 256, 0, st>>>(p);
  else if (cache->dtype == MCPU_INT8)
    kv::gather_kernel<__nv_bfloat16, kv::kInt8><<<grid, 256, 0, st>>>(p);
  else if (half)
    kv::gather_kernel<__half, kv::kE4M3><<<grid, 256, 0, st>>>(p);
  else
    kv::gather_kernel<__nv_bfloat16, kv::kE4M3><<<grid, 256, 0, st>>>(p);
  return from_cuda(cudaGetLastError(), "gather_cache launch");
}
