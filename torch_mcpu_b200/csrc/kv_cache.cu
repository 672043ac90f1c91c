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
// Every result is the correctly rounded one.  A quantised value that lands on
// the wrong side of a rounding border is a whole 8-bit step off, and a key
// that is rounded the wrong way before it is quantised moves its row's scale
// and with it the whole row; so the fast fp32 results are used only where they
// lie further from a border than their error bound, and the few others
// (about 2^-13 of the rotated values, 2^-17 of the quantised ones) are computed
// again in 64 bits and rounded once (through an odd fp32, which lies on no
// border of the shorter types).
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
  int q_heads, kv_heads, D, R, lanes_log2, neox;
  long long rows_per_block;
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

// Out of line: the common path keeps its registers.
template <typename T>
__device__ __noinline__ float rotate_exact(float a, float c, float b, float s) {
  const double bs = static_cast<double>(b) * static_cast<double>(s);
  return up<T>(down<T>(to_odd(static_cast<double>(a) * static_cast<double>(c) - bs)));
}

// a*c - b*s (or + with s negated) rounded once to T, as its fp32 value.
template <typename T>
__device__ __forceinline__ float rotate(float a, float c, float b, float s) {
  const float p = __fmul_rn(b, s);
  const float r = __fmaf_rn(a, c, -p);
  if constexpr (sizeof(T) == 4) {
    return r;
  } else {
    // |r - exact| <= 2^-24 (|p| + |r|).  The border of T that r's bits fall
    // next to: the dropped bits replaced by 100..0.
    constexpr bool kBf16 = sizeof(T) == 2 && static_cast<int>(std::is_same<T, __nv_bfloat16>::value);
    constexpr uint32_t kDropped = kBf16 ? 0xFFFFu : 0x1FFFu;
    const uint32_t u = __float_as_uint(r);
    const float border = __uint_as_float((u & ~kDropped) | ((kDropped + 1) >> 1));
    const float mag = fabsf(p) + fabsf(r);
    bool near = fabsf(r - border) <= mag * 1.1920929e-7f;  // 2^-23: twice the bound
    if constexpr (kBf16)
      near = near || fabsf(r) < 1e-30f;  // products that may have lost bits to underflow
    else
      near = near || fabsf(r) < 6.2e-5f;  // fp16 subnormals: their borders lie elsewhere
    if (near) return rotate_exact<T>(a, c, b, s);
    return up<T>(down<T>(r));
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// The two 8-bit forms of x / s, rounded once.  inv = 1 / s (one rounding), so
// x * inv is within 2^-23 of x / s; usable where s is far from underflow.
struct Scale {
  float s, inv;
  bool plain;  // fp32 arithmetic is safe
  __device__ __forceinline__ explicit Scale(float v)
      : s(v), inv(1.0f / v), plain(!(v < 1e-30f) && v < 1e30f) {}
};

template <int KIND>
__device__ __noinline__ float quotient_exact(float x, float s) {
  const double y = static_cast<double>(x) / static_cast<double>(s);
  if (KIND == kInt8) return static_cast<float>(rint(fmin(fmax(y, -127.0), 127.0)));
  return to_odd(fmin(fmax(y, -448.0), 448.0));
}

// fp32 value whose conversion to the 8-bit type gives the rounding of x / s.
template <int KIND>
__device__ __forceinline__ float quotient(float x, const Scale& sc) {
  float t = x * sc.inv;
  if (sc.s == 0.0f) return 0.0f;  // a row of zeros
  bool near;
  if constexpr (KIND == kE4M3) {
    // above 2^-6 e4m3 keeps 3 bits of the fraction; below it is subnormal
    const uint32_t u = __float_as_uint(t);
    const float border = __uint_as_float((u & 0xFFF00000u) | 0x80000u);
    near = fabsf(t - border) <= fabsf(t) * 2.3841858e-7f || (fabsf(t) < 0.015625f && t != 0.0f);
  } else {
    t = fminf(fmaxf(t == t ? t : 0.0f, -127.0f), 127.0f);
    const float q = rintf(t);
    near = fabsf(t - q) > 0.49996f;
    t = q;
  }
  if ((near || !sc.plain) && x == x && fabsf(x) <= 3.4028235e38f && sc.s == sc.s && fabsf(sc.s) <= 3.4028235e38f)
    return quotient_exact<KIND>(x, sc.s);
  return t;
}

// 8 values -> 8 bytes.
template <int KIND>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], const Scale& sc) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = quotient<KIND>(x[4 * h + i], sc);
    if constexpr (KIND == kE4M3) {
      uint16_t lo, hi;  // the first source goes to the upper byte; saturates, NaN stays NaN
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(t[1]), "f"(t[0]));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(t[3]), "f"(t[2]));
      w[h] = static_cast<uint32_t>(lo) | static_cast<uint32_t>(hi) << 16;
    } else {
      // whole numbers: adding 1.5 * 2^23 leaves them in the low bits
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) b[i] = __float_as_uint(t[i] + 12582912.0f);
      w[h] = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    }
  }
  return make_uint2(w[0], w[1]);
}

// ---------------------------------------------------------------- 8 values at a time
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

// One block walks tokens; its threads are split into groups of 2^lanes_log2
// lanes, one row (head) each.  gridDim.y splits a token's rows where there are
// too few tokens to fill the GPU.
template <typename T, int CACHE, bool ROPE, bool VEC>
__global__ void __launch_bounds__(kThreads) rows_kernel(const __grid_constant__ Params p) {
  const int lanes = 1 << p.lanes_log2;
  const int g = threadIdx.x & (lanes - 1), slot_in_block = threadIdx.x >> p.lanes_log2;
  const int groups = kThreads >> p.lanes_log2;
  const bool active = g < p.D / 16;
  const bool turns = ROPE && g < p.R / 16;
  // where this thread's 16 values lie in a row
  int at0 = 16 * g, at1 = 16 * g + 8;
  if (ROPE && p.neox && turns) at0 = 8 * g, at1 = 8 * g + p.R / 2;
  const int q_rows = ROPE ? p.q_heads : 0;
  const int rows = q_rows + p.kv_heads + (CACHE == kNoCache ? 0 : p.kv_heads);
  const int row0 = static_cast<int>(blockIdx.y * p.rows_per_block);
  const int row1 = min(rows, static_cast<int>(row0 + p.rows_per_block));
  for (long long t = blockIdx.x; t < p.tokens; t += gridDim.x) {
    float cs[8], sn[8];
    bool rope_ok = true;
    if constexpr (ROPE) {
      const long long pos = p.positions[t];
      rope_ok = pos >= 0 && pos < p.max_position;
      if (!rope_ok && g == 0 && slot_in_block == 0) atomicOr(&g_kv_error, 1);
      if (turns && rope_ok) {
        const float* row = p.table + pos * p.R + 8 * g;
        load8<float, true>(row, cs);
        load8<float, true>(row + p.R / 2, sn);
      }
    }
    long long block = 0, inside = 0;
    bool cached = false;
    if constexpr (CACHE != kNoCache) {
      const long long s = p.slots[t];
      if (s >= 0) {  // negative: a padded token, nothing is written
        block = s / p.c.block_size;
        inside = s - block * p.c.block_size;
        cached = block < p.c.num_blocks && rope_ok;
        if (block >= p.c.num_blocks && g == 0 && slot_in_block == 0) atomicOr(&g_kv_error, 1);
      }
    }
    for (int base = row0; base < row1; base += groups) {  // every lane takes every turn: the maxima are shuffled
      const int r = base + slot_in_block;
      const bool is_q = r < q_rows;
      const bool is_k = !is_q && r < q_rows + p.kv_heads;
      const bool here = r < row1 && active && (is_q ? rope_ok : CACHE == kNoCache ? rope_ok : cached);
      const int h = is_q ? r : is_k ? r - q_rows : r - q_rows - p.kv_heads;
      float x0[8], x1[8];
      const Rows& src = is_q ? p.q : is_k ? p.k : p.v;
      T* in = reinterpret_cast<T*>(const_cast<void*>(src.in)) + t * src.tok_stride + h * src.head_stride;
      if (here) {
        load8<T, VEC>(in + at0, x0);
        load8<T, VEC>(in + at1, x1);
        if (ROPE && turns && (is_q || is_k)) {
          if (p.neox) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float a = x0[i], b = x1[i];
              x0[i] = rotate<T>(a, cs[i], b, sn[i]);
              x1[i] = rotate<T>(b, cs[i], a, -sn[i]);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float a = x0[2 * i], b = x0[2 * i + 1];
              x0[2 * i] = rotate<T>(a, cs[i], b, sn[i]);
              x0[2 * i + 1] = rotate<T>(b, cs[i], a, -sn[i]);
              a = x1[2 * i], b = x1[2 * i + 1];
              x1[2 * i] = rotate<T>(a, cs[4 + i], b, sn[4 + i]);
              x1[2 * i + 1] = rotate<T>(b, cs[4 + i], a, -sn[4 + i]);
            }
          }
        }
      }
      if (CACHE == kNoCache || is_q) {
        if (here && turns) {
          store8<T, VEC>(in + at0, x0);
          store8<T, VEC>(in + at1, x1);
        }
      }
      if constexpr (CACHE == kSame) {
        if (here && !is_q) {
          const int64_t* st = is_k ? p.c.key_stride : p.c.value_stride;
          T* out = static_cast<T*>(is_k ? p.c.key : p.c.value) + block * st[0] + inside * st[1] + h * st[2];
          store8<T, true>(out + at0, x0);
          store8<T, true>(out + at1, x1);
        }
      }
      if constexpr (CACHE == kE4M3 || CACHE == kInt8) {
        if (__any_sync(kFull, here && !is_q)) {
          const bool is_kv = here && !is_q;
          const int64_t* ss = is_k ? p.c.k_scale_stride : p.c.v_scale_stride;
          float* scale = (is_k ? p.c.k_scale : p.c.v_scale) + block * ss[0] + inside * ss[1] + h * ss[2];
          float s = 0.0f;
          if (p.c.scale_mode == MCPU_KV_SCALE_TOKEN) {
            float m = 0.0f;
            if (is_kv) {
#pragma unroll
              for (int i = 0; i < 8; ++i) m = max_nan(m, max_nan(fabsf(x0[i]), fabsf(x1[i])));
            }
            for (int o = lanes >> 1; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(kFull, m, o));
            s = __fdiv_rn(m, CACHE == kE4M3 ? 448.0f : 127.0f);
            if (is_kv && g == 0) *scale = s;
          } else if (is_kv) {
            s = *scale;
          }
          if (is_kv) {
            const Scale sc(s);
            const int64_t* st = is_k ? p.c.key_stride : p.c.value_stride;
            uint8_t* out = static_cast<uint8_t*>(is_k ? p.c.key : p.c.value) + block * st[0] + inside * st[1] + h * st[2];
            *reinterpret_cast<uint2*>(out + at0) = quantise8<CACHE>(x0, sc);
            *reinterpret_cast<uint2*>(out + at1) = quantise8<CACHE>(x1, sc);
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
      *pa = down<T>(rotate<T>(a, c, b, s));
      *pb = down<T>(rotate<T>(b, c, a, -s));
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

// Dequantises 16 values held in 16 bytes to two 16-byte vectors of T.
template <typename T, int KIND>
__device__ __forceinline__ void dequantise16(const uint4& q, float s, uint4 (&out)[2]) {
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
    lo *= s, hi *= s;
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

// One warp per token: finds its sequence (32-way search of the offsets, one
// step up to 32 sequences), looks its page up once, and moves all heads' key
// and value, 16 values per lane and step.
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
      uint4 o[2];
      dequantise16<T, KIND>(a, sk, o);
      kd[0] = o[0], kd[1] = o[1];
      dequantise16<T, KIND>(e, sv, o);
      vd[0] = o[0], vd[1] = o[1];
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
  const int lanes_needed = p.D / 16;
  p.lanes_log2 = 0;
  while ((1 << p.lanes_log2) < lanes_needed) ++p.lanes_log2;
  const int groups = kThreads >> p.lanes_log2;
  const int rows = (ROPE ? p.q_heads : 0) + p.kv_heads + (CACHE == kNoCache ? 0 : p.kv_heads);
  // Few tokens: one turn of the row loop per block, so a token's rows are in
  // flight together; many: a block keeps a token's cosines for all its rows.
  const long long fill = 16LL * sm_count();
  long long parts = (rows + groups - 1) / groups;
  if (p.tokens * parts > fill) parts = std::max<long long>(1, fill / p.tokens);
  p.rows_per_block = (rows + parts - 1) / parts;
  p.rows_per_block = (p.rows_per_block + groups - 1) / groups * groups;
  const dim3 grid(static_cast<unsigned>(std::min<long long>(p.tokens, fill)),
                  static_cast<unsigned>((rows + p.rows_per_block - 1) / p.rows_per_block));
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
