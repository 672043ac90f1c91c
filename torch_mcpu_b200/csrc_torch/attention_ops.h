// The attention path's operators on tensors: the checks that need a tensor's
// shape, strides and type, and the call into the C entry points
// (include/mcpu_ops.h).  Used twice: by the mcpu:: registrations of the
// PrivateUse1 device and by the Python functions on CUDA tensors.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>

#include <algorithm>
#include <array>
#include <cstring>
#include <optional>
#include <tuple>

#include "mcpu_ops.h"

namespace mcpu_torch {
namespace attention {

// The entry points, and the stream a tensor's work goes on.
struct Api {
  decltype(&mcpu_rotary_embedding) rotary;
  decltype(&mcpu_rotary_reshape_and_cache) write;
  decltype(&mcpu_gather_cache) gather;
  decltype(&mcpu_tree_attention) attend;
  decltype(&mcpu_tree_attention_workspace_bytes) workspace;
  decltype(&mcpuGetLastErrorString) error;
  c10::DeviceType device;
  orStream_t (*stream)(c10::DeviceIndex);
};

using Opt = std::optional<at::Tensor>;

inline void ok(const Api& api, orError_t e, const char* op) {
  TORCH_CHECK(e == orSuccess, op, " failed: ", api.error());
}

inline void on_device(const Api& api, const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(t.device().type() == api.device, op, ": ", name, " must be a device tensor (got device ", t.device(),
              "); the mcpu B200 ops have no CPU fallback");
}
inline void same_device(const at::Tensor& t, const at::Tensor& first, const char* op, const char* name) {
  TORCH_CHECK(t.device() == first.device(), op, ": ", name, " is on ", t.device(), ", expected ", first.device());
}
inline void same_device(const Opt& t, const at::Tensor& first, const char* op, const char* name) {
  if (t) same_device(*t, first, op, name);
}

// Operators of serving: they have no gradient to give, and what is rotated in place would falsify others'.
inline void no_gradient(const at::Tensor& t, const char* op, const char* name) {
  TORCH_CHECK(!t.requires_grad() || !c10::GradMode::is_enabled(), op, ": ", name,
              " requires a gradient, which this operator does not have; call it under torch.no_grad()");
}
inline void no_gradient(const Opt& t, const char* op, const char* name) {
  if (t) no_gradient(*t, op, name);
}
inline void no_gradient(const at::Tensor& key_cache, const at::Tensor& value_cache, const Opt& k_scale, const Opt& v_scale,
                        const char* op) {
  no_gradient(key_cache, op, "key_cache");
  no_gradient(value_cache, op, "value_cache");
  no_gradient(k_scale, op, "k_scale");
  no_gradient(v_scale, op, "v_scale");
}

// A tensor the call has written: autograd, where it has saved it for another operator, is to know.  Tensors of inference
// mode count no versions.
inline void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// [tokens, heads * head_size] or [tokens, heads, head_size] with contiguous heads.
struct Heads {
  int64_t tokens = 0, heads = 0, token_stride = 0, head_stride = 0;
};
inline Heads heads_of(const at::Tensor& t, int64_t head_size, const char* op, const char* name) {
  Heads h;
  if (t.dim() == 2) {
    TORCH_CHECK(head_size > 0 && t.size(1) % head_size == 0 && (t.stride(1) == 1 || t.size(1) <= 1), op, ": ", name,
                " must be [tokens, heads * ", head_size, "] with contiguous rows");
    h = {t.size(0), t.size(1) / head_size, t.stride(0), head_size};
  } else {
    TORCH_CHECK(t.dim() == 3 && t.size(2) == head_size && (t.stride(2) == 1 || head_size <= 1), op, ": ", name,
                " must be [tokens, heads, ", head_size, "] with contiguous heads");
    h = {t.size(0), t.size(1), t.stride(0), t.stride(1)};
  }
  return h;
}

// Written tensors: no two of their elements in one place.  (stride, count) of each dimension outside `reach` elements.
template <size_t N>
void disjoint(std::array<std::pair<int64_t, int64_t>, N> dims, int64_t reach, const char* op, const char* name) {
  std::sort(dims.begin(), dims.end());
  for (const auto& d : dims) {
    if (d.second <= 1) continue;
    TORCH_CHECK(d.first >= reach, op, ": ", name, " is written and must not overlap itself");
    reach += (d.second - 1) * d.first;
  }
}

// Where a strided tensor lies, in bytes: its first address, what is contiguous, and (stride, count) of the dimensions outside
// of that, largest stride first.
struct Place {
  intptr_t at = 0;
  int64_t inner = 0;
  std::array<std::pair<int64_t, int64_t>, 3> dims{};
  int n = 0;
  int64_t reach(int from) const {
    int64_t r = inner;
    for (int i = from; i < n; ++i) r += (dims[i].second - 1) * dims[i].first;
    return r;
  }
};
template <size_t N>
Place place_of(const at::Tensor& t, const std::array<std::pair<int64_t, int64_t>, N>& dims, int64_t inner) {
  const int64_t size = static_cast<int64_t>(t.element_size());
  Place p;
  p.at = reinterpret_cast<intptr_t>(t.const_data_ptr());
  p.inner = inner * size;
  for (const auto& d : dims) {
    if (d.second == 0) p.inner = 0;
    if (d.second > 1 && d.first != 0) p.dims[p.n++] = {d.first * size, d.second};  // an expanded dimension adds no place
  }
  std::sort(p.dims.begin(), p.dims.begin() + p.n, [](const auto& a, const auto& b) { return a.first > b.first; });
  while (p.n > 0 && p.dims[p.n - 1].first == p.inner) p.inner *= p.dims[--p.n].second;
  return p;
}
inline int64_t down_div(int64_t a, int64_t b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }
// Whether the dimensions of a from i on and those of b from j on, b lying `off` bytes behind a, share a byte.  Dimensions of
// one stride are taken together, so views of one tensor are decided in a few steps; others after `steps` count as apart.
inline bool meet(const Place& a, int i, const Place& b, int j, int64_t off, int& steps) {
  if (off >= a.reach(i) || -off >= b.reach(j)) return false;
  if (i == a.n && j == b.n) return true;
  if (--steps < 0) return false;
  const int64_t sa = i < a.n ? a.dims[i].first : 0, sb = j < b.n ? b.dims[j].first : 0;
  if (sa < sb) return meet(b, j, a, i, -off, steps);
  const bool both = sa == sb;  // not 0: one of the two has a dimension left
  const int64_t ra = a.reach(i + 1), rb = b.reach(both ? j + 1 : j);
  // the k-th of a against b, or of one stride those that are k apart
  const int64_t from = std::max(down_div(off - ra, sa) + 1, both ? 1 - b.dims[j].second : 0);
  const int64_t to = std::min(down_div(off + rb - 1, sa), a.dims[i].second - 1);
  for (int64_t k = from; k <= to && steps >= 0; ++k)
    if (meet(a, i + 1, b, both ? j + 1 : j, off - k * sa, steps)) return true;
  return false;
}
inline bool overlap(const Place& a, const Place& b) {
  if (a.inner == 0 || b.inner == 0) return false;
  int steps = 4096;
  return meet(a, 0, b, 0, b.at - a.at, steps);
}
using Dim = std::pair<int64_t, int64_t>;
inline Place place_of(const at::Tensor& t, const Heads& h, int64_t inner) {
  return place_of<2>(t, {Dim{h.token_stride, h.tokens}, Dim{h.head_stride, h.heads}}, inner);
}
inline Place place_of(const at::Tensor& t) {  // up to 3 dimensions and a contiguous one
  std::array<Dim, 3> dims{};
  for (int i = 0; i < 3; ++i) dims[i] = i < t.dim() ? Dim{t.stride(i), t.size(i)} : Dim{0, 1};
  return place_of<3>(t, dims, t.dim() > 3 ? t.size(3) : 1);
}

inline int half_code(at::ScalarType t, const char* op) {
  TORCH_CHECK(t == at::kBFloat16 || t == at::kHalf, op, ": bfloat16 or float16 tensors expected, got ", t);
  return t == at::kHalf ? MCPU_FLOAT16 : MCPU_BFLOAT16;
}

inline void check_table(const at::Tensor& positions, int64_t tokens, const at::Tensor& table, const char* op) {
  TORCH_CHECK(positions.scalar_type() == at::kLong && positions.dim() == 1 && positions.size(0) == tokens &&
                  positions.is_contiguous(),
              op, ": positions must be a contiguous int64 [", tokens, "] tensor");
  TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous(), op,
              ": cos_sin_cache must be a contiguous float32 [max_position, rotary_dim] tensor");
}
inline void check_int32(const at::Tensor& t, int64_t n, const char* op, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), op, ": ", name,
              " must be a contiguous int32 [", n, "] tensor");
}
inline void check_block_table(const at::Tensor& t, const char* op) {
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1) &&
                  (t.size(0) <= 1 || t.stride(0) >= t.size(1)),
              op, ": block_table must be an int32 [batch, blocks] tensor with contiguous rows");
}

inline mcpuKvCache cache_of(const at::Tensor& key_cache, const at::Tensor& value_cache, const Opt& k_scale,
                            const Opt& v_scale, at::ScalarType dtype, bool writes, const char* op) {
  mcpuKvCache c{};
  const int code = half_code(dtype, op);
  TORCH_CHECK(key_cache.dim() == 4 && value_cache.sizes() == key_cache.sizes(), op,
              ": key_cache and value_cache must both be [num_blocks, block_size, kv_heads, head_size]");
  const auto kind = key_cache.scalar_type();
  const bool small = kind == at::kFloat8_e4m3fn || kind == at::kChar;
  TORCH_CHECK(value_cache.scalar_type() == kind && (kind == dtype || small), op, ": the caches must hold ", dtype,
              ", float8_e4m3fn or int8 (got ", kind, ", ", value_cache.scalar_type(), ")");
  const auto sz = key_cache.sizes();
  const auto ks = key_cache.strides(), vs = value_cache.strides();
  TORCH_CHECK((ks[3] == 1 && vs[3] == 1) || sz[3] <= 1, op, ": cache rows must be contiguous");
  TORCH_CHECK(sz[1] < (1LL << 31) && sz[2] < (1LL << 31) && sz[3] < (1LL << 31), op, ": bad cache sizes");
  if (writes) {
    TORCH_CHECK(!overlap(place_of(key_cache), place_of(value_cache)), op, ": key_cache and value_cache are written and must not overlap");
    disjoint<3>({Dim{ks[0], sz[0]}, Dim{ks[1], sz[1]}, Dim{ks[2], sz[2]}}, sz[3], op, "key_cache");
    disjoint<3>({Dim{vs[0], sz[0]}, Dim{vs[1], sz[1]}, Dim{vs[2], sz[2]}}, sz[3], op, "value_cache");
  }
  c.key = key_cache.data_ptr(), c.value = value_cache.data_ptr();
  c.num_blocks = sz[0];
  c.block_size = static_cast<int32_t>(sz[1]), c.kv_heads = static_cast<int32_t>(sz[2]);
  c.head_size = static_cast<int32_t>(sz[3]);
  for (int i = 0; i < 3; ++i) c.key_stride[i] = ks[i], c.value_stride[i] = vs[i];
  if (!small) {
    TORCH_CHECK(!k_scale && !v_scale, op, ": a ", kind, " cache has no scales");
    c.dtype = code, c.scale_mode = MCPU_KV_SCALE_NONE;
    return c;
  }
  c.dtype = kind == at::kChar ? MCPU_INT8 : MCPU_FLOAT8_E4M3;
  TORCH_CHECK(k_scale && v_scale, op, ": a ", kind, " cache needs k_scale and v_scale");
  TORCH_CHECK(k_scale->scalar_type() == at::kFloat && v_scale->scalar_type() == at::kFloat &&
                  k_scale->sizes() == v_scale->sizes(),
              op, ": k_scale and v_scale must be float32 tensors of one shape");
  c.k_scale = static_cast<float*>(k_scale->data_ptr()), c.v_scale = static_cast<float*>(v_scale->data_ptr());
  if (k_scale->dim() == 3 && k_scale->sizes() == sz.slice(0, 3)) {
    c.scale_mode = MCPU_KV_SCALE_TOKEN;
    for (int i = 0; i < 3; ++i) c.k_scale_stride[i] = k_scale->stride(i), c.v_scale_stride[i] = v_scale->stride(i);
    if (writes) {
      TORCH_CHECK(!overlap(place_of(*k_scale), place_of(*v_scale)), op, ": k_scale and v_scale are written and must not overlap");
      const int64_t *k3 = c.k_scale_stride, *v3 = c.v_scale_stride;
      disjoint<3>({Dim{k3[0], sz[0]}, Dim{k3[1], sz[1]}, Dim{k3[2], sz[2]}}, 1, op, "k_scale");
      disjoint<3>({Dim{v3[0], sz[0]}, Dim{v3[1], sz[1]}, Dim{v3[2], sz[2]}}, 1, op, "v_scale");
    }
  } else if (k_scale->numel() == 1) {
    c.scale_mode = MCPU_KV_SCALE_GIVEN;
  } else {
    TORCH_CHECK(k_scale->dim() == 1 && k_scale->size(0) == sz[2], op, ": scales must have 1, [", sz[2], "] or [", sz[0], ", ",
                sz[1], ", ", sz[2], "] elements, got ", k_scale->sizes());
    c.scale_mode = MCPU_KV_SCALE_GIVEN;
    c.k_scale_stride[2] = k_scale->stride(0), c.v_scale_stride[2] = v_scale->stride(0);
  }
  return c;
}

inline void rotary_embedding(const Api& api, const at::Tensor& positions, const at::Tensor& query, const Opt& key,
                             int64_t head_size, const at::Tensor& table, bool is_neox) {
  const char* op = "rotary_embedding";
  on_device(api, query, op, "query");
  same_device(positions, query, op, "positions");
  same_device(key, query, op, "key");
  same_device(table, query, op, "cos_sin_cache");
  no_gradient(query, op, "query");
  no_gradient(key, op, "key");
  no_gradient(table, op, "cos_sin_cache");
  const auto type = query.scalar_type();
  TORCH_CHECK((type == at::kFloat || type == at::kBFloat16 || type == at::kHalf) && (!key || key->scalar_type() == type), op,
              ": query and key must both be float32, bfloat16 or float16");
  const Heads q = heads_of(query, head_size, op, "query");
  check_table(positions, q.tokens, table, op);
  const int64_t part = table.size(1);
  TORCH_CHECK(part <= head_size, op, ": rotary_dim ", part, " exceeds head_size ", head_size);
  disjoint<2>({Dim{q.token_stride, q.tokens}, Dim{q.head_stride, q.heads}}, part, op, "query");
  Heads k;
  if (key) {
    k = heads_of(*key, head_size, op, "key");
    TORCH_CHECK(k.tokens == q.tokens, op, ": key has ", k.tokens, " tokens, query ", q.tokens);
    TORCH_CHECK(!overlap(place_of(query, q, part), place_of(*key, k, part)), op, ": query and key are written and must not overlap");
    disjoint<2>({Dim{k.token_stride, k.tokens}, Dim{k.head_stride, k.heads}}, part, op, "key");
  }
  ok(api,
     api.rotary(positions.const_data_ptr<int64_t>(), q.tokens, query.data_ptr(), static_cast<int>(q.heads), q.token_stride,
                q.head_stride, key ? key->data_ptr() : nullptr, static_cast<int>(k.heads), k.token_stride, k.head_stride,
                static_cast<int>(part), table.const_data_ptr<float>(), table.size(0), is_neox,
                type == at::kFloat ? MCPU_FLOAT32 : type == at::kHalf ? MCPU_FLOAT16 : MCPU_BFLOAT16,
                api.stream(query.device().index())),
     op);
  written(query);
  if (key) written(*key);
}

// table without a value: the write alone.
inline void write(const Api& api, const Opt& positions, const Opt& query, const at::Tensor& key, const at::Tensor& value,
                  const Opt& table, bool is_neox, const at::Tensor& key_cache, const at::Tensor& value_cache,
                  const at::Tensor& slot_mapping, const Opt& k_scale, const Opt& v_scale) {
  const char* op = table ? "rotary_reshape_and_cache" : "reshape_and_cache";
  on_device(api, key, op, "key");
  same_device(positions, key, op, "positions");
  same_device(query, key, op, "query");
  same_device(value, key, op, "value");
  same_device(table, key, op, "cos_sin_cache");
  same_device(key_cache, key, op, "key_cache");
  same_device(value_cache, key, op, "value_cache");
  same_device(slot_mapping, key, op, "slot_mapping");
  same_device(k_scale, key, op, "k_scale");
  same_device(v_scale, key, op, "v_scale");
  no_gradient(query, op, "query");
  no_gradient(key, op, "key");
  no_gradient(value, op, "value");
  no_gradient(table, op, "cos_sin_cache");
  no_gradient(key_cache, value_cache, k_scale, v_scale, op);
  const auto type = key.scalar_type();
  TORCH_CHECK(value.scalar_type() == type && (!query || query->scalar_type() == type), op,
              ": query, key and value must have one type");
  const mcpuKvCache c = cache_of(key_cache, value_cache, k_scale, v_scale, type, true, op);
  const Heads k = heads_of(key, c.head_size, op, "key"), v = heads_of(value, c.head_size, op, "value");
  TORCH_CHECK(k.heads == c.kv_heads && v.heads == c.kv_heads && v.tokens == k.tokens, op, ": key and value must be [", k.tokens,
              ", ", c.kv_heads, ", ", c.head_size, "], as the cache is");
  TORCH_CHECK(slot_mapping.scalar_type() == at::kLong && slot_mapping.dim() == 1 && slot_mapping.size(0) == k.tokens &&
                  slot_mapping.is_contiguous(),
              op, ": slot_mapping must be a contiguous int64 [", k.tokens, "] tensor");
  Heads q;
  int64_t part = 0;
  if (table) {
    TORCH_CHECK(positions, op, ": positions are needed");
    check_table(*positions, k.tokens, *table, op);
    part = table->size(1);
    TORCH_CHECK(part > 0 && part <= c.head_size, op, ": rotary_dim ", part, " must be in 1..head_size (", c.head_size, ")");
    if (query) {
      q = heads_of(*query, c.head_size, op, "query");
      TORCH_CHECK(q.tokens == k.tokens, op, ": query has ", q.tokens, " tokens, key ", k.tokens);
      disjoint<2>({Dim{q.token_stride, q.tokens}, Dim{q.head_stride, q.heads}}, part, op, "query");
      const Place place = place_of(*query, q, part);
      TORCH_CHECK(!overlap(place, place_of(key, k, c.head_size)) && !overlap(place, place_of(value, v, c.head_size)), op,
                  ": query is written and must not overlap key or value");
    }
  }
  ok(api,
     api.write(table ? positions->const_data_ptr<int64_t>() : nullptr, k.tokens, table && query ? query->data_ptr() : nullptr,
               static_cast<int>(q.heads), q.token_stride, q.head_stride, key.const_data_ptr(), k.token_stride, k.head_stride,
               value.const_data_ptr(), v.token_stride, v.head_stride, static_cast<int>(part),
               table ? table->const_data_ptr<float>() : nullptr, table ? table->size(0) : 0, is_neox, half_code(type, op),
               slot_mapping.const_data_ptr<int64_t>(), &c, api.stream(key.device().index())),
     op);
  if (table && query) written(*query);
  written(key_cache);
  written(value_cache);
  if (c.scale_mode == MCPU_KV_SCALE_TOKEN) {
    written(*k_scale);
    written(*v_scale);
  }
}

inline void gather_cache(const Api& api, const at::Tensor& key_cache, const at::Tensor& value_cache,
                         const at::Tensor& block_table, const at::Tensor& cu_seq_lens, const at::Tensor& key_out,
                         const at::Tensor& value_out, const Opt& k_scale, const Opt& v_scale, const Opt& seq_starts) {
  const char* op = "gather_cache";
  on_device(api, key_cache, op, "key_cache");
  same_device(value_cache, key_cache, op, "value_cache");
  same_device(block_table, key_cache, op, "block_table");
  same_device(cu_seq_lens, key_cache, op, "cu_seq_lens");
  same_device(key_out, key_cache, op, "key_out");
  same_device(value_out, key_cache, op, "value_out");
  same_device(k_scale, key_cache, op, "k_scale");
  same_device(v_scale, key_cache, op, "v_scale");
  same_device(seq_starts, key_cache, op, "seq_starts");
  no_gradient(key_cache, value_cache, k_scale, v_scale, op);
  no_gradient(key_out, op, "key_out");
  no_gradient(value_out, op, "value_out");
  TORCH_CHECK(value_out.scalar_type() == key_out.scalar_type() && value_out.sizes() == key_out.sizes(), op,
              ": key_out and value_out must have one shape and type");
  const mcpuKvCache c = cache_of(key_cache, value_cache, k_scale, v_scale, key_out.scalar_type(), false, op);
  TORCH_CHECK(key_out.dim() == 3 && key_out.size(1) == c.kv_heads && key_out.size(2) == c.head_size &&
                  key_out.is_contiguous() && value_out.is_contiguous(),
              op, ": outputs must be contiguous [tokens, ", c.kv_heads, ", ", c.head_size, "] tensors");
  TORCH_CHECK(!overlap(place_of<0>(key_out, {}, key_out.numel()), place_of<0>(value_out, {}, value_out.numel())), op,
              ": key_out and value_out are written and must not overlap");
  check_block_table(block_table, op);
  const int64_t batch = block_table.size(0), width = block_table.size(1);
  check_int32(cu_seq_lens, batch + 1, op, "cu_seq_lens");
  if (seq_starts) check_int32(*seq_starts, batch, op, "seq_starts");
  ok(api,
     api.gather(&c, block_table.const_data_ptr<int32_t>(), std::max(block_table.stride(0), width), width, batch,
                cu_seq_lens.const_data_ptr<int32_t>(), seq_starts ? seq_starts->const_data_ptr<int32_t>() : nullptr,
                key_out.data_ptr(), value_out.data_ptr(), key_out.size(0), half_code(key_out.scalar_type(), op),
                api.stream(key_cache.device().index())),
     op);
  written(key_out);
  written(value_out);
}

inline std::tuple<at::Tensor, at::Tensor> tree_attention(
    const Api& api, const at::Tensor& query, const at::Tensor& key_cache, const at::Tensor& value_cache,
    const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& cu_query_lens, int64_t max_query_len,
    double scale, const Opt& tree_mask, const Opt& k_scale, const Opt& v_scale, const Opt& out_given, bool return_lse) {
  const char* op = "tree_attention";
  on_device(api, query, op, "query");
  same_device(key_cache, query, op, "key_cache");
  same_device(value_cache, query, op, "value_cache");
  same_device(block_table, query, op, "block_table");
  same_device(seq_lens, query, op, "seq_lens");
  same_device(cu_query_lens, query, op, "cu_query_lens");
  same_device(tree_mask, query, op, "tree_mask");
  same_device(k_scale, query, op, "k_scale");
  same_device(v_scale, query, op, "v_scale");
  same_device(out_given, query, op, "out");
  no_gradient(query, op, "query");
  no_gradient(out_given, op, "out");
  no_gradient(key_cache, value_cache, k_scale, v_scale, op);
  const auto type = query.scalar_type();
  const mcpuKvCache c = cache_of(key_cache, value_cache, k_scale, v_scale, type, false, op);
  TORCH_CHECK(query.dim() == 3 && query.size(2) == c.head_size && query.stride(2) == 1, op,
              ": query must be [tokens, heads, ", c.head_size, "] with contiguous heads of the cache's size");
  const int64_t tokens = query.size(0), heads = query.size(1);
  TORCH_CHECK(c.kv_heads > 0 && heads > 0 && heads % c.kv_heads == 0, op, ": ", heads, " query heads cannot share ", c.kv_heads,
              " key / value heads evenly");
  check_block_table(block_table, op);
  const int64_t batch = block_table.size(0), width = block_table.size(1);
  check_int32(seq_lens, batch, op, "seq_lens");
  check_int32(cu_query_lens, batch + 1, op, "cu_query_lens");
  int64_t words = 0, mask_stride = 0;
  if (tree_mask) {
    const at::Tensor& m = *tree_mask;
    TORCH_CHECK(m.scalar_type() == at::kLong && m.dim() == 2 && m.size(0) == tokens && m.size(1) >= 1 &&
                    (m.stride(1) == 1 || m.size(1) == 1) && (tokens <= 1 || m.stride(0) >= m.size(1)),
                op, ": tree_mask must be an int64 [", tokens, ", words] tensor with contiguous rows");
    words = m.size(1);
    mask_stride = std::max(m.stride(0), words);
  }
  at::Tensor out, lse;
  if (out_given) {
    out = *out_given;
    TORCH_CHECK(out.sizes() == query.sizes() && out.scalar_type() == type && out.stride(2) == 1, op, ": out must be a ", type, " ",
                query.sizes(), " tensor with contiguous heads");
    disjoint<2>({Dim{out.stride(0), tokens}, Dim{out.stride(1), heads}}, c.head_size, op, "out");
    TORCH_CHECK((out.const_data_ptr() == query.const_data_ptr() && out.strides() == query.strides()) ||
                    !overlap(place_of(out), place_of(query)),
                op, ": out is written and must be query itself or not overlap it");
  } else {
    out = at::empty(query.sizes(), query.options());
  }
  if (return_lse) lse = at::empty({tokens, heads}, query.options().dtype(at::kFloat));
  uint64_t need = 0;
  ok(api, api.workspace(max_query_len, static_cast<int>(heads), c.kv_heads, c.head_size, &need), op);
  const at::Tensor work = at::empty({static_cast<int64_t>(need)}, query.options().dtype(at::kByte));
  ok(api,
     api.attend(query.const_data_ptr(), query.stride(0), query.stride(1), tokens, static_cast<int>(heads), out.data_ptr(),
                out.stride(0), out.stride(1), return_lse ? lse.data_ptr<float>() : nullptr, half_code(type, op), &c,
                block_table.const_data_ptr<int32_t>(), std::max(block_table.stride(0), width), width, batch,
                seq_lens.const_data_ptr<int32_t>(), cu_query_lens.const_data_ptr<int32_t>(), max_query_len,
                tree_mask ? tree_mask->const_data_ptr<int64_t>() : nullptr, mask_stride, words, static_cast<float>(scale),
                work.data_ptr(), need, api.stream(query.device().index())),
     op);
  if (out_given) written(out);
  return {out, lse};
}

}  // namespace attention
}  // namespace mcpu_torch
