// The attention path on the mcpu device: schemas with vLLM's argument order,
// bodies in attention_ops.h.
#include <torch/library.h>

#include "attention_ops.h"
#include "mcpu_torch.h"

namespace mcpu_torch {
namespace {

const attention::Api kApi = {&mcpu_rotary_embedding,  &mcpu_rotary_reshape_and_cache,
                             &mcpu_gather_cache,      &mcpu_tree_attention,
                             &mcpu_tree_attention_workspace_bytes, &mcpuGetLastErrorString,
                             c10::DeviceType::PrivateUse1, &current_stream_handle};

// The tensors' device as the current one while a call is enqueued.
struct OnDevice {
  explicit OnDevice(const at::Tensor& t) : before(current_device()), here(t.device().index()) {
    if (t.device().type() != c10::DeviceType::PrivateUse1) here = before;
    if (here != before) orSetDevice(here);
  }
  ~OnDevice() {
    if (here != before) orSetDevice(before);
  }
  c10::DeviceIndex before, here;
};

void rotary_embedding(const at::Tensor& positions, at::Tensor& query, const std::optional<at::Tensor>& key, int64_t head_size,
                      const at::Tensor& cos_sin_cache, bool is_neox) {
  OnDevice on(query);
  attention::rotary_embedding(kApi, positions, query, key, head_size, cos_sin_cache, is_neox);
}
void reshape_and_cache(const at::Tensor& key, const at::Tensor& value, at::Tensor& key_cache, at::Tensor& value_cache,
                       const at::Tensor& slot_mapping, const std::optional<at::Tensor>& k_scale,
                       const std::optional<at::Tensor>& v_scale) {
  OnDevice on(key);
  attention::write(kApi, std::nullopt, std::nullopt, key, value, std::nullopt, true, key_cache, value_cache, slot_mapping, k_scale,
                   v_scale);
}
void rotary_reshape_and_cache(const at::Tensor& positions, const std::optional<at::Tensor>& query, const at::Tensor& key,
                              const at::Tensor& value, const at::Tensor& cos_sin_cache, bool is_neox, at::Tensor& key_cache,
                              at::Tensor& value_cache, const at::Tensor& slot_mapping, const std::optional<at::Tensor>& k_scale,
                              const std::optional<at::Tensor>& v_scale) {
  OnDevice on(key);
  attention::write(kApi, positions, query, key, value, cos_sin_cache, is_neox, key_cache, value_cache, slot_mapping, k_scale,
                   v_scale);
}
void gather_cache(const at::Tensor& key_cache, const at::Tensor& value_cache, const at::Tensor& block_table,
                  const at::Tensor& cu_seq_lens, at::Tensor& key_out, at::Tensor& value_out,
                  const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                  const std::optional<at::Tensor>& seq_starts) {
  OnDevice on(key_cache);
  attention::gather_cache(kApi, key_cache, value_cache, block_table, cu_seq_lens, key_out, value_out, k_scale, v_scale, seq_starts);
}
std::tuple<at::Tensor, at::Tensor> tree_attention(const at::Tensor& query, const at::Tensor& key_cache,
                                                  const at::Tensor& value_cache, const at::Tensor& block_table,
                                                  const at::Tensor& seq_lens, const at::Tensor& cu_query_lens,
                                                  int64_t max_query_len, double scale, const std::optional<at::Tensor>& tree_mask,
                                                  const std::optional<at::Tensor>& k_scale,
                                                  const std::optional<at::Tensor>& v_scale) {
  OnDevice on(query);
  return attention::tree_attention(kApi, query, key_cache, value_cache, block_table, seq_lens, cu_query_lens, max_query_len, scale,
                                   tree_mask, k_scale, v_scale, std::nullopt, true);
}

}  // namespace
}  // namespace mcpu_torch

TORCH_LIBRARY_FRAGMENT(mcpu, m) {
  m.def("rotary_embedding(Tensor positions, Tensor(a!) query, Tensor(b!)? key, int head_size, Tensor cos_sin_cache, "
        "bool is_neox) -> ()");
  m.def("reshape_and_cache(Tensor key, Tensor value, Tensor(a!) key_cache, Tensor(b!) value_cache, Tensor slot_mapping, "
        "Tensor(c!)? k_scale=None, Tensor(d!)? v_scale=None) -> ()");
  m.def("rotary_reshape_and_cache(Tensor positions, Tensor(a!)? query, Tensor key, Tensor value, Tensor cos_sin_cache, "
        "bool is_neox, Tensor(b!) key_cache, Tensor(c!) value_cache, Tensor slot_mapping, Tensor(d!)? k_scale=None, "
        "Tensor(e!)? v_scale=None) -> ()");
  m.def("gather_cache(Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor cu_seq_lens, Tensor(a!) key_out, "
        "Tensor(b!) value_out, Tensor? k_scale=None, Tensor? v_scale=None, Tensor? seq_starts=None) -> ()");
  m.def("tree_attention(Tensor query, Tensor key_cache, Tensor value_cache, Tensor block_table, Tensor seq_lens, "
        "Tensor cu_query_lens, int max_query_len, float scale, Tensor? tree_mask=None, Tensor? k_scale=None, "
        "Tensor? v_scale=None) -> (Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(mcpu, PrivateUse1, m) {
  using namespace mcpu_torch;
  m.impl("rotary_embedding", rotary_embedding);
  m.impl("reshape_and_cache", reshape_and_cache);
  m.impl("rotary_reshape_and_cache", rotary_reshape_and_cache);
  m.impl("gather_cache", gather_cache);
  m.impl("tree_attention", tree_attention);
}
