// The attention entry points of the C-ABI, and the kernels for a cache of the heads' own type.
#include "attention_launch.hpp"

namespace iris_amd {
namespace calls {
IRIS_ATTENTION_CALLS(, 0)
IRIS_ATTENTION_CALLS(extern, IRIS_DTYPE_E4M3)
IRIS_ATTENTION_CALLS(extern, IRIS_DTYPE_E5M2)

namespace {
// f(the codes' type) for a cache in 8 bits
template <class F>
int with_codes(const iris_cache_scales* s, F f) {
  if (!s) return hipErrorInvalidValue;
  if (s->code == IRIS_DTYPE_E4M3) return f(std::integral_constant<int, IRIS_DTYPE_E4M3>{});
  if (s->code == IRIS_DTYPE_E5M2) return f(std::integral_constant<int, IRIS_DTYPE_E5M2>{});
  return hipErrorInvalidValue;
}
}  // namespace
}  // namespace calls
}  // namespace iris_amd

using namespace iris_amd::calls;

extern "C" int64_t iris_attention_workspace_elems(int32_t head_dim) {
  if (head_dim <= 0 || head_dim > MAX_HEAD_DIM) return 0;
  return COUNTERS + ROW_SLOTS * row_slot(head_dim);
}

extern "C" int iris_attention_launch(const iris_attention_args* args, void* stream) {
  return args ? launch_call<0>(*args, nullptr, stream) : hipErrorInvalidValue;
}
extern "C" int iris_attention_plan(const iris_attention_args* args, int32_t num_cus, iris_attention_plan_info* plan) {
  return args && plan && num_cus >= 0 ? plan_call<0>(*args, nullptr, num_cus, plan) : hipErrorInvalidValue;
}
extern "C" int iris_attention_kernel_info(const iris_attention_args* args, int* n_regs, int* n_spills) {
  return args && n_regs && n_spills ? info_call<0>(*args, nullptr, n_regs, n_spills) : hipErrorInvalidValue;
}

extern "C" int iris_quantized_attention_launch(const iris_attention_args* args, const iris_cache_scales* scales, void* stream) {
  if (!args) return hipErrorInvalidValue;
  return with_codes(scales, [&](auto ct) { return launch_call<ct.value>(*args, scales, stream); });
}
extern "C" int iris_quantized_attention_plan(const iris_attention_args* args, const iris_cache_scales* scales, int32_t num_cus,
                                             iris_attention_plan_info* plan) {
  if (!args || !plan || num_cus < 0) return hipErrorInvalidValue;
  return with_codes(scales, [&](auto ct) { return plan_call<ct.value>(*args, scales, num_cus, plan); });
}
extern "C" int iris_quantized_attention_item(const iris_attention_args* args, const iris_cache_scales* scales, int32_t num_cus, int64_t place, int64_t* item) {
  if (!args || !item || num_cus < 0) return hipErrorInvalidValue;
  return with_codes(scales, [&](auto ct) { return item_call<ct.value>(*args, scales, num_cus, place, item); });
}
extern "C" int iris_quantized_attention_kernel_info(const iris_attention_args* args, const iris_cache_scales* scales, int* n_regs, int* n_spills) {
  if (!args || !n_regs || !n_spills) return hipErrorInvalidValue;
  return with_codes(scales, [&](auto ct) { return info_call<ct.value>(*args, scales, n_regs, n_spills); });
}
