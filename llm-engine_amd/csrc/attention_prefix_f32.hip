// Shared-prefix attention of fp32 accuracy: fp32 activations or an fp32 cache, or
// two 16-bit types.
#include "attention_prefix_wg.h"

namespace le {

hipError_t attention_prefix_f32(const PrefixParams& p, int act_dtype, int kv_dtype, hipStream_t stream) {
  return with_dtype(act_dtype, [&](auto act) {
    return with_dtype(kv_dtype, [&](auto kv) {
      using ACT = decltype(act);
      using KV = decltype(kv);
      if constexpr (!std::is_same_v<ACT, KV> || sizeof(KV) == 4) {
        return p.head_dim == 64 ? pfx::launch_prefix<ACT, KV, 64>(p, stream)
                                : pfx::launch_prefix<ACT, KV, 128>(p, stream);
      } else {
        return hipErrorInvalidValue;  // attention_prefix has these
      }
    });
  });
}

}  // namespace le
