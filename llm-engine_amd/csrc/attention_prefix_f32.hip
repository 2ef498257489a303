// Shared-prefix attention on the fp32 MFMA: fp32 activations or an fp32 cache.
#include "attention_prefix_wg.h"

namespace le {

hipError_t attention_prefix_f32(const PrefixParams& p, int act_dtype, int kv_dtype, hipStream_t stream) {
  return with_dtype(act_dtype, [&](auto act) {
    return with_dtype(kv_dtype, [&](auto kv) {
      using ACT = decltype(act);
      using KV = decltype(kv);
      if constexpr (std::is_same_v<pfx::operand<ACT, KV>, float>) {
        return p.head_dim == 64 ? pfx::launch_prefix<ACT, KV, 64>(p, stream)
                                : pfx::launch_prefix<ACT, KV, 128>(p, stream);
      } else {
        return hipErrorInvalidValue;  // attention_prefix has these
      }
    });
  });
}

}  // namespace le
