// Shared-prefix attention with q and a cache of one 16-bit type (bf16 or fp16
// MFMA); attention_prefix_f32.hip has every other pair of types.
#include "attention_prefix_wg.h"

namespace le {

hipError_t attention_prefix(const PrefixParams& p, int act_dtype, int kv_dtype, hipStream_t stream) {
  if (act_dtype != kv_dtype || kv_dtype == kDtF32) return attention_prefix_f32(p, act_dtype, kv_dtype, stream);
  return with_dtype16(kv_dtype, [&](auto kv) {
    using KV = decltype(kv);
    return p.head_dim == 64 ? pfx::launch_prefix<KV, KV, 64>(p, stream) : pfx::launch_prefix<KV, KV, 128>(p, stream);
  });
}

}  // namespace le
