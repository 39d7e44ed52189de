// The 8-bit cache's attention for bf16 activations and int8 codes.
#include "kv8_attn.hpp"

namespace slhip {

template <> int kv8_attn_launch<SLHIP_BF16, SLHIP_KV8_I8, kPlain>(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    return kv8_attn_by_dim<SLHIP_BF16, SLHIP_KV8_I8, kPlain>(a, p, st);
}

}  // namespace slhip
