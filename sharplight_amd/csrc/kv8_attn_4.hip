// The 8-bit cache's attention for f32 activations and int8 codes, scores capped, sloped or scaled by a factor that is not positive.
#include "kv8_attn.hpp"

namespace slhip {

template <> int kv8_attn_launch<SLHIP_F32, SLHIP_KV8_I8, kReshaped>(const Kv8AttnArgs& a, const Kv8AttnPlan& p, hipStream_t st)
{
    return kv8_attn_by_dim<SLHIP_F32, SLHIP_KV8_I8, kReshaped>(a, p, st);
}

}  // namespace slhip
