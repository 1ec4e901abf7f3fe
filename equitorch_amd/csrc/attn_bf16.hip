#include "attn_impl.h"

namespace cgtp {
void attn_launch_bf16(const cgtp_attn_args& a, const AttnScratch* w, hipStream_t s) { launch_type<bf16_t>(a, w, s); }
}  // namespace cgtp
