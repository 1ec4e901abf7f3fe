#include "attn_impl.h"

namespace cgtp {
void attn_launch_f32(const cgtp_attn_args& a, const AttnScratch* w, hipStream_t s) { launch_type<float>(a, w, s); }
}  // namespace cgtp
