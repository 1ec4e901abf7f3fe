#include "attn_impl.h"

namespace cgtp {
template void attn_launch<bf16_t, false, true>(const AttnLaunch&, const AttnScratch*, hipStream_t);
}  // namespace cgtp
