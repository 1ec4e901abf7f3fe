#include "attn_impl.h"

namespace cgtp {
template void attn_launch<f16_t, false, false>(const AttnLaunch&, const AttnScratch*, hipStream_t);
}  // namespace cgtp
