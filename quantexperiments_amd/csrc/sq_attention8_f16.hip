// attention kernels over an 8-bit cache for fp16
#include "sq_attention8.h"

namespace sq {
int attn8_launch_f16(const Attn8Shared& a, const AttnPlan& p, hipStream_t s) { return attn8_launch<SQ_F16>(a, p, s); }
}  // namespace sq
