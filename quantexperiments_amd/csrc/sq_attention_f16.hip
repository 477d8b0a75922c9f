// attention kernels for fp16
#include "sq_attention.h"

namespace sq {
int attn_launch_f16(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { return attn_launch<SQ_F16>(a, p, s); }
}  // namespace sq
