// attention kernels for bf16
#include "sq_attention.h"

namespace sq {
int attn_launch_bf16(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { return attn_launch<SQ_BF16>(a, p, s); }
}  // namespace sq
