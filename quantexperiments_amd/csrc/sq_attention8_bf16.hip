// attention kernels over an 8-bit cache for bf16
#include "sq_attention8.h"

namespace sq {
int attn8_launch_bf16(const Attn8Shared& a, const AttnPlan& p, hipStream_t s) { return attn8_launch<SQ_BF16>(a, p, s); }
}  // namespace sq
