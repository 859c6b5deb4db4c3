// attention_bf16.hip — the attention kernels of bfloat16 tensors.
#include "attention_kernels.h"

void tohip::launch_attention_bf16(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { launch_attention<kBF16>(a, p, s); }
void tohip::launch_prefix_bf16(const AttnArgs& pre, const AttnPlan& p0, const AttnArgs& own, const AttnPlan& p1, hipStream_t s) {
    launch_prefix<kBF16>(pre, p0, own, p1, s);
}
