// attention_f32.hip — the attention kernels of float32 tensors.
#include "attention_kernels.h"

void tohip::launch_attention_f32(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { launch_attention<kF32>(a, p, s); }
void tohip::launch_prefix_f32(const AttnArgs& pre, const AttnPlan& p0, const AttnArgs& own, const AttnPlan& p1, hipStream_t s) {
    launch_prefix<kF32>(pre, p0, own, p1, s);
}
