// attention_f16.hip — the attention kernels of float16 tensors.
#include "attention_kernels.h"

void tohip::launch_attention_f16(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { launch_attention<kF16>(a, p, s); }
