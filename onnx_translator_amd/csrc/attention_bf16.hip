// attention_bf16.hip — the attention kernels of bfloat16 tensors.
#include "attention_kernels.h"

void tohip::launch_attention_bf16(const AttnArgs& a, const AttnPlan& p, hipStream_t s) { launch_attention<kBF16>(a, p, s); }
