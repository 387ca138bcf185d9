// Instances of the general attention kernels (attention.h): f32, relative bias.
#include "attention.h"

DTF_ATTN_INSTANCE(run_f32_rel, float, kRel)
