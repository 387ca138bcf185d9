// Instances of the general attention kernels (attention.h): f32, key bias, with or without a relative one.
#include "attention.h"

DTF_ATTN_INSTANCE(run_f32_keys, float, kKeys)
