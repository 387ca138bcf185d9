// Instances of the general attention kernels (attention.h): bf16, key bias, with or without a relative one.
#include "attention.h"

DTF_ATTN_TWO_PARTS(kKeys)
DTF_ATTN_INSTANCE(run_bf16_keys, unsigned short, kKeys)
