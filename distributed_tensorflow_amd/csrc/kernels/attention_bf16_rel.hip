// Instances of the general attention kernels (attention.h): bf16, relative bias.
#include "attention.h"

DTF_ATTN_TWO_PARTS(kRel)
DTF_ATTN_INSTANCE(run_bf16_rel, unsigned short, kRel)
