// Instances of the general attention kernels (attention.h): bf16, no bias.
#include "attention.h"

DTF_ATTN_INSTANCE(run_bf16_plain, unsigned short, kPlain)
