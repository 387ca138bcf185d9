// bf16 instances of the general attention kernels (attention.h).
#include "attention.h"

namespace dtf {
namespace attn {
int fwd_bf16(const Args& a, hipStream_t s) { return dispatch_fwd<unsigned short>(a, s); }
int bwd_bf16(const Args& a, hipStream_t s) { return dispatch_bwd<unsigned short>(a, s); }
}  // namespace attn
}  // namespace dtf
