// fp32 instances of the general attention kernels (attention.h).
#include "attention.h"

namespace dtf {
namespace attn {
int fwd_f32(const Args& a, hipStream_t s) { return dispatch_fwd<float>(a, s); }
int bwd_f32(const Args& a, hipStream_t s) { return dispatch_bwd<float>(a, s); }
}  // namespace attn
}  // namespace dtf
