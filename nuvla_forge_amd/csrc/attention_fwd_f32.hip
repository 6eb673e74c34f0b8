// Attention's forward kernels for fp32.
#include "attention_fwd.h"

namespace nf {
namespace attn {
template int launch_fwd<float>(const FwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
