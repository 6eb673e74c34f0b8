// Attention's forward kernels for f16.
#include "attention_fwd.h"

namespace nf {
namespace attn {
template int launch_fwd<f16>(const FwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
