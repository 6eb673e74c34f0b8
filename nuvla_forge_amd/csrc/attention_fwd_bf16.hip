// Attention's forward kernels for bf16.
#include "attention_fwd.h"

namespace nf {
namespace attn {
template int launch_fwd<bf16>(const FwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
