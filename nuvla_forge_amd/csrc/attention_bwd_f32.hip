// Attention's backward kernels for fp32.
#include "attention_bwd.h"

namespace nf {
namespace attn {
template int launch_bwd<float>(const BwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
