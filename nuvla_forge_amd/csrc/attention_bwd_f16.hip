// Attention's backward kernels for f16.
#include "attention_bwd.h"

namespace nf {
namespace attn {
template int launch_bwd<f16>(const BwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
