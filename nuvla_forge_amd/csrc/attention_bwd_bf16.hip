// Attention's backward kernels for bf16.
#include "attention_bwd.h"

namespace nf {
namespace attn {
template int launch_bwd<bf16>(const BwdArgs &, const Sizes &, hipStream_t);
}  // namespace attn
}  // namespace nf
