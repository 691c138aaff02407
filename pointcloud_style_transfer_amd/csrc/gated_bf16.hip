// The gated linear layer's products with bfloat16 operands (gated_core.h).
#define PCST_GATED_IMPL
#include "gated_core.h"

namespace pcst {
namespace gated {
template <>
int fwd<EBF16>(const FwdCall& c, void* stream) {
  return fwd_out<EBF16, EBF16::T>(c, as_stream(stream));
}
template <>
int bwd<EBF16>(const BwdCall& c, void* stream) {
  return bwd_impl<EBF16>(c, as_stream(stream));
}
}  // namespace gated
}  // namespace pcst
