// The gated linear layer's products with float16 operands (gated_core.h).
#define PCST_GATED_IMPL
#include "gated_core.h"

namespace pcst {
namespace gated {
template <>
int fwd<EF16>(const FwdCall& c, void* stream) {
  return fwd_out<EF16, EF16::T>(c, as_stream(stream));
}
template <>
int bwd<EF16>(const BwdCall& c, void* stream) {
  return bwd_impl<EF16>(c, as_stream(stream));
}
}  // namespace gated
}  // namespace pcst
