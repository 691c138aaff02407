// The gated linear layer's products with float32 operands (gated_core.h).
#define PCST_GATED_IMPL
#include "gated_core.h"

namespace pcst {
namespace gated {
template <>
int fwd<EF32>(const FwdCall& c, void* stream) {
  return fwd_out<EF32, EF32::T>(c, as_stream(stream));
}
template <>
int bwd<EF32>(const BwdCall& c, void* stream) {
  return bwd_impl<EF32>(c, as_stream(stream));
}
}  // namespace gated
}  // namespace pcst
