// The gated linear layer's forward on e4m3 operands with a scale for each row (gated_core.h).
#define PCST_GATED_IMPL
#include "gated_core.h"

namespace pcst {
namespace gated {
template <>
int fwd<EE4M3>(const FwdCall& c, void* stream) {
  hipStream_t s = as_stream(stream);
  if (c.out_type == kBF16) return fwd_out<EE4M3, __bf16>(c, s);
  return fwd_out<EE4M3, _Float16>(c, s);
}
}  // namespace gated
}  // namespace pcst
