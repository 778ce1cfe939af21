// F16 instantiations of the varlen attention gradient's kernels
// (varlen_backward_kernel.h).
#include "varlen_backward_kernel.h"

namespace va {

template <>
void launch_varlen_backward<false, 64>(const VarlenBwdParams& p, hipStream_t st) {
  launch_varlen_backward_d<false, 64>(p, st);
}
template <>
void launch_varlen_backward<false, 128>(const VarlenBwdParams& p, hipStream_t st) {
  launch_varlen_backward_d<false, 128>(p, st);
}

}  // namespace va
