// BF16 instantiations of the varlen attention gradient's kernels
// (varlen_backward_kernel.h).
#include "varlen_backward_kernel.h"

namespace va {

template <>
void launch_varlen_backward<true, 64>(const VarlenBwdParams& p, hipStream_t st) {
  launch_varlen_backward_d<true, 64>(p, st);
}
template <>
void launch_varlen_backward<true, 128>(const VarlenBwdParams& p, hipStream_t st) {
  launch_varlen_backward_d<true, 128>(p, st);
}

}  // namespace va
