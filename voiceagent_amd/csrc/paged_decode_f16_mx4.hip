// F16 instantiations of the paged decode over MXFP4 pools (paged_decode_mx4.h).
#include "paged_decode_mx4.h"

namespace va {

template <>
bool launch_paged_decode_mx4<F16>(int D, int G, const DecodeMx4Params& p, dim3 grid,
                                   hipStream_t s) {
  return dispatch_mx4_d<F16>(D, G, p, grid, s);
}

}  // namespace va
