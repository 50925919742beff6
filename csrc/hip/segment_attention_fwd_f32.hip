// Segment attention forward: fp32, exact products.
#include "segment_attention_fwd.h"

namespace dgmc {
namespace segattn {
void fwd_f32(const Args& a, int axes, int nw, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_fwd<F32, 32, 1, false>(a, axes, st)
            : launch_fwd<F32, 32, 4, false>(a, axes, st);
  else if (a.D <= 64)
    nw == 1 ? launch_fwd<F32, 64, 1, false>(a, axes, st)
            : launch_fwd<F32, 64, 4, false>(a, axes, st);
  else
    nw == 1 ? launch_fwd<F32, 128, 1, false>(a, axes, st)
            : launch_fwd<F32, 128, 4, false>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
