// Segment attention backward, dq: fp32, exact products.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dq_f32(const Args& a, int axes, int nw, int nblk, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_dq<F32, 32, 1>(a, axes, nblk, st)
            : launch_dq<F32, 32, 4>(a, axes, nblk, st);
  else if (a.D <= 64)
    nw == 1 ? launch_dq<F32, 64, 1>(a, axes, nblk, st)
            : launch_dq<F32, 64, 4>(a, axes, nblk, st);
  else
    nw == 1 ? launch_dq<F32, 128, 1>(a, axes, nblk, st)
            : launch_dq<F32, 128, 4>(a, axes, nblk, st);
}
}  // namespace segattn
}  // namespace dgmc
