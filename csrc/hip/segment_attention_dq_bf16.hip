// Segment attention backward, dq: bf16.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dq_bf16(const Args& a, int axes, int nw, int nblk, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_dq<Bf16, 32, 1>(a, axes, nblk, st)
            : launch_dq<Bf16, 32, 4>(a, axes, nblk, st);
  else if (a.D <= 64)
    nw == 1 ? launch_dq<Bf16, 64, 1>(a, axes, nblk, st)
            : launch_dq<Bf16, 64, 4>(a, axes, nblk, st);
  else
    nw == 1 ? launch_dq<Bf16, 128, 1>(a, axes, nblk, st)
            : launch_dq<Bf16, 128, 4>(a, axes, nblk, st);
}
}  // namespace segattn
}  // namespace dgmc
