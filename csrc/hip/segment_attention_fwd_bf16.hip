// Segment attention forward: bf16, inference (short segments: FINE).
#include "segment_attention_fwd.h"

namespace dgmc {
namespace segattn {
void fwd_bf16(const Args& a, int axes, int nw, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_fwd<Bf16, 32, 1, true>(a, axes, st)
            : launch_fwd<Bf16, 32, 4, false>(a, axes, st);
  else if (a.D <= 64)
    nw == 1 ? launch_fwd<Bf16, 64, 1, true>(a, axes, st)
            : launch_fwd<Bf16, 64, 4, false>(a, axes, st);
  else
    nw == 1 ? launch_fwd<Bf16, 128, 1, true>(a, axes, st)
            : launch_fwd<Bf16, 128, 4, false>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
