// Segment attention forward: fp32 in three bf16 planes.
#include "segment_attention_fwd.h"

namespace dgmc {
namespace segattn {
void fwd_x6(const Args& a, int axes, hipStream_t st) {
  // (four waves; short segments and wide heads take the exact products)
  a.D <= 32 ? launch_fwd<X6, 32, 4, false>(a, axes, st)
            : launch_fwd<X6, 64, 4, false>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
