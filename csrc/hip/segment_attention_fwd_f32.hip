// fp32 instances of the segment attention forward.
#include "segment_attention_fwd.h"

namespace dgmc {
namespace segattn {
void fwd_f32(const Args& a, int axes, int nw, hipStream_t st) {
  run_fwd<float, false>(a, axes, nw, st);
}
}  // namespace segattn
}  // namespace dgmc
