// bf16 instances of the segment attention forward.
#include "segment_attention_fwd.h"

namespace dgmc {
namespace segattn {
void fwd_bf16(const Args& a, int axes, int nw, hipStream_t st) {
  run_fwd<__bf16, false>(a, axes, nw, st);
}
}  // namespace segattn
}  // namespace dgmc
