// bf16 instances of the segment attention backward.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void bwd_bf16(const Args& a, int axes, int nwq, int nwk, int nblk,
              hipStream_t st) {
  run_bwd<__bf16>(a, axes, nwq, nwk, nblk, st);
}
}  // namespace segattn
}  // namespace dgmc
