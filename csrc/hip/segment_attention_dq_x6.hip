// Segment attention backward, dq: fp32 in three bf16 planes, without a table.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dq_x6(const Args& a, hipStream_t st) {
  a.D <= 32 ? launch_dq<X6, 32, 4>(a, 0, 0, st)
            : launch_dq<X6, 64, 4>(a, 0, 0, st);
}
}  // namespace segattn
}  // namespace dgmc
