// Segment attention backward, dkv: fp32 in three bf16 planes.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dkv_x6(const Args& a, int axes, hipStream_t st) {
  a.D <= 32 ? launch_dkv<X6, 32, 4>(a, axes, st)
            : launch_dkv<X6, 64, 4>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
