// Segment attention backward, dkv: bf16.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dkv_bf16(const Args& a, int axes, int nw, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_dkv<Bf16, 32, 1>(a, axes, st)
            : launch_dkv<Bf16, 32, 4>(a, axes, st);
  else if (a.D <= 64)
    nw == 1 ? launch_dkv<Bf16, 64, 1>(a, axes, st)
            : launch_dkv<Bf16, 64, 4>(a, axes, st);
  else
    nw == 1 ? launch_dkv<Bf16, 128, 1>(a, axes, st)
            : launch_dkv<Bf16, 128, 4>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
