// Segment attention backward, dkv: fp32, exact products.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dkv_f32(const Args& a, int axes, int nw, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_dkv<F32, 32, 1>(a, axes, st)
            : launch_dkv<F32, 32, 4>(a, axes, st);
  else if (a.D <= 64)
    nw == 1 ? launch_dkv<F32, 64, 1>(a, axes, st)
            : launch_dkv<F32, 64, 4>(a, axes, st);
  else
    nw == 1 ? launch_dkv<F32, 128, 1>(a, axes, st)
            : launch_dkv<F32, 128, 4>(a, axes, st);
}
}  // namespace segattn
}  // namespace dgmc
