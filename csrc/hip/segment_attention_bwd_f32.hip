// fp32 instances of the segment attention backward.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dq_f32(const Args& a, int axes, int nw, int nblk, hipStream_t st) {
  run_dq<float>(a, axes, nw, nblk, st);
}
void dkv_f32(const Args& a, int axes, int nw, hipStream_t st) {
  run_dkv<float>(a, axes, nw, st);
}
}  // namespace segattn
}  // namespace dgmc
