// bf16 instances of the segment attention backward.
#include "segment_attention_bwd.h"

namespace dgmc {
namespace segattn {
void dq_bf16(const Args& a, int axes, int nw, int nblk, hipStream_t st) {
  run_dq<__bf16>(a, axes, nw, nblk, st);
}
void dkv_bf16(const Args& a, int axes, int nw, hipStream_t st) {
  run_dkv<__bf16>(a, axes, nw, st);
}
}  // namespace segattn
}  // namespace dgmc
