// Entry points of the attentional operators (segment_attention.hip,
// layer_norm.hip, match_logprob.hip); attentional.cpp puts the autograd
// nodes around them.
#pragma once

#include <ATen/ATen.h>

#include <tuple>

namespace dgmc {

using OptTensor = c10::optional<at::Tensor>;

// Bucket layout of a bias table: half-width, log2 of the buckets per octave,
// first distance of the last bucket.
struct BucketLayout {
  int64_t half, mbits;
  double dmax;
};

namespace segattn {

// `x6`: long fp32 segments on the bf16 matrix cores, three terms an operand.
// (out, lo, stat): lo (bf16 rest of out's rounding, bf16 only) and stat (fp32
// [Nq, H, 2], the softmax's maximum and 1 / sum) are empty unless `train`.
std::tuple<at::Tensor, at::Tensor, at::Tensor> forward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& ptr_q, const at::Tensor& ptr_k, double scale,
    double cap, const OptTensor& bias, const OptTensor& pos_q,
    const OptTensor& pos_k, const BucketLayout& layout, bool x6, bool train);

// (dq, dk, dv, dbias): dbias (fp32) is empty without a bias.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> backward(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& v, const at::Tensor& out, const at::Tensor& lo,
    const at::Tensor& stat, const at::Tensor& ptr_q, const at::Tensor& ptr_k,
    double scale, double cap, const OptTensor& bias, const OptTensor& pos_q,
    const OptTensor& pos_k, const BucketLayout& layout, bool x6);

}  // namespace segattn

// x: [..., C].  (y, s, stat): s is empty without a residual, stat [rows, 2]
// (mean, rstd) empty unless `train`.
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd(
    const at::Tensor& x, const OptTensor& residual, const OptTensor& weight,
    const OptTensor& bias, double eps, bool train);

// (dx, dw, db): dw and db fp32, empty unless `with_weight`.
std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_bwd(
    const at::Tensor& dy, const OptTensor& ds, const at::Tensor& s,
    const at::Tensor& stat, const OptTensor& weight, bool with_weight);

// (logp [R], entropy [R], top_lp [R, k], top_idx [R, k], stat): stat [R, 2]
// is empty unless `train`.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
match_logprob_fwd(const at::Tensor& z, const at::Tensor& y,
                  const OptTensor& n, int64_t k, bool train);

// dz [R, V], contiguous, in z's type.
at::Tensor match_logprob_bwd(const OptTensor& gl, const OptTensor& gh,
                             const at::Tensor& z, const at::Tensor& y,
                             const OptTensor& n, const at::Tensor& logp,
                             const at::Tensor& ent, const at::Tensor& stat);

}  // namespace dgmc
