// Segment attention: entry points, the join of split keys and the sum of the
// bias table's gradient.  The kernels are in segment_attention_{fwd,bwd}.h,
// instantiated per type in segment_attention_{fwd,bwd}_{bf16,f32}.hip.
#include "segment_attention.h"

namespace dgmc {
namespace segattn {

void fwd_bf16(const Args& a, int axes, int nw, hipStream_t st);
void fwd_f32(const Args& a, int axes, int nw, hipStream_t st);
void bwd_bf16(const Args& a, int axes, int nwq, int nwk, int nblk,
              hipStream_t st);
void bwd_f32(const Args& a, int axes, int nwq, int nwk, int nblk,
             hipStream_t st);

constexpr int kMaxSplits = 64;        // one per lane of the joining wave

// One wave per (row, head): o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s
// over the splits in order.
template <typename T>
__global__ __launch_bounds__(256) void join_kernel(const Args a) {
  const int64_t rows = (int64_t)a.Nq * a.H;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f;
  if (lane < a.splits) {
    m = a.part_ml[(lane * rows + row) * 2];
    l = a.part_ml[(lane * rows + row) * 2 + 1];
  }
  const float M = wave_max(m);
  // (a split without a finite score has l = 0: weight 0)
  const float w = l == 0.f ? 0.f : exp2_(m - M);
  const float L = wave_sum(w * l);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  float o[2] = {0.f, 0.f};
  for (int s = 0; s < a.splits; ++s) {
    const float ws = lane_of(w, s);
    const float* p = a.part_o + (s * rows + row) * a.D;
#pragma unroll
    for (int k = 0; k < 2; ++k)
      if (lane + 64 * k < a.D && ws != 0.f) o[k] += ws * p[lane + 64 * k];
  }
  T* out = (T*)a.out + row * a.D;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (lane + 64 * k < a.D) out[lane + 64 * k] = (T)(o[k] * inv);
  if (lane == 0 && a.lse) a.lse[row] = L == 0.f ? INFINITY : M + log2f(L);
}

// dT[head][c] = sum over the workgroups' parts, in order.  One workgroup per
// head: 4 lanes groups of 64 slots each take every fourth part.
__global__ __launch_bounds__(256) void bias_sum_kernel(
    const float* __restrict__ part, float* __restrict__ out, int nblk, int KV,
    int G, int slots, int nb, int half, int axes) {
  __shared__ float red[4][kSlots];
  const int head = blockIdx.x, kvh = head / G, g = head % G;
  const int s = threadIdx.x & 63, p = threadIdx.x >> 6;
  float sum = 0.f;
  if (s < slots)
    for (int b = p; b < nblk; b += 4)
      sum += part[(((int64_t)b * KV + kvh) * G + g) * slots + s];
  red[p][s] = sum;
  __syncthreads();
  if (threadIdx.x >= nb) return;
  const int c = threadIdx.x, w = 2 * half + 1, W = w + 1;
  const int y = c % w, x = axes == 1 ? 0 : c / w;
  const int ys = y < half ? y : y + 1, xs = x < half ? x : x + 1;
  const int t = axes == 1 ? ys : xs * W + ys;
  out[(int64_t)head * nb + c] =
      (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]);
}

static void check_heads(const at::Tensor& t, const char* name,
                        const at::Tensor& like) {
  TORCH_CHECK(t.dim() == 3, "segment_attention: ", name,
              " must be [nodes, heads, dim]");
  TORCH_CHECK(t.is_cuda() && t.device() == like.device(),
              "segment_attention: ", name, " must be on ", like.device());
  TORCH_CHECK(t.scalar_type() == like.scalar_type(), "segment_attention: ",
              name, " must be ", like.scalar_type());
  TORCH_CHECK(t.numel() == 0 || t.size(2) == 1 || t.stride(2) == 1,
              "segment_attention: ", name,
              "'s last dimension must be contiguous");
}

static void check_index(const at::Tensor& t, const char* name, int dim,
                        const at::Tensor& like) {
  TORCH_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt &&
                  t.dim() == dim && t.is_contiguous(),
              "segment_attention: ", name, " must be a contiguous ", dim,
              "-d int32 tensor on ", like.device());
}

// 16-byte loads of whole rows: base, row and head strides and the width are
// multiples of 16 bytes.
static int rows16(const at::Tensor& t) {
  const int64_t e = 16 / t.element_size();
  return t.size(2) % e == 0 && t.stride(0) % e == 0 && t.stride(1) % e == 0 &&
         aligned16(t.data_ptr());
}

static Args make_args(const at::Tensor& q, const at::Tensor& k,
                      const at::Tensor& v, const at::Tensor& ptr_q,
                      const at::Tensor& ptr_k, double scale, double cap,
                      const c10::optional<at::Tensor>& bias,
                      const c10::optional<at::Tensor>& pos_q,
                      const c10::optional<at::Tensor>& pos_k, int64_t half,
                      int64_t mbits, double dmax, int& axes) {
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  check_heads(v, "v", q);
  TORCH_CHECK(q.scalar_type() == at::kFloat ||
                  q.scalar_type() == at::kBFloat16,
              "segment_attention: unsupported dtype ", q.scalar_type());
  TORCH_CHECK(k.sizes() == v.sizes(), "segment_attention: k and v differ in "
              "shape");
  TORCH_CHECK(q.size(2) == k.size(2) && q.size(2) >= 1 && q.size(2) <= 128,
              "segment_attention: head dimensions must agree, 1 to 128");
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 &&
                  q.size(1) % k.size(1) == 0 && q.size(1) / k.size(1) <= 32,
              "segment_attention: query heads must be a multiple (at most "
              "32) of the key heads");
  check_index(ptr_q, "ptr_q", 1, q);
  check_index(ptr_k, "ptr_k", 1, q);
  TORCH_CHECK(ptr_q.size(0) >= 1 && ptr_q.size(0) == ptr_k.size(0),
              "segment_attention: ptr_q and ptr_k must have equal lengths");
  Args a = {};
  a.q = q.data_ptr(); a.k = k.data_ptr(); a.v = v.data_ptr();
  a.q_sn = q.stride(0); a.q_sh = q.stride(1);
  a.k_sn = k.stride(0); a.k_sh = k.stride(1);
  a.v_sn = v.stride(0); a.v_sh = v.stride(1);
  a.B = (int)ptr_q.size(0) - 1;
  a.H = (int)q.size(1); a.KV = (int)k.size(1); a.G = a.H / a.KV;
  a.D = (int)q.size(2);
  // 32-bit row numbers and launch sizes (threads of a launch < 2^32).
  const int64_t lim = (int64_t)1 << 31;
  TORCH_CHECK(q.size(0) < lim - 4096 && k.size(0) < lim - 4096 &&
                  (q.size(0) * a.G + 64 * (int64_t)a.B + 64) * a.KV <
                      ((int64_t)1 << 30) &&
                  (k.size(0) + 64 * (int64_t)a.B + 64) * a.KV <
                      ((int64_t)1 << 30),
              "segment_attention: too many rows for one call");
  a.Nq = (int)q.size(0); a.Nk = (int)k.size(0);
  a.ptr_q = ptr_q.data_ptr<int>(); a.ptr_k = ptr_k.data_ptr<int>();
  a.scale = (float)scale; a.cap = (float)cap;
  a.vec_q = rows16(q); a.vec_k = rows16(k); a.vec_v = rows16(v);
  a.splits = 1;
  axes = 0;
  if (bias.has_value()) {
    TORCH_CHECK(pos_q.has_value() && pos_k.has_value(),
                "segment_attention: bias needs pos_q and pos_k");
    check_index(*pos_q, "pos_q", 2, q);
    check_index(*pos_k, "pos_k", 2, q);
    axes = (int)pos_q->size(1);
    const int64_t w = 2 * half + 1;
    TORCH_CHECK((axes == 1 || axes == 2) && pos_k->size(1) == axes &&
                    pos_q->size(0) == q.size(0) &&
                    pos_k->size(0) == k.size(0),
                "segment_attention: positions must be [nodes, 1 or 2]");
    TORCH_CHECK(half >= 0 && (axes == 1 ? half <= 31 : half <= 3) &&
                    mbits >= 0 && mbits <= 3 && dmax <= (1 << 22),
                "segment_attention: unsupported bucket layout");
    TORCH_CHECK(bias->scalar_type() == at::kFloat &&
                    bias->device() == q.device() && bias->is_contiguous() &&
                    bias->dim() == 2 && bias->size(0) == a.H &&
                    bias->size(1) == (axes == 1 ? w : w * w),
                "segment_attention: bias must be a contiguous fp32 [heads, "
                "buckets] table");
    a.bias = bias->data_ptr<float>();
    a.pos_q = pos_q->data_ptr<int>(); a.pos_k = pos_k->data_ptr<int>();
    a.half = (int)half; a.mbits = (int)mbits; a.nb = (int)bias->size(1);
    a.slots = axes == 1 ? a.half * 2 + 2
                        : (a.half * 2 + 2) * (a.half * 2 + 2);
    a.dmax = (float)dmax;
    a.dmul = 2.f / (float)(1 << mbits);
  }
  return a;
}

// Waves sharing the staged tiles: 4 where the mean segment has rows for
// them, 1 (one wave walks a small segment alone) otherwise.
static int waves_for(int64_t rows, int64_t B) {
  return rows > 64 * std::max<int64_t>(B, 1) ? 4 : 1;
}

std::tuple<at::Tensor, at::Tensor> segment_attention_fwd(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& ptr_q, const at::Tensor& ptr_k, double scale,
    double cap, const c10::optional<at::Tensor>& bias,
    const c10::optional<at::Tensor>& pos_q,
    const c10::optional<at::Tensor>& pos_k, int64_t half, int64_t mbits,
    double dmax, bool with_lse) {
  int axes;
  Args a = make_args(q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q, pos_k,
                     half, mbits, dmax, axes);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor out = at::empty({a.Nq, a.H, a.D}, q.options());
  at::Tensor lse = at::empty({with_lse ? a.Nq : 0, a.H}, f32);
  if (a.Nq == 0) return {out, lse};
  a.out = out.data_ptr();
  a.lse = with_lse ? lse.data_ptr<float>() : nullptr;
  const int nw = waves_for((int64_t)a.Nq * a.G, a.B);
  // Few rows over long segments: the keys are split until about four
  // workgroups per CU run, each of two tiles at least.
  const int64_t tiles =
      std::max<int64_t>(a.Nq / (32 / a.G * nw), std::min(a.B, a.Nq)) * a.KV;
  const int64_t keys = a.Nk / std::max(a.B, 1);
  if (tiles < 512)
    a.splits = (int)std::max<int64_t>(
        1, std::min<int64_t>({(1024 + tiles - 1) / std::max<int64_t>(tiles, 1),
                              keys / 128, kMaxSplits}));
  at::Tensor po, pml;
  if (a.splits > 1) {
    po = at::empty({a.splits, a.Nq, a.H, a.D}, f32);
    pml = at::empty({a.splits, a.Nq, a.H, 2}, f32);
    a.part_o = po.data_ptr<float>();
    a.part_ml = pml.data_ptr<float>();
  }
  const bool f = q.scalar_type() == at::kFloat;
  f ? fwd_f32(a, axes, nw, stream()) : fwd_bf16(a, axes, nw, stream());
  if (a.splits > 1) {
    const int64_t rows = (int64_t)a.Nq * a.H;
    const dim3 grid((unsigned)((rows + 3) / 4));
    if (f)
      join_kernel<float><<<grid, 256, 0, stream()>>>(a);
    else
      join_kernel<__bf16><<<grid, 256, 0, stream()>>>(a);
    DGMC_CHECK_LAUNCH();
  }
  return {out, lse};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor>
segment_attention_bwd(const at::Tensor& dout, const at::Tensor& q,
                      const at::Tensor& k, const at::Tensor& v,
                      const at::Tensor& out, const at::Tensor& lse,
                      const at::Tensor& ptr_q, const at::Tensor& ptr_k,
                      double scale, double cap,
                      const c10::optional<at::Tensor>& bias,
                      const c10::optional<at::Tensor>& pos_q,
                      const c10::optional<at::Tensor>& pos_k, int64_t half,
                      int64_t mbits, double dmax) {
  int axes;
  Args a = make_args(q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q, pos_k,
                     half, mbits, dmax, axes);
  check_heads(dout, "dout", q);
  TORCH_CHECK(dout.sizes() == q.sizes() && out.sizes() == q.sizes() &&
                  out.scalar_type() == q.scalar_type() &&
                  out.device() == q.device() && out.is_contiguous(),
              "segment_attention: dout and out must have q's shape");
  TORCH_CHECK(lse.device() == q.device() && lse.is_contiguous() &&
                  lse.scalar_type() == at::kFloat && lse.dim() == 2 &&
                  lse.size(0) == a.Nq && lse.size(1) == a.H,
              "segment_attention: lse must be fp32 [nodes, heads]");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor dq = at::empty({a.Nq, a.H, a.D}, q.options());
  at::Tensor dk = at::empty({a.Nk, a.KV, a.D}, q.options());
  at::Tensor dv = at::empty({a.Nk, a.KV, a.D}, q.options());
  at::Tensor dbias = axes ? at::empty({a.H, a.nb}, f32) : at::empty({0}, f32);
  if (a.Nq == 0) {
    dk.zero_();
    dv.zero_();
    dbias.zero_();
    return {dq, dk, dv, dbias};
  }
  at::Tensor delta = at::empty({a.Nq, a.H}, f32);
  a.o = out.data_ptr();
  a.dout = dout.data_ptr();
  a.g_sn = dout.stride(0); a.g_sh = dout.stride(1);
  a.vec_g = rows16(dout); a.vec_o = rows16(out);
  a.lse = lse.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  a.dq = dq.data_ptr();
  a.dk = a.Nk ? dk.data_ptr() : nullptr;
  a.dv = a.Nk ? dv.data_ptr() : nullptr;
  const int nwq = waves_for((int64_t)a.Nq * a.G, a.B);
  const int nwk = waves_for(a.Nk, a.B);
  // Workgroups of the dq kernel with a table: each keeps its LDS columns
  // over all of its tiles.
  int nblk = 0;
  at::Tensor part;
  if (axes) {
    const int nslot = a.Nq / (32 / a.G * nwq) + a.B + 1;
    nblk = std::max(1, std::min(nslot, 2048 / (a.KV * nwq)));
    part = at::empty({nblk, a.KV, a.G, a.slots}, f32);
    a.part_bias = part.data_ptr<float>();
  }
  q.scalar_type() == at::kFloat
      ? bwd_f32(a, axes, nwq, nwk, nblk, stream())
      : bwd_bf16(a, axes, nwq, nwk, nblk, stream());
  if (axes) {
    bias_sum_kernel<<<a.H, 256, 0, stream()>>>(
        a.part_bias, dbias.data_ptr<float>(), nblk, a.KV, a.G, a.slots, a.nb,
        a.half, axes);
    DGMC_CHECK_LAUNCH();
  }
  return {dq, dk, dv, dbias};
}

}  // namespace segattn
}  // namespace dgmc
