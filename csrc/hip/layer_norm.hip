// Layer norm over the last dimension, forward and backward:
//
//   s = x + residual (optional, rounded to x's type: the sum is an output)
//   y = (s - mean) rstd w + b
//   dx = rstd (g - mean(g) - xhat mean(g xhat)) + ds,  g = dy w
//   dw = sum_rows dy xhat,  db = sum_rows dy
//
// Memory bound: forward reads x (and the residual) and writes y (and s)
// once, backward reads dy, s (and ds) and writes dx once.  A row is held in
// the registers of a group of TPR lanes (16-byte vectors, or single values
// where a row is not made of them), so mean and variance are two exact
// passes over registers and nothing is read twice; sums are fp32.  The
// weight gradients are kept per column in the lanes' registers over all the
// rows a workgroup walks, joined over its row groups through LDS and added
// over the workgroups in order by a second kernel: no atomics, the same bits
// every run.
//
// Measured (38960 x 256 bf16 with residual, 80 MB each way; a large copy runs
// at 4.8 TB/s): forward 24 us, 3.3 TB/s, backward 20 and its fold 4; no load
// is in flight while a row is reduced, and 4870 groups of rows are 2.4 rounds
// of 2048 workgroups that take the time of 3.  20 x 256 fp32: 10 us, a launch.
#include "attentional.h"
#include "common.h"

namespace dgmc {

namespace {

constexpr int kLnThreads = 256;
// Rows wider than the registers' share are refused (8 vectors x 256 lanes
// of 16 bytes, or 32 single values).
constexpr int kLnMaxCols = 8192;

// Sum over the TPR lanes that share a row (every lane gets it).
template <int TPR>
__device__ __forceinline__ float ln_sum(float v, float* red) {
  v = quad_sum(v);                       // lane exchanges of up to 16 lanes
  v += dpp_mov<0x141>(v);                // are VALU modifiers, no LDS trip
  if constexpr (TPR >= 16) v += dpp_mov<0x140>(v);
  if constexpr (TPR >= 32) v += __shfl_xor(v, 16);
  if constexpr (TPR >= 64) v += __shfl_xor(v, 32);
  if constexpr (TPR > 64) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wave] = v;
    __syncthreads();
    v = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return v;
}

// Column of element e of vector i of lane t.
template <int TPR, int N>
__device__ __forceinline__ int ln_col(int t, int i, int e) {
  return (i * TPR + t) * N + e;
}

// NV vectors of N values a lane: x[i][e] (zeros past C).
template <typename T, int TPR, int NV, int N>
__device__ __forceinline__ void ln_load(const T* row, int t, int C,
                                        float (&x)[NV][N]) {
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = ln_col<TPR, N>(t, i, 0);
    if (c < C) {
      load_vec<T, N>(row + c, x[i]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i][e] = 0.f;
    }
  }
}

struct LnArgs {
  const void *x, *res, *dy, *ds;
  void *y, *s, *dx;
  const float *w, *b;
  float2* stat;                 // [rows] (mean, rstd)
  float* part;                  // [blocks][2][C]
  int64_t rows;
  int C;
  float eps;
};

// A workgroup walks rows blockIdx.x RPB + k gridDim.x RPB; weight and bias
// stay in registers.
template <typename T, int TPR, int NV, int N>
__global__ __launch_bounds__(kLnThreads) void ln_fwd_kernel(const LnArgs a) {
  __shared__ float red[4];
  constexpr int RPB = kLnThreads / TPR;
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = min(ln_col<TPR, N>(t, i, e), a.C - 1);
      w[i][e] = a.w ? a.w[c] : 1.f;
      b[i][e] = a.b ? a.b[c] : 0.f;
    }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows;
       r0 += (int64_t)gridDim.x * RPB) {
    const int64_t r = r0 + grp;
    const bool live = r < a.rows;
    const int C = live ? a.C : 0;
    float x[NV][N];
    ln_load<T, TPR, NV, N>((const T*)a.x + r * a.C, t, C, x);
    if (a.res != nullptr) {
      float q[NV][N];
      ln_load<T, TPR, NV, N>((const T*)a.res + r * a.C, t, C, q);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int e = 0; e < N; ++e)
          x[i][e] = Cvt<T>::to_f(Cvt<T>::from_f(x[i][e] + q[i][e]));
        const int c = ln_col<TPR, N>(t, i, 0);
        if (c < C) store_vec<T, N>((T*)a.s + r * a.C + c, x[i]);
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) sum += x[i][e];
    const float mean = ln_sum<TPR>(sum, red) / a.C;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float d = x[i][e] - mean;
        sum += ln_col<TPR, N>(t, i, e) < C ? d * d : 0.f;
      }
    const float rstd = 1.f / sqrtf(ln_sum<TPR>(sum, red) / a.C + a.eps);
    if (live && t == 0 && a.stat) a.stat[r] = make_float2(mean, rstd);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ln_col<TPR, N>(t, i, 0);
#pragma unroll
      for (int e = 0; e < N; ++e)
        x[i][e] = fmaf((x[i][e] - mean) * rstd, w[i][e], b[i][e]);
      if (c < C) store_vec<T, N>((T*)a.y + r * a.C + c, x[i]);
    }
  }
}

template <typename T, int TPR, int NV, int N>
__global__ __launch_bounds__(kLnThreads) void ln_bwd_kernel(const LnArgs a) {
  __shared__ float red[4];
  extern __shared__ __attribute__((aligned(16))) float cols[];
  constexpr int RPB = kLnThreads / TPR;
  const int t = threadIdx.x % TPR, grp = threadIdx.x / TPR;
  float dw[NV][N], db[NV][N], w[NV][N];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int c = ln_col<TPR, N>(t, i, e);
      dw[i][e] = db[i][e] = 0.f;
      w[i][e] = c < a.C ? (a.w ? a.w[c] : 1.f) : 0.f;
    }
  for (int64_t r0 = (int64_t)blockIdx.x * RPB; r0 < a.rows;
       r0 += (int64_t)gridDim.x * RPB) {
    const int64_t r = r0 + grp;
    const bool live = r < a.rows;
    const int C = live ? a.C : 0;
    float x[NV][N], g[NV][N];
    ln_load<T, TPR, NV, N>((const T*)a.x + r * a.C, t, C, x);
    ln_load<T, TPR, NV, N>((const T*)a.dy + r * a.C, t, C, g);
    const float2 st = live ? a.stat[r] : make_float2(0.f, 0.f);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) {
        x[i][e] = (x[i][e] - st.x) * st.y;
        db[i][e] += g[i][e];
        // (g is 0 past the row's end: nothing enters from there)
        dw[i][e] = fmaf(g[i][e], x[i][e], dw[i][e]);
        g[i][e] *= w[i][e];
        s1 += g[i][e];
        s2 = fmaf(g[i][e], x[i][e], s2);
      }
    s1 = ln_sum<TPR>(s1, red) / a.C;
    s2 = ln_sum<TPR>(s2, red) / a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = ln_col<TPR, N>(t, i, 0);
      if (c >= C) continue;
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e)
        o[e] = st.y * (g[i][e] - s1 - x[i][e] * s2);
      if (a.ds != nullptr) {
        float q[N];
        load_vec<T, N>((const T*)a.ds + r * a.C + c, q);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] += q[e];
      }
      store_vec<T, N>((T*)a.dx + r * a.C + c, o);
    }
  }
  if (a.part == nullptr) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.C;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    if constexpr (RPB > 1) {
      // cols[grp][C]: group by group into the first one's order
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int c = ln_col<TPR, N>(t, i, e);
          if (c < a.C) cols[grp * a.C + c] = k ? db[i][e] : dw[i][e];
        }
      __syncthreads();
      for (int c = threadIdx.x; c < a.C; c += kLnThreads) {
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < RPB; ++q) s += cols[q * a.C + c];
        part[k * a.C + c] = s;
      }
    } else {
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int c = ln_col<TPR, N>(t, i, e);
          if (c < a.C) part[k * a.C + c] = k ? db[i][e] : dw[i][e];
        }
    }
  }
}

// out[c] = sum over the blocks' parts in a fixed order: 32 columns a
// workgroup, each by 32 threads that take every 32nd part.
constexpr int kLnWays = 32;

__global__ __launch_bounds__(32 * kLnWays) void ln_fold_kernel(
    const float* __restrict__ part, float* __restrict__ dw,
    float* __restrict__ db, int blocks, int C) {
  __shared__ float red[kLnWays][32];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), p = threadIdx.x >> 5;
  float s = 0.f;
  if (c < 2 * C) {
#pragma unroll 8
    for (int b = p; b < blocks; b += kLnWays)
      s += part[(int64_t)b * 2 * C + c];
  }
  red[p][threadIdx.x & 31] = s;
  __syncthreads();
  if (p != 0 || c >= 2 * C) return;
#pragma unroll
  for (int q = 1; q < kLnWays; ++q) s += red[q][threadIdx.x];
  if (c < C) {
    if (dw) dw[c] = s;
  } else if (db) {
    db[c - C] = s;
  }
}

// Lanes and vectors for a row of C: the fewest lanes (a power of two, at
// least 8) that hold it in one vector each, then more vectors of a wave,
// then of the workgroup.
template <typename T, int N, typename F>
void ln_pick(int C, F f) {
  const int v = (C + N - 1) / N;
#define LN_CASE(cond, tpr, nv) \
  if (cond) return f(std::integral_constant<int, tpr>(), \
                     std::integral_constant<int, nv>())
  LN_CASE(v <= 8, 8, 1);
  LN_CASE(v <= 16, 16, 1);
  LN_CASE(v <= 32, 32, 1);
  LN_CASE(v <= 64, 64, 1);
  LN_CASE(v <= 128, 64, 2);
  LN_CASE(v <= 256, 64, 4);
  if constexpr (N == 1) {
    LN_CASE(v <= 1024, 64, 16);
    LN_CASE(v <= 2048, 256, 8);
    LN_CASE(v <= 8192, 256, 32);
  } else {
    LN_CASE(v <= 512, 256, 2);
    LN_CASE(v <= 1024, 256, 4);
    if constexpr (N == 4) LN_CASE(v <= 2048, 256, 8);
  }
#undef LN_CASE
  TORCH_CHECK(false, "layer_norm: ", C, " columns");
}

template <typename T, typename F>
void ln_width(bool vec, int C, F f) {
  if (vec)
    ln_pick<T, 16 / (int)sizeof(T)>(C, [&](auto tpr, auto nv) {
      f(tpr, nv, std::integral_constant<int, 16 / (int)sizeof(T)>());
    });
  else
    ln_pick<T, 1>(C, [&](auto tpr, auto nv) {
      f(tpr, nv, std::integral_constant<int, 1>());
    });
}

// Rows of whole 16-byte vectors.
bool ln_vec(const at::Tensor& t) {
  return t.numel() == 0 || (aligned16(t.data_ptr()) &&
                            t.size(-1) * t.element_size() % 16 == 0);
}

void ln_check(const at::Tensor& t, const at::Tensor& x, const char* name) {
  TORCH_CHECK(t.device() == x.device() &&
                  t.scalar_type() == x.scalar_type() && t.sizes() == x.sizes(),
              "layer_norm: ", name, " must be like x");
}

int64_t ln_cols(const at::Tensor& x) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= kLnMaxCols,
              "layer_norm: x must be [..., 1 to ", kLnMaxCols, "]");
  return x.size(-1);
}

void ln_check_w(const OptTensor& w, const at::Tensor& x) {
  TORCH_CHECK(!w.has_value() ||
                  (w->device() == x.device() &&
                   w->scalar_type() == at::kFloat && w->is_contiguous() &&
                   w->dim() == 1 && w->size(0) == x.size(-1)),
              "layer_norm: weight and bias must be fp32 [columns]");
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_fwd(
    const at::Tensor& x_in, const OptTensor& residual_in,
    const OptTensor& weight, const OptTensor& bias, double eps, bool train) {
  const int64_t C = ln_cols(x_in);
  const at::Tensor x = x_in.contiguous();
  OptTensor residual;
  if (residual_in.has_value()) {
    ln_check(*residual_in, x, "residual");
    residual = residual_in->contiguous();
  }
  ln_check_w(weight, x);
  ln_check_w(bias, x);
  TORCH_CHECK(weight.has_value() || !bias.has_value(),
              "layer_norm: bias needs weight");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
  at::Tensor y = at::empty_like(x);
  at::Tensor s = residual.has_value() ? at::empty_like(x)
                                      : at::empty({0}, x.options());
  const int64_t rows = x.numel() / C;
  at::Tensor stat =
      at::empty({train ? rows : 0, 2}, x.options().dtype(at::kFloat));
  if (rows == 0) return {y, s, stat};
  LnArgs a = {};
  a.x = x.data_ptr();
  a.y = y.data_ptr();
  a.res = residual.has_value() ? residual->data_ptr() : nullptr;
  a.s = residual.has_value() ? s.data_ptr() : nullptr;
  a.w = weight.has_value() ? weight->data_ptr<float>() : nullptr;
  a.b = bias.has_value() ? bias->data_ptr<float>() : nullptr;
  a.stat = train ? (float2*)stat.data_ptr<float>() : nullptr;
  a.rows = rows;
  a.C = (int)C;
  a.eps = (float)eps;
  const bool vec = ln_vec(x) && (!residual.has_value() || ln_vec(*residual));
  DGMC_DISPATCH_FLOAT(x.scalar_type(), T, [&] {
    ln_width<T>(vec, a.C, [&](auto tpr, auto nv, auto n) {
      constexpr int rpb = kLnThreads / tpr();
      // 2048 workgroups (eight a CU, all resident) at most.
      const int64_t blocks =
          std::min<int64_t>((a.rows + rpb - 1) / rpb, 2048);
      ln_fwd_kernel<T, tpr(), nv(), n()>
          <<<dim3((unsigned)blocks), kLnThreads, 0, stream()>>>(a);
    });
    DGMC_CHECK_LAUNCH();
  });
  return {y, s, stat};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_bwd(
    const at::Tensor& dy_in, const OptTensor& ds_in, const at::Tensor& s_in,
    const at::Tensor& stat, const OptTensor& weight, bool with_weight) {
  const int C = (int)ln_cols(s_in);
  const at::Tensor s = s_in.contiguous(), dy = dy_in.contiguous();
  ln_check(dy, s, "dy");
  OptTensor ds;
  if (ds_in.has_value()) {
    ln_check(*ds_in, s, "ds");
    ds = ds_in->contiguous();
  }
  const int64_t rows = s.numel() / C;
  ln_check_w(weight, s);
  TORCH_CHECK(stat.device() == s.device() && stat.is_contiguous() &&
                  stat.scalar_type() == at::kFloat && stat.dim() == 2 &&
                  stat.size(0) == rows && stat.size(1) == 2,
              "layer_norm: stat must be fp32 [rows, 2]");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(s.device());
  const auto f32 = s.options().dtype(at::kFloat);
  at::Tensor dx = at::empty_like(s);
  at::Tensor dw = at::empty({with_weight ? C : 0}, f32);
  at::Tensor db = at::empty({with_weight ? C : 0}, f32);
  if (rows == 0) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  LnArgs a = {};
  a.x = s.data_ptr();
  a.dy = dy.data_ptr();
  a.ds = ds.has_value() ? ds->data_ptr() : nullptr;
  a.dx = dx.data_ptr();
  a.w = weight.has_value() ? weight->data_ptr<float>() : nullptr;
  a.stat = (float2*)stat.data_ptr<float>();
  a.rows = rows;
  a.C = C;
  const bool vec = ln_vec(s) && ln_vec(dy) && (!ds.has_value() || ln_vec(*ds));
  at::Tensor part;
  int blocks = 0;
  DGMC_DISPATCH_FLOAT(s.scalar_type(), T, [&] {
    ln_width<T>(vec, C, [&](auto tpr, auto nv, auto n) {
      constexpr int rpb = kLnThreads / tpr();
      // 1024 workgroups (four a CU) at most: their parts are folded.
      blocks = (int)std::min<int64_t>((a.rows + rpb - 1) / rpb, 1024);
      if (with_weight) {
        part = at::empty({blocks, 2, C}, f32);
        a.part = part.data_ptr<float>();
      }
      const size_t lds = with_weight && rpb > 1 ? rpb * C * 4 : 0;
      ln_bwd_kernel<T, tpr(), nv(), n()>
          <<<blocks, kLnThreads, lds, stream()>>>(a);
    });
    DGMC_CHECK_LAUNCH();
  });
  if (with_weight) {
    ln_fold_kernel<<<(2 * C + 31) / 32, 32 * kLnWays, 0, stream()>>>(
        a.part, dw.data_ptr<float>(), db.data_ptr<float>(), blocks, C);
    DGMC_CHECK_LAUNCH();
  }
  return {dx, dw, db};
}

}  // namespace dgmc
