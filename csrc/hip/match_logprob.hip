// Log-probabilities of given matches, row entropies and best alternatives of
// a score matrix, and the scores' gradient:
//
//   p_ij = exp(z_ij - lse_i) over the row's valid columns j < n_i
//   logp_i = z_i,y - lse_i,  H_i = -sum_j p_ij log p_ij
//   top: the k largest z_ij, ties to the lower column, as log p and column
//   dz_ij = gl_i ([j = y_i] - p_ij) - gh_i p_ij (log p_ij + H_i)
//
// Memory bound: the forward reads the scores once, the backward reads them
// and writes the gradient once.  A row (or a part of a long one) stays in
// its lanes' registers as loaded, so maximum, sum, sum of p log p and the
// selection are passes over registers, not over memory; all sums are fp32
// around the row's maximum.
//
// Selection.  The workgroup's lanes form 64 groups; the k-th largest of the
// groups' maxima bounds the k-th largest score from below, few more than k
// scores reach it, and those are compacted (LDS counter) and ranked by
// (score, column), whatever order they were compacted in.  More than kLpCand
// of them (many equal scores) fall back to k rounds of an exact arg-max over
// the registers.
//
// Rows past one workgroup's registers are cut into parts; a second kernel
// joins the parts' maxima, sums and selections.
//
// Measured (4500 x 19572 fp32, ten alternatives): forward 109 us for 352 MB
// (3.2 TB/s: two workgroups a CU, whose loads stop while they rank), backward
// 110 us for 705 MB, part of it still cached.  4608 x 19: 5 and 3 us.
#include "attentional.h"
#include "common.h"

namespace dgmc {

namespace {

constexpr int kLpMaxTop = 32;
constexpr int kLpCand = 256;      // candidates ranked at once
constexpr int kLpSmall = 256;     // columns of the wave-level kernel

struct LpArgs {
  const void* z;
  void* dz;
  const int64_t* y;
  const int* n;                   // [rows] valid columns, or null
  const float *gl, *gh;           // gradients of logp and entropy, or null
  float *logp, *ent, *top_lp;
  int64_t* top_idx;
  float2* stat;                   // [rows] (max, log of the sum)
  float4* part;                   // [rows][parts] (max, sum, sum e d, -)
  float* part_v;                  // [rows][parts][k]
  int* part_i;
  int64_t rows, stride;
  int V, k, parts, width;         // width: columns of a part
};

__device__ __forceinline__ int lp_valid(const LpArgs& a, int64_t r) {
  return a.n == nullptr ? a.V : min(max(a.n[r], 0), a.V);
}

// (v, j) before (w, i): the larger score, then the lower column; column -1:
// none.
__device__ __forceinline__ bool lp_before(float v, int j, float w, int i) {
  return j >= 0 && (i < 0 || v > w || (v == w && j < i));
}
__device__ __forceinline__ void lp_take(float& v, int& j, float w, int i) {
  if (lp_before(w, i, v, j)) {
    v = w;
    j = i;
  }
}

// e^d and its sums: l += e^d, t += d e^d (0 where e^d is).
__device__ __forceinline__ void lp_add(float d, float& l, float& t) {
  const float e = __expf(d);
  l += e;
  t = fmaf(e, fmaxf(d, -1e30f), t);
}

// Outputs of a row from its maximum m, l and t (l = 0: no score above -inf;
// NaN or +inf scores make l NaN).  Returns the log of the sum.
template <typename T>
__device__ __forceinline__ void lp_finish(const LpArgs& a, int64_t r, int nv,
                                          float m, float l, float t) {
  const int64_t y = a.y[r];
  const float ll = logf(l);
  float lp = 0.f;                       // no match given
  if (y >= 0 && y < a.V) {
    lp = -INFINITY;                     // masked, or an empty row
    if (y < nv && l != 0.f)
      lp = Cvt<T>::to_f(((const T*)a.z)[r * a.stride + y]) - m - ll;
  }
  a.logp[r] = lp;
  a.ent[r] = l == 0.f ? 0.f : ll - t / l;
  // (an empty row: p = exp(z - 0 - inf) = 0)
  if (a.stat)
    a.stat[r] = l == 0.f ? make_float2(0.f, INFINITY) : make_float2(m, ll);
}

__device__ __forceinline__ void lp_put(const LpArgs& a, int64_t r, int q,
                                       float v, int j, float m, float ll) {
  a.top_lp[r * a.k + q] = j < 0 ? -INFINITY : v - m - ll;
  a.top_idx[r * a.k + q] = j;
}

// --------------------------------------------------------------------------
// Rows of up to 256 columns: TPR lanes a row, NV values a lane.
// --------------------------------------------------------------------------
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(256) void lp_small_kernel(const LpArgs a) {
  const int t0 = threadIdx.x % TPR;
  const int64_t r = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
  const bool live = r < a.rows;
  const int nv = live ? lp_valid(a, r) : 0;
  const T* row = (const T*)a.z + (live ? r * a.stride : 0);
  float x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int j = t0 + i * TPR;
    x[i] = j < nv ? Cvt<T>::to_f(row[j]) : -INFINITY;
  }
  float m = x[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) m = fmaxf(m, x[i]);
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i) lp_add(x[i] - ms, l, t);
#pragma unroll
  for (int o = 1; o < TPR; o <<= 1) {
    l += __shfl_xor(l, o);
    t += __shfl_xor(t, o);
  }
  if (live && t0 == 0) lp_finish<T>(a, r, nv, ms, l, t);
  const float ll = logf(l);
  float pv = INFINITY;
  int pj = -1;
  bool first = true;
  for (int q = 0; q < a.k; ++q) {
    float v = -INFINITY;
    int best = -1;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      // behind the one before, and a score at all
      const int j = t0 + i * TPR;
      const bool ok =
          x[i] > -INFINITY && (first || lp_before(pv, pj, x[i], j)) &&
          !(j == pj);
      if (ok) lp_take(v, best, x[i], j);
    }
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1)
      lp_take(v, best, __shfl_xor(v, o), __shfl_xor(best, o));
    if (live && t0 == 0) lp_put(a, r, q, v, best, ms, ll);
    // (once none is left, none comes back: pj stays the last column)
    if (best >= 0) {
      pv = v;
      pj = best;
      first = false;
    } else {
      pv = -INFINITY;
    }
  }
}

// --------------------------------------------------------------------------
// Longer rows: a workgroup of NT threads per row part, NV 16-byte vectors a
// lane.  Vectors lie on 16-byte boundaries; the one or two that hang over
// the part's ends are read value by value.
// --------------------------------------------------------------------------
template <int NT>
__device__ __forceinline__ void lp_block_sum(float& l, float& t,
                                             float (*red)[2]) {
  l = wave_sum(l);
  t = wave_sum(t);
  if ((threadIdx.x & 63) == 0) {
    red[threadIdx.x >> 6][0] = l;
    red[threadIdx.x >> 6][1] = t;
  }
  __syncthreads();
  l = t = 0.f;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    l += red[w][0];
    t += red[w][1];
  }
}

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT, 4) void lp_row_kernel(const LpArgs a) {
  constexpr int N = Vec16<T>::N;
  constexpr int GS = NT / 64;                  // lanes of one of 64 groups
  __shared__ float gmax[64], red[NT / 64][2];
  __shared__ int ranks[NT / 64][64];
  __shared__ float cand_v[kLpCand];
  __shared__ int cand_j[kLpCand], count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t r = blockIdx.x / a.parts;
  const int p = blockIdx.x % a.parts;
  const int nv_row = lp_valid(a, r);
  const T* row = (const T*)a.z + r * a.stride;
  const int c0 = p * a.width, c1 = min(c0 + a.width, nv_row);
  const int cv = min(c0 + a.width, a.V);       // readable end
  // Column of element 0 of vector 0 (a 16-byte boundary).
  const int shift =
      (int)(((uintptr_t)(row + c0) & 15u) / (unsigned)sizeof(T));
  const int b0 = c0 - shift;
  // The row's first whole vector, for lanes without one of their own (parts
  // begin on vectors, so every part has the row's shift).
  const int inner = shift ? N - shift : 0;
  if (tid == 0) count = 0;

  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = b0 + (i * NT + tid) * N;
    const bool whole = c >= c0 && c + N <= cv;
    raw[i] = *reinterpret_cast<const uint4*>(row + (whole ? c : inner));
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = b0 + (i * NT + tid) * N;
    if ((c < c0 || c + N > cv) && c < cv) {
      T e[N];
#pragma unroll
      for (int k = 0; k < N; ++k)
        e[k] = c + k >= c0 && c + k < cv ? row[c + k] : Cvt<T>::from_f(0.f);
      __builtin_memcpy(&raw[i], e, 16);
    }
  }
  // Masked columns and empty slots become -inf once, here.
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = b0 + (i * NT + tid) * N;
    if (c < c0 || c + N > c1) {
      T e[N];
      __builtin_memcpy(e, &raw[i], 16);
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (c + k < c0 || c + k >= c1) e[k] = Cvt<T>::from_f(-INFINITY);
      __builtin_memcpy(&raw[i], e, 16);
    }
  }
  auto value = [&](int i, int k) {
    return Cvt<T>::to_f(reinterpret_cast<const T*>(&raw[i])[k]);
  };

  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) m = fmaxf(m, value(i, k));
  const float lane_max = m;
  // (opaque between the passes: the vectors are unpacked anew, not kept as
  // twice the registers)
  auto again = [&] {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      asm volatile("" : "+v"(raw[i].x), "+v"(raw[i].y), "+v"(raw[i].z),
                   "+v"(raw[i].w));
  };
  again();
#pragma unroll
  for (int o = 1; o < GS; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (tid % GS == 0) gmax[tid / GS] = m;
  __syncthreads();
  const float gm = gmax[lane];
  m = wave_max(gm);
  const float ms = m == -INFINITY ? 0.f : m;
  // Each wave ranks the 64 maxima against its share of them (equal ones by
  // group number).
  if (a.k > 0) {
    int rank = 0;
#pragma unroll
    for (int q = 0; q < 64 / (NT / 64); ++q) {
      const int o = (tid >> 6) * (64 / (NT / 64)) + q;
      const float w = gmax[o];
      rank += w > gm || (w == gm && o < lane);
    }
    ranks[tid >> 6][lane] = rank;
  }
  float l = 0.f, t = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) lp_add(value(i, k) - ms, l, t);
  again();
  lp_block_sum<NT>(l, t, red);                 // (a barrier: ranks are there)
  if (tid == 0) {
    if (a.parts > 1)
      a.part[r * a.parts + p] = make_float4(m, l, t, 0.f);
    else
      lp_finish<T>(a, r, nv_row, ms, l, t);
  }
  if (a.k == 0) return;

  int rank = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) rank += ranks[w][lane];
  // The k-th largest of the 64 maxima.
  const float ll = logf(l),
              thr = lane_of(gm, __ffsll(__ballot(rank == a.k - 1)) - 1);
  auto put = [&](int q, float v, int j) {
    if (a.parts > 1) {
      a.part_v[(r * a.parts + p) * a.k + q] = v;
      a.part_i[(r * a.parts + p) * a.k + q] = j;
    } else {
      lp_put(a, r, q, v, j, ms, ll);
    }
  };
  // (about k lanes of the workgroup hold a candidate)
  if (lane_max >= thr && lane_max > -INFINITY)
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float v = value(i, k);
      if (v >= thr && v > -INFINITY) {
        const int s = atomicAdd(&count, 1);
        if (s < kLpCand) {
          cand_v[s] = v;
          cand_j[s] = b0 + (i * NT + tid) * N + k;
        }
      }
    }
  __syncthreads();
  const int n = count;
  if (n <= 64) {
    // One wave, a candidate a lane, the others' values by readlane.
    if (tid >= 64) return;
    const bool own = lane < n;
    const float v = own ? cand_v[lane] : -INFINITY;
    const int j = own ? cand_j[lane] : -1;
    int q = 0;
    for (int o = 0; o < n; ++o)
      q += lp_before(lane_of(v, o), __builtin_amdgcn_readlane(j, o), v, j);
    if (own ? q < a.k : lane < a.k) put(own ? q : lane, v, j);
    return;
  }
  if (n <= kLpCand) {
    for (int c = tid; c < max(n, a.k); c += NT) {
      if (c >= n) {
        put(c, -INFINITY, -1);
        continue;
      }
      const float v = cand_v[c];
      const int j = cand_j[c];
      int q = 0;
#pragma unroll 4
      for (int o = 0; o < n; ++o)
        q += lp_before(cand_v[o], cand_j[o], v, j);
      if (q < a.k) put(q, v, j);
    }
    return;
  }
  // Many equal scores: k rounds of an exact arg-max behind the last pick.
  float pv = INFINITY;
  int pj = -1;
  for (int q = 0; q < a.k; ++q) {
    float v = -INFINITY;
    int best = -1;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int k = 0; k < N; ++k) {
        const float w = value(i, k);
        const int j = b0 + (i * NT + tid) * N + k;
        if (w >= thr && w > -INFINITY &&
            (q == 0 || (j != pj && lp_before(pv, pj, w, j))))
          lp_take(v, best, w, j);
      }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      lp_take(v, best, __shfl_xor(v, o), __shfl_xor(best, o));
    __syncthreads();
    if (lane == 0) {
      cand_v[tid >> 6] = v;
      cand_j[tid >> 6] = best;
    }
    __syncthreads();
    v = cand_v[0];
    best = cand_j[0];
    for (int w = 1; w < NT / 64; ++w) lp_take(v, best, cand_v[w], cand_j[w]);
    if (tid == 0) put(q, v, best);
    pv = v;
    pj = best;
  }
}

// Parts -> row: one wave a row.
template <typename T>
__global__ __launch_bounds__(64) void lp_join_kernel(const LpArgs a) {
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x;
  const float4* part = a.part + r * a.parts;
  float m = -INFINITY;
  for (int p = lane; p < a.parts; p += 64) m = fmaxf(m, part[p].x);
  m = wave_max(m);
  const float ms = m == -INFINITY ? 0.f : m;
  float l = 0.f, t = 0.f;
  for (int p = lane; p < a.parts; p += 64) {
    const float4 s = part[p];
    // sum e^(z - ms) (z - ms) = e^(mp - ms) (t_p + (mp - ms) l_p)
    const float d = (s.x == -INFINITY ? 0.f : s.x) - ms, e = __expf(d);
    l += s.y == 0.f ? 0.f : e * s.y;
    t += s.y == 0.f ? 0.f : e * fmaf(fmaxf(d, -1e30f), s.y, s.z);
  }
  l = wave_sum(l);
  t = wave_sum(t);
  if (lane == 0) lp_finish<T>(a, r, lp_valid(a, r), ms, l, t);
  const float ll = logf(l);
  const int n = a.parts * a.k;
  const float* pv_ = a.part_v + r * n;
  const int* pi_ = a.part_i + r * n;
  float pv = INFINITY;
  int pj = -1;
  for (int q = 0; q < a.k; ++q) {
    float v = -INFINITY;
    int best = -1;
    for (int c = lane; c < n; c += 64) {
      const float w = pv_[c];
      const int j = pi_[c];
      if (j >= 0 && (q == 0 || (pj >= 0 && j != pj && lp_before(pv, pj, w, j))))
        lp_take(v, best, w, j);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      lp_take(v, best, __shfl_xor(v, o), __shfl_xor(best, o));
    if (lane == 0) lp_put(a, r, q, v, best, ms, ll);
    pv = v;
    pj = best;
  }
}

// --------------------------------------------------------------------------
// Backward
// --------------------------------------------------------------------------
struct LpRow {
  float m, ll, gl, gh, ent;
  int64_t y;
  int nv;
};

__device__ __forceinline__ LpRow lp_row(const LpArgs& a, int64_t r) {
  LpRow w;
  const float2 s = a.stat[r];
  w.m = s.x;
  w.ll = s.y;
  w.y = a.y[r];
  w.nv = lp_valid(a, r);
  // No gradient from the logp of a row without a given match, nor from that
  // of a masked one (the constant -inf; so in every empty row).
  w.gl = a.gl != nullptr && w.y >= 0 && w.y < a.V && a.logp[r] != -INFINITY
             ? a.gl[r]
             : 0.f;
  w.gh = a.gh != nullptr ? a.gh[r] : 0.f;
  w.ent = a.ent[r];
  return w;
}

__device__ __forceinline__ float lp_grad(const LpRow& w, float z, int j) {
  const float lp = z - w.m - w.ll, p = __expf(lp);
  // (p = 0 takes p log p to 0; NaN stays NaN)
  const float plp = p * fmaxf(lp, -1e30f);
  float g = -w.gl * p - w.gh * fmaf(p, w.ent, plp);
  if (j == w.y) g += w.gl;
  return j < w.nv ? g : 0.f;
}

// One value a thread at a time (short rows, rows whose score and gradient
// vectors do not fall on the same 16-byte boundaries).
constexpr int64_t kLpFlatBlocks = 1 << 23;     // (2^31 threads)

template <typename T>
__global__ __launch_bounds__(256) void lp_bwd_flat_kernel(const LpArgs a) {
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
       e < a.rows * a.V; e += (int64_t)gridDim.x * 256) {
    const int64_t r = e / a.V;
    const int j = (int)(e - r * a.V);
    const LpRow w = lp_row(a, r);
    ((T*)a.dz)[e] = Cvt<T>::from_f(
        lp_grad(w, Cvt<T>::to_f(((const T*)a.z)[r * a.stride + j]), j));
  }
}

// One workgroup per 4 vectors a lane of one row.
constexpr int kLpBwdVec = 4;

template <typename T>
__global__ __launch_bounds__(256) void lp_bwd_kernel(const LpArgs a) {
  constexpr int N = Vec16<T>::N;
  const int64_t r = blockIdx.x / a.parts;
  const int p = blockIdx.x % a.parts;
  const T* row = (const T*)a.z + r * a.stride;
  T* out = (T*)a.dz + r * a.V;
  const int shift = (int)(((uintptr_t)row & 15u) / (unsigned)sizeof(T));
  const int b0 = p * 256 * kLpBwdVec * N - shift, inner = shift ? N - shift : 0;
  uint4 raw[kLpBwdVec];
#pragma unroll
  for (int i = 0; i < kLpBwdVec; ++i) {
    const int c = b0 + (i * 256 + (int)threadIdx.x) * N;
    raw[i] = *reinterpret_cast<const uint4*>(
        row + (c >= 0 && c + N <= a.V ? c : inner));
  }
  const LpRow w = lp_row(a, r);
#pragma unroll
  for (int i = 0; i < kLpBwdVec; ++i) {
    const int c = b0 + (i * 256 + (int)threadIdx.x) * N;
    if (c >= 0 && c + N <= a.V) {
      const T* e = reinterpret_cast<const T*>(&raw[i]);
      float g[N];
#pragma unroll
      for (int k = 0; k < N; ++k) g[k] = lp_grad(w, Cvt<T>::to_f(e[k]), c + k);
      store_vec<T, N>(out + c, g);
    } else {
#pragma unroll
      for (int k = 0; k < N; ++k)
        if (c + k >= 0 && c + k < a.V)
          out[c + k] =
              Cvt<T>::from_f(lp_grad(w, Cvt<T>::to_f(row[c + k]), c + k));
    }
  }
}

void lp_check(const at::Tensor& z, const at::Tensor& y,
              const OptTensor& n) {
  TORCH_CHECK(z.is_cuda() && z.dim() == 2 && z.size(1) >= 1 &&
                  z.size(1) < (1 << 30) &&
                  (z.size(1) == 1 || z.stride(1) == 1),
              "match_log_probs: scores must be [rows, columns] with "
              "contiguous rows");
  TORCH_CHECK(y.device() == z.device() && y.scalar_type() == at::kLong &&
                  y.dim() == 1 && y.size(0) == z.size(0) && y.is_contiguous(),
              "match_log_probs: target must be int64 [rows]");
  TORCH_CHECK(!n.has_value() ||
                  (n->device() == z.device() &&
                   n->scalar_type() == at::kInt && n->dim() == 1 &&
                   n->size(0) == z.size(0) && n->is_contiguous()),
              "match_log_probs: n_cols must be int32 [rows]");
}

template <typename T, int NT, int NV>
void lp_rows(LpArgs& a, const at::TensorOptions& f32, hipStream_t st) {
  // (a vector less than the registers hold: room for the misaligned start)
  a.width = (NT * NV - 1) * Vec16<T>::N;
  a.parts = (a.V + a.width - 1) / a.width;
  TORCH_CHECK(a.rows * a.parts < (1 << 23) * (int64_t)(512 / NT),
              "match_log_probs: too many rows for one call");
  at::Tensor part, pv, pi;
  if (a.parts > 1) {
    part = at::empty({a.rows, a.parts, 4}, f32);
    pv = at::empty({a.rows, a.parts, a.k}, f32);
    pi = at::empty({a.rows, a.parts, a.k}, f32.dtype(at::kInt));
    a.part = (float4*)part.data_ptr<float>();
    a.part_v = pv.data_ptr<float>();
    a.part_i = pi.data_ptr<int>();
  }
  lp_row_kernel<T, NT, NV>
      <<<dim3((unsigned)(a.rows * a.parts)), NT, 0, st>>>(a);
  DGMC_CHECK_LAUNCH();
  if (a.parts > 1) {
    lp_join_kernel<T><<<dim3((unsigned)a.rows), 64, 0, st>>>(a);
    DGMC_CHECK_LAUNCH();
  }
}

template <typename T, int TPR, int NV>
void lp_small(const LpArgs& a, hipStream_t st) {
  const int64_t blocks = (a.rows + 256 / TPR - 1) / (256 / TPR);
  TORCH_CHECK(blocks < (1 << 24),
              "match_log_probs: too many rows for one call");
  lp_small_kernel<T, TPR, NV><<<dim3((unsigned)blocks), 256, 0, st>>>(a);
  DGMC_CHECK_LAUNCH();
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor>
match_logprob_fwd(const at::Tensor& z, const at::Tensor& y,
                  const OptTensor& n, int64_t k, bool train) {
  lp_check(z, y, n);
  TORCH_CHECK(k >= 0 && k <= kLpMaxTop && k <= z.size(1),
              "match_log_probs: top must be 0 to ", kLpMaxTop,
              " and at most the columns");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(z.device());
  const auto f32 = z.options().dtype(at::kFloat);
  const int64_t R = z.size(0);
  at::Tensor logp = at::empty({R}, f32), ent = at::empty({R}, f32);
  at::Tensor top_lp = at::empty({R, k}, f32);
  at::Tensor top_idx = at::empty({R, k}, z.options().dtype(at::kLong));
  at::Tensor stat = at::empty({train ? R : 0, 2}, f32);
  if (R == 0) return {logp, ent, top_lp, top_idx, stat};
  LpArgs a = {};
  a.z = z.data_ptr();
  a.y = y.data_ptr<int64_t>();
  a.n = n.has_value() ? n->data_ptr<int>() : nullptr;
  a.logp = logp.data_ptr<float>();
  a.ent = ent.data_ptr<float>();
  a.top_lp = top_lp.data_ptr<float>();
  a.top_idx = top_idx.data_ptr<int64_t>();
  a.stat = train ? (float2*)stat.data_ptr<float>() : nullptr;
  a.rows = R;
  a.stride = z.stride(0);
  a.V = (int)z.size(1);
  a.k = (int)k;
  a.parts = 1;
  const hipStream_t st = stream();
  DGMC_DISPATCH_FLOAT(z.scalar_type(), T, [&] {
    constexpr int N = Vec16<T>::N;
    constexpr int S = N / 4;        // 8, 16, 32 .. 64 values a lane
    const int vals = a.V + 2 * N;   // (with room for a misaligned start)
    if (a.V <= 16) lp_small<T, 16, 1>(a, st);
    else if (a.V <= 32) lp_small<T, 16, 2>(a, st);
    else if (a.V <= 64) lp_small<T, 16, 4>(a, st);
    else if (a.V <= kLpSmall) lp_small<T, 64, 4>(a, st);
    else if (vals <= 256 * 8) lp_rows<T, 256, 2 / S>(a, f32, st);
    else if (vals <= 256 * 16) lp_rows<T, 256, 4 / S>(a, f32, st);
    else if (vals <= 256 * 32) lp_rows<T, 256, 8 / S>(a, f32, st);
    else if (vals <= 512 * 24) lp_rows<T, 512, 6 / S>(a, f32, st);
    else if (vals <= 512 * 40) lp_rows<T, 512, 10 / S>(a, f32, st);
    else lp_rows<T, 512, 16 / S>(a, f32, st);
  });
  return {logp, ent, top_lp, top_idx, stat};
}

at::Tensor match_logprob_bwd(const OptTensor& gl,
                             const OptTensor& gh,
                             const at::Tensor& z, const at::Tensor& y,
                             const OptTensor& n,
                             const at::Tensor& logp, const at::Tensor& ent,
                             const at::Tensor& stat) {
  lp_check(z, y, n);
  const int64_t R = z.size(0);
  for (const auto* t : {&gl, &gh})
    TORCH_CHECK(!t->has_value() ||
                    ((*t)->device() == z.device() && (*t)->is_contiguous() &&
                     (*t)->scalar_type() == at::kFloat &&
                     (*t)->dim() == 1 && (*t)->size(0) == R),
                "match_log_probs: gradients must be fp32 [rows]");
  for (const auto* t : {&logp, &ent, &stat})
    TORCH_CHECK(t->device() == z.device() && t->is_contiguous() &&
                    t->scalar_type() == at::kFloat &&
                    t->numel() == (t == &stat ? 2 * R : R),
                "match_log_probs: saved statistics do not fit the scores");
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(z.device());
  at::Tensor dz = at::empty({R, z.size(1)}, z.options());
  if (R == 0) return dz;
  LpArgs a = {};
  a.z = z.data_ptr();
  a.dz = dz.data_ptr();
  a.y = y.data_ptr<int64_t>();
  a.n = n.has_value() ? n->data_ptr<int>() : nullptr;
  a.gl = gl.has_value() ? gl->data_ptr<float>() : nullptr;
  a.gh = gh.has_value() ? gh->data_ptr<float>() : nullptr;
  a.logp = logp.data_ptr<float>();
  a.ent = ent.data_ptr<float>();
  a.stat = (float2*)stat.data_ptr<float>();
  a.rows = R;
  a.stride = z.stride(0);
  a.V = (int)z.size(1);
  const hipStream_t st = stream();
  DGMC_DISPATCH_FLOAT(z.scalar_type(), T, [&] {
    constexpr int N = Vec16<T>::N;
    const bool same = aligned16(a.z) && aligned16(a.dz) &&
                      (a.stride - a.V) % N == 0;
    if (a.V > kLpSmall && same) {
      const int width = 256 * kLpBwdVec * N;
      a.parts = (a.V + N + width - 1) / width;
      TORCH_CHECK(R * a.parts < (1 << 24),
                  "match_log_probs: too many rows for one call");
      lp_bwd_kernel<T>
          <<<dim3((unsigned)(R * a.parts)), 256, 0, st>>>(a);
    } else {
      const int64_t blocks =
          std::min<int64_t>((R * a.V + 255) / 256, kLpFlatBlocks);
      lp_bwd_flat_kernel<T><<<dim3((unsigned)blocks), 256, 0, st>>>(a);
    }
    DGMC_CHECK_LAUNCH();
  });
  return dz;
}

}  // namespace dgmc
