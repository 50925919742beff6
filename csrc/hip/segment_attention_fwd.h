// Forward kernel of the segment attention (segment_attention.h), one pass
// over the keys with the running maximum and sum of the softmax.
//
// A wave owns RW packed rows (one query x head per lane column), NW waves
// share the K / V tiles of KT keys staged in LDS (double-buffered, the next
// tile's global loads in flight over the current one's products).  Scores
// S^T = K Q^T put a row's KT scores into the two lanes l, l ^ 32; the
// running maximum moves only when a tile exceeds it by 2^8 (the rescale of
// the output accumulators is skipped otherwise; P <= 2^8 changes no
// relative rounding), the sum is kept per lane and joined once at the end.
// P is rounded to bf16 for the bf16 product (fp32: not at all); maximum,
// sum and outputs are fp32.
#pragma once

#include "segment_attention.h"

namespace dgmc {
namespace segattn {

template <typename T, int DP, int NW, int KT, int POS>
__global__ __launch_bounds__(NW * 64, sizeof(T) == 2 ? 2 : 1) void fwd_kernel(
    const Args a) {
  constexpr int CH = DP * (int)sizeof(T) / 16;   // 16-byte chunks per row
  constexpr int NT = NW * 64;
  constexpr int LD = KT * CH / NT;               // chunks a thread stages
  static_assert(LD * NT == KT * CH, "staging");
  constexpr int TB = KT * CH * 16;               // bytes of one tile
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  DGMC_LDS float* kpos = (DGMC_LDS float*)(lds + 4 * TB);   // [2][2][KT]
  DGMC_LDS float* tab = kpos + (POS ? 4 * KT : 0);          // [G][kSlots]

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, slot = blockIdx.x / a.KV;
  const int split = blockIdx.y;
  const int QW = 32 / a.G, TQ = QW * NW;
  const int seg = find_segment(a.ptr_q, a.B, a.Nq, TQ, slot);
  int q_lo, q_hi, k_lo = 0, k_hi = 0;
  seg_range(a.ptr_q, seg, a.B, a.Nq, q_lo, q_hi);
  q_lo += (slot - (seg_begin(a.ptr_q, seg, a.Nq) / TQ + seg)) * TQ;
  if (q_lo >= q_hi) return;
  if (seg < a.B) seg_range(a.ptr_k, seg, a.B, a.Nk, k_lo, k_hi);

  // This lane's packed row.
  const int g = c % a.G;
  const int64_t qi = (int64_t)q_lo + wave * QW + c / a.G;
  const bool live = c < QW * a.G && qi < q_hi;
  const int head = kvh * a.G + g;
  const T* qrow = (const T*)a.q + qi * a.q_sn + (int64_t)head * a.q_sh;
  u32x4 qf[CH / 2];
#pragma unroll
  for (int s = 0; s < CH / 2; ++s)
    qf[s] = load_chunk<T>(qrow, 2 * s + h, a.D, live, a.vec_q);
  float px = 0.f, py = 0.f;
  const Bucket bk(a);
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    if (live) {
      px = load_pos(a.pos_q, qi, POS, 0);
      if (POS == 2) py = load_pos(a.pos_q, qi, POS, 1);
    }
  }
  const DGMC_LDS float* mytab = tab + g * kSlots;
  const int W = 2 * a.half + 2;

  // Key tiles [t0, t1) of this split.
  const int ntile = (k_hi - k_lo + KT - 1) / KT;
  const int per = (ntile + a.splits - 1) / a.splits;
  const int t0 = min(split * per, ntile), t1 = min(t0 + per, ntile);

  const T* kbase = (const T*)a.k + (int64_t)kvh * a.k_sh;
  const T* vbase = (const T*)a.v + (int64_t)kvh * a.v_sh;
  u32x4 kr[LD], vr[LD];
  float pr[2] = {0.f, 0.f};
  auto fetch = [&](int t) {
    const int k0 = k_lo + t * KT;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int e = tid + i * NT, row = e / CH, ch = e % CH;
      const int64_t j = (int64_t)k0 + row;
      const bool ok = j < k_hi;
      kr[i] = load_chunk<T>(kbase + j * a.k_sn, ch, a.D, ok, a.vec_k);
      vr[i] = load_chunk<T>(vbase + j * a.v_sn, ch, a.D, ok, a.vec_v);
    }
    if constexpr (POS > 0) {
      if (tid < KT && k0 + tid < k_hi) {
        pr[0] = load_pos(a.pos_k, (int64_t)k0 + tid, POS, 0);
        if (POS == 2) pr[1] = load_pos(a.pos_k, (int64_t)k0 + tid, POS, 1);
      }
    }
  };
  auto stage = [&](int buf) {
    DGMC_LDS char* kt = lds + buf * 2 * TB;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int e = tid + i * NT, row = e / CH, ch = e % CH;
      const int off = (row * CH + (ch ^ swz<CH>(row))) * 16;
      *(DGMC_LDS u32x4*)(kt + off) = kr[i];
      *(DGMC_LDS u32x4*)(kt + TB + off) = vr[i];
    }
    if constexpr (POS > 0) {
      if (tid < KT) {
        kpos[(buf * 2 + 0) * KT + tid] = pr[0];
        if (POS == 2) kpos[(buf * 2 + 1) * KT + tid] = pr[1];
      }
    }
  };

  f32x16 acc[DP / 32];
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[k][r] = 0.f;
  float m = -INFINITY, l = 0.f;
  const float s1 = a.cap > 0.f ? a.scale / a.cap : a.scale * kLog2e;
  const float s2 = a.cap * kLog2e;

  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const int buf = (t - t0) & 1;
    stage(buf);
    if (t + 1 < t1) fetch(t + 1);
    __syncthreads();
    const DGMC_LDS char* kt = lds + buf * 2 * TB;
    f32x16 z[KT / 32];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) z[u][r] = 0.f;
#pragma unroll
      for (int s = 0; s < CH / 2; ++s)
        z[u] = Mma<T>::dot(lds_chunk<CH>(kt, 32 * u + c, 2 * s + h), qf[s],
                           z[u]);
    }
    if (a.cap > 0.f) {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          z[u][r] = s2 * tanh_<sizeof(T) == 4>(z[u][r] * s1);
    } else {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[u][r] *= s1;
    }
    if constexpr (POS > 0) {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int row = 32 * u + 8 * r4 + 4 * h;
          const f32x4 kx =
              *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 0) * KT + row);
          f32x4 ky = kx;
          if (POS == 2)
            ky = *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 1) * KT + row);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            int s = bk.slot(kx[r] - px);
            if (POS == 2) s = s * W + bk.slot(ky[r] - py);
            z[u][4 * r4 + r] += mytab[s];
          }
        }
      }
    }
    const int left = k_hi - (k_lo + t * KT);
    if (left < KT) {
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * u + 8 * (r >> 2) + 4 * h + (r & 3) >= left)
            z[u][r] = -INFINITY;
    }
    float mt = z[0][0];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) mt = fmaxf(mt, z[u][r]);
    mt = max_half(mt);
    if (__any(mt > m + 8.f)) {
      const float mn = fmaxf(m, mt);
      const float al = mn == m ? 1.f : exp2_(m - mn);
      l *= al;
#pragma unroll
      for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[k][r] *= al;
      m = mn;
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
      for (int r = 0; r < 16; ++r) z[u][r] = exp2_(z[u][r] - ms);
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) s += z[u][r];
      l += s;
      Mma<T>::template accum<DP>(acc, kt + TB, 32 * u, z[u]);
    }
  }
  l = sum_half(l);
  if (!live) return;
  const int64_t row = qi * a.H + head;
  if (a.splits > 1) {
    const int64_t prow = (int64_t)split * a.Nq * a.H + row;
    if (h == 0) {
      a.part_ml[prow * 2] = m;
      a.part_ml[prow * 2 + 1] = l;
    }
    float* po = a.part_o + prow * a.D;
#pragma unroll
    for (int k = 0; k < DP / 32; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = 32 * k + 8 * (r >> 2) + 4 * h + (r & 3);
        if (d < a.D) po[d] = acc[k][r];
      }
    return;
  }
  // l is 0 only without a key of finite score: such a row is 0.
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (h == 0 && a.lse) a.lse[row] = l == 0.f ? INFINITY : m + log2f(l);
  T* orow = (T*)a.out + row * a.D;
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int d = 32 * k + 8 * r4 + 4 * h;
      T o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (T)(acc[k][4 * r4 + r] * inv);
      if (a.D % 4 == 0) {
        if (d < a.D) __builtin_memcpy(__builtin_assume_aligned(
                         orow + d, 4 * sizeof(T)), o, 4 * sizeof(T));
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (d + r < a.D) orow[d + r] = o[r];
      }
    }
}

template <typename T, int DP, int NW>
void launch_fwd(const Args& a, int axes, hipStream_t st) {
  // Tiles of 64 keys while both buffers of K and V fit 64 KB of LDS.
  constexpr int KT = (NW > 1 && DP * (int)sizeof(T) <= 256) ? 64 : 32;
  const int TQ = 32 / a.G * NW;
  const dim3 grid((a.Nq / TQ + a.B + 1) * a.KV, a.splits), blk(NW * 64);
  const size_t sm = 4 * KT * DP * sizeof(T) +
                    (axes ? 16 * KT + a.G * kSlots * 4 : 0);
  auto kern = axes == 0   ? fwd_kernel<T, DP, NW, KT, 0>
              : axes == 1 ? fwd_kernel<T, DP, NW, KT, 1>
                          : fwd_kernel<T, DP, NW, KT, 2>;
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<grid, blk, sm, st>>>(a);
  DGMC_CHECK_LAUNCH();
}

template <typename T>
void run_fwd(const Args& a, int axes, int nw, hipStream_t st) {
  if (a.D <= 32)
    nw == 1 ? launch_fwd<T, 32, 1>(a, axes, st)
            : launch_fwd<T, 32, 4>(a, axes, st);
  else if (a.D <= 64)
    nw == 1 ? launch_fwd<T, 64, 1>(a, axes, st)
            : launch_fwd<T, 64, 4>(a, axes, st);
  else
    nw == 1 ? launch_fwd<T, 128, 1>(a, axes, st)
            : launch_fwd<T, 128, 4>(a, axes, st);
}

}  // namespace segattn
}  // namespace dgmc
