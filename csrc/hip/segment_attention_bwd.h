// Backward kernels of the segment attention (segment_attention.h): with
// p_ij recomputed from the forward's log-sum-exp,
//
//   delta_i = <do_i, o_i>,  dz_ij = p_ij (<do_i, v_j> - delta_i)
//   dT[h, b] = sum of dz_ij over the pairs in bucket b
//   ds_ij = dz_ij (1 - tanh^2) scale,   dq = ds k,  dk = ds^T q,  dv = p^T do
//
// Two kernels, each owning its output rows (no atomics, a fixed order of
// every sum): dq_kernel has a query per lane column and walks the keys
// (writing delta on the way), dkv_kernel a key per column and walks the
// packed query rows of the whole head group, so shared key heads need no
// second reduction.  Each recomputes the scores: 7 products in place of 5,
// against atomics on dq.
//
// The table's gradient: every lane adds its dz into its own LDS column of
// [slots][64] (no address is shared: no conflicts and a fixed order); a
// workgroup keeps its columns over all the tiles it walks and sums them
// once, a last kernel adds the workgroups' parts in order.
#pragma once

#include "segment_attention.h"

namespace dgmc {
namespace segattn {

// Scores of one 32 x 32 block in log2 units, from the raw products; `t`
// receives tanh where the scores are capped.
template <bool EXACT>
__device__ __forceinline__ void cap_scores(const Args& a, f32x16& z,
                                           f32x16& t) {
  if (a.cap > 0.f) {
    const float s1 = a.scale / a.cap, s2 = a.cap * kLog2e;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      t[r] = tanh_<EXACT>(z[r] * s1);
      z[r] = s2 * t[r];
    }
  } else {
    const float s1 = a.scale * kLog2e;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] *= s1;
  }
}

template <typename T, int DP, int NW, int POS>
__global__ __launch_bounds__(NW * 64, 1) void dq_kernel(const Args a,
                                                        int nslot) {
  constexpr int KT = 32;
  constexpr int CH = DP * (int)sizeof(T) / 16;
  constexpr int NT = NW * 64;
  constexpr int LD = (KT * CH + NT - 1) / NT;
  constexpr int TB = KT * CH * 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  DGMC_LDS float* kpos = (DGMC_LDS float*)(lds + 4 * TB);   // [2][2][KT]
  DGMC_LDS float* tab = kpos + (POS ? 4 * KT : 0);          // [G][kSlots]
  DGMC_LDS float* hist = tab + (POS ? a.G * kSlots : 0);    // [NW][slots][64]

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, blk = blockIdx.x / a.KV;
  const int nblk = gridDim.x / a.KV;
  const int QW = 32 / a.G, TQ = QW * NW;
  const int g = c % a.G, W = 2 * a.half + 2;
  const int head = kvh * a.G + g;
  const Bucket bk(a);
  const DGMC_LDS float* mytab = tab + g * kSlots;
  DGMC_LDS float* myhist = hist + wave * a.slots * 64 + lane;
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    for (int s = 0; s < a.slots; ++s) myhist[s * 64] = 0.f;
  }
  const T* kbase = (const T*)a.k + (int64_t)kvh * a.k_sh;
  const T* vbase = (const T*)a.v + (int64_t)kvh * a.v_sh;

  for (int slot = blk; slot < nslot; slot += nblk) {
    const int seg = find_segment(a.ptr_q, a.B, a.Nq, TQ, slot);
    int q_lo, q_hi, k_lo = 0, k_hi = 0;
    seg_range(a.ptr_q, seg, a.B, a.Nq, q_lo, q_hi);
    q_lo += (slot - (seg_begin(a.ptr_q, seg, a.Nq) / TQ + seg)) * TQ;
    if (q_lo >= q_hi) continue;
    if (seg < a.B) seg_range(a.ptr_k, seg, a.B, a.Nk, k_lo, k_hi);

    const int64_t qi = (int64_t)q_lo + wave * QW + c / a.G;
    const bool live = c < QW * a.G && qi < q_hi;
    const int64_t row = qi * a.H + head;
    const T* qrow = (const T*)a.q + qi * a.q_sn + (int64_t)head * a.q_sh;
    const T* grow = (const T*)a.dout + qi * a.g_sn + (int64_t)head * a.g_sh;
    const T* orow = (const T*)a.o + row * a.D;
    u32x4 qf[CH / 2], gf[CH / 2];
    float dl = 0.f;
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) {
      qf[s] = load_chunk<T>(qrow, 2 * s + h, a.D, live, a.vec_q);
      gf[s] = load_chunk<T>(grow, 2 * s + h, a.D, live, a.vec_g);
      dl += Mma<T>::chunk_dot(
          gf[s], load_chunk<T>(orow, 2 * s + h, a.D, live, a.vec_o));
    }
    dl = sum_half(dl);
    const float lse = live ? a.lse[row] : INFINITY;
    if (live && h == 0) a.delta[row] = dl;
    float px = 0.f, py = 0.f;
    if (POS > 0 && live) {
      px = load_pos(a.pos_q, qi, POS, 0);
      if (POS == 2) py = load_pos(a.pos_q, qi, POS, 1);
    }

    const int ntile = (k_hi - k_lo + KT - 1) / KT;
    u32x4 kr[LD], vr[LD];
    float pr[2] = {0.f, 0.f};
    auto fetch = [&](int t) {
      const int k0 = k_lo + t * KT;
#pragma unroll
      for (int i = 0; i < LD; ++i) {
        const int e = tid + i * NT, rw = e / CH, ch = e % CH;
        const int64_t j = (int64_t)k0 + rw;
        const bool ok = rw < KT && j < k_hi;
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
        const int e = tid + i * NT, rw = e / CH, ch = e % CH;
        if (LD * NT == KT * CH || rw < KT) {
          const int off = (rw * CH + (ch ^ swz<CH>(rw))) * 16;
          *(DGMC_LDS u32x4*)(kt + off) = kr[i];
          *(DGMC_LDS u32x4*)(kt + TB + off) = vr[i];
        }
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

    if (ntile > 0) fetch(0);
    __syncthreads();       // the previous slot's last tile has been read
    for (int t = 0; t < ntile; ++t) {
      const int buf = t & 1;
      stage(buf);
      if (t + 1 < ntile) fetch(t + 1);
      __syncthreads();
      const DGMC_LDS char* kt = lds + buf * 2 * TB;
      f32x16 z, dp, th;
#pragma unroll
      for (int r = 0; r < 16; ++r) z[r] = dp[r] = th[r] = 0.f;
#pragma unroll
      for (int s = 0; s < CH / 2; ++s) {
        z = Mma<T>::dot(lds_chunk<CH>(kt, c, 2 * s + h), qf[s], z);
        dp = Mma<T>::dot(lds_chunk<CH>(kt + TB, c, 2 * s + h), gf[s], dp);
      }
      cap_scores<sizeof(T) == 4>(a, z, th);
      int sl[16];
      if constexpr (POS > 0) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int rw = 8 * r4 + 4 * h;
          const f32x4 kx =
              *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 0) * KT + rw);
          f32x4 ky = kx;
          if (POS == 2)
            ky = *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 1) * KT + rw);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            int s = bk.slot(kx[r] - px);
            if (POS == 2) s = s * W + bk.slot(ky[r] - py);
            sl[4 * r4 + r] = s;
            z[4 * r4 + r] += mytab[s];
          }
        }
      }
      const int left = k_hi - (k_lo + t * KT);
      if (left < KT) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (8 * (r >> 2) + 4 * h + (r & 3) >= left) z[r] = -INFINITY;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r)
        z[r] = exp2_(z[r] - lse) * (dp[r] - dl);
      if constexpr (POS > 0) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          __hip_atomic_fetch_add(myhist + sl[r] * 64, z[r], __ATOMIC_RELAXED,
                                 __HIP_MEMORY_SCOPE_WORKGROUP);
      }
      if (a.cap > 0.f) {
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] *= fmaf(-th[r], th[r], 1.f);
      }
      Mma<T>::template accum<DP>(acc, kt, 0, z);
    }
    if (live && a.dq != nullptr) {
      T* drow = (T*)a.dq + row * a.D;
#pragma unroll
      for (int k = 0; k < DP / 32; ++k)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int d = 32 * k + 8 * (r >> 2) + 4 * h + (r & 3);
          if (d < a.D) drow[d] = (T)(acc[k][r] * a.scale);
        }
    }
  }
  if constexpr (POS > 0) {
    // Columns of this workgroup in a fixed order, started at a lane's own
    // (64 different banks).
    __syncthreads();
    const int RW = QW * a.G;
    for (int e = tid; e < a.G * a.slots; e += NT) {
      const int gg = e / a.slots, s = e % a.slots;
      float sum = 0.f;
      for (int w = 0; w < NW; ++w)
        for (int j = 0; j < 64; ++j) {
          const int col = (j + s) & 63;
          if ((col & 31) < RW && (col & 31) % a.G == gg)
            sum += hist[(w * a.slots + s) * 64 + col];
        }
      a.part_bias[((int64_t)blk * a.KV + kvh) * a.G * a.slots + e] = sum;
    }
  }
}

template <typename T, int DP, int NW, int POS>
__global__ __launch_bounds__(NW * 64, 1) void dkv_kernel(const Args a) {
  constexpr int QT = 32;                         // packed rows per tile
  constexpr int CH = DP * (int)sizeof(T) / 16;
  constexpr int NT = NW * 64;
  constexpr int LD = (QT * CH + NT - 1) / NT;
  constexpr int TB = QT * CH * 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  DGMC_LDS float* rowv = (DGMC_LDS float*)(lds + 4 * TB);   // [2][4][QT]
  DGMC_LDS float* tab = rowv + 8 * QT;                      // [G][kSlots]

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, slot = blockIdx.x / a.KV;
  const int QW = 32 / a.G, RW = QW * a.G;
  const int seg = find_segment(a.ptr_k, a.B, a.Nk, 32 * NW, slot);
  int k_lo, k_hi, q_lo = 0, q_hi = 0;
  seg_range(a.ptr_k, seg, a.B, a.Nk, k_lo, k_hi);
  k_lo += (slot - (seg_begin(a.ptr_k, seg, a.Nk) / (32 * NW) + seg)) * 32 *
          NW;
  if (k_lo >= k_hi) return;
  if (seg < a.B) seg_range(a.ptr_q, seg, a.B, a.Nq, q_lo, q_hi);

  const int64_t kj = (int64_t)k_lo + wave * 32 + c;
  const bool live = kj < k_hi;
  const T* krow = (const T*)a.k + kj * a.k_sn + (int64_t)kvh * a.k_sh;
  const T* vrow = (const T*)a.v + kj * a.v_sn + (int64_t)kvh * a.v_sh;
  u32x4 kf[CH / 2], vf[CH / 2];
#pragma unroll
  for (int s = 0; s < CH / 2; ++s) {
    kf[s] = load_chunk<T>(krow, 2 * s + h, a.D, live, a.vec_k);
    vf[s] = load_chunk<T>(vrow, 2 * s + h, a.D, live, a.vec_v);
  }
  float px = 0.f, py = 0.f;
  const Bucket bk(a);
  const int W = 2 * a.half + 2;
  int gb[16];                     // the accumulator rows' tables
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    if (live) {
      px = load_pos(a.pos_k, kj, POS, 0);
      if (POS == 2) py = load_pos(a.pos_k, kj, POS, 1);
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      gb[r] = ((8 * (r >> 2) + 4 * h + (r & 3)) % a.G) * kSlots;
  }

  const int ntile = (q_hi - q_lo + QW - 1) / QW;
  u32x4 qr[LD], gr[LD];
  float rv[4] = {INFINITY, 0.f, 0.f, 0.f};
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int e = tid + i * NT, rw = e / CH, ch = e % CH;
      const int64_t qi = (int64_t)q_lo + t * QW + rw / a.G;
      const int head = kvh * a.G + rw % a.G;
      const bool ok = rw < RW && qi < q_hi;
      qr[i] = load_chunk<T>((const T*)a.q + qi * a.q_sn + head * a.q_sh, ch,
                            a.D, ok, a.vec_q);
      gr[i] = load_chunk<T>((const T*)a.dout + qi * a.g_sn + head * a.g_sh,
                            ch, a.D, ok, a.vec_g);
    }
    if (tid < QT) {
      const int64_t qi = (int64_t)q_lo + t * QW + tid / a.G;
      const bool ok = tid < RW && qi < q_hi;
      const int64_t row = qi * a.H + kvh * a.G + tid % a.G;
      rv[0] = ok ? a.lse[row] : INFINITY;      // p = 0 in a row not there
      rv[1] = ok ? a.delta[row] : 0.f;
      if (POS > 0) {
        rv[2] = ok ? load_pos(a.pos_q, qi, POS, 0) : 0.f;
        if (POS == 2) rv[3] = ok ? load_pos(a.pos_q, qi, POS, 1) : 0.f;
      }
    }
  };
  auto stage = [&](int buf) {
    DGMC_LDS char* qt = lds + buf * 2 * TB;
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const int e = tid + i * NT, rw = e / CH, ch = e % CH;
      if (LD * NT == QT * CH || rw < QT) {
        const int off = (rw * CH + (ch ^ swz<CH>(rw))) * 16;
        *(DGMC_LDS u32x4*)(qt + off) = qr[i];
        *(DGMC_LDS u32x4*)(qt + TB + off) = gr[i];
      }
    }
    if (tid < QT) {
#pragma unroll
      for (int k = 0; k < 2 + POS; ++k)
        rowv[(buf * 4 + k) * QT + tid] = rv[k];
    }
  };

  f32x16 ak[DP / 32], av[DP / 32];
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) ak[k][r] = av[k][r] = 0.f;

  if (ntile > 0) fetch(0);
  for (int t = 0; t < ntile; ++t) {
    const int buf = t & 1;
    stage(buf);
    if (t + 1 < ntile) fetch(t + 1);
    __syncthreads();
    const DGMC_LDS char* qt = lds + buf * 2 * TB;
    const DGMC_LDS float* rw = rowv + buf * 4 * QT;
    f32x16 z, dp, th;
#pragma unroll
    for (int r = 0; r < 16; ++r) z[r] = dp[r] = th[r] = 0.f;
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) {
      z = Mma<T>::dot(lds_chunk<CH>(qt, c, 2 * s + h), kf[s], z);
      dp = Mma<T>::dot(lds_chunk<CH>(qt + TB, c, 2 * s + h), vf[s], dp);
    }
    cap_scores<sizeof(T) == 4>(a, z, th);
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const int o = 8 * r4 + 4 * h;
      const f32x4 ls = *(const DGMC_LDS f32x4*)(rw + o);
      const f32x4 de = *(const DGMC_LDS f32x4*)(rw + QT + o);
      if constexpr (POS > 0) {
        const f32x4 qx = *(const DGMC_LDS f32x4*)(rw + 2 * QT + o);
        f32x4 qy = qx;
        if (POS == 2) qy = *(const DGMC_LDS f32x4*)(rw + 3 * QT + o);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          int s = bk.slot(px - qx[r]);
          if (POS == 2) s = s * W + bk.slot(py - qy[r]);
          z[4 * r4 + r] += tab[gb[4 * r4 + r] + s];
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 4 * r4 + r;
        z[i] = exp2_(z[i] - ls[r]);
        dp[i] = z[i] * (dp[i] - de[r]);
      }
    }
    if (a.cap > 0.f) {
#pragma unroll
      for (int r = 0; r < 16; ++r) dp[r] *= fmaf(-th[r], th[r], 1.f);
    }
    Mma<T>::template accum<DP>(av, qt + TB, 0, z);
    Mma<T>::template accum<DP>(ak, qt, 0, dp);
  }
  if (!live) return;
  T* dk = (T*)a.dk + (kj * a.KV + kvh) * a.D;
  T* dv = (T*)a.dv + (kj * a.KV + kvh) * a.D;
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int d = 32 * k + 8 * (r >> 2) + 4 * h + (r & 3);
      if (d < a.D) {
        dk[d] = (T)(ak[k][r] * a.scale);
        dv[d] = (T)av[k][r];
      }
    }
}

template <typename T, int DP, int NW, int POS>
void launch_dq(const Args& a, int nblk, hipStream_t st) {
  const int TQ = 32 / a.G * NW, nslot = a.Nq / TQ + a.B + 1;
  const size_t sm = 4 * 32 * DP * sizeof(T) +
                    (POS ? 16 * 32 + a.G * kSlots * 4 +
                               (size_t)NW * a.slots * 256 : 0);
  auto kern = dq_kernel<T, DP, NW, POS>;
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<dim3((POS ? nblk : nslot) * a.KV), dim3(NW * 64), sm, st>>>(a,
                                                                    nslot);
  DGMC_CHECK_LAUNCH();
}

template <typename T, int DP, int NW, int POS>
void launch_dkv(const Args& a, hipStream_t st) {
  const size_t sm = 4 * 32 * DP * sizeof(T) + 8 * 32 * 4 +
                    (POS ? a.G * kSlots * 4 : 0);
  auto kern = dkv_kernel<T, DP, NW, POS>;
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<dim3((a.Nk / (32 * NW) + a.B + 1) * a.KV), dim3(NW * 64), sm, st>>>(
      a);
  DGMC_CHECK_LAUNCH();
}

template <typename T, int DP, int NW>
void dq_axes(const Args& a, int axes, int nblk, hipStream_t st) {
  axes == 0   ? launch_dq<T, DP, NW, 0>(a, nblk, st)
  : axes == 1 ? launch_dq<T, DP, NW, 1>(a, nblk, st)
              : launch_dq<T, DP, NW, 2>(a, nblk, st);
}
template <typename T, int DP, int NW>
void dkv_axes(const Args& a, int axes, hipStream_t st) {
  axes == 0   ? launch_dkv<T, DP, NW, 0>(a, st)
  : axes == 1 ? launch_dkv<T, DP, NW, 1>(a, st)
              : launch_dkv<T, DP, NW, 2>(a, st);
}
template <typename T, int DP>
void bwd_dim(const Args& a, int axes, int nwq, int nwk, int nblk,
             hipStream_t st) {
  nwq == 1 ? dq_axes<T, DP, 1>(a, axes, nblk, st)
           : dq_axes<T, DP, 4>(a, axes, nblk, st);
  if (a.dk == nullptr) return;
  nwk == 1 ? dkv_axes<T, DP, 1>(a, axes, st)
           : dkv_axes<T, DP, 4>(a, axes, st);
}

// The dq kernel first: it writes the rows' delta.
template <typename T>
void run_bwd(const Args& a, int axes, int nwq, int nwk, int nblk,
             hipStream_t st) {
  a.D <= 32   ? bwd_dim<T, 32>(a, axes, nwq, nwk, nblk, st)
  : a.D <= 64 ? bwd_dim<T, 64>(a, axes, nwq, nwk, nblk, st)
              : bwd_dim<T, 128>(a, axes, nwq, nwk, nblk, st);
}

}  // namespace segattn
}  // namespace dgmc
