// Backward kernels of the segment attention (segment_attention.h): with
// p_ij recomputed from the forward's row maximum and sum,
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
// against atomics on dq.  P and dS enter their bf16 products rounded to bf16
// (an error of the output's own rounding's size, averaged over the keys), on
// short segments as two bf16 terms (no error to average there, and products
// are not what takes the time).
//
// The table's gradient: every lane adds its dz into its own LDS column of
// [slots][64] (no address is shared at a time: no conflicts and a fixed
// order); a workgroup keeps its columns over all the tiles it walks and sums
// them once, a last kernel adds the workgroups' parts in order.
//
// Measured (dq / dkv).  4847 x 4893 rows, fp32 as x6, 4 heads of 64: 231 /
// 316 us, 156 TFLOP/s of fp32 products - the matrix cores, six products for
// one; with a table dq takes exact products: 579 us.  24 graphs of 1 to 1350
// nodes, bf16, 8 heads on 2 key heads of 128, cap and table: 151 / 165 us;
// vector units busy 34 / 26 % of it, matrix cores 9 / 12 %: the time is that
// of the workgroups with the most tiles (dq: 42 against 23 on average).  1024
// graphs of 3 to 19 nodes, fp32, two position axes: 42 / 39 us (dq: vector
// units busy 18 %, matrix cores 15 %), 512 pairs of 30 to 80 nodes, bf16: 54 /
// 40 us; latency of one wave's chain.
#pragma once

#include "segment_attention.h"

namespace dgmc {
namespace segattn {

// hist[sl[r]] += v[r] in a lane's own LDS column, four at a time and in
// order.  A plain read, add, write: ds_add_f32 took 120 cycles and more a
// wave (ragged case: 552 us, without the table 139 us).  Equal slots among
// the four take the earlier ones' values along and the last write counts;
// where all four are one slot in every lane (nodes in order, far apart) they
// are added first.
//
// HC = 32: lanes l and l ^ 32 (one query's) share a column, one half of the
// wave after the other - half the LDS, and the waves that fit beside it are
// what a short segment's time depends on.
template <int HC>
__device__ __forceinline__ void add_slots(DGMC_LDS float* hist,
                                          const int (&sl)[4],
                                          const float (&v)[4]) {
  const int a = sl[0], b = sl[1], c = sl[2], d = sl[3];
  const auto halves = [&](auto add) {
    if constexpr (HC == 64) {
      add();
    } else {
      if ((threadIdx.x & 32) == 0) add();
      asm volatile("" ::: "memory");     // (one thread's two cases are two)
      if ((threadIdx.x & 32) != 0) add();
      asm volatile("" ::: "memory");
    }
  };
  if (__all(a == b && b == c && c == d)) {
    const float all = (v[0] + v[1]) + (v[2] + v[3]);
    halves([&] { hist[a * HC] += all; });
    return;
  }
  const float va = v[0], vb = v[1] + (a == b ? va : 0.f);
  const float vc = v[2] + (b == c ? vb : a == c ? va : 0.f);
  const float vd = v[3] + (c == d ? vc : b == d ? vb : a == d ? va : 0.f);
  halves([&] {
    const float ha = hist[a * HC], hb = hist[b * HC], hc = hist[c * HC],
                hd = hist[d * HC];
    hist[a * HC] = ha + va;
    hist[b * HC] = hb + vb;
    hist[c * HC] = hc + vc;
    hist[d * HC] = hd + vd;
  });
}

// Columns of a wave's table sums.
constexpr int hist_cols(int nw) { return nw == 1 ? 32 : 64; }

// Wide heads at two waves per SIMD: registers are short.
template <typename P>
constexpr bool tight(int DP) {
  return P::kPlanes == 1 && sizeof(typename P::S) == 2 && DP == 128;
}

template <typename P, int DP, int NW, int POS>
__global__ __launch_bounds__(
    NW * 64,
    sizeof(typename P::S) == 2 || (NW == 1 && DP <= 64) ? 2 : 1) void
dq_kernel(const Args a, int ntiles) {
  using T = typename P::T;
  using S = typename P::S;
  constexpr bool kTight = tight<P>(DP);
  constexpr int KT = 32;
  constexpr int CH = DP * (int)sizeof(S) / 16;
  constexpr int NT = NW * 64;
  constexpr int TB = P::kPlanes * KT * CH * 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  const int NB = stage_bufs<P, NW>(a);
  DGMC_LDS float* kpos = (DGMC_LDS float*)(lds + 2 * NB * TB);  // [NB][2][KT]
  DGMC_LDS float* tab = kpos + (POS ? 2 * NB * KT : 0);          // [G][kTab]
  DGMC_LDS float* hist = tab + (POS ? a.G * kTab : 0);    // [NW][slots][HC]
  constexpr int HC = hist_cols(NW);

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, blk = blockIdx.x / a.KV;
  const int nblk = gridDim.x / a.KV;
  const int QW = 32 / a.G, TQ = QW * NW;
  const int cq = div_group(a, c), g = c - cq * a.G, W = 2 * a.half + 2;
  const int head = kvh * a.G + g, qo = wave * QW + cq;
  const Bucket bk(a);
  const DGMC_LDS float* mytab = tab + g * kTab;
  DGMC_LDS float* myhist = hist + wave * a.slots * HC + (lane & (HC - 1));
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    for (int s = 0; s < a.slots; ++s) myhist[s * HC] = 0.f;
  }
  const S* kbase = (const S*)a.k + (int64_t)kvh * a.k_sh;
  const S* vbase = (const S*)a.v + (int64_t)kvh * a.v_sh;
  const bool capped = a.cap > 0.f;
  const float s1 = capped ? a.scale / a.cap : a.scale * kLog2e;
  const float s2 = a.cap * kLog2e;
  const bool plain = plain_scores<POS>(a, s1);
  constexpr bool kOther = sizeof(S) == 4 && NW > 1 && POS > 0;
  const int rows0 = row_base<CH>(), cols0 = P::template cols<CH>();

  for (int it = blk; it < ntiles * a.splits; it += nblk) {
    const int split = it % a.splits;
    const int q_lo = it / a.splits * TQ, q_hi = min(q_lo + TQ, a.Nq);
    const int qi = q_lo + qo;
    const bool live = c < QW * a.G && qi < q_hi;
    const int64_t row = (int64_t)qi * a.H + head;
    u32x4 qf[P::kPlanes][CH / 2], gf[P::kPlanes][CH / 2];
    load_frags<P>(qf,
                  (const S*)a.q + (int64_t)q_lo * a.q_sn +
                      (int64_t)kvh * a.G * a.q_sh,
                  a.q_sp, (qo * a.q_sn + g * a.q_sh) * (int64_t)sizeof(S),
                  live, a.D);
    load_frags<P>(gf,
                  (const S*)a.dout + (int64_t)q_lo * a.g_sn +
                      (int64_t)kvh * a.G * a.g_sh,
                  a.g_sp, (qo * a.g_sn + g * a.g_sh) * (int64_t)sizeof(S),
                  live, a.D);
    const int wrows = min(QW, q_hi - q_lo - wave * QW);
    const Rows w =
        Rows::find<NW>(a.ptr_q, a.ptr_k, a.B, a.Nq, a.Nk, q_lo, q_hi, qi,
                       wrows > 0 ? (wrows - 1) * a.G : -1);
    const int ntile = (w.hi - w.lo + KT - 1) / KT;
    const int per = split_tiles(a, ntile);
    if (split > 0 && split * per >= ntile) continue;
    put_splits(a, it / a.splits * a.KV + kvh, split, ntile, per);
    const int k_lo = w.lo + split * per * KT;
    const int k_hi = min(k_lo + per * KT, w.hi);

    // delta, in two parts of the output for bf16 (its rounding's rest).
    float dl = 0.f;
    {
      const int64_t ob = ((int64_t)q_lo * a.H + kvh * a.G) * a.D;
      const int64_t oo = ((int64_t)qo * a.H + g) * a.D * (int64_t)sizeof(T);
      if constexpr (P::kPlanes > 1) {
        // (the planes' sum is the value)
        u32x4 of[CH];
        load_row8(of, (const T*)a.o + ob, oo, live, a.D, a.vec_o);
#pragma unroll
        for (int s = 0; s < CH / 2; ++s)
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            const bf16x8 x = __builtin_bit_cast(bf16x8, gf[2 - p][s]);
            const f32x4 y0 = __builtin_bit_cast(f32x4, of[2 * s]),
                        y1 = __builtin_bit_cast(f32x4, of[2 * s + 1]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              dl = fmaf((float)x[i], y0[i], dl);
              dl = fmaf((float)x[4 + i], y1[i], dl);
            }
          }
      } else {
        u32x4 of[CH / 2];
        load_row(of, (const T*)a.o + ob, oo, live, a.D, a.vec_o);
#pragma unroll
        for (int s = 0; s < CH / 2; ++s) dl += P::chunk_dot(gf[0][s], of[s]);
        if constexpr (sizeof(T) == 2) {
          load_row(of, (const T*)a.out_lo + ob, oo, live, a.D, a.vec_o);
#pragma unroll
          for (int s = 0; s < CH / 2; ++s)
            dl += P::chunk_dot(gf[0][s], of[s]);
        }
      }
    }
    dl = sum_half(dl);
    // p / st.y, so also dz / st.y, is summed: 1 / sum is a row's own factor.
    const float2 st = live ? a.stat[row] : make_float2(INFINITY, 0.f);
    if (live && h == 0 && split == 0) a.delta[row] = dl;
    const bool scaled = !plain || __any(st.x < INFINITY && fabsf(st.x) > kFar);
    const float ex = scaled ? 1.f : s1;
    float px = 0.f, py = 0.f;
    if (POS > 0 && live) {
      px = load_pos(a.pos_q, qi, POS, 0);
      if (POS == 2) py = load_pos(a.pos_q, qi, POS, 1);
    }

    int pr[2] = {0, 0};
    auto fetch = [&](int k0, int e, int buf) {
      using St = Stager<P, KT, CH, NT>;
      const int left = e - k0;
      DGMC_LDS char* kt = lds + buf * 2 * TB;
      const auto ok = [&](int r) { return r < left; };
      St::fill(kbase + (int64_t)k0 * a.k_sn, a.k_sp, a.D, kt, ok,
               [&](int r) { return r * (a.k_sn * (int)sizeof(S)); });
      St::fill(vbase + (int64_t)k0 * a.v_sn, a.v_sp, a.D, kt + TB,
               ok, [&](int r) { return r * (a.v_sn * (int)sizeof(S)); });
      if constexpr (POS > 0) {
        if (tid < KT && tid < left) {
          pr[0] = a.pos_k[((int64_t)k0 + tid) * POS];
          if (POS == 2) pr[1] = a.pos_k[((int64_t)k0 + tid) * POS + 1];
        }
      }
    };
    auto put_pos = [&](int buf) {
      if constexpr (POS > 0) {
        if (tid < KT) {
          kpos[(buf * 2 + 0) * KT + tid] = to_pos(pr[0]);
          if (POS == 2) kpos[(buf * 2 + 1) * KT + tid] = to_pos(pr[1]);
        }
      }
    };

    // Passes as in the forward; the table's gradient is whole after the first
    // (no sum over a tile enters a dz).
    for (int pass = w.b0 - 1;; ++pass) {
      int p_lo, p_hi;
      w.pass_range(a.ptr_k, a.B, a.Nk, pass, k_lo, k_hi, p_lo, p_hi);
      f32x16 acc[DP / 32];
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) acc[k] = f32x16{};
      stage_barrier();     // the last tile staged before has been read
      if (p_lo < p_hi) fetch(p_lo, p_hi, 0);
      for (int k0 = p_lo, buf = 0; k0 < p_hi; k0 += KT, buf ^= NB - 1) {
        if (NB == 1 && k0 > p_lo) {
          stage_barrier();
          fetch(k0, p_hi, 0);
        }
        put_pos(buf);
        stage_barrier();
        if (NB == 2 && k0 + KT < p_hi) fetch(k0 + KT, p_hi, buf ^ 1);
        if (w.skip(k0, KT)) continue;
        const int rows = lane_base<CH>(rows0 + buf * 2 * TB);
        const int cols = lane_base<CH>(cols0 + buf * 2 * TB);
        f32x16 z, dp;
        if constexpr (kTight) {
          row_dot2<P, CH, KT>(
              z, dp, lds, TB, rows, [&](int s) { return qf[0][s]; },
              [&](int s) { return gf[0][s]; });
        } else {
          z = row_dot<P, CH, KT, true>(lds, rows, qf);
          dp = row_dot<P, CH, KT, true>(lds + TB, rows, gf);
        }
        const bool whole = w.whole(k0, KT, p_hi);
        const unsigned n = w.count(p_hi);
        const int j0 = k0 + 4 * h - w.r_lo;
        int one = 0;
        bool same = false;
        float bias1 = 0.f, sum1 = 0.f;
        if constexpr (POS == 1 && NW > 1) {
          same = one_bucket<true>(bk, kpos + buf * 2 * KT, px, live, one);
          if (same) bias1 = mytab[one];
        }
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          float v[4], t[4] = {0.f, 0.f, 0.f, 0.f};
          int sl[4] = {0, 0, 0, 0};
#pragma unroll
          for (int r = 0; r < 4; ++r) v[r] = z[4 * r4 + r];
          if (scaled) {
#pragma unroll
            for (int r = 0; r < 4; ++r) v[r] = mul_(v[r], s1);
          }
          if (capped) {
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              t[r] = tanh_<sizeof(T) == 4>(v[r]);
              v[r] = mul_(s2, t[r]);
            }
          }
          if constexpr (POS > 0) {
            if (same) {
#pragma unroll
              for (int r = 0; r < 4; ++r) v[r] += bias1;
            } else {
              const int o = 8 * r4 + 4 * h;
              const f32x4 kx =
                  *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 0) * KT + o);
              f32x4 ky = kx;
              if (POS == 2)
                ky = *(const DGMC_LDS f32x4*)(kpos + (buf * 2 + 1) * KT + o);
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                sl[r] = bk.slot(kx[r] - px);
                if (POS == 2) sl[r] = sl[r] * W + bk.slot(ky[r] - py);
                v[r] += mytab[sl[r]];
              }
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            float x = fmaf(v[r], ex, -st.x);
            // (the forward's scores were x6 products, other bits than these)
            if (kOther) x = x > 9.f ? 9.f : x;
            v[r] = exp2_(x) * (dp[4 * r4 + r] - dl);
          }
          if (!whole) {
            // (selected, not multiplied away: a masked key may hold NaN)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if ((unsigned)(j0 + 8 * r4 + r) >= n) v[r] = t[r] = 0.f;
          }
          if constexpr (POS > 0) {
            if (same) {
              sum1 += (v[0] + v[1]) + (v[2] + v[3]);
            } else if (pass < w.b0) {
              const float dz[4] = {v[0] * st.y, v[1] * st.y, v[2] * st.y,
                                   v[3] * st.y};
              add_slots<HC>(myhist, sl, dz);
            }
          }
#pragma unroll
          for (int r = 0; r < 4; ++r)
            z[4 * r4 + r] = v[r] * fmaf(-t[r], t[r], 1.f);
        }
        if constexpr (POS == 1 && NW > 1) {
          if (same && pass < w.b0) myhist[one * HC] += sum1 * st.y;
        }
        P::template accum<DP, KT, NW == 1>(acc, lds, cols, z);
      }
      const bool redo = pass < w.b0 && w.b1 > w.b0 &&
                        any_lane<NW>(live && not_finite(acc));
      if (!redo && live && (pass < w.b0 || w.seg == pass)) {
        if (per < ntile)        // joined by join_kernel
          put_acc<DP>(a.part_o + ((int64_t)split * a.Nq * a.H + row) * a.D,
                      acc, a.D, st.y);
        else
          put_acc<DP>((T*)a.dq + row * a.D, acc, a.D, a.scale * st.y);
      }
      if (pass < w.b0 ? !redo : pass == w.b1) break;
    }
  }
  if constexpr (POS > 0) {
    // Columns of this workgroup in a fixed order, started at a lane's own
    // (different banks).
    __syncthreads();
    const int RW = QW * a.G;
    for (int e = tid; e < a.G * a.slots; e += NT) {
      const int gg = e / a.slots, s = e % a.slots;
      float sum = 0.f;
      for (int wv = 0; wv < NW; ++wv) {
#pragma unroll 8
        for (int j = 0; j < HC; ++j) {
          const int col = (j + s) & (HC - 1), cc = col & 31;
          const float x = hist[(wv * a.slots + s) * HC + col];
          sum += cc < RW && cc - div_group(a, cc) * a.G == gg ? x : 0.f;
        }
      }
      a.part_bias[((int64_t)blk * a.KV + kvh) * a.G * a.slots + e] = sum;
    }
  }
}

template <typename P, int DP, int NW, int POS>
__global__ __launch_bounds__(
    NW * 64,
    sizeof(typename P::S) == 2 || (NW == 1 && DP <= 64) ? 2 : 1) void
dkv_kernel(const Args a) {
  using T = typename P::T;
  using S = typename P::S;
  constexpr int QT = 32;                         // packed rows per tile
  constexpr int CH = DP * (int)sizeof(S) / 16;
  constexpr int NT = NW * 64;
  constexpr int TB = P::kPlanes * QT * CH * 16;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  const int NB = stage_bufs<P, NW>(a);
  // Of every row: maximum, delta, 1 / sum, position.
  DGMC_LDS float* rowv = (DGMC_LDS float*)(lds + 2 * NB * TB);  // [NB][5][QT]
  DGMC_LDS int* toff = (DGMC_LDS int*)(rowv + 5 * NB * QT);     // [QT]
  DGMC_LDS int* far_rows = toff + QT;              // [2, of 4: see kFar]
  // Wide heads: the lanes' own rows of V and the last KL chunks of K, too
  // many for the registers (a spilled one's load in the loop waits for the
  // next tile's, in order: 14 segments of 30 to 1350 nodes, 297 us; so 204).
  constexpr bool VL = tight<P>(DP);
  constexpr int KL = VL ? 2 : 0, OWN = VL ? CH / 2 + KL : 0;
  DGMC_LDS u32x4* own = (DGMC_LDS u32x4*)(far_rows + 4);    // [OWN][NT]
  DGMC_LDS float* tab = (DGMC_LDS float*)(own + OWN * NT);  // [G][kTab]

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, split = blockIdx.y;
  const int QW = 32 / a.G, RW = QW * a.G;
  const int k_lo = blockIdx.x / a.KV * 32 * NW;
  const int k_hi = min(k_lo + 32 * NW, a.Nk);
  const int ko = wave * 32 + c, kj = k_lo + ko;
  const bool live = kj < k_hi;
  u32x4 kf[P::kPlanes][CH / 2], vf[P::kPlanes][CH / 2];
  load_frags<P>(kf,
                (const S*)a.k + (int64_t)k_lo * a.k_sn +
                    (int64_t)kvh * a.k_sh,
                a.k_sp, ko * a.k_sn * (int64_t)sizeof(S), live, a.D);
  load_frags<P>(vf,
                (const S*)a.v + (int64_t)k_lo * a.v_sn +
                    (int64_t)kvh * a.v_sh,
                a.v_sp, ko * a.v_sn * (int64_t)sizeof(S), live, a.D);
  if constexpr (VL) {
#pragma unroll
    for (int s = 0; s < CH / 2; ++s) own[s * NT + tid] = vf[0][s];
#pragma unroll
    for (int s = CH / 2 - KL; s < CH / 2; ++s)
      own[(s + KL) * NT + tid] = kf[0][s];
  }
  const int wrows = min(32, k_hi - k_lo - wave * 32);
  const Rows w = Rows::find<NW>(a.ptr_k, a.ptr_q, a.B, a.Nk, a.Nq, k_lo, k_hi,
                                kj, wrows > 0 ? wrows - 1 : -1);
  // The queries of this split.
  const int ntile = (w.hi - w.lo + QW - 1) / QW;
  const int per = split_tiles(a, ntile);
  if (split > 0 && split * per >= ntile) return;
  put_splits(a, blockIdx.x, split, ntile, per);
  const int q_lo = w.lo + split * per * QW;
  const int q_hi = min(q_lo + per * QW, w.hi);

  float px = 0.f, py = 0.f;
  const Bucket bk(a);
  const int W = 2 * a.half + 2;
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    if (tid < QT) toff[tid] = (tid - div_group(a, tid) * a.G) * kTab;
    if (live) {
      px = load_pos(a.pos_k, kj, POS, 0);
      if (POS == 2) py = load_pos(a.pos_k, kj, POS, 1);
    }
  }

  const S* qbase = (const S*)a.q + (int64_t)kvh * a.G * a.q_sh;
  const S* gbase = (const S*)a.dout + (int64_t)kvh * a.G * a.g_sh;
  float rv[3] = {INFINITY, 0.f, 0.f};
  int rp[2] = {0, 0};
  auto fetch = [&](int q0, int e, int buf) {
    using St = Stager<P, QT, CH, NT>;
    const int left = e - q0;
    DGMC_LDS char* qt = lds + buf * 2 * TB;
    const auto ok = [&](int r) { return r < RW && div_group(a, r) < left; };
    const auto off = [&](int r, int64_t sn, int64_t sh) {
      const int i = div_group(a, r);
      return (i * sn + (r - i * a.G) * sh) * (int64_t)sizeof(S);
    };
    // (first: a wait among these few is not one for the tile)
    if (tid < QT) {
      const int i = div_group(a, tid), qi = q0 + i;
      const bool there = tid < RW && qi < e;
      const int64_t row = (int64_t)qi * a.H + kvh * a.G + tid - i * a.G;
      // (p = 0 in a row not there)
      const float2 st = there ? a.stat[row] : make_float2(INFINITY, 0.f);
      rv[0] = st.x;
      rv[1] = there ? a.delta[row] : 0.f;
      rv[2] = st.y;
      if (POS > 0) {
        // (rows not there: the first one's)
        const int64_t i = there ? qi : q0;
        rp[0] = a.pos_q[i * POS];
        if (POS == 2) rp[1] = a.pos_q[i * POS + 1];
      }
    }
    St::fill(qbase + (int64_t)q0 * a.q_sn, a.q_sp, a.D, qt, ok,
             [&](int r) { return off(r, a.q_sn, a.q_sh); });
    St::fill(gbase + (int64_t)q0 * a.g_sn, a.g_sp, a.D, qt + TB, ok,
             [&](int r) { return off(r, a.g_sn, a.g_sh); });
  };
  auto put_rows = [&](int buf) {
    if (tid < QT) {
      const bool far = __any(rv[0] < INFINITY && fabsf(rv[0]) > kFar);
      if (tid == 0) far_rows[buf] = far;
#pragma unroll
      for (int k = 0; k < 3 + POS; ++k)
        rowv[(buf * 5 + k) * QT + tid] = k < 3 ? rv[k] : to_pos(rp[k - 3]);
    }
  };
  const bool capped = a.cap > 0.f;
  const float s1 = capped ? a.scale / a.cap : a.scale * kLog2e;
  const float s2 = a.cap * kLog2e;
  const bool plain = plain_scores<POS>(a, s1);
  const int rows0 = row_base<CH>(), cols0 = P::template cols<CH>();

  // Passes as in the forward.
  for (int pass = w.b0 - 1;; ++pass) {
    int p_lo, p_hi;
    w.pass_range(a.ptr_q, a.B, a.Nq, pass, q_lo, q_hi, p_lo, p_hi);
    f32x16 ak[DP / 32], av[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) ak[k] = av[k] = f32x16{};
    if (pass >= w.b0) stage_barrier();
    if (p_lo < p_hi) fetch(p_lo, p_hi, 0);
    for (int q0 = p_lo, buf = 0; q0 < p_hi; q0 += QW, buf ^= NB - 1) {
      if (NB == 1 && q0 > p_lo) {
        stage_barrier();
        fetch(q0, p_hi, 0);
      }
      put_rows(buf);
      stage_barrier();
      if (NB == 2 && q0 + QW < p_hi) fetch(q0 + QW, p_hi, buf ^ 1);
      if (w.skip(q0, QW)) continue;
      const DGMC_LDS float* rw = rowv + buf * 5 * QT;
      const bool scaled = !plain || far_rows[buf] != 0;
      const float ex = scaled ? 1.f : s1;
      const int rows = lane_base<CH>(rows0 + buf * 2 * TB);
      const int cols = lane_base<CH>(cols0 + buf * 2 * TB);
      f32x16 z, dp;
      if constexpr (VL) {
        row_dot2<P, CH, QT>(
            z, dp, lds, TB, rows,
            [&](int s) {
              return s < CH / 2 - KL ? kf[0][s] : own[(s + KL) * NT + tid];
            },
            [&](int s) { return own[s * NT + tid]; });
      } else {
        z = row_dot<P, CH, QT, false>(lds, rows, kf);
        dp = row_dot<P, CH, QT, false>(lds + TB, rows, vf);
      }
      const bool whole = w.whole(q0, QW, p_hi);
      const unsigned n = w.count(p_hi) * a.G;
      const int j0 = (q0 - w.r_lo) * a.G + 4 * h;
      int one = 0;
      bool same = false;
      if constexpr (POS == 1 && NW > 1)
        same = one_bucket<false>(bk, rw + 3 * QT, px, live, one);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const int o = 8 * r4 + 4 * h;
        const f32x4 mx = *(const DGMC_LDS f32x4*)(rw + o);
        const f32x4 de = *(const DGMC_LDS f32x4*)(rw + QT + o);
        const f32x4 inv = *(const DGMC_LDS f32x4*)(rw + 2 * QT + o);
        float p[4], t[4] = {0.f, 0.f, 0.f, 0.f}, ds[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = z[4 * r4 + r];
        if (scaled) {
#pragma unroll
          for (int r = 0; r < 4; ++r) p[r] = mul_(p[r], s1);
        }
        if (capped) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            t[r] = tanh_<sizeof(T) == 4>(p[r]);
            p[r] = mul_(s2, t[r]);
          }
        }
        if constexpr (POS > 0) {
          // (toff: the row's head's table)
          const i32x4 to = *(const DGMC_LDS i32x4*)(toff + o);
          if (same) {
#pragma unroll
            for (int r = 0; r < 4; ++r) p[r] += tab[one + to[r]];
          } else {
            const f32x4 qx = *(const DGMC_LDS f32x4*)(rw + 3 * QT + o);
            f32x4 qy = qx;
            if (POS == 2) qy = *(const DGMC_LDS f32x4*)(rw + 4 * QT + o);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              int s = bk.slot(px - qx[r]);
              if (POS == 2) s = s * W + bk.slot(py - qy[r]);
              p[r] += tab[s + to[r]];
            }
          }
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          p[r] = exp2_(fmaf(p[r], ex, -mx[r])) * inv[r];
          ds[r] = p[r] * (dp[4 * r4 + r] - de[r]);
        }
        if (!whole) {
          // Packed rows of other segments (selected, not multiplied away:
          // they may hold NaN; rows from RW on have p = 0).
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if ((unsigned)(j0 + 8 * r4 + r) >= n) p[r] = ds[r] = t[r] = 0.f;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          z[4 * r4 + r] = p[r];
          dp[4 * r4 + r] = ds[r] * fmaf(-t[r], t[r], 1.f);
        }
      }
      P::template accum<DP, QT, NW == 1>(av, lds + TB, cols, z);
      P::template accum<DP, QT, NW == 1>(ak, lds, cols, dp);
    }
    const bool redo =
        pass < w.b0 && w.b1 > w.b0 &&
        any_lane<NW>(live && (not_finite(ak) || not_finite(av)));
    if (!redo && live && (pass < w.b0 || w.seg == pass)) {
      const int64_t row = (int64_t)kj * a.KV + kvh;
      if (per < ntile) {        // joined by join_kernel
        const int64_t all = (int64_t)a.Nk * a.KV;
        float* p = a.part_o + (split * all + row) * a.D;
        put_acc<DP>(p, ak, a.D, 1.f);
        put_acc<DP>(p + a.splits * all * a.D, av, a.D, 1.f);
      } else {
        put_acc<DP>((T*)a.dk + row * a.D, ak, a.D, a.scale);
        put_acc<DP>((T*)a.dv + row * a.D, av, a.D, 1.f);
      }
    }
    if (pass < w.b0 ? !redo : pass == w.b1) return;
  }
}

template <typename P, int DP, int NW>
void launch_dq(const Args& a, int axes, int nblk, hipStream_t st) {
  constexpr int B = P::kPlanes * (int)sizeof(typename P::S);
  const int TQ = 32 / a.G * NW, ntiles = (a.Nq + TQ - 1) / TQ;
  const int NB = NW == 1 ? a.bufs : 2;
  const size_t sm = NB * (2 * 32 * DP * B + (axes ? 8 * 32 : 0)) +
                    (axes ? a.G * kTab * 4 +
                                (size_t)NW * a.slots * hist_cols(NW) * 4
                          : 0);
  auto kern = dq_kernel<P, DP, NW, 0>;
  if constexpr (P::kPlanes == 1) {     // (x6: without a table only)
    if (axes == 1) kern = dq_kernel<P, DP, NW, 1>;
    if (axes == 2) kern = dq_kernel<P, DP, NW, 2>;
  }
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<dim3((axes ? nblk : ntiles * a.splits) * a.KV), dim3(NW * 64), sm,
         st>>>(a, ntiles);
  DGMC_CHECK_LAUNCH();
}

template <typename P, int DP, int NW>
void launch_dkv(const Args& a, int axes, hipStream_t st) {
  constexpr int B = P::kPlanes * (int)sizeof(typename P::S);
  const int NB = NW == 1 ? a.bufs : 2;
  const size_t sm = NB * (2 * 32 * DP * B + 5 * 32 * 4) + 36 * 4 +
                    (tight<P>(DP) ? (8 + 2) * NW * 64 * 16 : 0) +
                    (axes ? a.G * kTab * 4 : 0);
  auto kern = axes == 0   ? dkv_kernel<P, DP, NW, 0>
              : axes == 1 ? dkv_kernel<P, DP, NW, 1>
                          : dkv_kernel<P, DP, NW, 2>;
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<dim3((a.Nk + 32 * NW - 1) / (32 * NW) * a.KV, a.splits),
         dim3(NW * 64), sm, st>>>(a);
  DGMC_CHECK_LAUNCH();
}

}  // namespace segattn
}  // namespace dgmc
