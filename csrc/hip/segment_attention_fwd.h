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
// sum and outputs are fp32.  FINE (bf16): P enters as two bf16 terms - in
// training, where the rounding rest of the output is kept beside it too,
// because the backward's delta = <do, o> multiplies whole rows of P and its
// error does not average out over the keys (the table's gradient would lose
// 2 of bf16's 8 bits); and on short segments, whose few keys average nothing
// out and whose time is latency, not products.
//
// Measured.  19388 x 19572 rows, 4 heads of 64, bf16: 470 us with its join,
// 0.83 PFLOP/s.  Per 32 x 64 scores the vector unit has 830 cycles of work
// (exp2 takes 16 a wave) and the matrix cores 512; counters find them busy 65
// and 40 % of the time: for the most part one runs after the other.  4847 x
// 4893 rows, fp32 as x6: 148 us, 164 TFLOP/s, matrix cores; with a table 184.
// One row in each of four graphs of 14000 to 20000 nodes, bf16, heads of 128:
// 23 us, 75 MB at 3.2 TB/s (474 workgroups of one wave, a tile in flight
// each).  1024 graphs of 3 to 19 nodes, fp32, heads of 64: 27 us, the chain of
// dependent loads (segment search, rows, tiles) and 64 matrix cycles for every
// fp32 product.
#pragma once

#include "segment_attention.h"

namespace dgmc {
namespace segattn {

// Waves per SIMD the registers are cut to.
template <typename P>
constexpr int fwd_waves(int DP) {
  return P::kPlanes > 1 ? 2 : sizeof(typename P::S) == 2 ? DP <= 64 ? 4 : 2 : 1;
}

template <typename P, int DP, int NW, int KT, int POS, bool FINE>
__global__ __launch_bounds__(NW * 64, fwd_waves<P>(DP)) void fwd_kernel(
    const Args a) {
  using T = typename P::T;
  using S = typename P::S;
  constexpr int CH = DP * (int)sizeof(S) / 16;   // 16-byte chunks per row
  constexpr int NT = NW * 64;
  constexpr int TB = P::kPlanes * KT * CH * 16;  // bytes of one tile
  constexpr int UB = 32 * CH * 16;               // bytes of 32 rows
  // Long fp32 rows with a table: 32 keys are summed from 0 and then added.
  // The output's error is the backward's delta's, which misses the sum of a
  // row's p dp by as much, and the table's gradient adds up what all rows
  // miss (1079 x 726 rows, 3 buckets: 2e-6 of it, so 6e-7).
  constexpr bool kBlocked = sizeof(T) == 4 && NW > 1 && POS > 0;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  DGMC_LDS char* lds = (DGMC_LDS char*)smem;
  const int NB = stage_bufs<P, NW>(a);
  DGMC_LDS float* kpos = (DGMC_LDS float*)(lds + 2 * NB * TB);  // [NB][2][KT]
  DGMC_LDS float* tab = kpos + (POS ? 2 * NB * KT : 0);          // [G][kTab]

  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int h = lane >> 5, c = lane & 31;
  const int kvh = blockIdx.x % a.KV, split = blockIdx.y;
  const int QW = 32 / a.G, TQ = QW * NW;
  const int q_lo = blockIdx.x / a.KV * TQ, q_hi = min(q_lo + TQ, a.Nq);

  // This lane's packed row.
  const int cq = div_group(a, c), g = c - cq * a.G;
  const int qo = wave * QW + cq, qi = q_lo + qo;
  const bool live = c < QW * a.G && qi < q_hi;
  const int head = kvh * a.G + g;
  u32x4 qf[P::kPlanes][CH / 2];
  load_frags<P>(qf,
                (const S*)a.q + (int64_t)q_lo * a.q_sn +
                    (int64_t)kvh * a.G * a.q_sh,
                a.q_sp, (qo * a.q_sn + g * a.q_sh) * (int64_t)sizeof(S), live,
                a.D);
  const int wrows = min(QW, q_hi - q_lo - wave * QW);
  const Rows w = Rows::find<NW>(a.ptr_q, a.ptr_k, a.B, a.Nq, a.Nk, q_lo, q_hi,
                                qi, wrows > 0 ? (wrows - 1) * a.G : -1);
  // The keys of this split.
  const int ntile = (w.hi - w.lo + KT - 1) / KT;
  const int per = split_tiles(a, ntile);
  if (split > 0 && split * per >= ntile) return;
  put_splits(a, blockIdx.x, split, ntile, per);
  const int k_lo = w.lo + split * per * KT;
  const int k_hi = min(k_lo + per * KT, w.hi);

  float px = 0.f, py = 0.f;
  const Bucket bk(a);
  if constexpr (POS > 0) {
    load_table(a, kvh, tab, POS);
    if (live) {
      px = load_pos(a.pos_q, qi, POS, 0);
      if (POS == 2) py = load_pos(a.pos_q, qi, POS, 1);
    }
  }
  const DGMC_LDS float* mytab = tab + g * kTab;
  const int W = 2 * a.half + 2;

  const S* kbase = (const S*)a.k + (int64_t)kvh * a.k_sh;
  const S* vbase = (const S*)a.v + (int64_t)kvh * a.v_sh;
  int pr[2] = {0, 0};
  // Start the loads of keys [k0, e) into buffer `buf`; their positions wait
  // in registers.
  auto fetch = [&](int k0, int e, int buf) {
    using St = Stager<P, KT, CH, NT>;
    const int left = e - k0;
    DGMC_LDS char* kt = lds + buf * 2 * TB;
    const auto ok = [&](int r) { return r < left; };
    St::fill(kbase + (int64_t)k0 * a.k_sn, a.k_sp, a.D, kt, ok,
             [&](int r) { return r * (a.k_sn * (int)sizeof(S)); });
    St::fill(vbase + (int64_t)k0 * a.v_sn, a.v_sp, a.D, kt + TB, ok,
             [&](int r) { return r * (a.v_sn * (int)sizeof(S)); });
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

  const float s1 = a.cap > 0.f ? a.scale / a.cap : a.scale * kLog2e;
  const float s2 = a.cap * kLog2e;
  const bool plain = plain_scores<POS>(a, s1);
  const float ex = plain ? s1 : 1.f;
  const int rows0 = row_base<CH>(), cols0 = P::template cols<CH>();

  // Pass b0 - 1: all rows over all keys of the tile; passes b0 .. b1 (only
  // after a non-finite result): segment by segment.
  for (int pass = w.b0 - 1;; ++pass) {
    int p_lo, p_hi;
    w.pass_range(a.ptr_k, a.B, a.Nk, pass, k_lo, k_hi, p_lo, p_hi);
    f32x16 acc[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) acc[k] = f32x16{};
    float m = -INFINITY, l = 0.f;
    if (pass >= w.b0) stage_barrier();
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
      f32x16 z[KT / 32];
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
        z[u] = row_dot<P, CH, KT, true>(lds + u * UB, rows, qf);
      if (!plain) {
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) z[u][r] = mul_(z[u][r], s1);
        if (a.cap > 0.f) {
#pragma unroll
          for (int u = 0; u < KT / 32; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              z[u][r] = mul_(s2, tanh_<sizeof(T) == 4>(z[u][r]));
        }
      }
      if constexpr (POS > 0) {
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
          if constexpr (POS == 1 && NW > 1) {
            int s;
            if (one_bucket<true>(bk, kpos + buf * 2 * KT + 32 * u, px, live,
                                 s)) {
              const float t = mytab[s];
#pragma unroll
              for (int r = 0; r < 16; ++r) z[u][r] += t;
              continue;
            }
          }
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
      if (!w.whole(k0, KT, p_hi)) {
        const unsigned n = w.count(p_hi);
        const int j0 = k0 + 4 * h - w.r_lo;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if ((unsigned)(j0 + 32 * u + 8 * (r >> 2) + (r & 3)) >= n)
              z[u][r] = -INFINITY;
      }
      float mt = z[0][0];
#pragma unroll
      for (int u = 0; u < KT / 32; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) mt = fmaxf(mt, z[u][r]);
      mt = mul_(max_half(mt), ex);
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
      float e = ex;
      if (plain && __any(fabsf(ms) > kFar)) {
        e = 1.f;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u)
#pragma unroll
          for (int r = 0; r < 16; ++r) z[u][r] = mul_(z[u][r], s1);
      }
#pragma unroll
      for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          z[u][r] = exp2_(fmaf(z[u][r], e, -ms));
        l = P::template sum<FINE>(z[u], l);
        if constexpr (kBlocked) {
          f32x16 blk[DP / 32];
#pragma unroll
          for (int k = 0; k < DP / 32; ++k) blk[k] = f32x16{};
          P::template accum<DP, KT, FINE>(blk, lds + TB + u * UB, cols, z[u]);
#pragma unroll
          for (int k = 0; k < DP / 32; ++k)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[k][r] += blk[k][r];
        } else {
          P::template accum<DP, KT, FINE>(acc, lds + TB + u * UB, cols, z[u]);
        }
      }
    }
    l = sum_half(l);
    const bool redo = pass < w.b0 && w.b1 > w.b0 &&
                      any_lane<NW>(live && not_finite(acc));
    const int64_t row = (int64_t)qi * a.H + head;
    if (!redo && live && (pass < w.b0 || w.seg == pass)) {
      if (per < ntile) {        // joined by join_kernel
        const int64_t prow = (int64_t)split * a.Nq * a.H + row;
        if (h == 0) {
          a.part_ml[prow * 2] = m;
          a.part_ml[prow * 2 + 1] = l;
        }
        put_acc<DP>(a.part_o + prow * a.D, acc, a.D, 1.f);
      } else {
        // l is 0 only without a key of finite score: such a row is 0.
        const float inv = row_stat(m, l).y;
        if (h == 0 && a.stat) a.stat[row] = row_stat(m, l);
        T* orow = (T*)a.out + row * a.D;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const int d = 32 * k + 8 * r4 + 4 * h;
            T o[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = (T)(acc[k][4 * r4 + r] * inv);
            put4(orow, d, a.D, o);
            if (FINE && a.out_lo) {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                o[r] = (T)(acc[k][4 * r4 + r] * inv - (float)o[r]);
              put4((T*)a.out_lo + row * a.D, d, a.D, o);
            }
          }
      }
    }
    if (pass < w.b0 ? !redo : pass == w.b1) return;
  }
}

template <typename P, int DP, int NW, bool FINE>
void launch_fwd(const Args& a, int axes, hipStream_t st) {
  constexpr int B = P::kPlanes * (int)sizeof(typename P::S);
  constexpr int KT = fwd_keys(DP, NW, B);
  const int TQ = 32 / a.G * NW;
  const dim3 grid((a.Nq + TQ - 1) / TQ * a.KV, a.splits), blk(NW * 64);
  const int NB = NW == 1 ? a.bufs : 2;
  const size_t sm =
      NB * (2 * KT * DP * B + (axes ? 8 * KT : 0)) + (axes ? a.G * kTab * 4 : 0);
  auto kern = axes == 0   ? fwd_kernel<P, DP, NW, KT, 0, FINE>
              : axes == 1 ? fwd_kernel<P, DP, NW, KT, 1, FINE>
                          : fwd_kernel<P, DP, NW, KT, 2, FINE>;
  allow_lds(reinterpret_cast<const void*>(kern), sm);
  kern<<<grid, blk, sm, st>>>(a);
  DGMC_CHECK_LAUNCH();
}

}  // namespace segattn
}  // namespace dgmc
