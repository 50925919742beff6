// Attention inside the segments (graphs) of a packed node batch, gfx950:
// shared pieces of the forward and backward kernels.
//
//   z_ij = cap tanh(scale <q_i, k_j> / cap) + T[h, bucket(pos_j - pos_i)]
//   p_i  = softmax_j z_ij over the keys j of row i's segment,  o_i = p_i v
//
// (cap and the bias table T are optional; a row without keys, or whose
// scores are all -inf, gives 0).  Heads h share key head h / G.
//
// Packed rows.  The G query heads of one key head are rows of the same
// tile: row c of a wave's 32 is query c / G, head c % G (c < RW = G floor(32
// / G)), so every K / V tile staged in LDS serves all of them, a single new
// query fills G rows, and dK / dV sum over the group inside one workgroup.
//
// Tiles are consecutive packed rows, whatever segments they belong to: a
// tile visits the keys from its first row's segment to its last row's, and
// where it spans several segments each lane masks by its own row's key range
// (a wave skips key tiles outside all of its rows).  Small graphs so share a
// tile (9-node graphs: 3 to 4 a wave) and the grid depends on N only - no
// plan, no host copy of ptr, and a captured graph may change ptr between
// replays.  A masked pair's weight is 0, but 0 times a NaN or inf of another
// segment is NaN in a product that sums over the tile: a tile of several
// segments that ends with a non-finite result is done again segment by
// segment, each on its own rows alone, so segments never touch each other.
// Rows find their segments on the device: a 64-way wave search for
// the tile's first row (two dependent loads for B <= 4096), then the next 64
// boundaries, one a lane, searched in registers.
//
// Matrix products.  32 x 32 accumulators: lane l holds column l & 31 and
// rows 8 (r / 4) + 4 (l >> 5) + r % 4.  Scores are formed TRANSPOSED to the
// axis that is reduced next (the forward keeps one query per lane, so a
// row's maximum and sum are in-lane plus one exchange), and the
// accumulator's rows then serve directly as the K index of the second
// product: its other operand is read from LDS in that same row order
// (bf16: ds_read_b64_tr_b16, 4 rows a time; fp32: one value a lane), no
// lane exchange of P.  bf16 runs on v_mfma_f32_32x32x16_bf16; fp32 either on
// v_mfma_f32_32x32x2_f32 (exact products, fp32 sums) or, where segments are
// long, as "x6": every operand as three bf16 terms (hi + mid + lo = all 24
// bits), the six largest of their nine products on the bf16 instruction -
// 192 matrix cycles in place of 512 for the same 32 x 32 x 16 block, terms
// from 2^-24 on dropped.  The operands' planes are written once by a kernel
// of their own, P and dS are split in registers.
//
// Bucket of an offset d = pos_j - pos_i on one axis: b(|d|) with `steps` =
// 2^m buckets per octave, read off the float 2 (|d| / steps + 1): its
// exponent and top m mantissa bits ARE the bucket number (exact integer
// arithmetic up to 2^23; larger distances fall into the last bucket).  The
// sign selects the upper or lower half.  The table sits in LDS with one
// unused slot between the halves (so the sign is one xor-add).
#pragma once

#include "common.h"

namespace dgmc {
namespace segattn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef short i16x8 __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSlots = 64;            // slots of one head's bias table
constexpr int kTab = kSlots + 1;      // its LDS row: one slot, many banks
// Finite biases below this count as it: times log2(e) they stay finite, so
// a row masked everywhere by a type's lowest value is uniform, not empty.
constexpr float kLowest = -1e38f;

struct Args {
  const void *q, *k, *v, *o, *dout;
  void *out, *out_lo, *dq, *dk, *dv;  // out_lo: bf16 rest of out (training)
  // Softmax statistics [Nq, H]: (maximum, 1 / sum) of 2^(z log2(e) - maximum).
  // Apart: in one log-sum-exp a maximum of -1e9 would swallow the sum's log.
  float2* stat;
  float* delta;                       // [Nq, H]
  // Splits: [S][Nq, H, D] (dk, dv: [2][S][Nk, KV, D]), [S][Nq, H, 2] and
  // the number of every [tile, KV]'s.
  float *part_o, *part_ml;
  int* part_n;
  float *part_bias;                   // [blocks][KV][G][kSlots]
  const int *ptr_q, *ptr_k;
  const float* bias;                  // [H, nb]
  const int *pos_q, *pos_k;           // [N, axes]
  int64_t q_sn, q_sh, k_sn, k_sh, v_sn, v_sh, g_sn, g_sh;
  int64_t q_sp, k_sp, v_sp, g_sp;     // between the planes (x6)
  int B, Nq, Nk, H, KV, G, gmul, D, nb, half, mbits, slots;
  float scale, cap, dmax, dmul;
  int vec_o;                          // o has 16-byte rows
  int splits, chunk;                  // most splits, least tiles of one
  int bufs;                           // see stage_bufs
};

// Tiles of one split of an axis of n tiles: an even share of the splits, at
// least `chunk` (a join costs more than a short split gains).
__device__ __forceinline__ int split_tiles(const Args& a, int n) {
  return max(a.chunk, (n + a.splits - 1) / a.splits);
}

// Leaves the number of splits of `n` tiles, `per` each, to the join.
__device__ __forceinline__ void put_splits(const Args& a, int where, int split,
                                           int n, int per) {
  if (a.splits > 1 && split == 0 && threadIdx.x == 0)
    a.part_n[where] = (n + per - 1) / per;
}

// First row of segment `b` (clamped to [0, N]; the first segment starts at
// row 0, "segment" B is the tail behind the last one).
__device__ __forceinline__ int seg_begin(const int* ptr, int b, int N) {
  return b == 0 ? 0 : min(max(ptr[b], 0), N);
}

// Segment of a (wave-uniform) row: the last b in [0, B] that begins at or
// before it.
__device__ __forceinline__ int segment_of(const int* ptr, int B, int N,
                                          int row) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B + 1;
  while (n > 1) {
    const int step = (n + 63) >> 6;
    bool ok = lane * step < n;
    if (ok) ok = seg_begin(ptr, lo + lane * step, N) <= row;
    const int adv = (max(__popcll(__ballot(ok)), 1) - 1) * step;
    lo += adv;
    n = min(step, n - adv);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Segment of every lane's own `row`, at or behind a row of segment b0.
__device__ __forceinline__ int lane_segment(const int* ptr, int B, int N,
                                            int b0, int row) {
  const int lane = threadIdx.x & 63;
  int seg = b0;
  for (int base = b0 + 1;; base += 64) {
    const int e = base + lane <= B ? seg_begin(ptr, base + lane, N)
                                   : 0x7fffffff;
    int n = 0;                    // boundaries at or before the row
#pragma unroll
    for (int s = 32; s > 0; s >>= 1)
      if (__shfl(e, n + s - 1) <= row) n += s;
    // (readlane: a shuffle in this condition needs lane 63 to be in it)
    if (n == 63 && __builtin_amdgcn_readlane(e, 63) <= row) n = 64;
    seg += n;
    if (!__any(n == 64)) return seg;
  }
}

// Rows [lo, hi) of segment `seg` on the other side (none of the tail's).
__device__ __forceinline__ void seg_range(const int* ptr, int seg, int B,
                                          int N, int& lo, int& hi) {
  const int b = min(seg, B);
  lo = b == 0 && B == 0 ? N : seg_begin(ptr, b, N);
  hi = b < B ? min(max(ptr[b + 1], lo), N) : lo;
}

// What a wave knows of its tile's own rows [t_lo, t_hi) and the other side's:
// the segments [b0, b1] and other rows [lo, hi) of the whole tile, the lane's
// own segment and range [r_lo, r_hi), and the ranges of the wave's first and
// last row (ranges ascend with the rows, so these bound all of them).
struct Rows {
  int b0, b1, lo, hi;
  int seg, r_lo, r_hi, f_lo, f_hi, l_lo, l_hi;

  // `row`: the lane's row (clamped into the tile); `last`: the lane of the
  // wave's last row, -1 for a wave without rows.
  template <int NW>
  __device__ __forceinline__ static Rows find(const int* own, const int* other,
                                              int B, int N, int No, int t_lo,
                                              int t_hi, int row, int last) {
    Rows w;
    w.b0 = segment_of(own, B, N, t_lo);
    w.seg = lane_segment(own, B, N, w.b0, min(row, t_hi - 1));
    const int l = max(last, 0);
    w.b1 = NW == 1 ? __builtin_amdgcn_readlane(w.seg, l)
                   : __builtin_amdgcn_readfirstlane(
                         lane_segment(own, B, N, w.b0, t_hi - 1));
    int x = 0, y = 0, z = 0;
    if (NW > 1) {
      seg_range(other, w.b0, B, No, x, z);
      seg_range(other, w.b1, B, No, z, y);
    }
    seg_range(other, w.seg, B, No, w.r_lo, w.r_hi);
    w.f_lo = __builtin_amdgcn_readlane(w.r_lo, 0);
    w.f_hi = __builtin_amdgcn_readlane(w.r_hi, 0);
    w.l_lo = __builtin_amdgcn_readlane(w.r_lo, l);
    w.l_hi = __builtin_amdgcn_readlane(w.r_hi, l);
    w.lo = NW == 1 ? w.f_lo : __builtin_amdgcn_readfirstlane(x);
    w.hi = max(NW == 1 ? w.l_hi : __builtin_amdgcn_readfirstlane(y), w.lo);
    if (last < 0) w.seg = -1, w.f_lo = w.l_hi = 0;   // (skips every tile)
    return w;
  }
  // No row of the wave reaches other rows [x, x + n).
  __device__ __forceinline__ bool skip(int x, int n) const {
    return x >= l_hi || x + n <= f_lo;
  }
  // Every row of the wave takes all of them, and all are staged: a pass ends
  // at `end`, inside a tile where a segment of its own starts inside one.
  __device__ __forceinline__ bool whole(int x, int n, int end) const {
    return x >= l_lo && x + n <= min(f_hi, end);
  }
  // Other rows of the lane's own that are staged: [r_lo, min(r_hi, end)).
  __device__ __forceinline__ unsigned count(int end) const {
    return max(min(r_hi, end) - r_lo, 0);
  }
  // Pass `pass` of a tile cut to [s_lo, s_hi): all of it (pass < b0) or the
  // segment's own part.
  __device__ __forceinline__ void pass_range(const int* other, int B, int No,
                                             int pass, int s_lo, int s_hi,
                                             int& p_lo, int& p_hi) const {
    p_lo = s_lo;
    p_hi = s_hi;
    if (pass < b0) return;
    seg_range(other, pass, B, No, p_lo, p_hi);
    p_lo = max(p_lo, s_lo);
    p_hi = min(p_hi, s_hi);
  }
};

// Whether an accumulator of this lane is not finite.
template <int M>
__device__ __forceinline__ bool not_finite(const f32x16 (&acc)[M]) {
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < M; ++k)
#pragma unroll
    for (int r = 0; r < 16; ++r) s = fmaf(acc[k][r], 0.f, s);
  return s != 0.f;
}

// Workgroup-wide any().
template <int NW>
__device__ __forceinline__ bool any_lane(bool v) {
  if constexpr (NW == 1) return __any(v);
  else return __syncthreads_or(v);
}

// A value the compiler cannot see through: what is computed from it inside a
// loop stays there and holds no register across it.
__device__ __forceinline__ int opaque(int v) {
  asm volatile("" : "+v"(v));
  return v;
}
// A lane's LDS address in this buffer: one register and an xor a read where
// rows are long (registers are short there), all of them kept otherwise.
template <int CH>
__device__ __forceinline__ int lane_base(int v) {
  return CH > 8 ? opaque(v) : v;
}

// 16-byte chunk swizzle of an LDS tile row with CH chunks: both 16-byte
// column reads over 16 rows and transposing reads of 4 rows spread over all
// banks.  Linear over xor of row numbers without common bits, so a lane's
// address is its own base xor a constant, plus a constant.
template <int CH>
__host__ __device__ constexpr int swz(int row) {
  if constexpr (CH >= 16) return ((row & 3) << 2) | ((row >> 2) & 3);
  else if constexpr (CH == 8)
    return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
  else return (row >> 2) & 3;
}

template <int CH>
__host__ __device__ constexpr int swz_xor(int row, int chunk) {
  return (swz<CH>(row) ^ chunk) * 16;
}

// x / G and x % G for x < 32 (gmul = ceil(1024 / G): the excess stays under
// 1 / 32, below the next multiple).
__device__ __forceinline__ int div_group(const Args& a, int x) {
  return (x * a.gmul) >> 10;
}

// v of lanes l and l ^ 32 (one VALU swap of the halves; the two results as
// scalars before the casts: a bit cast of a vector's element took element 0).
__device__ __forceinline__ void halves(float v, float& a, float& b) {
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const unsigned x = r[0], y = r[1];
  a = __builtin_bit_cast(float, x);
  b = __builtin_bit_cast(float, y);
}
__device__ __forceinline__ float max_half(float v) {
  float a, b;
  halves(v, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float sum_half(float v) {
  float a, b;
  halves(v, a, b);
  return a + b;
}
__device__ __forceinline__ float exp2_(float x) {
  return __builtin_amdgcn_exp2f(x);
}
// A product that is rounded before what is added to it.
__device__ __forceinline__ float mul_(float x, float y) {
#pragma clang fp contract(off)
  return x * y;
}

// Weights are 2^(z ex - m), one fma: of plain scores (no cap, no table) z is
// the product alone and ex its scale.  Where a maximum is past kFar, that
// product's own rounding, which m has and the fma has not, would be an
// exponent of its own (a score of 2^31: up to 128, the weight inf): such
// scores are scaled and rounded first.  Forward and backward round alike, so
// that no weight of a row passes the forward's largest.
constexpr float kFar = 16777216.f;
template <int POS>
__device__ __forceinline__ bool plain_scores(const Args& a, float s1) {
  return POS == 0 && a.cap <= 0.f && s1 > 0.f;
}

// A row's statistics; without a key of finite score p is 0 everywhere.
__device__ __forceinline__ float2 row_stat(float m, float l) {
  return l == 0.f ? make_float2(INFINITY, 0.f) : make_float2(m, 1.f / l);
}

// One 16-byte chunk of a row of D elements (zeros outside).
template <typename T>
__device__ __forceinline__ u32x4 load_chunk(const T* row, int ch, int D,
                                            bool valid, int vec) {
  constexpr int E = 16 / sizeof(T);
  u32x4 r = {0u, 0u, 0u, 0u};
  const int d0 = ch * E;
  if (!valid || d0 >= D) return r;
  if (vec) return *reinterpret_cast<const u32x4*>(row + d0);
  T tmp[E];
#pragma unroll
  for (int e = 0; e < E; ++e) tmp[e] = d0 + e < D ? row[d0 + e] : T(0.f);
  __builtin_memcpy(&r, tmp, 16);
  return r;
}

// --------------------------------------------------------------------------
// Staging.  A tile is ROWS x CH 16-byte chunks, chunk ch of row r at slot
// (r, ch ^ swz(r)).  Rows are 16-byte chunks (the entry points pack other
// layouts first) and go straight from global memory to LDS
// (buffer_load_dwordx4 ... lds: no register in between, the loads of the
// next tile stay in flight over the current one's products); a lane fills
// slot (r, s) with chunk s ^ swz(r) and lanes without a row (or past the
// width) carry an offset beyond the buffer's range, which reads zeros.
// --------------------------------------------------------------------------
constexpr unsigned kNoRow = 0x80000000u;   // past every buffer's range

template <typename P, int ROWS, int CH, int NT>
struct Stager {
  using S = typename P::S;
  static constexpr int E = 16 / (int)sizeof(S);
  static constexpr int N = (ROWS * CH + NT - 1) / NT;
  static constexpr bool kFull = N * NT == ROWS * CH;

  // `ok(row)`: the row is there, at `off(row)` bytes from `base` (below
  // 2^31); planes `sp` elements apart.
  template <typename Ok, typename Off>
  __device__ __forceinline__ static void fill(const S* base, int64_t sp,
                                              int D, DGMC_LDS char* tile,
                                              Ok ok, Off off) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // (a wave's many slots are computed anew every tile, a few are kept)
    const int tid = N > 2 ? opaque(threadIdx.x) : threadIdx.x;
#pragma unroll
    for (int p = 0; p < P::kPlanes; ++p) {
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<S*>(base + p * sp), 0, 0x80000000u, 0x00020000);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (!kFull && i * NT + wave * 64 >= ROWS * CH) continue;
        const int r = (tid + i * NT) / CH;
        const int ch = ((tid + i * NT) % CH) ^ swz<CH>(r);
        const unsigned o =
            ok(r) && ch * E < D ? (unsigned)off(r) + ch * 16 : kNoRow;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs,
            (DGMC_LDS void*)(tile +
                             (p * ROWS * CH + i * NT + wave * 64) * 16),
            16, o, 0, 0, 0);
      }
    }
  }
};

// The 16-byte chunks h, h + 2, .. of this lane's own row: at `off` bytes from
// the wave-uniform `base`, zeros where it is not `live`.  All loads are
// issued before the first is needed (no branch around them).
template <typename T, int N>
__device__ __forceinline__ void load_row(u32x4 (&f)[N], const T* base,
                                         int64_t off, bool live, int D,
                                         int vec) {
  constexpr int E = 16 / (int)sizeof(T);
  const int h = (threadIdx.x >> 5) & 1;
  if (vec) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<T*>(base), 0, 0x80000000u, 0x00020000);
#pragma unroll
    for (int s = 0; s < N; ++s) {
      const int ch = 2 * s + h;
      f[s] = __builtin_amdgcn_raw_buffer_load_b128(
          rs, live && ch * E < D ? (unsigned)off + ch * 16 : kNoRow, 0, 0);
    }
  } else {
#pragma unroll
    for (int s = 0; s < N; ++s)
      f[s] = load_chunk<T>((const T*)((const char*)base + off), 2 * s + h, D,
                           live, 0);
  }
}

// Of an fp32 row, the elements that load_row takes of a bf16 one: chunks 4 s
// + 2 h and the next.
template <int N>
__device__ __forceinline__ void load_row8(u32x4 (&f)[N], const float* base,
                                          int64_t off, bool live, int D,
                                          int vec) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int s = 0; s < N; ++s)
    f[s] = load_chunk<float>((const float*)((const char*)base + off),
                             4 * (s >> 1) + 2 * h + (s & 1), D, live, vec);
}

// An MFMA operand of own rows: load_row of every plane.
template <typename P, int N>
__device__ __forceinline__ void load_frags(u32x4 (&f)[P::kPlanes][N],
                                           const typename P::S* base,
                                           int64_t sp, int64_t off, bool live,
                                           int D) {
#pragma unroll
  for (int p = 0; p < P::kPlanes; ++p)
    load_row(f[p], base + p * sp, off, live, D, 1);
}

// Every wave's staged data (and LDS reads) done, then the barrier.  (The
// wait as a builtin: the compiler so knows that nothing is in flight behind
// it, and does not wait for older loads with the next tile's among them.)
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);      // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// load(t) and use(t) for t = 0 .. N - 1, every load kAhead steps ahead of its
// use and no further: where registers are short the compiler otherwise loads
// and waits one step at a time.
constexpr int kAhead = 2;
template <int N, typename L, typename U>
__device__ __forceinline__ void stepped(L load, U use) {
#pragma unroll
  for (int t = 0; t < kAhead; ++t) load(t);
#pragma unroll
  for (int t = 0; t < N; ++t) {
    if (t + kAhead < N) load(t + kAhead);
    __builtin_amdgcn_sched_barrier(0);
    use(t);
  }
}

// --------------------------------------------------------------------------
// Matrix core policies.  `rows` and `cols` are a lane's byte offsets into a
// staged tile for the two ways it is read: row operand (16-byte chunks of
// row c) and transposed operand of accum().
// --------------------------------------------------------------------------
// bf16 tensors: one plane.
struct Bf16 {
  using T = __bf16;                 // of the tensors
  using S = __bf16;                 // staged
  static constexpr int kPlanes = 1;
  template <int CH> __device__ __forceinline__ static int cols() {
    const int lane = threadIdx.x & 63;
    const int row = 4 * (lane >> 5) + ((lane >> 2) & 3);
    const int ch = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    return row * CH * 16 + ((ch ^ swz<CH>(row)) * 16) + 8 * (lane & 1);
  }
  // acc += A B for one pair of 16-byte chunks (K = 16).
  __device__ __forceinline__ static f32x16 dot(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(
        __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
        0);
  }
  // Transposed operand: columns of block k, rows of K half c.
  template <int CH>
  __device__ __forceinline__ static bf16x8 col_frag(const DGMC_LDS char* tile,
                                                    int cols, int c, int k) {
    i16x4 v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = 16 * c + 8 * i;
      v[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (DGMC_LDS i16x4*)(tile + (cols ^ swz_xor<CH>(row, 4 * k)) +
                            row * CH * 16));
    }
    const i16x8 both = __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5,
                                               6, 7);
    return __builtin_bit_cast(bf16x8, both);
  }
  // acc[blk] += tile^T p: 32 rows of the tile (planes of ROWS rows) are the K
  // index, in the accumulator's row order.  FINE: p as the sum of two bf16
  // terms.
  template <int DP, int ROWS, bool FINE = false>
  __device__ __forceinline__ static void accum(f32x16 (&acc)[DP / 32],
                                               const DGMC_LDS char* tile,
                                               int cols, f32x16 p) {
    constexpr int CH = DP / 8;
    if constexpr (CH >= 16) {
      bf16x8 a[2 * (DP / 32)], b[2], lo_b[2];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        b[i >> 3][i & 7] = (__bf16)p[i];
        if (FINE)
          lo_b[i >> 3][i & 7] = (__bf16)(p[i] - (float)b[i >> 3][i & 7]);
      }
      stepped<2 * (DP / 32)>(
          [&](int t) {
            a[t] = col_frag<CH>(tile, cols, t / (DP / 32), t % (DP / 32));
          },
          [&](int t) {
            const int c = t / (DP / 32), k = t % (DP / 32);
            acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[t], b[c],
                                                             acc[k], 0, 0, 0);
            if constexpr (FINE)
              acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  a[t], lo_b[c], acc[k], 0, 0, 0);
          });
      return;
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8 b, lo_b;
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = (__bf16)p[8 * c + i];
      if constexpr (FINE) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          lo_b[i] = (__bf16)(p[8 * c + i] - (float)b[i]);
      }
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        const bf16x8 a = col_frag<CH>(tile, cols, c, k);
        acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc[k], 0, 0,
                                                         0);
        if constexpr (FINE)
          acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, lo_b, acc[k], 0,
                                                           0, 0);
      }
    }
  }
  // l + the sum of p as the product takes it: rounded, two a v_dot2 (FINE:
  // the fp32 values).
  template <bool FINE>
  __device__ __forceinline__ static float sum(f32x16 p, float l) {
    float s[2] = {l, 0.f};
    if constexpr (FINE) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r & 1] += p[r];
    } else {
      const bf16x2 one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const bf16x2 v = {(__bf16)p[r], (__bf16)p[r + 1]};
        s[(r >> 1) & 1] = __builtin_amdgcn_fdot2_f32_bf16(v, one,
                                                          s[(r >> 1) & 1],
                                                          false);
      }
    }
    return s[0] + s[1];
  }
  __device__ __forceinline__ static float chunk_dot(u32x4 a, u32x4 b) {
    const bf16x8 x = __builtin_bit_cast(bf16x8, a),
                 y = __builtin_bit_cast(bf16x8, b);
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += (float)x[i] * (float)y[i];
    return s;
  }
};

// fp32 tensors, exact products.
struct F32 {
  using T = float;
  using S = float;
  static constexpr int kPlanes = 1;
  template <int CH> __device__ __forceinline__ static int cols() {
    const int lane = threadIdx.x & 63, row = 4 * (lane >> 5), d = lane & 31;
    return row * CH * 16 + (((d >> 2) ^ swz<CH>(row)) * 16) + 4 * (d & 3);
  }
  __device__ __forceinline__ static f32x16 dot(u32x4 a, u32x4 b, f32x16 c) {
    const f32x4 x = __builtin_bit_cast(f32x4, a),
                y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    return c;
  }
  template <int DP, int ROWS, bool FINE = false>
  __device__ __forceinline__ static void accum(f32x16 (&acc)[DP / 32],
                                               const DGMC_LDS char* tile,
                                               int cols, f32x16 p) {
    constexpr int CH = DP / 4;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = 8 * (r >> 2) + (r & 3);
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        const float a = *(const DGMC_LDS float*)(
            tile + (cols ^ swz_xor<CH>(row, 8 * k)) + row * CH * 16);
        acc[k] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, p[r], acc[k], 0, 0,
                                                      0);
      }
    }
  }
  template <bool FINE>
  __device__ __forceinline__ static float sum(f32x16 p, float l) {
    float s[4] = {l, 0.f, 0.f, 0.f};
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r & 3] += p[r];
    return (s[0] + s[1]) + (s[2] + s[3]);
  }
  __device__ __forceinline__ static float chunk_dot(u32x4 a, u32x4 b) {
    const f32x4 x = __builtin_bit_cast(f32x4, a),
                y = __builtin_bit_cast(f32x4, b);
    return (x[0] * y[0] + x[1] * y[1]) + (x[2] * y[2] + x[3] * y[3]);
  }
};

// Terms of an x6 product, the smallest first: lo hi, hi lo, mid mid, mid hi,
// hi mid, hi hi.
__host__ __device__ constexpr int x6_a(int t) {
  return t == 0 ? 2 : t == 2 || t == 3 ? 1 : 0;
}
__host__ __device__ constexpr int x6_b(int t) {
  return t == 1 ? 2 : t == 2 || t == 4 ? 1 : 0;
}

// fp32 tensors in three bf16 planes.
struct X6 {
  using T = float;
  using S = __bf16;
  static constexpr int kPlanes = 3;
  template <int CH> __device__ __forceinline__ static int cols() {
    return Bf16::cols<CH>();
  }
  template <int DP, int ROWS, bool FINE = false>
  __device__ __forceinline__ static void accum(f32x16 (&acc)[DP / 32],
                                               const DGMC_LDS char* tile,
                                               int cols, f32x16 p) {
    constexpr int CH = DP / 8;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      bf16x8 b[3];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = p[8 * c + i];
        b[0][i] = (__bf16)x;
        const float r = x - (float)b[0][i];
        b[1][i] = (__bf16)r;
        b[2][i] = (__bf16)(r - (float)b[1][i]);
      }
#pragma unroll
      for (int k = 0; k < DP / 32; ++k) {
        bf16x8 a[3];
#pragma unroll
        for (int q = 0; q < 3; ++q)
          a[q] = Bf16::col_frag<CH>(tile + q * ROWS * CH * 16, cols, c, k);
#pragma unroll
        for (int t = 0; t < 6; ++t)
          acc[k] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              a[x6_a(t)], b[x6_b(t)], acc[k], 0, 0, 0);
      }
    }
  }
  template <bool FINE>
  __device__ __forceinline__ static float sum(f32x16 p, float l) {
    return F32::sum<FINE>(p, l);
  }
};

// Row operand: chunks h, h + 2, .. of row c of a staged block of 32 rows.
// KEYS: the staged rows are the keys (x6 adds its terms in one order of query
// and key, so that a score has the same bits in every kernel).
template <int CH>
__device__ __forceinline__ int row_base() {
  const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
  return c * CH * 16 + ((h ^ swz<CH>(c)) * 16);
}
template <typename P, int CH, int ROWS, bool KEYS>
__device__ __forceinline__ f32x16 row_dot(
    const DGMC_LDS char* tile, int rows,
    const u32x4 (&f)[P::kPlanes][CH / 2]) {
  f32x16 acc = {};
#pragma unroll
  for (int s = 0; s < CH / 2; ++s) {
    u32x4 a[P::kPlanes];
#pragma unroll
    for (int p = 0; p < P::kPlanes; ++p)
      a[p] = *(const DGMC_LDS u32x4*)(tile + (rows ^ (32 * s)) +
                                      p * ROWS * CH * 16);
    if constexpr (P::kPlanes == 1) {
      acc = P::dot(a[0], f[0][s], acc);
    } else {
#pragma unroll
      for (int t = 0; t < 6; ++t)
        acc = KEYS ? Bf16::dot(a[x6_a(t)], f[x6_b(t)][s], acc)
                   : Bf16::dot(a[x6_b(t)], f[x6_a(t)][s], acc);
    }
  }
  return acc;
}

// Two row products of the backward: z of tile 0 with fz(s), dp of the tile TB
// bytes on with fd(s), the chunks of the lane's own rows.
template <typename P, int CH, int ROWS, typename Z, typename D>
__device__ __forceinline__ void row_dot2(f32x16& z, f32x16& dp,
                                         const DGMC_LDS char* lds, int TB,
                                         int rows, Z fz, D fd) {
  constexpr int N = CH / 2;
  u32x4 a[2 * N], b[2 * N];
  z = dp = f32x16{};
  stepped<2 * N>(
      [&](int t) {
        const int s = t % N;
        a[t] = *(const DGMC_LDS u32x4*)(lds + (t < N ? 0 : TB) +
                                        (rows ^ (32 * s)));
        b[t] = t < N ? fz(s) : fd(s);
      },
      [&](int t) {
        f32x16& acc = t < N ? z : dp;
        acc = P::dot(a[t], b[t], acc);
      });
}

// Four values of an output row of D at d (d % 4 == 0).
template <typename T>
__device__ __forceinline__ void put4(T* row, int d, int D, const T* v) {
  if (D % 4 == 0) {
    if (d < D)
      __builtin_memcpy(__builtin_assume_aligned(row + d, 4 * sizeof(T)), v,
                       4 * sizeof(T));
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (d + r < D) row[d + r] = v[r];
  }
}

// A wave's accumulators -> its lanes' output rows.
template <int DP, typename T>
__device__ __forceinline__ void put_acc(T* row, const f32x16 (&acc)[DP / 32],
                                        int D, float scale) {
  const int h = (threadIdx.x >> 5) & 1;
#pragma unroll
  for (int k = 0; k < DP / 32; ++k)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      T o[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = (T)(acc[k][4 * r4 + r] * scale);
      put4(row, 32 * k + 8 * r4 + 4 * h, D, o);
    }
}

// --------------------------------------------------------------------------
// Scores
// --------------------------------------------------------------------------
// tanh: v_exp / v_rcp (about 1 ulp each) of 1 - 2 / (e^2x + 1), whose
// cancellation leaves an absolute error of 1e-7 near 0, times the cap in a
// score.  bf16 takes that up to a cap of 64, where it is the 2^-17 that
// weights of two terms are rounded to (wider caps are taken in fp32; the
// series in these kernels cost 3 % of every capped call).  fp32 (EXACT) takes
// the odd series up to |x| < 0.25 (to x^9; the next term is 8.5e-9 of x
// there) so small scores keep their relative precision.
template <bool EXACT>
__device__ __forceinline__ float tanh_(float x) {
  const float e = exp2_(x * (2.f * kLog2e));
  const float t = fmaf(-2.f, __builtin_amdgcn_rcpf(e + 1.f), 1.f);
  if constexpr (EXACT) {
    const float y = x * x;
    float s = fmaf(y, 62.f / 2835.f, -17.f / 315.f);
    s = fmaf(y, s, 2.f / 15.f);
    s = fmaf(y, s, -1.f / 3.f);
    const float small = fmaf(x * y, s, x);
    return fabsf(x) < 0.25f ? small : t;
  } else {
    return t;
  }
}

// Bucket slot of offset d (float, exact) on one axis: 0 .. 2 half + 1.
struct Bucket {
  float dmin, dmax, dmul;
  int shift, width, K;
  // (0 - dmax: +0 where there is one bucket, whose offsets so have no sign)
  __device__ __forceinline__ explicit Bucket(const Args& a)
      : dmin(0.f - a.dmax), dmax(a.dmax), dmul(a.dmul), shift(23 - a.mbits),
        width(5 + a.mbits), K(a.half + 1) {}
  __device__ __forceinline__ int slot(float d) const {
    const float c = __builtin_amdgcn_fmed3f(d, dmin, dmax);
    const float x = fmaf(fabsf(c), dmul, 2.f);
    const int t = __builtin_amdgcn_ubfe(__builtin_bit_cast(unsigned, x),
                                        shift, width);
    const int s = __builtin_bit_cast(int, c) >> 31;
    return (t ^ s) + K;
  }
};

// Positions as floats, clamped to +-2^23 (their differences are exact).
// (What is fetched for the next tile is converted when it is put there: a
// conversion right behind its load would wait for the whole tile.)
__device__ __forceinline__ float to_pos(int p) {
  return (float)min(max(p, -(1 << 23)), 1 << 23);
}
__device__ __forceinline__ float load_pos(const int* pos, int64_t i, int axes,
                                          int axis) {
  return to_pos(pos[i * axes + axis]);
}

// LDS buffers of the staged tiles: two, or (a.bufs) one where a wave walks
// the few fp32 tiles of short segments alone - what it then waits for them is
// less than what the waves gain that fit beside it (1024 graphs of 3 to 19
// nodes, heads of 64: forward 37 -> 26 us, dkv 46 -> 39; heads of 128: dq 190
// -> 81).  Few rows of long segments stream through two.
template <typename P, int NW>
__device__ __forceinline__ int stage_bufs(const Args& a) {
  return NW == 1 && sizeof(typename P::S) == 4 ? a.bufs : 2;
}

// Keys of a forward tile: 64 where four waves share it and both buffers of K
// and V stay within 64 KB of LDS.
constexpr int fwd_keys(int DP, int nw, int row_bytes) {
  return nw > 1 && DP * row_bytes <= 256 ? 64 : 32;
}

// Dynamic LDS past 64 KB has to be asked for.
inline void allow_lds(const void* kernel, size_t bytes) {
  TORCH_CHECK(bytes <= 160 * 1024, "segment_attention: ", bytes,
              " bytes of LDS");
  if (bytes > 64 * 1024)
    DGMC_CHECK_HIP(hipFuncSetAttribute(
        kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
}

// The group's bias tables -> LDS slots, times log2(e).
__device__ __forceinline__ void load_table(const Args& a, int kvh,
                                           DGMC_LDS float* tab, int axes) {
  const int W = 2 * a.half + 2, w = 2 * a.half + 1;
  for (int e = threadIdx.x; e < a.G * kSlots; e += blockDim.x) {
    const int g = e / kSlots, s = e % kSlots;
    int c = -1;
    if (axes == 1) {
      if (s < W && s != a.half) c = s < a.half ? s : s - 1;
    } else if (s < W * W) {
      const int x = s / W, y = s % W;
      if (x != a.half && y != a.half)
        c = (x < a.half ? x : x - 1) * w + (y < a.half ? y : y - 1);
    }
    float v = 0.f;
    if (c >= 0) {
      v = a.bias[(int64_t)(kvh * a.G + g) * a.nb + c];
      if (v < kLowest && v > -INFINITY) v = kLowest;
      v *= kLog2e;
    }
    tab[g * kTab + s] = v;
  }
}

// Whether all offsets between this lane's position `p` and the 16 x 2 other
// positions `o` of a 32-row block (this half's at o + 4 h) fall into one
// bucket, in every lane of the wave that `live`s; `s`: the bucket.  Slots
// ascend with the offset, so the least and the greatest position tell (a
// neighbour's rows may be among them: they can only say no).  Blocks of nodes
// in order that lie far apart share a bucket: one look-up and one sum then
// serve 16 pairs of a lane.  KEY: offsets are o - p, else p - o.
template <bool KEY>
__device__ __forceinline__ bool one_bucket(const Bucket& bk,
                                           const DGMC_LDS float* o, float p,
                                           bool live, int& s) {
  const int h = (threadIdx.x >> 5) & 1;
  float mn = INFINITY, mx = -INFINITY;
#pragma unroll
  for (int r4 = 0; r4 < 4; ++r4) {
    const f32x4 x = *(const DGMC_LDS f32x4*)(o + 8 * r4 + 4 * h);
    mn = fminf(fminf(mn, fminf(x[0], x[1])), fminf(x[2], x[3]));
    mx = fmaxf(fmaxf(mx, fmaxf(x[0], x[1])), fmaxf(x[2], x[3]));
  }
  mn = -max_half(-mn);
  mx = max_half(mx);
  s = bk.slot(KEY ? mn - p : p - mn);
  return __all(!live || s == bk.slot(KEY ? mx - p : p - mx));
}

}  // namespace segattn
}  // namespace dgmc
