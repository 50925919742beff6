// Segment attention: entry points, copies of inputs, the join of split keys
// and the sum of the bias table's gradient.  The kernels are in
// segment_attention_{fwd,bwd}.h, instantiated per kernel and type in
// segment_attention_{fwd,dq,dkv}_*.hip.
#include "attentional.h"
#include "segment_attention.h"

namespace dgmc {
namespace segattn {

void fwd_bf16(const Args& a, int axes, int nw, hipStream_t st);
void fwd_bf16_fine(const Args& a, int axes, int nw, hipStream_t st);
void fwd_f32(const Args& a, int axes, int nw, hipStream_t st);
void fwd_x6(const Args& a, int axes, hipStream_t st);
void dq_bf16(const Args& a, int axes, int nw, int nblk, hipStream_t st);
void dq_f32(const Args& a, int axes, int nw, int nblk, hipStream_t st);
void dq_x6(const Args& a, hipStream_t st);
void dkv_bf16(const Args& a, int axes, int nw, hipStream_t st);
void dkv_f32(const Args& a, int axes, int nw, hipStream_t st);
void dkv_x6(const Args& a, int axes, hipStream_t st);

// Copies of strided [N, heads, D] tensors in the form the kernels read: rows
// padded with zeros to DC, a whole number of chunks of E values, one chunk a
// thread.
struct Copies {
  const void* src[4];
  void* dst[4];
  int64_t sn[4], sh[4], n[4];       // strides, chunks (0: none to make)
  int heads[4];
  int D;
};

// This thread's chunk of tensor blockIdx.y; false: there is none.
template <typename T, int E>
__device__ __forceinline__ bool copy_chunk(const Copies& p, int64_t& e,
                                           T (&x)[E]) {
  const int t = blockIdx.y, ce = (p.D + E - 1) / E;
  e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= p.n[t]) return false;
  const int64_t row = e / ce;
  const int d0 = (int)(e - row * ce) * E;
  const int64_t i = row / p.heads[t];
  const int hd = (int)(row - i * p.heads[t]);
  const T* src = (const T*)p.src[t] + i * p.sn[t] + hd * p.sh[t] + d0;
  if (d0 + E <= p.D && aligned16(src)) {
    __builtin_memcpy(x, __builtin_assume_aligned(src, 16), E * sizeof(T));
  } else {
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = d0 + k < p.D ? src[k] : (T)0.f;
  }
  return true;
}

// Rows that are not 16-byte chunks: the same values, padded.
template <typename T>
__global__ __launch_bounds__(256) void pad_kernel(const Copies p) {
  constexpr int E = 16 / sizeof(T);
  int64_t e;
  T x[E];
  if (!copy_chunk(p, e, x)) return;
  T* dst = (T*)p.dst[blockIdx.y] + e * E;
  __builtin_memcpy(__builtin_assume_aligned(dst, 16), x, 16);
}

// fp32 -> bf16 planes [3][N][heads][D8] (hi, mid, lo).
__global__ __launch_bounds__(256) void planes_kernel(const Copies p) {
  const int t = blockIdx.y;
  int64_t e;
  float x[8];
  if (!copy_chunk(p, e, x)) return;
  bf16x8 v[3];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    __bf16 h, m, l;
    split3_bf16(x[k], h, m, l);
    // (the terms of inf and NaN stay in the first: inf - inf is NaN)
    const bool fin = fabsf(x[k]) < INFINITY;
    v[0][k] = h;
    v[1][k] = fin ? m : (__bf16)0.f;
    v[2][k] = fin ? l : (__bf16)0.f;
  }
#pragma unroll
  for (int q = 0; q < 3; ++q)
    *(bf16x8*)((__bf16*)p.dst[t] + (q * p.n[t] + e) * 8) = v[q];
}

constexpr int kMaxSplits = 512;

// Join of the split rows (FWD: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M)
// l_s; DQ, DKV: plain sums), in a fixed order of the splits.  A workgroup
// takes rows of one tile of the kernel whose splits it joins (that kernel
// left the number of the tile's splits); 1 << lt threads a row, 8 values
// each, and `ways` (a power of two) such groups share the splits of a row,
// kJoin of them loaded at a time; their sums are added in order.
enum { FWD, DQ, DKV };
constexpr int kJoin = 4;

template <typename T, int MODE>
__global__ __launch_bounds__(256) void join_kernel(const Args a, int per_tile,
                                                   int ways, int lt) {
  __shared__ float red[256][9];
  __shared__ float2 wml[64];
  const int ns = a.part_n[blockIdx.x];
  if (ns <= 1) return;
  const int kvh = blockIdx.x % a.KV;
  const int N = MODE == DKV ? a.Nk : a.Nq;
  const int lo = blockIdx.x / a.KV * per_tile, hi = min(lo + per_tile, N);
  const int G = MODE == DKV ? 1 : a.G, heads = G * a.KV;
  const int rows = (hi - lo) * G;
  const int64_t all = (int64_t)N * heads;
  const int tid = threadIdx.x, tpr = 1 << lt, d0 = (tid & (tpr - 1)) * 8;
  const int grp = tid >> lt, rpr = (256 >> lt) / ways;
  const int rr = grp / ways, way = grp % ways;
  const bool vec = a.D % 4 == 0 && d0 + 8 <= a.D;
  const float* part =
      a.part_o + (MODE == DKV ? blockIdx.y * a.splits * all * a.D : 0);
  for (int r0 = blockIdx.z * rpr; r0 < rows; r0 += rpr * gridDim.z) {
    const int r = r0 + rr;
    const bool live = r < rows;
    const int64_t row = (int64_t)(lo + r / G) * heads + kvh * G + r % G;
    float M = -INFINITY, L = 0.f, o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) o[k] = 0.f;
    for (int s0 = way; live && s0 < ns; s0 += kJoin * ways) {
      float2 ml[kJoin];
      f32x4 x[kJoin], y[kJoin];
#pragma unroll
      for (int i = 0; i < kJoin; ++i) {
        const int s = s0 + i * ways;
        ml[i] = make_float2(-INFINITY, 0.f);
        x[i] = y[i] = f32x4{};
        if (s >= ns) continue;
        if (MODE == FWD)
          ml[i] = *(const float2*)(a.part_ml + (s * all + row) * 2);
        const float* p = part + (s * all + row) * a.D + d0;
        if (vec) {
          x[i] = *(const f32x4*)p;
          y[i] = *(const f32x4*)(p + 4);
        } else {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (d0 + k < a.D) x[i][k] = p[k];
            if (d0 + 4 + k < a.D) y[i][k] = p[4 + k];
          }
        }
      }
      float wt[kJoin];
      if (MODE == FWD) {
        float m = M;
#pragma unroll
        for (int i = 0; i < kJoin; ++i) m = fmaxf(m, ml[i].x);
        const float ms = m == -INFINITY ? 0.f : m, f = exp2_(M - ms);
        L *= f;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] *= f;
        M = m;
#pragma unroll
        for (int i = 0; i < kJoin; ++i) {
          wt[i] = exp2_(ml[i].x - ms);
          L = fmaf(wt[i], ml[i].y, L);
        }
      }
#pragma unroll
      for (int i = 0; i < kJoin; ++i)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[k] = MODE == FWD ? fmaf(wt[i], x[i][k], o[k]) : o[k] + x[i][k];
          o[4 + k] =
              MODE == FWD ? fmaf(wt[i], y[i][k], o[4 + k]) : o[4 + k] + y[i][k];
        }
    }
    if (ways > 1) {
#pragma unroll
      for (int k = 0; k < 8; ++k) red[tid][k] = o[k];
      if ((tid & (tpr - 1)) == 0) wml[grp] = make_float2(M, L);
      __syncthreads();
      if (way == 0) {
        if (MODE == FWD) {
          for (int w = 1; w < ways; ++w) M = fmaxf(M, wml[grp + w].x);
          const float ms = M == -INFINITY ? 0.f : M;
          L = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k) o[k] = 0.f;
          for (int w = 0; w < ways; ++w) {
            const float2 x = wml[grp + w];
            const float f = exp2_(x.x - ms);
            L = fmaf(f, x.y, L);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              o[k] = fmaf(f, red[tid + tpr * w][k], o[k]);
          }
        } else {
          for (int w = 1; w < ways; ++w)
#pragma unroll
            for (int k = 0; k < 8; ++k) o[k] += red[tid + tpr * w][k];
        }
      }
      __syncthreads();
    }
    if (!live || way != 0) continue;
    const float f = MODE == FWD ? row_stat(M, L).y
                    : MODE == DKV && blockIdx.y == 1 ? 1.f
                                                     : a.scale;
    T* out = (T*)(MODE == FWD  ? a.out
                  : MODE == DQ ? a.dq
                               : (blockIdx.y ? a.dv : a.dk)) +
             row * a.D;
    T v[8], v_lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[k] = (T)(o[k] * f);
      v_lo[k] = (T)(o[k] * f - (float)v[k]);
    }
    put4(out, d0, a.D, v);
    put4(out, d0 + 4, a.D, v + 4);
    if (MODE == FWD && a.out_lo) {
      T* lo_row = (T*)a.out_lo + row * a.D;
      put4(lo_row, d0, a.D, v_lo);
      put4(lo_row, d0 + 4, a.D, v_lo + 4);
    }
    if (MODE == FWD && a.stat && d0 == 0) a.stat[row] = row_stat(M, L);
  }
}

template <int MODE>
static void join(const Args& a, bool f32, int per_tile) {
  const int N = MODE == DKV ? a.Nk : a.Nq;
  const int G = MODE == DKV ? 1 : a.G;
  const int lt = a.D > 64 ? 4 : a.D > 32 ? 3 : 2, groups = 256 >> lt;
  int ways = 1;
  while (ways < groups && kJoin * ways < a.splits) ways *= 2;
  // (workgroups along z share a tile's rows, groups / ways a round)
  const dim3 grid((N + per_tile - 1) / per_tile * a.KV, MODE == DKV ? 2 : 1,
                  std::min((per_tile * G * ways + groups - 1) / groups, 128));
  if (f32)
    join_kernel<float, MODE><<<grid, 256, 0, stream()>>>(a, per_tile, ways,
                                                         lt);
  else
    join_kernel<__bf16, MODE><<<grid, 256, 0, stream()>>>(a, per_tile, ways,
                                                          lt);
  DGMC_CHECK_LAUNCH();
}

// dT[head][c] = sum over the workgroups' parts, in a fixed order: one
// workgroup per head, 16 threads a slot, each of which takes every 16th part
// (eight loads in flight); their sums are added in order.
constexpr int kSumWays = 16;

__global__ __launch_bounds__(kSlots * kSumWays) void bias_sum_kernel(
    const float* __restrict__ part, float* __restrict__ out, int nblk, int KV,
    int G, int slots, int nb, int half, int axes) {
  __shared__ float red[kSumWays][kSlots];
  const int head = blockIdx.x, kvh = head / G, g = head % G;
  const int s = threadIdx.x & 63, p = threadIdx.x >> 6;
  const float* src = part + ((int64_t)kvh * G + g) * slots + min(s, slots - 1);
  const int64_t step = (int64_t)KV * G * slots;
  float sum = 0.f;
#pragma unroll 8
  for (int b = p; b < nblk; b += kSumWays) sum += src[b * step];
  red[p][s] = sum;
  __syncthreads();
  if ((int)threadIdx.x >= nb) return;
  const int c = threadIdx.x, w = 2 * half + 1, W = w + 1;
  const int y = c % w, x = axes == 1 ? 0 : c / w;
  const int ys = y < half ? y : y + 1, xs = x < half ? x : x + 1;
  const int t = axes == 1 ? ys : xs * W + ys;
  sum = 0.f;
  for (int k = 0; k < kSumWays; ++k) sum += red[k][t];
  out[(int64_t)head * nb + c] = sum;
}

constexpr double kMaxCapBf16 = 64.0;      // see tanh_

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
// multiples of 16 bytes, and a tile (128 rows, 32 heads) spans less than the
// 2^31 bytes of a buffer's offsets.
static bool rows16(const at::Tensor& t) {
  const int64_t e = 16 / t.element_size();
  return t.size(2) % e == 0 && t.stride(0) % e == 0 && t.stride(1) % e == 0 &&
         aligned16(t.data_ptr()) &&
         (128 * t.stride(0) + 32 * t.stride(1) + 128) * t.element_size() <
             ((int64_t)1 << 31);
}

static Args make_args(const at::Tensor& q, const at::Tensor& k,
                      const at::Tensor& v, const at::Tensor& ptr_q,
                      const at::Tensor& ptr_k, double scale, double cap,
                      const OptTensor& bias, const OptTensor& pos_q,
                      const OptTensor& pos_k, const BucketLayout& layout,
                      int& axes) {
  const int64_t half = layout.half, mbits = layout.mbits;
  const double dmax = layout.dmax;
  check_heads(q, "q", q);
  check_heads(k, "k", q);
  check_heads(v, "v", q);
  TORCH_CHECK(q.scalar_type() == at::kFloat ||
                  q.scalar_type() == at::kBFloat16,
              "segment_attention: unsupported dtype ", q.scalar_type());
  TORCH_CHECK(q.scalar_type() == at::kFloat || cap <= kMaxCapBf16,
              "segment_attention: caps over ", kMaxCapBf16, " need fp32");
  TORCH_CHECK(k.sizes() == v.sizes(), "segment_attention: k and v differ in "
              "shape");
  TORCH_CHECK(q.size(2) == k.size(2) && q.size(2) >= 1 && q.size(2) <= 128,
              "segment_attention: head dimensions must agree, 1 to 128");
  TORCH_CHECK(k.size(1) >= 1 && q.size(1) >= 1 &&
                  q.size(1) % k.size(1) == 0 && q.size(1) / k.size(1) <= 32,
              "segment_attention: query heads must be a multiple (at most "
              "32) of the key heads");
  // (a tile's rows, also of a copy in eights, lie within 2^31 bytes)
  TORCH_CHECK(q.size(1) * ((q.size(2) + 7) / 8 * 8) <= 1 << 21,
              "segment_attention: rows of more than 2^21 values");
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
  a.gmul = (1024 + a.G - 1) / a.G;
  a.D = (int)q.size(2);
  // 32-bit row numbers and launch sizes (threads of a launch < 2^32).
  const int64_t lim = (int64_t)1 << 31;
  TORCH_CHECK(q.size(0) < lim - 4096 && k.size(0) < lim - 4096 &&
                  q.size(0) * a.H < ((int64_t)1 << 30) &&
                  k.size(0) * a.KV < ((int64_t)1 << 30),
              "segment_attention: too many rows for one call");
  a.Nq = (int)q.size(0); a.Nk = (int)k.size(0);
  a.ptr_q = ptr_q.data_ptr<int>(); a.ptr_k = ptr_k.data_ptr<int>();
  a.scale = (float)scale; a.cap = (float)cap;
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

// See stage_bufs.
static void pick_bufs(Args& a, bool f32) {
  a.bufs = f32 && waves_for((int64_t)a.Nq * a.G, a.B) == 1 &&
                   waves_for(a.Nk, a.B) == 1
               ? 1
               : 2;
}

// Whether an fp32 call takes the x6 kernels: long segments on both sides (the
// planes cost a pass over the tensors and 1.5 times their memory), heads of
// up to 64 (wider ones' planes exceed the LDS beside the table's columns).
static bool takes_x6(const Args& a, bool x6) {
  return x6 && a.D <= 64 && waves_for((int64_t)a.Nq * a.G, a.B) == 4 &&
         waves_for(a.Nk, a.B) == 4;
}

// Points q, k, v (and dout, if defined) of `a` to copies of them: all of them
// to their planes (`six`), else those whose rows are not 16-byte chunks to
// padded ones.  The result keeps the copies alive.
static at::Tensor make_copies(Args& a, bool six, const at::Tensor& q,
                              const at::Tensor& k, const at::Tensor& v,
                              const at::Tensor& dout) {
  const bool f = q.scalar_type() == at::kFloat;
  const int E = six ? 8 : f ? 4 : 8, planes = six ? 3 : 1;
  const int64_t DC = (a.D + E - 1) / E * E;
  const at::Tensor* ts[4] = {&q, &k, &v, &dout};
  Copies p = {};
  p.D = a.D;
  int64_t total = 0, most = 0;
  for (int t = 0; t < 4; ++t) {
    if (!ts[t]->defined() || (!six && rows16(*ts[t]))) continue;
    p.heads[t] = (int)ts[t]->size(1);
    p.n[t] = ts[t]->size(0) * p.heads[t] * DC / E;
    total += planes * p.n[t] * E;
    most = std::max(most, p.n[t]);
  }
  if (most == 0) return at::Tensor();
  at::Tensor ws = at::empty({total}, q.options().dtype(
                                         six ? at::kBFloat16
                                             : q.scalar_type()));
  char* w = (char*)ws.data_ptr();
  auto add = [&](int t, const void*& ptr, int64_t& sn, int64_t& sh,
                 int64_t& sp) {
    if (p.n[t] == 0) return;
    p.src[t] = ptr;
    p.dst[t] = w;
    p.sn[t] = sn;
    p.sh[t] = sh;
    ptr = w;
    sn = p.heads[t] * DC;
    sh = DC;
    sp = p.n[t] * E;
    w += planes * p.n[t] * 16;
  };
  add(0, a.q, a.q_sn, a.q_sh, a.q_sp);
  add(1, a.k, a.k_sn, a.k_sh, a.k_sp);
  add(2, a.v, a.v_sn, a.v_sh, a.v_sp);
  add(3, a.dout, a.g_sn, a.g_sh, a.g_sp);
  const dim3 grid((unsigned)((most + 255) / 256), 4);
  six ? planes_kernel<<<grid, 256, 0, stream()>>>(p)
  : f ? pad_kernel<float><<<grid, 256, 0, stream()>>>(p)
      : pad_kernel<__bf16><<<grid, 256, 0, stream()>>>(p);
  DGMC_CHECK_LAUNCH();
  return ws;
}

// Splits of the other axis (`n` rows in tiles of `tile`) where the `tiles`
// of the own axis are too few or too uneven to fill the chip: up to two
// rounds of the workgroups of four waves that it holds at `waves` a SIMD
// (knowledge graphs' evaluation, 4 a SIMD: 1024 workgroups 540 us, 2048 516;
// 2 a SIMD: 1024 444 us of the ragged case, 1536 509, 768 487), no split
// under 16 tiles (ragged case: 8 650 us, 16 604, 32 659), 8 where one wave
// walks them (new entities: 16 44 us, 8 35).  None where the mean segment is
// short: a join with nothing to join takes 4 us.  False: none.
static bool split_axis(Args& a, int64_t tiles, int64_t n, int tile, int nw,
                       int waves) {
  tiles = std::max<int64_t>(tiles, 1) * a.KV;
  a.chunk = nw == 4 ? 16 : 8;
  a.splits = 1;
  if (waves_for(n, a.B) == 1) return false;
  a.splits = (int)std::max<int64_t>(
      1, std::min<int64_t>({(512 * waves + tiles - 1) / tiles,
                            n / ((int64_t)tile * a.chunk), kMaxSplits}));
  return a.splits > 1;
}

// Workspace of the splits: `outs` outputs and, for the forward (ml), maxima
// and sums of `rows` rows each, then the number of every tile's splits.
static at::Tensor part_workspace(Args& a, int64_t rows, int outs, bool ml,
                                 int64_t tiles, const at::Tensor& like) {
  const int64_t no = outs * a.splits * rows * a.D;
  const int64_t nml = ml ? 2 * a.splits * rows : 0;
  // (pairs of floats and 16-byte rows keep their alignment)
  const int64_t no4 = (no + 3) / 4 * 4;
  at::Tensor ws = at::empty({no4 + nml + tiles * a.KV},
                            like.options().dtype(at::kFloat));
  a.part_o = ws.data_ptr<float>();
  a.part_ml = a.part_o + no4;
  a.part_n = (int*)(a.part_ml + nml);
  return ws;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> forward(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
    const at::Tensor& ptr_q, const at::Tensor& ptr_k, double scale,
    double cap, const OptTensor& bias, const OptTensor& pos_q,
    const OptTensor& pos_k, const BucketLayout& layout, bool x6,
    bool train) {
  int axes;
  Args a = make_args(q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q, pos_k,
                     layout, axes);
  const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
  const auto f32 = q.options().dtype(at::kFloat);
  at::Tensor out = at::empty({a.Nq, a.H, a.D}, q.options());
  at::Tensor stat = at::empty({train ? a.Nq : 0, a.H, 2}, f32);
  // bf16 training keeps the rest of the output's rounding for delta.
  const bool f = q.scalar_type() == at::kFloat, fine = train && !f;
  at::Tensor lo = at::empty({fine ? a.Nq : 0, a.H, a.D}, q.options());
  if (a.Nq == 0) return {out, lo, stat};
  a.out = out.data_ptr();
  a.out_lo = fine ? lo.data_ptr() : nullptr;
  a.stat = train ? (float2*)stat.data_ptr<float>() : nullptr;
  const int nw = waves_for((int64_t)a.Nq * a.G, a.B);
  const bool six = f && takes_x6(a, x6);
  pick_bufs(a, f);
  const int DP = a.D <= 32 ? 32 : a.D <= 64 ? 64 : 128;
  const int TQ = 32 / a.G * nw,
            KT = fwd_keys(DP, nw, six ? 6 : f ? 4 : 2);
  const at::Tensor ws = make_copies(a, six, q, k, v, at::Tensor());
  at::Tensor part;
  if (split_axis(a, a.Nq / TQ, a.Nk, KT, nw, f || DP > 64 ? 2 : 4))
    part = part_workspace(a, (int64_t)a.Nq * a.H, 1, true,
                          (a.Nq + TQ - 1) / TQ, q);
  six    ? fwd_x6(a, axes, stream())
  : f    ? fwd_f32(a, axes, nw, stream())
  : fine ? fwd_bf16_fine(a, axes, nw, stream())
         : fwd_bf16(a, axes, nw, stream());
  if (a.splits > 1) join<FWD>(a, f, TQ);
  return {out, lo, stat};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> backward(
    const at::Tensor& dout, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& v, const at::Tensor& out, const at::Tensor& lo,
    const at::Tensor& stat, const at::Tensor& ptr_q, const at::Tensor& ptr_k,
    double scale, double cap, const OptTensor& bias, const OptTensor& pos_q,
    const OptTensor& pos_k, const BucketLayout& layout, bool x6) {
  int axes;
  Args a = make_args(q, k, v, ptr_q, ptr_k, scale, cap, bias, pos_q, pos_k,
                     layout, axes);
  check_heads(dout, "dout", q);
  TORCH_CHECK(dout.sizes() == q.sizes() && out.sizes() == q.sizes() &&
                  out.scalar_type() == q.scalar_type() &&
                  out.device() == q.device() && out.is_contiguous(),
              "segment_attention: dout and out must have q's shape");
  TORCH_CHECK(stat.device() == q.device() && stat.is_contiguous() &&
                  stat.scalar_type() == at::kFloat && stat.dim() == 3 &&
                  stat.size(0) == a.Nq && stat.size(1) == a.H &&
                  stat.size(2) == 2,
              "segment_attention: stat must be fp32 [nodes, heads, 2]");
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
  TORCH_CHECK(q.scalar_type() == at::kFloat ||
                  (lo.sizes() == q.sizes() && lo.is_contiguous() &&
                   lo.scalar_type() == q.scalar_type() &&
                   lo.device() == q.device()),
              "segment_attention: lo must have q's shape");
  a.o = out.data_ptr();
  a.out_lo = lo.data_ptr();
  a.dout = dout.data_ptr();
  a.g_sn = dout.stride(0); a.g_sh = dout.stride(1);
  a.vec_o = rows16(out);
  a.stat = (float2*)stat.data_ptr<float>();
  a.delta = delta.data_ptr<float>();
  a.dq = dq.data_ptr();
  a.dk = dk.data_ptr();
  a.dv = dv.data_ptr();
  const bool f = q.scalar_type() == at::kFloat;
  const int nwq = waves_for((int64_t)a.Nq * a.G, a.B);
  const int nwk = waves_for(a.Nk, a.B);
  const int TQ = 32 / a.G * nwq;
  const bool six = f && takes_x6(a, x6);
  pick_bufs(a, f);
  at::Tensor pq, pk, wsq;
  Args d = a;                         // of the dq kernel
  const at::Tensor ws = make_copies(a, six, q, k, v, dout);
  // A table's gradient sums dz over all rows, whose rounding has to average
  // out: x6 scores leave 4e-6 of it (1079 x 726 rows, 3 buckets), exact
  // products 6e-7, so the kernel that sums it takes those.
  const bool sixq = six && !axes;
  if (six && axes) wsq = make_copies(d, false, q, k, v, dout);
  else d = a;
  if (split_axis(d, d.Nq / TQ, d.Nk, 32, nwq, 2))
    pq = part_workspace(d, (int64_t)d.Nq * d.H, 1, false,
                        (d.Nq + TQ - 1) / TQ, q);
  // Workgroups of the dq kernel with a table: each keeps its LDS columns
  // over all of its tiles.  2048 waves: ragged case 149 us (1024 222, 4096
  // 168), one graph of 4096 nodes 222 (331, 248).
  int nblk = 0;
  at::Tensor part;
  if (axes) {
    const int items = (d.Nq + TQ - 1) / TQ * d.splits;
    nblk = std::max(1, std::min(items, 2048 / (d.KV * nwq)));
    part = at::empty({nblk, d.KV, d.G, d.slots}, f32);
    d.part_bias = part.data_ptr<float>();
  }
  sixq ? dq_x6(d, stream())
  : f  ? dq_f32(d, axes, nwq, nblk, stream())
       : dq_bf16(d, axes, nwq, nblk, stream());
  if (d.splits > 1) join<DQ>(d, f, TQ);
  if (a.Nk > 0) {
    if (split_axis(a, a.Nk / (32 * nwk), a.Nq, 32 / a.G, nwk, 2))
      pk = part_workspace(a, (int64_t)a.Nk * a.KV, 2, false,
                          (a.Nk + 32 * nwk - 1) / (32 * nwk), q);
    six ? dkv_x6(a, axes, stream())
    : f ? dkv_f32(a, axes, nwk, stream())
        : dkv_bf16(a, axes, nwk, stream());
    if (a.splits > 1) join<DKV>(a, f, 32 * nwk);
  }
  if (axes) {
    bias_sum_kernel<<<a.H, kSlots * kSumWays, 0, stream()>>>(
        d.part_bias, dbias.data_ptr<float>(), nblk, a.KV, a.G, a.slots, a.nb,
        a.half, axes);
    DGMC_CHECK_LAUNCH();
  }
  return {dq, dk, dv, dbias};
}

}  // namespace segattn
}  // namespace dgmc
