// cross_attention.hip -- attention of a batch of queries onto keys / values of another length:
//
//   S = scale q k^T over the keys that are not padding,  P = softmax(S),  out = P v       per head
//   backward: D = rowsum(dout * out),  dS = P * (dout v^T - D),
//             dv = P^T dout,  dq = scale dS k,  dk = scale dS^T q
//
// for float32, bfloat16 and float16, head widths up to 128, any lengths, per-batch key counts and
// / or a padding mask, and query heads that share key / value heads (h = g * hk).
// (reference: the attention of detection/GroupFree3D/models/transformer.py:36-76 with the
// key_padding_mask of models/multi_head_attention.py; csrc/attention.hip is the f32, unpadded core
// with dropout that the whole-layer call uses.)
//
// Rows.  The g query heads of one key head are rows of ONE product: row r of (batch, key head) is
// query r / g, head r % g of the group.  A single new query with 8 heads a group is then 8 rows of
// a tile instead of 8 one-row tiles, the keys are read once for all of them, and dk / dv sum over
// the group inside a workgroup: no atomics anywhere, equal results from run to run.
//
// Orientation.  Every product is arranged so that the lane that holds a score also holds it where
// the next product wants it.  Forward and dq compute S^T = K Q^T (32x32 tiles): a lane then has 16
// keys of ONE row, so maximum and sum are reductions over its own registers plus one exchange with
// the other half of the wave, the rescaling factor of a row is the lane's own, and the 16 values
// are, unmoved, the B operand of O^T += V^T P^T -- in a permuted key order that the A operand
// follows (a sum over keys does not care).  dk / dv compute S = Q K^T: a lane has 16 rows of one key
// and the same holds.  V^T, K^T, Q^T, dO^T fragments come from the row-major tiles by gfx950's LDS
// transpose read (16-bit) or 4-byte reads (f32).
//
// Numbers: scores, maxima, sums, O, dq, dk, dv accumulate in f32.  For 16-bit inputs P and dS are
// rounded to the input type where they enter the matrix instructions (relative error half an ulp
// per term).  float16 has five bits of exponent, too few for a backward pass as it stands -- a P of
// 16 384 even keys and a dS of small dout are subnormal or nothing, a dS of large dout infinite -- so
// there P is rounded as 2^15 P, and dS times a power of two, each row's for dq and each key's for dk,
// found on the way (fit_half).  All are taken out of the f32 sums again.  f32 runs on the f32 matrix
// instructions, nothing is rounded below 32 bits.
#include <algorithm>
#include <cstdint>

#include "decoder_ops.hpp"
#include "lds_dma.hpp"

#pragma clang fp contract(fast)

namespace btr {
namespace {

constexpr int kMaxShares = 1024;    // of a row's keys
constexpr int kFewShares = 8;
__host__ __device__ inline int up8(int v) { return (v + 7) & ~7; }
constexpr float kLog2e = 1.4426950408889634f;

struct XaArgs {
  int b, lq, lk, h, hk, g, d, gd, rows;          // rows = lq * g
  const void *q, *k, *v, *dout, *dout_dma;       // dout_dma: rows of gd elements that a DMA may read
  long long q_sb, q_sl, q_sh, k_sb, k_sl, k_sh, v_sb, v_sl, v_sh;   // element strides
  const int *lengths;                            // (b) or NULL
  const unsigned char *mask;                     // (b, lk), nonzero = padding, or NULL
  long long mask_sb;
  void *out;                                     // (b, lq, h, d)
  float *lse;      // (b * hk, rows): log2 of the row's sum of exp2(scale_log2 * s); +inf: no key;
                   // float16: less kPExp
  float *delta;    // (b * hk, rows): D
  void *dq, *dk, *dv;                            // contiguous, shaped like q, k, v
  float scale, scale_log2;
  int tiles, nsplit, chunk;                      // workgroup tiles, shares of the long axis, its length
  float *part, *part2;                           // partial results of the shares
};

// ------------------------------------------------------------------------------- f32 tiles in LDS
// Row-major [row][DP]; PITCH bytes a row, one 16-byte unit of padding.  (The 16-bit tiles: lds_dma.hpp.)
template <typename T, int DP>
struct Tile {
  static_assert(sizeof(T) == 4, "f32");
  static constexpr int V = Elem<T>::kVec;
  static constexpr int PITCH = DP * 4 + 16;
  static constexpr int UNITS = DP / V;           // 16-byte units of a row
  __device__ static __forceinline__ int unit_off(int row, int unit) {
    return row * PITCH + unit * 16;
  }
};

template <typename T>
__device__ __forceinline__ f32x16_t mma(typename Elem<T>::Vec a, typename Elem<T>::Vec b, f32x16_t c);
template <>
__device__ __forceinline__ f32x16_t mma<__bf16>(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
template <>
__device__ __forceinline__ f32x16_t mma<_Float16>(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
template <>   // f32: the 16 bytes are four reduction steps of two
__device__ __forceinline__ f32x16_t mma<float>(f32x4_t a, f32x4_t b, f32x16_t c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  return c;
}

// row of a 32x32 result tile that register v of lane half hh holds (its column is lane & 31)
__device__ __forceinline__ constexpr int acc_row(int v, int hh) {
  return (v & 3) + 8 * (v >> 2) + 4 * hh;
}

// first product: tile rows [row0, row0 + 32) x the register operand f (one row per lane & 31).  (All
// of the padded width: skipping the pieces beyond d -- 3 of 8 at d = 36 -- cost registers and time,
// dk / dv 50 -> 58 us.)
template <typename T, int DP>
__device__ __forceinline__ f32x16_t tile_times_rows(const char *tile, int row0, int l31, int hh,
                                                    const typename Elem<T>::Vec *f) {
  typedef Tile<T, DP> TL;
  f32x16_t acc = {};
#pragma unroll
  for (int j = 0; j < TL::UNITS / 2; ++j) {
    const auto a = *reinterpret_cast<const typename Elem<T>::Vec *>(
        tile + row0 * TL::PITCH + TL::unit_off(l31, 2 * j + hh));
    acc = mma<T>(a, f[j], acc);
  }
  return acc;
}

// second product: acc[nt] (32 columns of the tile x 32) += tile[row0 .. row0 + 32)^T w, w as the
// first product left it (register v: tile row acc_row(v, hh))
template <typename T, int DP>
__device__ __forceinline__ void tile_t_times(const char *tile, int row0, int lane,
                                             const f32x16_t &w, f32x16_t *acc) {
  typedef Tile<T, DP> TL;
  const int l31 = lane & 31, hh = lane >> 5;
  const char *t = tile + row0 * TL::PITCH;
#pragma unroll
  for (int s = 0; s < 16; ++s) {
    const float *row = reinterpret_cast<const float *>(t + acc_row(s, hh) * TL::PITCH);
#pragma unroll
    for (int nt = 0; nt < DP / 32; ++nt)
      acc[nt] = __builtin_amdgcn_mfma_f32_32x32x2f32(row[32 * nt + l31], w[s], acc[nt], 0, 0, 0);
  }
}

// value of the lane 32 away
__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32); }

// NR rows of a tile, global -> registers (a tile ahead) -> LDS
template <typename T, int DP, int NR, int THREADS>
struct Stage {
  typedef Tile<T, DP> TL;
  static constexpr int N = (NR * TL::UNITS + THREADS - 1) / THREADS;
  static constexpr bool EXACT = NR * TL::UNITS % THREADS == 0;
  typename Elem<T>::Vec r[N];
  // addr(row) -> pointer of the row (called for rows < limit only)
  template <typename F>
  __device__ __forceinline__ void fetch(F addr, int row0, int limit, int d, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + THREADS * i, row = e / TL::UNITS, col = (e % TL::UNITS) * TL::V;
      r[i] = typename Elem<T>::Vec{};
      if ((EXACT || row < NR) && row0 + row < limit && col < d)
        r[i] = load_row(addr(row0 + row), col, d);
    }
  }
  // rows whose bit in `live` is clear become zero whatever they hold (a padded row may hold NaN)
  __device__ __forceinline__ void store(char *tile, const unsigned long long *live, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + THREADS * i, row = e / TL::UNITS, unit = e % TL::UNITS;
      if (!EXACT && row >= NR) continue;
      typename Elem<T>::Vec v = r[i];
      if (live && !((live[row >> 6] >> (row & 63)) & 1)) v = typename Elem<T>::Vec{};
      *reinterpret_cast<typename Elem<T>::Vec *>(tile + TL::unit_off(row, unit)) = v;
    }
  }
};

// which keys of a tile take part, one bit each
template <int NR>
struct Live {
  static constexpr int W = (NR + 63) / 64;
  unsigned char m[W];
  __device__ __forceinline__ void fetch(const unsigned char *mask, int key0, int kend, int lane) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      const int key = key0 + 64 * i + lane;
      m[i] = mask && key < kend ? mask[key] : 0;
    }
  }
  __device__ __forceinline__ void words(int key0, int kend, int lane, unsigned long long *w) const {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = __ballot(key0 + 64 * i + lane < kend && m[i] == 0);
  }
};

// workgroup -> (tile, batch x key head, share).  Consecutive workgroups land on the eight XCDs in
// turn; all tiles of one (batch x key head, share) go to one XCD, whose L2 then serves their common
// keys, and those go to the XCDs in turn, so that batch entries of unequal length spread over all
// of them (with an eighth of the list per XCD, lengths of 1 024 .. 4 096 left 40 % of the chip idle).
__device__ __forceinline__ void place(const XaArgs &a, int &tile, int &bh, int &split) {
  const int units = gridDim.x / a.tiles, even = units / 8 * 8, id = blockIdx.x;
  int u;
  if (id < even * a.tiles) {
    const int j = id >> 3, q = j / a.tiles;
    u = (id & 7) + 8 * q;
    tile = j - q * a.tiles;
  } else {
    const int j = id - even * a.tiles, q = j / a.tiles;
    u = even + q;
    tile = j - q * a.tiles;
  }
  bh = u / a.nsplit;
  split = u - bh * a.nsplit;
}

template <typename T>
struct Rows {   // row r of (batch, key head) -> element offset of its query / its output
  const XaArgs &a;
  int b, kh;
  __device__ __forceinline__ const T *q(int r) const {
    const int l = r / a.g, hd = kh * a.g + r - l * a.g;
    return (const T *)a.q + b * a.q_sb + l * a.q_sl + hd * a.q_sh;
  }
  __device__ __forceinline__ long long o(int r) const {   // out, dout, dq: contiguous
    const int l = r / a.g, hd = kh * a.g + r - l * a.g;
    return (((long long)b * a.lq + l) * a.h + hd) * a.d;
  }
};

__device__ __forceinline__ int key_count(const XaArgs &a, int b) {
  int n = a.lk;
  if (a.lengths) n = min(n, max(a.lengths[b], 0));
  return n;
}

// four consecutive columns of a row
template <typename T>
__device__ __forceinline__ void store4(T *row, int c, int d, const float (&v)[4]) {
  typedef T U4 __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (c + 4 <= d) {
    U4 o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = (T)v[j];
    *reinterpret_cast<U4 *>(row + c) = o;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c + j < d) row[c + j] = (T)v[j];
  }
}

// float16's backward pass rounds P as 2^15 P <= 32 768 and dS as 2^up dS (fit_half).
template <typename T>
constexpr bool kHalf = false;
template <>
constexpr bool kHalf<_Float16> = true;
constexpr int kPExp = 15;
__device__ __forceinline__ int exp_above(float x) {   // |x| < 2^exp_above(x); 0 for 0, inf, NaN
  return __builtin_amdgcn_frexp_expf(x);
}
// dS as float16 takes it: 2^up dS, up one number per lane pair (32 apart) that share the sums `acc`.  It
// starts at kUpStart -- |dS| < 2^39, any of it fits float32 -- and goes down, for good, where a value
// leaves float16's range, to the power that puts the largest into [2^14, 2^15); the sums follow.  So the
// largest dS of a row or key decides, whatever the sizes of v and dout, and what it pushes below the
// type's smallest steps is 2^-39 of it.  (A maximum per two scores; the rest is for the few tiles that
// move it: 3 x 12 / 4 heads of 80, 333 x 1 777, dq 30 -> 32 us, dk / dv 45 -> 49 against powers from bounds,
// which did not hold.)  Returns by how much.  `on`: a lane whose sums are dropped has no say.
constexpr int kUpStart = 80;
template <int N>
__device__ __forceinline__ int fit_half(f32x16_t &ds, f32x16_t (&acc)[N], bool on) {
  float top = 0.f;
#pragma unroll
  for (int v = 0; v < 16; ++v) top = fmaxf(top, fabsf(ds[v]));
  const bool over = on && top > 65504.f;
  if (!__ballot(over)) return 0;
  top = over ? top : 0.f;
  top = fmaxf(top, __shfl_xor(top, 32));
  const int k = max(0, exp_above(top) - 15);     // (infinite: 0, nothing helps)
  const float f = __builtin_ldexpf(1.f, -k);
  ds *= f;
#pragma unroll
  for (int n = 0; n < N; ++n) acc[n] *= f;
  return k;
}
template <typename T>
__device__ __forceinline__ float lse_of(float m, float l) {   // l > 0, or NaN
  return l == 0.f ? INFINITY : m + __builtin_amdgcn_logf(l) - (kHalf<T> ? kPExp : 0);
}

constexpr int kMergePitch = 4;   // floats between rows beyond DP: rows land on different banks

// writes row r from the transposed accumulators (lane: row, 4 consecutive columns a register quad):
// the result and its log-sum-exp, or the share's unnormalised sums with (maximum in log2 units, sum)
template <typename T, int DP>
__device__ __forceinline__ void finish_row(const XaArgs &a, const Rows<T> &rows, int bh, int split,
                                           int r, int hh, float m, float l,
                                           const f32x16_t (&o)[DP / 32]) {
  const float mb = m * a.scale_log2;             // (-inf stays -inf)
  const bool share = a.nsplit > 1;
  const long long row = ((long long)split * a.b * a.hk + bh) * a.rows + r;
  const float inv = share ? 1.f : l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;   // (NaN stays NaN)
#pragma unroll
  for (int nt = 0; nt < DP / 32; ++nt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const float v4[4] = {o[nt][4 * gq] * inv, o[nt][4 * gq + 1] * inv, o[nt][4 * gq + 2] * inv,
                           o[nt][4 * gq + 3] * inv};
      const int c = 32 * nt + 8 * gq + 4 * hh;
      if (share)
        store4(a.part + row * a.d, c, a.d, v4);
      else
        store4((T *)a.out + rows.o(r), c, a.d, v4);
    }
  if (hh == 0) {
    if (share) {
      a.part2[2 * row] = mb;
      a.part2[2 * row + 1] = l;
    } else if (a.lse) {
      a.lse[(long long)bh * a.rows + r] = lse_of<T>(mb, l);
    }
  }
}

// the same for 32 WR rows whose keys WK waves each of the workgroup of four have shared: through LDS
// (om: 4 x 32 x (DP + 4) floats, the tiles' storage), added in wave order
template <typename T, int DP, int WR, int WK>
__device__ __forceinline__ void merge_rows(const XaArgs &a, const Rows<T> &rows, int bh, int split,
                                           int tile, int wr, int wk, int tid, float m, float l,
                                           const f32x16_t (&o)[DP / 32], float *om, float *mx,
                                           float *sm) {
  constexpr int LDO = DP + kMergePitch, PER = 256 / (32 * WR);   // threads a row
  const int lane = tid & 63, l31 = lane & 31, hh = lane >> 5, at = (wr * WK + wk) * 32 + l31;
  __syncthreads();                               // every wave is done with the tiles
#pragma unroll
  for (int nt = 0; nt < DP / 32; ++nt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq)
      *reinterpret_cast<f32x4_t *>(om + at * LDO + 32 * nt + 8 * gq + 4 * hh) =
          f32x4_t{o[nt][4 * gq], o[nt][4 * gq + 1], o[nt][4 * gq + 2], o[nt][4 * gq + 3]};
  if (hh == 0) {
    mx[at] = m * a.scale_log2;
    sm[at] = l;
  }
  __syncthreads();
  const int row = tid / PER, sub = tid % PER, rr = tile * 32 * WR + row;
  if (rr >= a.rows) return;
  const int first = (row >> 5) * WK * 32 + (row & 31);           // of its WK partial rows
  const bool share = a.nsplit > 1;
  const long long prow = ((long long)split * a.b * a.hk + bh) * a.rows + rr;
  float M = -INFINITY, L = 0.f, f[WK];
#pragma unroll
  for (int k = 0; k < WK; ++k) M = fmaxf(M, mx[first + 32 * k]);
#pragma unroll
  for (int k = 0; k < WK; ++k) {
    const float mk = mx[first + 32 * k];
    f[k] = mk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mk - M);
    L = fmaf(sm[first + 32 * k], f[k], L);
  }
  const float inv = share ? 1.f : L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
  for (int c = 4 * sub; c < a.d; c += 4 * PER) {
    f32x4_t t = {};
#pragma unroll
    for (int k = 0; k < WK; ++k)
      t += *reinterpret_cast<const f32x4_t *>(om + (first + 32 * k) * LDO + c) * f[k];
    const float v4[4] = {t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv};
    if (share)
      store4(a.part + prow * a.d, c, a.d, v4);
    else
      store4((T *)a.out + rows.o(rr), c, a.d, v4);
  }
  if (sub == 0) {
    if (share) {
      a.part2[2 * prow] = M;
      a.part2[2 * prow + 1] = L;
    } else if (a.lse) {
      a.lse[(long long)bh * a.rows + rr] = lse_of<T>(M, L);
    }
  }
}

// -------------------------------------------------------------------------------- forward
// WR waves along the rows (32 each) x WK along the keys, KT key subtiles of 32 per wave and tile.
//   WR 4, WK 1: many rows; the four waves share every K / V tile.
//   WR 1, WK 4: few rows (single queries).
// Bound by the f32 matrix instructions (64 columns wide for 33 .. 64) and, at a workgroup per CU, by
// their latency: 4 x 8 heads of 36, 256 queries, 1 024 keys 34 us and 6 for the join, 16 at the matrix
// pipe's rate.
template <typename T, int DP, int WR, int WK, int KT>
__global__ __launch_bounds__(256) void cross_attention_fwd_kernel(XaArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Vec Vec;
  constexpr int BKV = 32 * WK * KT, NT = DP / 32, TB = BKV * TL::PITCH;
  constexpr int MERGE = WK > 1 ? 4 * 32 * (DP + kMergePitch) * 4 : 0;
  constexpr int BYTES = 2 * TB > MERGE ? 2 * TB : MERGE;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  __shared__ float mx[WK > 1 ? 4 * 32 : 1], sm[WK > 1 ? 4 * 32 : 1];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  const int wr = w % WR, wk = w / WR;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kbeg = split * a.chunk, kend = min(key_count(a, b), kbeg + a.chunk);
  const T *kp = (const T *)a.k + b * a.k_sb + kh * a.k_sh;
  const T *vp = (const T *)a.v + b * a.v_sb + kh * a.v_sh;
  const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const Rows<T> rows{a, b, kh};
  const int r = tile * 32 * WR + 32 * wr + l31;

  Vec qf[TL::UNITS / 2];
#pragma unroll
  for (int j = 0; j < TL::UNITS / 2; ++j) {
    qf[j] = Vec{};
    if (r < a.rows) qf[j] = load_row(rows.q(r), (2 * j + hh) * TL::V, a.d);
  }
  f32x16_t o[NT] = {};
  float m = -INFINITY, l = 0.f;

  Stage<T, DP, BKV, 256> sk, sv;
  Live<BKV> lv;
  auto krow = [&](int key) { return kp + key * a.k_sl; };
  auto vrow = [&](int key) { return vp + key * a.v_sl; };
  if (kbeg < kend) {
    sk.fetch(krow, kbeg, kend, a.d, tid);
    sv.fetch(vrow, kbeg, kend, a.d, tid);
    lv.fetch(mask, kbeg, kend, lane);
  }
  char *kt = smem, *vt = smem + TB;
  for (int k0 = kbeg; k0 < kend; k0 += BKV) {
    unsigned long long live[Live<BKV>::W];
    lv.words(k0, kend, lane, live);
    lds_barrier();                               // the previous tile's reads are done
    sk.store(kt, mask ? live : nullptr, tid);
    sv.store(vt, mask ? live : nullptr, tid);
    if (k0 + BKV < kend) {                       // next tile's loads fly under this one's math
      sk.fetch(krow, k0 + BKV, kend, a.d, tid);
      sv.fetch(vrow, k0 + BKV, kend, a.d, tid);
      lv.fetch(mask, k0 + BKV, kend, lane);
    }
    lds_barrier();
    f32x16_t s[KT];
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int sub = wk * KT + t;
      const unsigned bits = (unsigned)(live[sub >> 1] >> (32 * (sub & 1)));
      s[t] = tile_times_rows<T, DP>(kt, 32 * sub, l31, hh, qf);
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (!((bits >> acc_row(v, hh)) & 1)) s[t][v] = -INFINITY;
      }
#pragma unroll
      for (int v = 0; v < 16; ++v) top = fmaxf(top, s[t][v]);
    }
    top = fmaxf(top, other_half(top));
    if (__ballot(top > m)) {                     // some row's maximum moved
      const float mn = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * a.scale_log2);
      m = mn;
      l *= f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[nt][v] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m * a.scale_log2;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        s[t][v] = __builtin_amdgcn_exp2f(fmaf(s[t][v], a.scale_log2, -base));
        l += s[t][v];
      }
      tile_t_times<T, DP>(vt, 32 * (wk * KT + t), lane, s[t], o);
    }
  }
  l += other_half(l);

  if constexpr (WK == 1) {
    if (r < a.rows) finish_row<T, DP>(a, rows, bh, split, r, hh, m, l, o);
  } else {
    merge_rows<T, DP, WR, WK>(a, rows, bh, split, tile, wr, wk, tid, m, l, o, (float *)smem, mx, sm);
  }
}

// Joins the shares.  A weight of a share without a finite score is its sum itself, which is 0, or NaN
// if its scores were.  Few shares: 32 threads a row, the shares in order.
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_join_few_kernel(XaArgs a) {
  const long long nrow = (long long)a.b * a.hk * a.rows;
  const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (row >= nrow) return;
  const int bh = (int)(row / a.rows), r = (int)(row - (long long)bh * a.rows);
  const int c = 4 * (threadIdx.x & 31);
  float m[kFewShares], l[kFewShares], M = -INFINITY, L = 0.f;
  f32x4_t p[kFewShares], t = {};
#pragma unroll
  for (int s = 0; s < kFewShares; ++s) {         // (every load in flight at once)
    const long long at = (s < a.nsplit ? s : 0) * nrow + row;
    m[s] = a.part2[2 * at];
    l[s] = a.part2[2 * at + 1];
    p[s] = load_row(a.part + at * a.d, c, a.d);
    if (s < a.nsplit) M = fmaxf(M, m[s]);
  }
#pragma unroll
  for (int s = 0; s < kFewShares; ++s)
    if (s < a.nsplit) {
      const float w = m[s] == -INFINITY ? l[s] : __builtin_amdgcn_exp2f(m[s] - M);
      t += p[s] * w;
      L = fmaf(l[s], w, L);
    }
  const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
  const Rows<T> rows{a, bh / a.hk, bh % a.hk};
  const float v4[4] = {t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv};
  store4((T *)a.out + rows.o(r), c, a.d, v4);
  if (c == 0 && a.lse) a.lse[row] = lse_of<T>(M, L);
}
// Many shares (of few rows): a workgroup a row, the weights once into LDS, then eight groups of 32
// threads add every eighth share, and the groups' sums are added in order.
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_join_kernel(XaArgs a) {
  __shared__ float wt[kMaxShares], red[8][128 + 4];
  const long long nrow = (long long)a.b * a.hk * a.rows, row = blockIdx.x;
  const int bh = (int)(row / a.rows), r = (int)(row - (long long)bh * a.rows);
  const int tid = threadIdx.x, g = tid >> 5, c = 4 * (tid & 31);
  float M = -INFINITY;
  for (int s = tid; s < a.nsplit; s += 256) {
    wt[s] = a.part2[2 * (s * nrow + row)];
    M = fmaxf(M, wt[s]);
  }
  for (int i = 32; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor(M, i));
  if ((tid & 63) == 0) red[0][tid >> 6] = M;
  __syncthreads();
  M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  for (int s = tid; s < a.nsplit; s += 256) {
    const float m = wt[s];
    wt[s] = m == -INFINITY ? a.part2[2 * (s * nrow + row) + 1] : __builtin_amdgcn_exp2f(m - M);
  }
  __syncthreads();
  f32x4_t t = {};
  float L = 0.f;
  for (int s = g; s < a.nsplit; s += 8) {
    const f32x4_t p = load_row(a.part + (s * nrow + row) * a.d, c, a.d);
    t += p * wt[s];
    L = fmaf(a.part2[2 * (s * nrow + row) + 1], wt[s], L);
  }
  *reinterpret_cast<f32x4_t *>(&red[g][c]) = t;
  if ((tid & 31) == 0) red[g][128] = L;
  __syncthreads();
  if (g) return;
  L = 0.f;
  t = f32x4_t{};
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    t += *reinterpret_cast<const f32x4_t *>(&red[k][c]);
    L += red[k][128];
  }
  const float inv = L > 0.f ? 1.f / L : L == 0.f ? 0.f : L;
  const Rows<T> rows{a, bh / a.hk, bh % a.hk};
  const float v4[4] = {t[0] * inv, t[1] * inv, t[2] * inv, t[3] * inv};
  store4((T *)a.out + rows.o(r), c, a.d, v4);
  if (tid == 0 && a.lse) a.lse[row] = lse_of<T>(M, L);
}

// -------------------------------------------------------------------------------- backward, dq
// As the forward: per tile S^T = K Q^T, dP^T = V dO^T, dS^T in place, dq^T += K^T dS^T.  D = rowsum
// (dO * O) comes first, from the same fragments, and is left for the dk / dv kernel.  (The sizes of
// the forward: 44 us and 5 for the shares' sum; 24 at the matrix pipe's rate.)
template <typename T, int DP, int WR, int WK, int KT>
__global__ __launch_bounds__(256) void cross_attention_bwd_q_kernel(XaArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Vec Vec;
  constexpr int BKV = 32 * WK * KT, NT = DP / 32, TB = BKV * TL::PITCH;
  constexpr int MERGE = WK > 1 ? 4 * 32 * (DP + kMergePitch) * 4 : 0;
  constexpr int BYTES = 2 * TB > MERGE ? 2 * TB : MERGE;
  __shared__ __attribute__((aligned(16))) char smem[BYTES];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  const int wr = w % WR, wk = w / WR;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kbeg = split * a.chunk, kend = min(key_count(a, b), kbeg + a.chunk);
  const T *kp = (const T *)a.k + b * a.k_sb + kh * a.k_sh;
  const T *vp = (const T *)a.v + b * a.v_sb + kh * a.v_sh;
  const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const Rows<T> rows{a, b, kh};
  const int r = tile * 32 * WR + 32 * wr + l31;

  Vec qf[TL::UNITS / 2], gf[TL::UNITS / 2];
  float delta = 0.f, lse = INFINITY;
#pragma unroll
  for (int j = 0; j < TL::UNITS / 2; ++j) {
    qf[j] = gf[j] = Vec{};
    if (r < a.rows) {
      const int c = (2 * j + hh) * TL::V;
      qf[j] = load_row(rows.q(r), c, a.d);
      gf[j] = load_row((const T *)a.dout + rows.o(r), c, a.d);
      const Vec of = load_row((const T *)a.out + rows.o(r), c, a.d);
#pragma unroll
      for (int i = 0; i < TL::V; ++i) delta = fmaf((float)gf[j][i], (float)of[i], delta);
    }
  }
  delta += other_half(delta);
  if (r < a.rows) {
    lse = a.lse[(long long)bh * a.rows + r];
    if (split == 0 && wk == 0 && hh == 0) a.delta[(long long)bh * a.rows + r] = delta;
  }
  f32x16_t dq[NT] = {};

  Stage<T, DP, BKV, 256> sk, sv;
  Live<BKV> lv;
  auto krow = [&](int key) { return kp + key * a.k_sl; };
  auto vrow = [&](int key) { return vp + key * a.v_sl; };
  if (kbeg < kend) {
    sk.fetch(krow, kbeg, kend, a.d, tid);
    sv.fetch(vrow, kbeg, kend, a.d, tid);
    lv.fetch(mask, kbeg, kend, lane);
  }
  char *kt = smem, *vt = smem + TB;
  for (int k0 = kbeg; k0 < kend; k0 += BKV) {
    unsigned long long live[Live<BKV>::W];
    lv.words(k0, kend, lane, live);
    lds_barrier();
    sk.store(kt, mask ? live : nullptr, tid);
    sv.store(vt, mask ? live : nullptr, tid);
    if (k0 + BKV < kend) {
      sk.fetch(krow, k0 + BKV, kend, a.d, tid);
      sv.fetch(vrow, k0 + BKV, kend, a.d, tid);
      lv.fetch(mask, k0 + BKV, kend, lane);
    }
    lds_barrier();
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      const int sub = wk * KT + t;
      const unsigned bits = (unsigned)(live[sub >> 1] >> (32 * (sub & 1)));
      f32x16_t s = tile_times_rows<T, DP>(kt, 32 * sub, l31, hh, qf);
      const f32x16_t dp = tile_times_rows<T, DP>(vt, 32 * sub, l31, hh, gf);
#pragma unroll
      for (int v = 0; v < 16; ++v)
        s[v] = __builtin_amdgcn_exp2f(fmaf(s[v], a.scale_log2, -lse)) * (dp[v] - delta);
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          if (!((bits >> acc_row(v, hh)) & 1)) s[v] = 0.f;
      }
      tile_t_times<T, DP>(kt, 32 * sub, lane, s, dq);
    }
  }
  const long long prow = ((long long)split * a.b * a.hk + bh) * a.rows;
  if constexpr (WK == 1) {
    if (r >= a.rows) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const float v4[4] = {dq[nt][4 * gq] * a.scale, dq[nt][4 * gq + 1] * a.scale,
                             dq[nt][4 * gq + 2] * a.scale, dq[nt][4 * gq + 3] * a.scale};
        const int c = 32 * nt + 8 * gq + 4 * hh;
        if (a.nsplit > 1)
          store4(a.part + (prow + r) * a.d, c, a.d, v4);
        else
          store4((T *)a.dq + rows.o(r), c, a.d, v4);
      }
  } else {
    constexpr int LDO = DP + kMergePitch, PER = 256 / (32 * WR);
    float *om = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int gq = 0; gq < 4; ++gq)
        *reinterpret_cast<f32x4_t *>(om + ((wr * WK + wk) * 32 + l31) * LDO + 32 * nt + 8 * gq +
                                     4 * hh) =
            f32x4_t{dq[nt][4 * gq], dq[nt][4 * gq + 1], dq[nt][4 * gq + 2], dq[nt][4 * gq + 3]};
    __syncthreads();
    const int row = tid / PER, sub = tid % PER, rr = tile * 32 * WR + row;
    if (rr >= a.rows) return;
    const int first = (row >> 5) * WK * 32 + (row & 31);
    for (int c = 4 * sub; c < a.d; c += 4 * PER) {
      f32x4_t t = {};
#pragma unroll
      for (int k = 0; k < WK; ++k)
        t += *reinterpret_cast<const f32x4_t *>(om + (first + 32 * k) * LDO + c);
      const float v4[4] = {t[0] * a.scale, t[1] * a.scale, t[2] * a.scale, t[3] * a.scale};
      if (a.nsplit > 1)
        store4(a.part + (prow + rr) * a.d, c, a.d, v4);
      else
        store4((T *)a.dq + rows.o(rr), c, a.d, v4);
    }
  }
}

// ----------------------------------------------------------------------------- backward, dk, dv
// Four waves x 32 keys; the rows pass by in tiles of 32.  S = Q K^T, dP = dO V^T with K and V rows
// in registers, then dv^T += dO^T P and dk^T += Q^T dS.  (The same sizes: 51 us and 8; 32.)
template <typename T, int DP>
__global__ __launch_bounds__(256) void cross_attention_bwd_kv_kernel(XaArgs a) {
  typedef Tile<T, DP> TL;
  typedef typename Elem<T>::Vec Vec;
  constexpr int BR = 32, NT = DP / 32, TB = BR * TL::PITCH;
  __shared__ __attribute__((aligned(16))) char smem[4 * TB];
  __shared__ __attribute__((aligned(16))) float stat[2][2][BR];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int nk = key_count(a, b);
  const int rbeg = split * a.chunk;
  int rend = min(a.rows, rbeg + a.chunk);
  if (tile * 128 >= nk) rend = rbeg;             // padding only: zeros
  const int key = tile * 128 + 32 * w + l31;
  const bool live = key < nk && !(a.mask && a.mask[b * a.mask_sb + key]);
  const Rows<T> rows{a, b, kh};

  Vec kf[TL::UNITS / 2], vf[TL::UNITS / 2];
#pragma unroll
  for (int j = 0; j < TL::UNITS / 2; ++j) {
    kf[j] = vf[j] = Vec{};
    if (live) {
      const int c = (2 * j + hh) * TL::V;
      kf[j] = load_row((const T *)a.k + b * a.k_sb + kh * a.k_sh + key * a.k_sl, c, a.d);
      vf[j] = load_row((const T *)a.v + b * a.v_sb + kh * a.v_sh + key * a.v_sl, c, a.d);
    }
  }
  f32x16_t dk[NT] = {}, dv[NT] = {};
  Stage<T, DP, BR, 256> sq, sg;
  float st = 0.f;
  auto qrow = [&](int r) { return rows.q(r); };
  auto grow = [&](int r) { return (const T *)a.dout + rows.o(r); };
  auto fetch = [&](int r0) {
    sq.fetch(qrow, r0, rend, a.d, tid);
    sg.fetch(grow, r0, rend, a.d, tid);
    if (tid < 2 * BR) {                          // lse (+inf beyond the rows: P = 0), then D
      const int r = r0 + (tid & (BR - 1));
      const float *src = tid < BR ? a.lse : a.delta;
      st = r < rend ? src[(long long)bh * a.rows + r] : tid < BR ? INFINITY : 0.f;
    }
  };
  if (rbeg < rend) fetch(rbeg);
  int buf = 0;
  for (int r0 = rbeg; r0 < rend; r0 += BR) {
    char *qt = smem + buf * 2 * TB, *gt = qt + TB;
    float *lse = stat[buf][0], *dl = stat[buf][1];
    sq.store(qt, nullptr, tid);
    sg.store(gt, nullptr, tid);
    if (tid < 2 * BR) (tid < BR ? lse : dl)[tid & (BR - 1)] = st;
    if (r0 + BR < rend) fetch(r0 + BR);
    lds_barrier();
    buf ^= 1;
    f32x16_t p = tile_times_rows<T, DP>(qt, 0, l31, hh, kf);
    f32x16_t ds = tile_times_rows<T, DP>(gt, 0, l31, hh, vf);
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const f32x4_t l4 = *reinterpret_cast<const f32x4_t *>(lse + 8 * gq + 4 * hh);
      const f32x4_t d4 = *reinterpret_cast<const f32x4_t *>(dl + 8 * gq + 4 * hh);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int v = 4 * gq + i;
        p[v] = live ? __builtin_amdgcn_exp2f(fmaf(p[v], a.scale_log2, -l4[i])) : 0.f;
        ds[v] = live ? p[v] * (ds[v] - d4[i]) : 0.f;
      }
    }
    tile_t_times<T, DP>(gt, 0, lane, p, dv);
    tile_t_times<T, DP>(qt, 0, lane, ds, dk);
  }
  if (key >= a.lk) return;
  const long long krow = (((long long)b * a.lk + key) * a.hk + kh) * a.d;
  const long long ptotal = (long long)a.b * a.lk * a.hk * a.d;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int c = 32 * nt + 8 * gq + 4 * hh;
      const float k4[4] = {dk[nt][4 * gq] * a.scale, dk[nt][4 * gq + 1] * a.scale,
                           dk[nt][4 * gq + 2] * a.scale, dk[nt][4 * gq + 3] * a.scale};
      const float v4[4] = {dv[nt][4 * gq], dv[nt][4 * gq + 1], dv[nt][4 * gq + 2],
                           dv[nt][4 * gq + 3]};
      if (a.nsplit > 1) {
        store4(a.part + split * ptotal + krow, c, a.d, k4);
        store4(a.part2 + split * ptotal + krow, c, a.d, v4);
      } else {
        store4((T *)a.dk + krow, c, a.d, k4);
        store4((T *)a.dv + krow, c, a.d, v4);
      }
    }
}

// out[i] = sum over the shares, in order; blockIdx.y picks one of two tensors.  ROWS: the share is
// laid out (batch, key head, row, d), the tensor (batch, query, head, d).  V elements at a time: 4
// where d is a multiple of 4, else 1.
template <typename T, bool ROWS, int V>
__global__ __launch_bounds__(256) void cross_attention_sum_kernel(XaArgs a, long long n, T *out0,
                                                                  T *out1) {
  typedef float F __attribute__((ext_vector_type(V), aligned(4)));
  const float *p = blockIdx.y ? a.part2 : a.part;
  T *out = blockIdx.y ? out1 : out0;
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * V; i < n;
       i += (long long)gridDim.x * 256 * V) {
    F t = 0.f;
    int s = 0;
    for (; s + 4 <= a.nsplit; s += 4) {            // (four loads in flight)
      F x[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) x[u] = *reinterpret_cast<const F *>(p + (s + u) * n + i);
#pragma unroll
      for (int u = 0; u < 4; ++u) t += x[u];
    }
    for (; s < a.nsplit; ++s) t += *reinterpret_cast<const F *>(p + s * n + i);
    long long dst = i;
    if (ROWS) {
      const long long row = i / a.d;
      const int bh = (int)(row / a.rows), r = (int)(row - (long long)bh * a.rows);
      const Rows<T> rows{a, bh / a.hk, bh % a.hk};
      dst = rows.o(r) + (i - row * a.d);
    }
    typedef T O __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    O o;
#pragma unroll
    for (int u = 0; u < V; ++u) o[u] = (T)t[u];
    *reinterpret_cast<O *>(out + dst) = o;
  }
}
template <typename T, bool ROWS>
void launch_sum(const XaArgs &a, long long n, T *out0, T *out1, hipStream_t hs) {
  const int v = a.d % 4 ? 1 : 4;
  const dim3 grid((unsigned)std::min<long long>(4096, (n / v + 255) / 256), out1 ? 2 : 1);
  if (v == 4)
    hipLaunchKernelGGL((cross_attention_sum_kernel<T, ROWS, 4>), grid, dim3(256), 0, hs, a, n, out0, out1);
  else
    hipLaunchKernelGGL((cross_attention_sum_kernel<T, ROWS, 1>), grid, dim3(256), 0, hs, a, n, out0, out1);
}

// =========================================================== 16-bit, aligned: tiles by LDS DMA
// Head widths of whole 16-byte units, rows on 16-byte boundaries (cross_attention_pack_kernel makes
// them so): the tiles go from memory to LDS by DMA (lds_dma.hpp; rows of 64 or 128 columns, of which
// the products take 32 NT), a tile ahead of their use, which frees the 32 staging registers a lane
// (two waves per SIMD fit: 332 -> 218 registers at D = 128) and the LDS write instructions.  Rows past
// the last key, masked keys and columns past d are loaded from beyond the buffer's bound, which reads
// as zero.
// rows x columns of a (row stride sl) matrix that a DMA may touch; anything else reads as zero
struct DmaSrc {
  const char *base;
  long long sl;                                  // bytes
  int d;                                         // bytes
};

// ROWS rows from row0 (those below `limit` and live) into `tile`, by THREADS threads
template <int D, int ROWS, int THREADS>
__device__ __forceinline__ void dma_tile(const DmaSrc &s, int row0, int limit,
                                         const unsigned long long *live, char *tile, int tid) {
  typedef Dma<D> DM;
  constexpr int N = ROWS * DM::UNITS / THREADS;
  static_assert(ROWS * DM::UNITS % THREADS == 0, "whole instructions");
  const int n = min(ROWS, limit - row0);
  const i32x4_t rsrc = dma_rsrc(s.base + row0 * s.sl, n > 0 ? (n - 1) * (int)s.sl + s.d : 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = i * THREADS + tid, row = e / DM::UNITS, u = (e % DM::UNITS) ^ DM::swz(row);
    int off = row * (int)s.sl + u * 16;
    if (u * 16 >= s.d) off = kFar;
    if (live && !((live[row >> 6] >> (row & 63)) & 1)) off = kFar;
    dma16(rsrc, off, tile + (i * THREADS + (tid & ~63)) * 16);
  }
}
// KT subtiles of 32 rows x the register operand.  The fragments are asked for in two batches ahead
// of the products: read one by one just before its product, each would cost an LDS round trip.
constexpr int row_of(int nt) { return nt <= 2 ? 64 : 128; }   // columns of a tile row in LDS
template <typename T, int NT, int KT>
__device__ __forceinline__ void dma_rows(const char *tile, int base, const typename Elem<T>::Vec *f,
                                         f32x16_t (&acc)[KT]) {
  constexpr int D = row_of(NT), J = 2 * NT, HALF = NT;
  typename Elem<T>::Vec x[J][KT];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int j = h * HALF; j < (h + 1) * HALF; ++j)
#pragma unroll
      for (int t = 0; t < KT; ++t)
        x[j][t] = *reinterpret_cast<const typename Elem<T>::Vec *>(
            tile + t * 32 * Dma<D>::PITCH + (base ^ (j << 5)));
    __builtin_amdgcn_sched_barrier(0);
  }
#pragma unroll
  for (int t = 0; t < KT; ++t) acc[t] = f32x16_t{};
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int t = 0; t < KT; ++t) acc[t] = mma<T>(x[j][t], f[j], acc[t]);
}
// acc[nt] += tile[32 rows]^T w: the next 16 rows' fragments are in flight during a step's products
template <typename T, int NT>
struct DmaT {
  static constexpr int D = row_of(NT);
  s16x4_t x[2][NT][2];
  __device__ __forceinline__ void load(const char *tile, int base, int s) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      x[s & 1][nt][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4)(tile + (base ^ (nt << 6)) + 16 * s * Dma<D>::PITCH));
      x[s & 1][nt][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(
          tile + (base ^ (nt << 6) ^ Dma<D>::kTrHi) + (16 * s + 8) * Dma<D>::PITCH));
    }
  }
  __device__ __forceinline__ void step(const f32x16_t &w, int s, f32x16_t *acc) {
    typename Elem<T>::Vec bv;
#pragma unroll
    for (int j = 0; j < 8; ++j) bv[j] = (T)w[8 * (s & 1) + j];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      union {
        s16x4_t s4[2];
        typename Elem<T>::Vec v;
      } u;
      u.s4[0] = x[s & 1][nt][0];
      u.s4[1] = x[s & 1][nt][1];
      acc[nt] = mma<T>(u.v, bv, acc[nt]);
    }
  }
};
// ... over KT subtiles; the first step's fragments have been loaded
template <typename T, int NT, int KT>
__device__ __forceinline__ void dma_t(DmaT<T, NT> &v, const char *tile, int base,
                                      const f32x16_t (&w)[KT], f32x16_t *acc) {
#pragma unroll
  for (int s = 0; s < 2 * KT; ++s) {
    if (s + 1 < 2 * KT) {
      v.load(tile, base, s + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    v.step(w[s >> 1], s, acc);
  }
}

// online softmax of one tile of KT x 32 scores a lane holds: maximum, rescaling, exponentials, sum
template <int KT, int NT>
__device__ __forceinline__ void online(f32x16_t (&s)[KT], float &m, float &l, f32x16_t (&o)[NT],
                                       float c) {
  float top = -INFINITY;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) top = fmaxf(top, s[t][v]);
  top = fmaxf(top, other_half(top));
  if (__ballot(top > m)) {                       // some row's maximum moved
    const float mn = fmaxf(m, top);
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * c);
    m = mn;
    l *= f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[nt][v] *= f;
  }
  const float base = m == -INFINITY ? 0.f : m * c;
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int v = 0; v < 16; ++v) {
      s[t][v] = __builtin_amdgcn_exp2f(fmaf(s[t][v], c, -base));
      l += s[t][v];
    }
}
template <int KT>
__device__ __forceinline__ void drop_dead(f32x16_t (&s)[KT], unsigned long long live, int hh) {
  if (~live == 0 || (KT == 1 && (unsigned)live == 0xffffffffu)) return;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const unsigned bits = (unsigned)(live >> (32 * t)) >> (4 * hh);
#pragma unroll
    for (int v = 0; v < 16; ++v) s[t][v] = bits & (1u << acc_row(v, 0)) ? s[t][v] : -INFINITY;
  }
}

// forward: WR waves x 32 rows share tiles of 64 keys, double-buffered, one barrier a tile.  Bound by
// the matrix pipe and the VALU in turns: a wave's exponentials run beside another's products as far
// as two or three waves a SIMD allow.  2 x 16 heads of 128 on 4 key heads, 4 096 queries, 16 384 keys,
// bf16: 1.03 ms, 1.07 PFLOP/s of the 1.5 that a large product reaches; 4 x 16 heads of 64, 2 048
// queries, 1 024 .. 4 096 keys: 125 - 140 us, 0.65 PFLOP/s (a score's VALU work is the same at half the
// products).
template <typename T, int NT, int WR>
__global__ __launch_bounds__(64 * WR, 2) void cross_attention_fwd_dma_kernel(XaArgs a) {
  typedef typename Elem<T>::Vec Vec;
  constexpr int D = row_of(NT), TB = 64 * Dma<D>::PITCH;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kbeg = split * a.chunk, kend = min(key_count(a, b), kbeg + a.chunk);
  const DmaSrc ks{(const char *)((const T *)a.k + b * a.k_sb + kh * a.k_sh), a.k_sl * 2, up8(a.d) * 2};
  const DmaSrc vs{(const char *)((const T *)a.v + b * a.v_sb + kh * a.v_sh), a.v_sl * 2, up8(a.d) * 2};
  const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const Rows<T> rows{a, b, kh};
  const int r = (tile * WR + w) * 32 + l31;
  Vec qf[2 * NT];
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) {
    qf[j] = Vec{};
    if (r < a.rows) qf[j] = load_row(rows.q(r), 16 * j + 8 * hh, a.d);
  }
  f32x16_t o[NT] = {};
  float m = -INFINITY, l = 0.f;
  const int rb = Dma<D>::row_base(l31, hh), tb = Dma<D>::tr_base(lane);

  Live<64> lv;
  unsigned long long live[1] = {0}, next[1] = {0};
  auto issue = [&](int k0, int buf) {
    dma_tile<D, 64, 64 * WR>(ks, k0, kend, mask ? next : nullptr, smem + buf * 2 * TB, tid);
    dma_tile<D, 64, 64 * WR>(vs, k0, kend, mask ? next : nullptr, smem + buf * 2 * TB + TB, tid);
  };
  lv.fetch(mask, kbeg, kend, lane);
  loads_done();
  if (kbeg < kend) {
    lv.words(kbeg, kend, lane, next);
    issue(kbeg, 0);
    if (mask) lv.fetch(mask, kbeg + 64, kend, lane);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += 64) {
    live[0] = next[0];
    dma_wait();
    lds_barrier();
    if (k0 + 64 < kend) {
      lv.words(k0 + 64, kend, lane, next);
      issue(k0 + 64, buf ^ 1);
      if (mask) lv.fetch(mask, k0 + 128, kend, lane);
    }
    const char *kt = smem + buf * 2 * TB, *vt = kt + TB;
    buf ^= 1;
    f32x16_t s[2];
    dma_rows<T, NT, 2>(kt, rb, qf, s);
    drop_dead<2>(s, live[0], hh);
    DmaT<T, NT> v;
    v.load(vt, tb, 0);
    online<2, NT>(s, m, l, o, a.scale_log2);
    dma_t<T, NT, 2>(v, vt, tb, s, o);
  }
  l += other_half(l);
  if (r < a.rows) finish_row<T, 32 * NT>(a, rows, bh, split, r, hh, m, l, o);
}

// few rows (32): every wave streams its own tiles of 32 keys -- wave w those of index w, w + 4, ..
// -- through its own double buffer, without a barrier until the four merge.  Bound by HBM: 64 KB a CU
// in flight.  (One query of 8 x 32 heads of 128 on 8 key heads, 8 192 .. 32 768 keys, bf16: 144 us,
// 4.65 TB/s, and 5 us for joining the shares.)
template <typename T, int NT>
__global__ __launch_bounds__(256) void cross_attention_fwd_stream_kernel(XaArgs a) {
  typedef typename Elem<T>::Vec Vec;
  constexpr int D = row_of(NT), TB = 32 * Dma<D>::PITCH, MERGE = 4 * 32 * (32 * NT + kMergePitch) * 4;
  __shared__ __attribute__((aligned(1024))) char smem[16 * TB > MERGE ? 16 * TB : MERGE];
  __shared__ float mx[4 * 32], sm[4 * 32];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kbeg = split * a.chunk, kend = min(key_count(a, b), kbeg + a.chunk);
  const DmaSrc ks{(const char *)((const T *)a.k + b * a.k_sb + kh * a.k_sh), a.k_sl * 2, up8(a.d) * 2};
  const DmaSrc vs{(const char *)((const T *)a.v + b * a.v_sb + kh * a.v_sh), a.v_sl * 2, up8(a.d) * 2};
  const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const Rows<T> rows{a, b, kh};
  const int r = tile * 32 + l31;
  Vec qf[2 * NT];
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) {
    qf[j] = Vec{};
    if (r < a.rows) qf[j] = load_row(rows.q(r), 16 * j + 8 * hh, a.d);
  }
  f32x16_t o[NT] = {};
  float m = -INFINITY, l = 0.f;
  const int rb = Dma<D>::row_base(l31, hh), tb = Dma<D>::tr_base(lane);
  const int wave = __builtin_amdgcn_readfirstlane(w);
  char *own = smem + wave * 4 * TB;

  Live<32> lv;
  unsigned long long live[1] = {0}, next[1] = {0};
  auto issue = [&](int k0, int buf) {
    dma_tile<D, 32, 64>(ks, k0, kend, mask ? next : nullptr, own + buf * 2 * TB, lane);
    dma_tile<D, 32, 64>(vs, k0, kend, mask ? next : nullptr, own + buf * 2 * TB + TB, lane);
  };
  const int first = kbeg + 32 * wave;
  lv.fetch(mask, first, min(kend, first + 32), lane);
  loads_done();
  if (first < kend) {
    lv.words(first, min(kend, first + 32), lane, next);
    issue(first, 0);
    if (mask) lv.fetch(mask, first + 128, min(kend, first + 160), lane);
  }
  int buf = 0;
  for (int k0 = first; k0 < kend; k0 += 128) {
    live[0] = next[0];
    if (k0 + 128 < kend) {
      lv.words(k0 + 128, min(kend, k0 + 160), lane, next);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the reads of the buffer it refills
      issue(k0 + 128, buf ^ 1);
      dma_wait<2 * 32 * Dma<D>::UNITS / 64>();
      if (mask) lv.fetch(mask, k0 + 256, min(kend, k0 + 288), lane);
    } else {
      dma_wait();
    }
    const char *kt = own + buf * 2 * TB, *vt = kt + TB;
    buf ^= 1;
    f32x16_t s[1];
    dma_rows<T, NT, 1>(kt, rb, qf, s);
    drop_dead<1>(s, live[0], hh);
    DmaT<T, NT> v;
    v.load(vt, tb, 0);
    online<1, NT>(s, m, l, o, a.scale_log2);
    dma_t<T, NT, 1>(v, vt, tb, s, o);
  }
  l += other_half(l);
  merge_rows<T, 32 * NT, 1, 4>(a, rows, bh, split, tile, 0, w, tid, m, l, o, (float *)smem, mx, sm);
}

// dq: WR waves x 32 rows share tiles of 64 keys as in the forward (the ragged batch: 155 - 170 us, 0.8
// PFLOP/s)
template <typename T, int NT, int WR>
__global__ __launch_bounds__(64 * WR, 2) void cross_attention_bwd_q_dma_kernel(XaArgs a) {
  typedef typename Elem<T>::Vec Vec;
  constexpr int D = row_of(NT), TB = 64 * Dma<D>::PITCH;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int kbeg = split * a.chunk, kend = min(key_count(a, b), kbeg + a.chunk);
  const DmaSrc ks{(const char *)((const T *)a.k + b * a.k_sb + kh * a.k_sh), a.k_sl * 2, up8(a.d) * 2};
  const DmaSrc vs{(const char *)((const T *)a.v + b * a.v_sb + kh * a.v_sh), a.v_sl * 2, up8(a.d) * 2};
  const unsigned char *mask = a.mask ? a.mask + b * a.mask_sb : nullptr;
  const Rows<T> rows{a, b, kh};
  const int r = (tile * WR + w) * 32 + l31;
  Vec qf[2 * NT], gf[2 * NT];
  float delta = 0.f, lse = INFINITY;
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) {
    qf[j] = gf[j] = Vec{};
    if (r < a.rows) {
      const int c = 16 * j + 8 * hh;
      qf[j] = load_row(rows.q(r), c, a.d);
      gf[j] = load_row((const T *)a.dout + rows.o(r), c, a.d);
      const Vec of = load_row((const T *)a.out + rows.o(r), c, a.d);
#pragma unroll
      for (int i = 0; i < 8; ++i) delta = fmaf((float)gf[j][i], (float)of[i], delta);
    }
  }
  delta += other_half(delta);
  if (r < a.rows) {
    lse = a.lse[(long long)bh * a.rows + r];
    if (split == 0 && hh == 0) a.delta[(long long)bh * a.rows + r] = delta;
  }
  int up = kUpStart;                             // float16: dS is rounded as 2^up dS
  if (kHalf<T>) lse += kPExp - up;               // (P comes out as 2^up P)
  f32x16_t dq[NT] = {};
  const int rb = Dma<D>::row_base(l31, hh), tb = Dma<D>::tr_base(lane);

  Live<64> lv;
  unsigned long long live[1] = {0}, next[1] = {0};
  auto issue = [&](int k0, int buf) {
    dma_tile<D, 64, 64 * WR>(ks, k0, kend, mask ? next : nullptr, smem + buf * 2 * TB, tid);
    dma_tile<D, 64, 64 * WR>(vs, k0, kend, mask ? next : nullptr, smem + buf * 2 * TB + TB, tid);
  };
  lv.fetch(mask, kbeg, kend, lane);
  loads_done();
  if (kbeg < kend) {
    lv.words(kbeg, kend, lane, next);
    issue(kbeg, 0);
    if (mask) lv.fetch(mask, kbeg + 64, kend, lane);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += 64) {
    live[0] = next[0];
    dma_wait();
    lds_barrier();
    if (k0 + 64 < kend) {
      lv.words(k0 + 64, kend, lane, next);
      issue(k0 + 64, buf ^ 1);
      if (mask) lv.fetch(mask, k0 + 128, kend, lane);
    }
    const char *kt = smem + buf * 2 * TB, *vt = kt + TB;
    buf ^= 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char *kt2 = kt + 32 * t * Dma<D>::PITCH;
      f32x16_t s[1], dp[1];
      dma_rows<T, NT, 1>(kt2, rb, qf, s);
      dma_rows<T, NT, 1>(vt + 32 * t * Dma<D>::PITCH, rb, gf, dp);
      DmaT<T, NT> kx;
      kx.load(kt2, tb, 0);
#pragma unroll
      for (int v = 0; v < 16; ++v)
        s[0][v] = __builtin_amdgcn_exp2f(fmaf(s[0][v], a.scale_log2, -lse)) * (dp[0][v] - delta);
      const unsigned bits = (unsigned)(live[0] >> (32 * t));
      if (bits != 0xffffffffu) {
#pragma unroll
        for (int v = 0; v < 16; ++v)
          s[0][v] = (bits >> (4 * hh)) & (1u << acc_row(v, 0)) ? s[0][v] : 0.f;
      }
      if constexpr (kHalf<T>) {
        const int down = fit_half(s[0], dq, true);
        up -= down;
        lse += (float)down;
      }
      dma_t<T, NT, 1>(kx, kt2, tb, s, dq);
    }
  }
  if (r >= a.rows) return;
  const long long prow = ((long long)split * a.b * a.hk + bh) * a.rows + r;
  if constexpr (kHalf<T>) {
    const float down = __builtin_ldexpf(1.f, -up);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) dq[nt] *= down;
  }
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const float v4[4] = {dq[nt][4 * gq] * a.scale, dq[nt][4 * gq + 1] * a.scale,
                           dq[nt][4 * gq + 2] * a.scale, dq[nt][4 * gq + 3] * a.scale};
      const int c = 32 * nt + 8 * gq + 4 * hh;
      if (a.nsplit > 1)
        store4(a.part + prow * a.d, c, a.d, v4);
      else
        store4((T *)a.dq + rows.o(r), c, a.d, v4);
    }
}

// dk, dv: WK waves x 32 keys, tiles of 64 rows.  A lane owns one key, its column of both results
// depends on no other key: what a padded key's lane computes is dropped at the end, nothing is
// selected on the way.  Rows past the end read as zeros (P = 1, but dout, dP - D and q are 0).  (The
// ragged batch: 210 - 235 us, 0.8 PFLOP/s.)
template <typename T, int NT, int WK>
__global__ __launch_bounds__(64 * WK, NT <= 2 ? 2 : 1) void cross_attention_bwd_kv_dma_kernel(XaArgs a) {
  typedef typename Elem<T>::Vec Vec;
  constexpr int D = row_of(NT), TB = 64 * Dma<D>::PITCH, THREADS = 64 * WK;
  constexpr int N = 64 * Dma<D>::UNITS / THREADS;
  __shared__ __attribute__((aligned(1024))) char smem[4 * TB];
  __shared__ __attribute__((aligned(1024))) float stat[2][2][64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l31 = lane & 31, hh = lane >> 5;
  int tile, bh, split;
  place(a, tile, bh, split);
  const int b = bh / a.hk, kh = bh - b * a.hk;
  const int nk = key_count(a, b);
  const int rbeg = split * a.chunk;
  int rend = min(a.rows, rbeg + a.chunk);
  if (tile * 32 * WK >= nk) rend = rbeg;         // padding only: zeros
  const int key = (tile * WK + w) * 32 + l31;
  const bool live = key < nk && !(a.mask && a.mask[b * a.mask_sb + key]);
  Vec kf[2 * NT], vf[2 * NT];
#pragma unroll
  for (int j = 0; j < 2 * NT; ++j) {
    kf[j] = vf[j] = Vec{};
    if (live && 16 * j + 8 * hh < a.d) {
      const int c = 16 * j + 8 * hh;
      kf[j] = *reinterpret_cast<const typename Elem<T>::VecU *>(
          (const T *)a.k + b * a.k_sb + kh * a.k_sh + key * a.k_sl + c);
      vf[j] = *reinterpret_cast<const typename Elem<T>::VecU *>(
          (const T *)a.v + b * a.v_sb + kh * a.v_sh + key * a.v_sl + c);
    }
  }
  int up = kUpStart;                             // float16: dS is rounded as 2^up dS, P as 2^kPExp P
  float ds_up = __builtin_ldexpf(1.f, up - kPExp);
  f32x16_t dk[NT] = {}, dv[NT] = {};
  const int rb = Dma<D>::row_base(l31, hh), tb = Dma<D>::tr_base(lane);

  const char *qb = (const char *)((const T *)a.q + b * a.q_sb + (long long)kh * a.g * a.q_sh);
  const char *gb = (const char *)((const T *)a.dout_dma +
                                  ((long long)b * a.lq * a.h + kh * a.g) * a.gd);
  // row r0 + row of the tile is query l0 + l, head hd of the group; (rem + row) / g by a multiplication
  // (exact: below 64 + g <= 192, times a reciprocal rounded up by less than g / 65 536)
  const int inv_g = (65536 + a.g - 1) / a.g;
  auto issue = [&](int r0, int buf) {
    char *qt = smem + buf * 2 * TB, *gt = qt + TB;
    const int l0 = r0 / a.g, rem = r0 - l0 * a.g;
    const i32x4_t qr = dma_rsrc(qb + 2 * (l0 * a.q_sl), kFar);
    const i32x4_t gr = dma_rsrc(gb + 2 * ((long long)l0 * a.h * a.gd), kFar);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * THREADS + tid, row = e / Dma<D>::UNITS;
      const int u = (e % Dma<D>::UNITS) ^ Dma<D>::swz(row);
      const int l = (rem + row) * inv_g >> 16, hd = rem + row - l * a.g;
      const bool in = r0 + row < rend && 8 * u < a.d;
      dma16(qr, in ? 2 * (l * (int)a.q_sl + hd * (int)a.q_sh + 8 * u) : kFar,
            qt + (i * THREADS + (tid & ~63)) * 16);
      dma16(gr, in ? 2 * ((l * a.h + hd) * a.gd + 8 * u) : kFar,
            gt + (i * THREADS + (tid & ~63)) * 16);
    }
    if (w < 2) {                                 // lse, D of the rows
      const float *src = (w ? a.delta : a.lse) + (long long)bh * a.rows + r0;
      dma4(dma_rsrc((const char *)src, (rend - r0) * 4), lane * 4, (char *)stat[buf][w ? 1 : 0]);
    }
  };
  loads_done();
  if (rbeg < rend) issue(rbeg, 0);
  int buf = 0;
  for (int r0 = rbeg; r0 < rend; r0 += 64) {
    dma_wait();
    lds_barrier();
    if (r0 + 64 < rend) issue(r0 + 64, buf ^ 1);
    const char *qt = smem + buf * 2 * TB, *gt = qt + TB;
    const float *lse = stat[buf][0], *dl = stat[buf][1];
    buf ^= 1;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const char *q2 = qt + 32 * t * Dma<D>::PITCH, *g2 = gt + 32 * t * Dma<D>::PITCH;
      f32x16_t p[1], ds[1];
      dma_rows<T, NT, 1>(q2, rb, kf, p);
      dma_rows<T, NT, 1>(g2, rb, vf, ds);
      DmaT<T, NT> gx;
      gx.load(g2, tb, 0);
#pragma unroll
      for (int gq = 0; gq < 4; ++gq) {
        const f32x4_t l4 = *reinterpret_cast<const f32x4_t *>(lse + 32 * t + 8 * gq + 4 * hh);
        const f32x4_t d4 = *reinterpret_cast<const f32x4_t *>(dl + 32 * t + 8 * gq + 4 * hh);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int v = 4 * gq + i;
          p[0][v] = __builtin_amdgcn_exp2f(fmaf(p[0][v], a.scale_log2, -l4[i]));
          ds[0][v] = p[0][v] * (ds[0][v] - d4[i]);
          if (kHalf<T>) ds[0][v] *= ds_up;
        }
      }
      if constexpr (kHalf<T>) {
        up -= fit_half(ds[0], dk, live);
        ds_up = __builtin_ldexpf(1.f, up - kPExp);
      }
      dma_t<T, NT, 1>(gx, g2, tb, p, dv);
      DmaT<T, NT> qx;
      qx.load(q2, tb, 0);
      dma_t<T, NT, 1>(qx, q2, tb, ds, dk);
    }
  }
  if (key >= a.lk) return;
  if constexpr (kHalf<T>) {
    const float down = __builtin_ldexpf(1.f, -up), p_down = __builtin_ldexpf(1.f, -kPExp);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      dk[nt] *= down;
      dv[nt] *= p_down;
    }
  }
  const long long krow = (((long long)b * a.lk + key) * a.hk + kh) * a.d;
  const long long ptotal = (long long)a.b * a.lk * a.hk * a.d;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int gq = 0; gq < 4; ++gq) {
      const int c = 32 * nt + 8 * gq + 4 * hh;
      float k4[4], v4[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        k4[i] = live ? dk[nt][4 * gq + i] * a.scale : 0.f;
        v4[i] = live ? dv[nt][4 * gq + i] : 0.f;
      }
      if (a.nsplit > 1) {
        store4(a.part + split * ptotal + krow, c, a.d, k4);
        store4(a.part2 + split * ptotal + krow, c, a.d, v4);
      } else {
        store4((T *)a.dk + krow, c, a.d, k4);
        store4((T *)a.dv + krow, c, a.d, v4);
      }
    }
}

// (batch, length, head, d) rows that do not lie on 16-byte boundaries in whole units -> contiguous ones
// that do, zeros behind them; up to four tensors (blockIdx.y)
struct XaPack {
  struct One {
    const void *src;
    void *dst;
    long long sb, sl, sh;
    int len, heads;
  } op[4];
  int b, d;
};
template <typename T>
__global__ __launch_bounds__(256) void cross_attention_pack_kernel(XaPack a) {
  const XaPack::One o = a.op[blockIdx.y];
  const int units = up8(a.d) / 8;
  const long long total = (long long)a.b * o.len * o.heads * units;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total;
       e += (long long)gridDim.x * 256) {
    const long long row = e / units, bl = row / o.heads;
    const int c = (int)(e - row * units) * 8, h = (int)(row - bl * o.heads);
    const long long b = bl / o.len, l = bl - b * o.len;
    reinterpret_cast<typename Elem<T>::Vec *>(o.dst)[e] =
        load_row((const T *)o.src + b * o.sb + l * o.sl + h * o.sh, c, a.d);
  }
}

// ------------------------------------------------------------------------------------ host
constexpr int kFewRows = 32;     // one tile of rows: the waves split the keys instead

struct Shares {
  int tiles, n, chunk;
};

// Shares of the long axis where the tiles alone do not fill the `slots` of resident workgroups, none
// shorter than `least`: their partial sums are as large as the result each, so not more of them than
// the rounds of workgroups call for -- the time of the rounds against 1 % of the whole per share (3
// x 1 777 keys, 999 rows of 80 columns, f16: 7 shares dk / dv 73 us with their sum, 3 shares 53).
// Not where the slots are full: 1 024 tiles on 768 in three shares cost 60 us of joins to save none.
Shares shares(int tiles, long long bh, int length, int step, int least, int slots) {
  const long long base = std::max<long long>(1, tiles * bh);
  const long long most = base >= slots ? 1 : std::min<long long>(64, length / least);
  long long best = 1;
  double time = 1e30;
  for (long long n = 1; n <= std::max<long long>(1, most); ++n) {
    const double t = (double)((base * n + slots - 1) / slots) / n + 0.01 * n;
    if (t < time) {
      time = t;
      best = n;
    }
  }
  const int chunk = std::max(step, cdiv(cdiv(length, best), step) * step);
  return {tiles, std::max(1, cdiv(length, chunk)), chunk};
}
// A few rows' forward streams the keys: about four workgroups per CU, which also evens out batch
// entries of unequal length.
Shares stream_shares(int tiles, long long bh, int length) {
  const long long base = std::max<long long>(1, tiles * bh);
  const long long n = std::max<long long>(
      1, std::min<long long>(base < 512 ? (1024 + base - 1) / base : 1, length / 256));
  const int chunk = std::max(128, cdiv(cdiv(length, n), 128) * 128);
  return {tiles, std::max(1, cdiv(length, chunk)), chunk};
}
bool few(int rows) { return rows <= kFewRows; }
// Rows of a workgroup of the DMA kernels.  Wide heads, bound by the tiles' way to LDS: 256 where those
// still give every CU two workgroups (the keys are read half as often).  Heads of up to 64 columns,
// bound by the VALU: 128, of which three fit a CU instead of one of 256 (ragged batch: 163 -> 133 us
// forward, 192 -> 157 us dq).
int dma_rows_per(const XaArgs &a) {
  return a.d > 64 && (long long)cdiv(a.rows, 256) * a.b * a.hk >= 512 ? 256 : 128;
}
// forward, dq: over the keys
Shares row_shares(const XaArgs &a, int dtype, bool fwd) {
  const long long bh = (long long)a.b * a.hk;
  if (few(a.rows) && (fwd || dtype == BTR_F32)) return stream_shares(1, bh, a.lk);
  const int per = dtype == BTR_F32 ? 128 : dma_rows_per(a);
  const int cu = dtype == BTR_F32 ? 1 : per == 256 ? 1 : a.d <= 64 ? 3 : 2;   // workgroups it holds
  return shares(cdiv(a.rows, per), bh, a.lk, 128, 256, 256 * cu);
}
// dk, dv: over the rows; two workgroups a CU for heads of up to 64 columns, one for wider ones
Shares key_shares(const XaArgs &a) {
  return shares(cdiv(a.lk, 128), (long long)a.b * a.hk, a.rows, 64, 128, a.d <= 64 ? 512 : 256);
}
// Rows a DMA may read where they are: whole 16-byte units on 16-byte boundaries, a tile's offsets
// below 2^31, and (keys) rows apart by at least a row.
bool aligned(int d, const void *p, long long sb, long long sl, long long sh) {
  return d % 8 == 0 && ((uintptr_t)p & 15) == 0 && ((sb | sl | sh) & 7) == 0 && sl <= (1 << 22) &&
         sh <= (1 << 22) && sl >= 0 && sh >= 0;
}
bool key_rows_ok(const XaArgs &a, const void *p, long long sb, long long sl, long long sh) {
  return aligned(a.d, p, sb, sl, sh) && sl >= a.d;
}
size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
size_t packed_bytes(const XaArgs &a, long long len, int heads) {
  return align256((size_t)a.b * len * heads * up8(a.d) * 2);
}
// What has to be packed before the DMA kernels run: K and V, for dk / dv also q and dout.  The
// workspace is counted with the same rule.
template <typename F>
void for_unaligned(const XaArgs &a, bool bwd, F f) {
  if (!key_rows_ok(a, a.k, a.k_sb, a.k_sl, a.k_sh)) f(0);
  if (!key_rows_ok(a, a.v, a.v_sb, a.v_sl, a.v_sh)) f(1);
  if (bwd && !aligned(a.d, a.q, a.q_sb, a.q_sl, a.q_sh)) f(2);
  if (bwd && !aligned(a.d, a.dout, 0, (long long)a.h * a.d, a.d)) f(3);
}
size_t pack_bytes(const XaArgs &a, int dtype, bool bwd) {
  size_t n = 0;
  if (dtype != BTR_F32)
    for_unaligned(a, bwd, [&](int i) {
      n += packed_bytes(a, i < 2 ? a.lk : a.lq, i < 2 ? a.hk : a.h);
    });
  return n;
}
template <typename T>
void pack(XaArgs &a, bool bwd, char *&ws, hipStream_t hs) {
  if constexpr (sizeof(T) == 2) {
    XaPack pk{};
    pk.b = a.b;
    pk.d = a.d;
    int n = 0;
    long long most = 0;
    const XaArgs in = a;
    for_unaligned(in, bwd, [&](int i) {
      const int len = i < 2 ? a.lk : a.lq, heads = i < 2 ? a.hk : a.h;
      const long long sl = (long long)heads * up8(a.d), sb = sl * len, sh = up8(a.d);
      const long long hd = (long long)in.h * in.d;
      if (i == 0) {
        pk.op[n++] = {in.k, ws, in.k_sb, in.k_sl, in.k_sh, len, heads};
        a.k = ws; a.k_sb = sb; a.k_sl = sl; a.k_sh = sh;
      } else if (i == 1) {
        pk.op[n++] = {in.v, ws, in.v_sb, in.v_sl, in.v_sh, len, heads};
        a.v = ws; a.v_sb = sb; a.v_sl = sl; a.v_sh = sh;
      } else if (i == 2) {
        pk.op[n++] = {in.q, ws, in.q_sb, in.q_sl, in.q_sh, len, heads};
        a.q = ws; a.q_sb = sb; a.q_sl = sl; a.q_sh = sh;
      } else {
        pk.op[n++] = {in.dout, ws, hd * in.lq, hd, in.d, len, heads};
        a.dout_dma = ws; a.gd = up8(a.d);
      }
      most = std::max(most, sb / 8 * a.b);
      ws += packed_bytes(a, len, heads);
    });
    if (n && most)
      hipLaunchKernelGGL((cross_attention_pack_kernel<T>),
                         dim3((unsigned)std::min<long long>(4096, (most + 255) / 256), n), dim3(256),
                         0, hs, pk);
  }
}

template <typename T, int DP>
void launch_fwd(const XaArgs &a, hipStream_t hs) {
  const dim3 grid((unsigned)((long long)a.tiles * a.b * a.hk * a.nsplit));
  if constexpr (sizeof(T) == 2) {
    constexpr int NT = DP / 32;
    if (few(a.rows))
      hipLaunchKernelGGL((cross_attention_fwd_stream_kernel<T, NT>), grid, dim3(256), 0, hs, a);
    else if (dma_rows_per(a) == 256)
      hipLaunchKernelGGL((cross_attention_fwd_dma_kernel<T, NT, 8>), grid, dim3(512), 0, hs, a);
    else
      hipLaunchKernelGGL((cross_attention_fwd_dma_kernel<T, NT, 4>), grid, dim3(256), 0, hs, a);
  } else {
    if (few(a.rows))
      hipLaunchKernelGGL((cross_attention_fwd_kernel<T, DP, 1, 4, 1>), grid, dim3(256), 0, hs, a);
    else
      hipLaunchKernelGGL((cross_attention_fwd_kernel<T, DP, 4, 1, 2>), grid, dim3(256), 0, hs, a);
  }
}
template <typename T, int DP>
void launch_bwd_q(const XaArgs &a, hipStream_t hs) {
  const dim3 grid((unsigned)((long long)a.tiles * a.b * a.hk * a.nsplit));
  if constexpr (sizeof(T) == 2) {
    if (dma_rows_per(a) == 256)
      hipLaunchKernelGGL((cross_attention_bwd_q_dma_kernel<T, DP / 32, 8>), grid, dim3(512), 0, hs, a);
    else
      hipLaunchKernelGGL((cross_attention_bwd_q_dma_kernel<T, DP / 32, 4>), grid, dim3(256), 0, hs, a);
  } else {
    if (few(a.rows))
      hipLaunchKernelGGL((cross_attention_bwd_q_kernel<T, DP, 1, 4, 1>), grid, dim3(256), 0, hs, a);
    else
      hipLaunchKernelGGL((cross_attention_bwd_q_kernel<T, DP, 4, 1, 2>), grid, dim3(256), 0, hs, a);
  }
}
template <typename T, int DP>
void launch_bwd_kv(const XaArgs &a, hipStream_t hs) {
  const dim3 grid((unsigned)((long long)a.tiles * a.b * a.hk * a.nsplit));
  if constexpr (sizeof(T) == 2)
    hipLaunchKernelGGL((cross_attention_bwd_kv_dma_kernel<T, DP / 32, 4>), grid, dim3(256), 0, hs, a);
  else
    hipLaunchKernelGGL((cross_attention_bwd_kv_kernel<T, DP>), grid, dim3(256), 0, hs, a);
}

#define BTR_XA_WIDTH(FN, ...)                  \
  do {                                         \
    if (a.d <= 32) FN<T, 32>(__VA_ARGS__);     \
    else if (a.d <= 64) FN<T, 64>(__VA_ARGS__);\
    else if (a.d <= 96) FN<T, 96>(__VA_ARGS__);\
    else FN<T, 128>(__VA_ARGS__);              \
  } while (0)

int check(const char *what, const btr_cross_attention_t *p, XaArgs &a) {
  BTR_REQUIRE(p, "%s: null description", what);
  BTR_REQUIRE(p->dtype >= BTR_F32 && p->dtype <= BTR_F16, "%s: unknown element type %d", what,
              p->dtype);
  BTR_REQUIRE(p->b >= 0 && p->lq >= 0 && p->lk >= 0 && p->h >= 1 && p->hk >= 1 &&
                  p->h % p->hk == 0,
              "%s: batch %d, queries %d, keys %d, heads %d on %d key heads", what, p->b, p->lq,
              p->lk, p->h, p->hk);
  BTR_REQUIRE(p->d >= 1 && p->d <= 128, "%s: head width %d (1 .. 128)", what, p->d);
  BTR_REQUIRE(p->h / p->hk <= 128 && (long long)p->h * up8(p->d) <= (1 << 22),
              "%s: %d heads on %d key heads", what, p->h, p->hk);
  BTR_REQUIRE(p->scale > 0.f && p->scale < INFINITY, "%s: scale %g", what, p->scale);
  a = XaArgs{};
  a.b = p->b; a.lq = p->lq; a.lk = p->lk; a.h = p->h; a.hk = p->hk; a.g = p->h / p->hk; a.d = p->d;
  const long long rows = (long long)p->lq * a.g;
  // a workgroup list and a row index of 32 bits (check_grid: the launches)
  BTR_REQUIRE(rows <= (1 << 30) && p->lk <= (1 << 30) &&
                  (rows / 32 + p->lk / 128 + 2) * (long long)p->b * p->hk <= (1 << 30),
              "%s: too many rows (%lld) or keys (%d)", what, rows, p->lk);
  a.rows = (int)rows;
  a.q = p->q; a.k = p->k; a.v = p->v;
  a.q_sb = p->q_sb; a.q_sl = p->q_sl; a.q_sh = p->q_sh;
  a.k_sb = p->k_sb; a.k_sl = p->k_sl; a.k_sh = p->k_sh;
  a.v_sb = p->v_sb; a.v_sl = p->v_sl; a.v_sh = p->v_sh;
  a.lengths = p->lengths;
  a.mask = p->mask;
  a.mask_sb = p->mask_sb;
  a.scale = p->scale;
  a.scale_log2 = p->scale * kLog2e;
  const bool some = p->b > 0 && p->lq > 0, keys = p->b > 0 && p->lk > 0;
  BTR_REQUIRE((!some || p->q) && (!keys || (p->k && p->v)), "%s: null pointer", what);
  return BTR_OK;
}

// a launch's thread numbers have 32 bits
int check_grid(const char *what, const XaArgs &a, int dtype, bool bwd) {
  const long long bh = (long long)a.b * a.hk;
  const auto threads = [&](const Shares &s, int per) { return s.tiles * bh * s.n * per; };
  const bool wide = dtype != BTR_F32 && dma_rows_per(a) == 256 && (bwd || !few(a.rows));
  long long most = threads(row_shares(a, dtype, !bwd), wide ? 512 : 256);
  if (bwd) most = std::max(most, threads(key_shares(a), 256));
  BTR_REQUIRE(most < 1ll << 32, "%s: batch %d, %d key heads, %d rows, %d keys: too many workgroups", what,
              a.b, a.hk, a.rows, a.lk);
  return BTR_OK;
}

size_t fwd_bytes(const XaArgs &a, int dtype) {
  const Shares s = row_shares(a, dtype, true);
  const size_t n = s.n == 1 ? 0 : (size_t)s.n * a.b * a.hk * a.rows;
  return pack_bytes(a, dtype, false) + align256(n * a.d * 4) + align256(n * 8);
}
size_t stats_bytes(const XaArgs &a) { return align256((size_t)a.b * a.hk * a.rows * 4); }   // D
size_t bwd_bytes(const XaArgs &a, int dtype) {   // this, what is packed, the shares of dq or of dk, dv
  const Shares q = row_shares(a, dtype, false), k = key_shares(a);
  size_t nq = 0, nk = 0;
  if (q.n > 1) nq = align256((size_t)q.n * a.b * a.hk * a.rows * a.d * 4);
  if (k.n > 1) nk = 2 * align256((size_t)k.n * a.b * a.lk * a.hk * a.d * 4);
  return stats_bytes(a) + pack_bytes(a, dtype, true) + std::max(nq, nk);
}

}  // namespace
}  // namespace btr

using namespace btr;

extern "C" size_t btr_cross_attention_fwd_workspace_bytes(const btr_cross_attention_t *p) {
  XaArgs a;
  if (check("cross_attention", p, a) != BTR_OK ||
      check_grid("cross_attention", a, p->dtype, false) != BTR_OK)
    return 0;
  return fwd_bytes(a, p->dtype);
}

extern "C" size_t btr_cross_attention_bwd_workspace_bytes(const btr_cross_attention_t *p,
                                                          const void *dout) {
  XaArgs a;
  if (check("cross_attention", p, a) != BTR_OK ||
      check_grid("cross_attention", a, p->dtype, true) != BTR_OK)
    return 0;
  a.dout = dout;
  return bwd_bytes(a, p->dtype);
}

extern "C" int btr_cross_attention_fwd(const btr_cross_attention_t *p, void *out, float *lse,
                                       void *workspace, size_t workspace_bytes,
                                       btr_stream_t stream) {
  XaArgs a;
  int rc = check("cross_attention_fwd", p, a);
  if (rc == BTR_OK) rc = check_grid("cross_attention_fwd", a, p->dtype, false);
  if (rc != BTR_OK) return rc;
  if (a.b == 0 || a.rows == 0) return BTR_OK;
  BTR_REQUIRE(out, "cross_attention_fwd: null pointer");
  const size_t need = fwd_bytes(a, p->dtype);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "cross_attention_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  BTR_REQUIRE(aligned16(workspace), "cross_attention_fwd: workspace off a 16-byte boundary");
  a.out = out;
  a.lse = lse;
  hipStream_t hs = as_stream(stream);
  char *ws = (char *)workspace;
  BTR_DISPATCH_DTYPE(p->dtype, pack<T>(a, false, ws, hs));
  const Shares s = row_shares(a, p->dtype, true);
  a.tiles = s.tiles; a.nsplit = s.n; a.chunk = s.chunk;
  const long long nrow = (long long)a.b * a.hk * a.rows;
  if (s.n > 1) {
    a.part = (float *)ws;
    a.part2 = (float *)(ws + align256((size_t)s.n * nrow * a.d * 4));
  }
  BTR_DISPATCH_DTYPE(p->dtype, BTR_XA_WIDTH(launch_fwd, a, hs));
  if (s.n > kFewShares)
    BTR_DISPATCH_DTYPE(p->dtype, hipLaunchKernelGGL((cross_attention_join_kernel<T>),
                                                    dim3((unsigned)nrow), dim3(256), 0, hs, a));
  else if (s.n > 1)
    BTR_DISPATCH_DTYPE(p->dtype, hipLaunchKernelGGL((cross_attention_join_few_kernel<T>),
                                                    dim3((unsigned)((nrow + 7) / 8)), dim3(256), 0,
                                                    hs, a));
  return check_launch("cross_attention_fwd");
}

extern "C" int btr_cross_attention_bwd(const btr_cross_attention_t *p, const void *out,
                                       const float *lse, const void *dout, void *dq, void *dk,
                                       void *dv, void *workspace, size_t workspace_bytes,
                                       btr_stream_t stream) {
  XaArgs a;
  int rc = check("cross_attention_bwd", p, a);
  if (rc == BTR_OK) rc = check_grid("cross_attention_bwd", a, p->dtype, true);
  if (rc != BTR_OK) return rc;
  if (a.b == 0) return BTR_OK;
  BTR_REQUIRE((a.rows == 0 || (out && lse && dout && dq)) && (a.lk == 0 || (dk && dv)),
              "cross_attention_bwd: null pointer");
  a.dout = a.dout_dma = dout;
  a.gd = a.d;
  const size_t need = bwd_bytes(a, p->dtype);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "cross_attention_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  BTR_REQUIRE(aligned16(workspace), "cross_attention_bwd: workspace off a 16-byte boundary");
  a.out = const_cast<void *>(out);
  a.lse = const_cast<float *>(lse);
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.delta = (float *)workspace;
  char *at = (char *)workspace + stats_bytes(a);
  hipStream_t hs = as_stream(stream);
  BTR_DISPATCH_DTYPE(p->dtype, pack<T>(a, true, at, hs));
  float *ws = (float *)at;
  if (a.rows > 0) {
    const Shares s = row_shares(a, p->dtype, false);
    XaArgs q = a;
    q.tiles = s.tiles; q.nsplit = s.n; q.chunk = s.chunk; q.part = ws;
    BTR_DISPATCH_DTYPE(p->dtype, BTR_XA_WIDTH(launch_bwd_q, q, hs));
    if (s.n > 1) {
      const long long n = (long long)a.b * a.hk * a.rows * a.d;
      BTR_DISPATCH_DTYPE(p->dtype, launch_sum<T, true>(q, n, (T *)dq, (T *)nullptr, hs));
    }
  }
  if (a.lk > 0) {
    const Shares s = key_shares(a);
    XaArgs k = a;
    const long long n = (long long)a.b * a.lk * a.hk * a.d;
    k.tiles = s.tiles; k.nsplit = s.n; k.chunk = s.chunk; k.part = ws;
    k.part2 = (float *)((char *)ws + align256((size_t)s.n * n * 4));
    BTR_DISPATCH_DTYPE(p->dtype, BTR_XA_WIDTH(launch_bwd_kv, k, hs));
    if (s.n > 1)
      BTR_DISPATCH_DTYPE(p->dtype, launch_sum<T, false>(k, n, (T *)dk, (T *)dv, hs));
  }
  return check_launch("cross_attention_bwd");
}
