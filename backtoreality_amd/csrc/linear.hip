// linear.hip -- a linear layer with its epilogue, forward and backward:
//
//   z = x W^T + bias,  y = act(z) [+ residual],   act = identity, ReLU, GELU (z Phi(z), erf form)
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = colsum(dz),  dresidual = dy
//
// x (m, k), W (n, k) as in torch.nn.Linear; float32, bfloat16, float16; any sizes and row strides.
// (reference: linear1 / linear2 and the projections of detection/GroupFree3D/models/
// transformer.py:36-76; csrc/sa_mlp.hip has the float32 GEMMs with BatchNorm around them.)
//
// The three products differ in whether the reduction runs along a row of the operand (x, W forward,
// dz for dx) or across its rows (W for dx; dz and x for dW).  Both kinds are staged the way memory
// has them and the second is read out of LDS with gfx950's transpose read, so nothing is ever
// transposed in memory.  Operands go to LDS by DMA (linear_dma_kernel); 16-bit rows that do not lie
// on 16-byte boundaries in whole 16-byte units are first copied to rows that do, in the workspace,
// f32 ones are split into three bf16 planes there.  Few rows (single tokens) or few outputs read the
// long operand once, straight into the matrix instructions (linear_rows_kernel).
//
// Numbers: every product accumulates in f32 and the epilogue works on the f32 sums; y is rounded
// once.  f32 operands are split into three bf16 terms (8 + 8 + 8 bits: exact up to the 24th) and
// multiplied as the six products above 2^-24, the smallest first, as one reduction six times as
// long, which the bf16 matrix pipe does 2.7 times faster than the f32 instructions do one; an
// infinite f32 element makes the sums it enters NaN, and one below 2^-108 has fewer bits (its last term
// is below 2^-126, the second from 2^-117).  What the backward needs of the activation is
// its slope act'(z), taken from the f32 sum in the forward's epilogue and kept in as many bits as x
// has: for GELU's of 16 bits a fixed-point number, off by 2^-16 at most (a bf16 slope, off by 2^-9 of
// itself, was a third of the gradients' error), and a floating-point one for the small slopes of the
// negative tail, off by 2^-10 of itself down to 2^-30, below which it is 0 (z < -6.6).  dz is rounded to
// the type of x before the two products that read it (dbias is summed from the f32 values); a float16
// GELU's, which its slopes push towards the type's smallest numbers, as dz times the power of two that
// fits the largest |dy|.
#include <algorithm>
#include <cstdint>

#include "decoder_ops.hpp"
#include "lds_dma.hpp"

#pragma clang fp contract(fast)

namespace btr {
namespace {

enum { kActNone = BTR_ACT_NONE, kActRelu = BTR_ACT_RELU, kActGelu = BTR_ACT_GELU };

// C (m, n) = A B^T over k.  TA / TB false: A[i * lda + kk]; true: A[kk * lda + i].
struct GemmArgs {
  int m, n, k;
  const void *a, *b;
  long long lda, ldb;
  const void *bias, *res;
  long long ldres;
  int act;
  void *c, *slope;           // contiguous (m, n); slope: act' of the sums (Slope), or NULL
  float *part;               // split reduction: (nsplit, m, n) partial sums
  int nsplit, chunk;         // shares of k, their length
  const float *unscale;      // float16: factor of the sums, or NULL (1)
  long long aplane, bplane;  // f32: elements from one bf16 plane of an operand to the next
  int mt, nt;                // tiles
};

template <typename T>
constexpr bool kHalf = false;
template <>
constexpr bool kHalf<_Float16> = true;

// what the matrix instructions eat: T itself, or three bf16 planes of f32
template <typename T>
struct Op {
  static constexpr int P = 1;
  typedef typename Elem<T>::Vec Frag;
};
template <>
struct Op<float> {
  static constexpr int P = 3;
  typedef bf16x8_t Frag;
};

template <typename T>
struct Matrix {
  typedef T E;
};
template <>
struct Matrix<float> {
  typedef __bf16 E;
};

__device__ __forceinline__ f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

constexpr float kBf16End = 0x1.ffp127f;   // from here on bf16 rounds to infinity
// f = h + m + l.  FAR, where an element is above bf16's largest value: its h is cut instead of rounded
// (rounded it would be infinite), and an infinite element keeps no rest.
template <bool FAR>
__device__ __forceinline__ void split3(f32x4_t f, bf16x4_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float size = __builtin_fabsf(f[i]);
    __bf16 h = (__bf16)f[i];
    if (FAR && size >= kBf16End && size < INFINITY)
      h = __builtin_bit_cast(__bf16, (unsigned short)(__float_as_uint(f[i]) >> 16));
    float r = f[i] - (float)h;
    if (FAR && size == INFINITY) r = 0.f;
    const __bf16 m = (__bf16)r;
    p[0][i] = h;
    p[1][i] = m;
    p[2][i] = (__bf16)(r - (float)m);
  }
}

__device__ __forceinline__ f32x4_t mfma16(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mfma16(f16x8_t a, f16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// eight consecutive elements -> fragments
template <typename V>
__device__ __forceinline__ void pack(const V (&v)[1], V (&f)[1]) { f[0] = v[0]; }
__device__ __forceinline__ void pack(const f32x4_t (&v)[2], bf16x8_t (&f)[3]) {
  bf16x4_t a[3], b[3];
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    top = fmaxf(fmaxf(top, __builtin_fabsf(v[0][i])), __builtin_fabsf(v[1][i]));
  if (__builtin_expect(__ballot(top >= kBf16End) != 0, 0)) {   // (per element: 33 -> 39 us at 32 x 4 096
    split3<true>(v[0], a);                                      // x 4 096)
    split3<true>(v[1], b);
  } else {
    split3<false>(v[0], a);
    split3<false>(v[1], b);
  }
#pragma unroll
  for (int p = 0; p < 3; ++p)
    f[p] = __builtin_shufflevector(a[p], b[p], 0, 1, 2, 3, 4, 5, 6, 7);
}

// GELU and its slope through the normal distribution's tail h = Phi(-|z|) and density phi:
//   z Phi(z) = max(z, 0) - |z| h,     (z Phi(z))' = [z > 0] + sign(z) (|z| phi(z) - h)
// (no cancellation: h is small where the rest is).  erfcx(x) = e^(x^2) erfc(x) is smooth -- t P(t)
// with t = 1 / (1 + c x) and polynomials P fitted here by reweighted least squares (Lawson) -- and h
// = e^(-z^2 / 2) erfcx(|z| / sqrt 2) / 2 keeps its relative error in the tail; phi shares the
// exponential.
// f32: degree 9 on x <= 14, 4e-8; the exponential's argument is rounded to 2^-24 of up to 100, which
// is added back to first order.  16 bits: degree 5 on x <= 9.5, 4e-5 (half an ulp is 5e-4 or more),
// no corrections: the 67 M elements of 16 384 x 4 096 are 20 us of a full chip's VALU per 10
// instructions.  |z| is cut at 30, where h and phi are 0, so that infinities meet no 0 times inf; NaN
// comes through the exponential.
template <bool F32>
__device__ __forceinline__ float gelu(float z, float &slope) {
  const float q = z * z, az = fminf(__builtin_fabsf(z), 30.f);
  float e, h;
  if (F32) {
    const float qe = fmaf(z, z, -q);
    const float a = q * -0.72134752044448170f, ae = fmaf(q, -0.72134752044448170f, -a);
    e = __builtin_amdgcn_exp2f(a);
    e = fmaf(e, fmaf(ae, 0.69314718055994531f, qe * -0.5f), e);
    if (!(q < 200.f)) e = q >= 200.f ? 0.f : q;  // (e is 0 from there on; NaN stays)
    const float t = __builtin_amdgcn_rcpf(fmaf(0.21213203435596426f, az, 1.f));
    float p = -0.12661709327829032f;
    p = fmaf(p, t, 0.4718284843770408f);
    p = fmaf(p, t, -0.4846959475126719f);
    p = fmaf(p, t, 0.5170530040780374f);
    p = fmaf(p, t, -0.07405165572695369f);
    p = fmaf(p, t, 0.20638609117498913f);
    p = fmaf(p, t, 0.15046865829841485f);
    p = fmaf(p, t, 0.1704237449651274f);
    p = fmaf(p, t, 0.16920475194603254f);
    h = 0.5f * e * (p * t);
  } else {                                       // (coefficients halved)
    e = __builtin_amdgcn_exp2f(q * -0.72134752044448170f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.38183766184073570f, az, 1.f));
    float p = -0.08940045184499485f;
    p = fmaf(p, t, 0.18426239198220193f);
    p = fmaf(p, t, 0.09526708661515707f);
    p = fmaf(p, t, 0.15783040089614615f);
    p = fmaf(p, t, 0.15202110402571496f);
    h = e * (p * t);
  }
  const float u = fmaf(az * 0.39894228040143268f, e, -h);
  const int bits = __float_as_int(z);            // (the sign bit in both places: z = 0 either way)
  slope = (bits >= 0 ? 1.f : 0.f) + __int_as_float(__float_as_int(u) ^ (bits & (int)0x80000000));
  return fmaf(-az, h, fmaxf(z, 0.f));
}
// act(z), and act'(z) into slope.  ReLU: the result itself, in T -- a z that T rounds to zero is off, and
// NaN is on, as where the rounded result is all that is kept.
template <typename T>
__device__ __forceinline__ float activate(float z, int act, float &slope) {
  if (act == kActGelu) return gelu<sizeof(T) == 4>(z, slope);
  if (act == kActRelu) {
    const float a = z > 0.f ? z : z != z ? z : 0.f;
    slope = (float)(T)a;
    return a;
  }
  slope = 1.f;
  return z;
}

// The slope as the backward gets it: f32 itself, or 16 bits.  GELU's:
//   code 0 .. 12 799: -2^-5 < slope <= -2^-30, the float's bits from 2^-30 on, 9 of its mantissa
//   up to 64 446:     slope * 40 960 + 18 200 for all others (-0.1291 .. 1.1291; 0 comes back as 0)
//   65 535:           NaN
// (What pads a row reads as 0, against a dy of 0.)  ReLU's: 1 or 0, and the result may stand in its place:
// on where it is positive or NaN.
constexpr unsigned kTailBits = 0x80000000u | (127u - 30u) << 23, kTailCodes = 25 * 512;   // of -2^-30
constexpr float kSlopeUnit = 40960.f, kSlopeZero = 18200.f;
template <typename T>
struct Slope {
  typedef unsigned short S;
  __device__ static __forceinline__ S keep(float d, int act) {
    if (act == kActRelu) return d > 0.f || d != d ? 1 : 0;
    const unsigned tail = __float_as_uint(d) - kTailBits + (1u << 13);   // (others wrap to large ones)
    const unsigned fixed = (unsigned)fminf(fmaf(d, kSlopeUnit, kSlopeZero + 0.5f), 65535.f);   // (NaN too)
    return (S)(tail < kTailCodes << 14 ? tail >> 14 : fixed);
  }
  __device__ static __forceinline__ float times(T dy, S v, int act) {   // dy act'
    constexpr int inf = kHalf<T> ? 0x7c00 : 0x7f80;
    if (act == kActRelu)                         // (an infinite dy stays out of it)
      return (short)v > 0 || (v & 0x7fff) > inf ? (float)dy : 0.f;
    float d = ((float)v - kSlopeZero) * (1.f / kSlopeUnit);
    if (v < kTailCodes) d = __uint_as_float(kTailBits + ((unsigned)v << 14));
    return (float)dy * (v != 0xffff ? d : __builtin_nanf(""));
  }
};
template <>
struct Slope<float> {
  typedef float S;
  __device__ static __forceinline__ S keep(float d, int) { return d; }
  __device__ static __forceinline__ float times(float dy, S v, int act) {
    if (act == kActRelu) return v > 0.f || v != v ? dy : 0.f;
    return dy * v;
  }
};

template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec bias_at(const GemmArgs &g, int col) {
  return g.bias ? load_row((const T *)g.bias, col, g.n) : typename Elem<T>::Vec{};
}
template <typename T>
__device__ __forceinline__ typename Elem<T>::Vec res_at(const GemmArgs &g, long long row, int col) {
  return g.res ? load_row((const T *)g.res + row * g.ldres, col, g.n) : typename Elem<T>::Vec{};
}
// V consecutive columns of one row: bias, activation, residual, one rounding
template <typename T>
__device__ __forceinline__ void epilogue(const GemmArgs &g, long long row, int col,
                                         const float (&s)[Elem<T>::kVec],
                                         typename Elem<T>::Vec bias, typename Elem<T>::Vec res) {
  constexpr int V = Elem<T>::kVec;
  typename Elem<T>::Vec y;
  typename Elem<typename Slope<T>::S>::Vec slope;
  float u = 1.f;
  if (kHalf<T> && g.unscale) u = *g.unscale;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float d;
    const float sum = kHalf<T> ? s[j] * u : s[j];
    y[j] = (T)(activate<T>(sum + (float)bias[j], g.act, d) + (float)res[j]);
    slope[j] = Slope<T>::keep(d, g.act);
  }
  if (g.slope) store_row((typename Slope<T>::S *)g.slope + row * g.n, col, g.n, slope);
  store_row((T *)g.c + row * g.n, col, g.n, y);
}

// workgroup -> tile and share.  Workgroups land on the eight XCDs in turn: each XCD gets a
// contiguous eighth of the tiles, and walks them in columns of eight row tiles, so that what its L2
// holds is read several times
template <int BM, int BN>
__device__ __forceinline__ void place(const GemmArgs &g, int &m0, int &n0, int &split) {
  const int total = gridDim.x, id = blockIdx.x, per = total / 8;
  int t = id < per * 8 ? (id & 7) * per + (id >> 3) : id;
  split = t / (g.mt * g.nt);
  t -= split * (g.mt * g.nt);
  const int band = t / (8 * g.nt), in = t - band * 8 * g.nt, bh = min(8, g.mt - band * 8);
  m0 = (band * 8 + in % bh) * BM;
  n0 = (in / bh) * BN;
}

// A wave's IM x IN accumulators leave through LDS, 32 rows at a time, as 16-byte row pieces.  A lane's
// pieces all lie in the same columns: their bias is read once, and a slab's residuals before its
// sums go through LDS (read piece by piece they cost a memory round trip each: 21 us a tile).
template <typename T, int IM, int IN>
__device__ __forceinline__ void leave(const GemmArgs &g, const f32x16_t (&acc)[IM][IN], float *slab,
                                      int row0, int col0, int split, int lane) {
  constexpr int V = Elem<T>::kVec, WN = 32 * IN, CP = WN + 4, PR = WN / V, NQ = 32 * PR / 64;
  static_assert(64 % PR == 0, "a lane keeps its columns");
  typedef typename Elem<T>::Vec Vec;
  const int col = (lane % PR) * V, gc = col0 + col;
  const bool whole = g.nsplit == 1;
  Vec bias = {}, res[NQ];
  if (whole && gc < g.n) bias = bias_at<T>(g, gc);
#pragma unroll
  for (int i = 0; i < IM; ++i) {
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int gr = row0 + 32 * i + lane / PR + 64 / PR * q;
      res[q] = Vec{};
      if (whole && gr < g.m && gc < g.n) res[q] = res_at<T>(g, gr, gc);
    }
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        slab[((v & 3) + 8 * (v >> 2) + 4 * (lane >> 5)) * CP + 32 * j + (lane & 31)] = acc[i][j][v];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      const int row = lane / PR + 64 / PR * q, gr = row0 + 32 * i + row;
      float s[V];
#pragma unroll
      for (int u = 0; u < V; u += 4) {
        const f32x4_t t = *reinterpret_cast<const f32x4_t *>(slab + row * CP + col + u);
#pragma unroll
        for (int x = 0; x < 4; ++x) s[u + x] = t[x];
      }
      if (gr < g.m && gc < g.n) {
        if (whole) {
          epilogue<T>(g, gr, gc, s, bias, res[q]);
        } else {
          float *dst = g.part + ((long long)split * g.m + gr) * g.n;
#pragma unroll
          for (int u = 0; u < V; u += 4)
            store_row(dst, gc + u, g.n, f32x4_t{s[u], s[u + 1], s[u + 2], s[u + 3]});
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// R rows (m / n axis) x 32 reduction steps of a 16-bit operand in LDS.  TR false: [R][32]; true:
// [32][R] in blocks of 128 (or 64) columns.
constexpr int kStep = 32;
template <typename T, bool TR, int R, int THREADS>
struct DmaPanel {
  static constexpr int D = TR ? (R >= 128 ? 128 : 64) : kStep;
  typedef Dma<D> DM;
  static constexpr int BLOCK = kStep * DM::PITCH, BYTES = R * kStep * 2;
  static constexpr int N = BYTES / 16 / THREADS;   // 16-byte units a thread moves
  int off[N];                                      // byte offsets from the step's first element
  // k position of unit i inside a step (its row / its column)
  __device__ static __forceinline__ int kpos(int i, int tid) {
    const int e = i * THREADS + tid;
    if (TR) return e % (BLOCK / 16) / DM::UNITS;
    return ((e % DM::UNITS) ^ DM::swz(e / DM::UNITS)) * 8;
  }
  __device__ __forceinline__ void init(long long ld, int r0, int rmax, int tid) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = i * THREADS + tid;
      if (TR) {
        const int blk = e / (BLOCK / 16), row = e % (BLOCK / 16) / DM::UNITS;
        const int col = blk * D + ((e % DM::UNITS) ^ DM::swz(row)) * 8;
        off[i] = r0 + col < rmax ? (row * (int)ld + col) * 2 : kFar;
      } else {
        const int row = e / DM::UNITS;
        off[i] = r0 + row < rmax ? row * (int)ld * 2 + kpos(i, tid) * 2 : kFar;
      }
    }
  }
  // the descriptor of the step at reduction index k0 (src: the operand's first row / column added)
  __device__ static __forceinline__ i32x4_t rsrc(const T *src, long long ld, int k0) {
    return dma_rsrc((const char *)(src + (TR ? k0 * ld : (long long)k0)), kFar);
  }
  // unit i of a step that has `left` reduction steps (none: zeros); wave: tid / 64, uniform
  __device__ __forceinline__ void issue(i32x4_t rs, int i, int left, char *lds, int tid,
                                        int wave) const {
    dma16(rs, kpos(i, tid) < left ? off[i] : kFar, lds + (i * THREADS + wave * 64) * 16);
  }
  // fragment: 32 rows at r0 (a multiple of 32), reduction steps 16 ks .. + 15; base: row_base / nat_base
  __device__ static __forceinline__ int base(int lane) {
    return TR ? DM::nat_base(lane) : DM::row_base(lane & 31, lane >> 5);
  }
  __device__ static __forceinline__ typename Elem<T>::Vec frag(const char *lds, int base, int r0,
                                                               int ks) {
    if constexpr (!TR) {
      return *reinterpret_cast<const typename Elem<T>::Vec *>(lds + r0 * DM::PITCH +
                                                              (base ^ (ks << 5)));
    } else {
      union {
        s16x4_t s[2];
        typename Elem<T>::Vec f;
      } u;
      const char *t = lds + r0 / D * BLOCK + 16 * ks * DM::PITCH;
      const int at = base ^ (r0 % D / 32 << 6);
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(t + at));
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (lds_s16x4)(t + (at ^ DM::kNatHi) + 4 * DM::PITCH));
      return u.f;
    }
  }
};

// 16 bits: BM x BN tile by GM x GN waves, 32 reduction steps at a time through a ring of NBUF tile
// pairs that DMA fills NBUF - 1 steps ahead, always: steps past the end are filled with zeros, so that
// the number of instructions in flight is a constant.  A group of 16 steps' fragments is read during
// the products of the group before.  The one barrier of a step stands in front of its SECOND group's
// products: every wave has then read all of this step's tiles (which are refilled during those
// products) and the next step's have landed (its first fragments are read during them as well).
// LDS reads and DMA instructions go out one between two products (in front of them they cost the
// matrix pipe their own issue time), and a wave among its products goes before one that has still
// to reach the barrier (s_setprio: 1 060 -> 1 170 TFLOP/s at 16 384 x 4 096 x 1 024 bf16).  The same
// loop with neither DMA nor LDS reads runs at 1 450 TFLOP/s, which is the clock's doing; the DMA
// costs 20 %, the reads 10 %.  256 x 256 tiles, a ring of four and one workgroup per CU for large
// products; 256 x 128 with a ring of three fits a CU twice and wins only where the large tile leaves
// CUs idle (8 192 x 4 096 x 1 024: 98 -> 79 us).
// f32 (T): the operands are bf16 planes (E), the reduction runs six times over k with the planes of
// kPlanes.
constexpr unsigned kPlanesA = 0x001102, kPlanesB = 0x010120;   // digit i: plane of the i-th pass
template <typename T, bool TA, bool TB, int BM, int BN, int GM, int GN, int NBUF, int OCC>
__global__ __launch_bounds__(64 * GM * GN, OCC) void linear_dma_kernel(GemmArgs g) {
  typedef typename Matrix<T>::E E;
  constexpr int THREADS = 64 * GM * GN, WM = BM / GM, WN = BN / GN, IM = WM / 32, IN = WN / 32;
  typedef DmaPanel<E, TA, BM, THREADS> PA;
  typedef DmaPanel<E, TB, BN, THREADS> PB;
  typedef typename Elem<E>::Vec Vec;
  constexpr int TILE = PA::BYTES + PB::BYTES, SLAB = GM * GN * 32 * (WN + 4) * 4;
  constexpr int NDMA = PA::N + PB::N;              // instructions a wave issues per step
  constexpr int NF = IM + IN, NP = IM * IN;        // fragments and products of a group
  constexpr int LQ = (NF + NP - 1) / NP, DQ = (NDMA + NP - 1) / NP;   // between two products, at most
  constexpr int PASSES = sizeof(T) == 4 ? 6 : 1;
  __shared__ __attribute__((aligned(1024))) char smem[NBUF * TILE > SLAB ? NBUF * TILE : SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int m0, n0, split;
  place<BM, BN>(g, m0, n0, split);
  const int kbeg = split * g.chunk, kend = min(g.k, kbeg + g.chunk);
  const int nk = kend > kbeg ? (kend - kbeg + kStep - 1) / kStep : 0, steps = nk * PASSES;
  const int wm = w / GN * WM, wn = w % GN * WN;
  const E *ap = (const E *)g.a + (TA ? (long long)m0 : m0 * g.lda);
  const E *bp = (const E *)g.b + (TB ? (long long)n0 : n0 * g.ldb);
  PA pa;
  PB pb;
  pa.init(g.lda, m0, g.m, tid);
  pb.init(g.ldb, n0, g.n, tid);
  const int ab = PA::base(lane), bb = PB::base(lane);

  f32x16_t acc[IM][IN] = {};
  Vec fa[2][IM], fb[2][IN];
  auto load = [&](int buf, int ks, int i) {        // fragment i of a group
    const char *la = smem + buf * TILE, *lb = la + PA::BYTES;
    if (i < IM) fa[ks][i] = PA::frag(la, ab, wm + 32 * i, ks);
    else fb[ks][i - IM] = PB::frag(lb, bb, wn + 32 * (i - IM), ks);
  };
  i32x4_t ra, rb;
  int ik = 0, pass = 0;                            // the next step to be asked for
  auto issue = [&](int buf, int i) {               // DMA instruction i of it
    char *la = smem + buf * TILE;
    const int k0 = kbeg + ik * kStep, left = pass < PASSES ? kend - k0 : 0;
    if (i == 0)
      ra = PA::rsrc(ap + (PASSES > 1 ? (kPlanesA >> (4 * pass) & 15) * g.aplane : 0), g.lda, k0);
    if (i == PA::N)
      rb = PB::rsrc(bp + (PASSES > 1 ? (kPlanesB >> (4 * pass) & 15) * g.bplane : 0), g.ldb, k0);
    if (i < PA::N) pa.issue(ra, i, left, la, tid, w);
    else pb.issue(rb, i - PA::N, left, la + PA::BYTES, tid, w);
    if (i == NDMA - 1 && ++ik >= nk) {
      ik = 0;
      ++pass;
    }
  };
  if (steps) {
#pragma unroll
    for (int t = 0; t < NBUF - 1; ++t)
#pragma unroll
      for (int i = 0; i < NDMA; ++i) issue(t, i);
    dma_wait<(NBUF - 2) * NDMA>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NDMA; ++i) issue(NBUF - 1, i);
#pragma unroll
    for (int i = 0; i < NF; ++i) load(0, 0, i);
  }
  int buf = 0;
  for (int step = 0; step < steps; ++step) {
    const int next = buf + 1 == NBUF ? 0 : buf + 1;
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      if (q == 0) __builtin_amdgcn_s_setprio(1);
      acc[q / IN][q % IN] = mfma(fa[0][q / IN], fb[0][q % IN], acc[q / IN][q % IN]);
#pragma unroll
      for (int i = q * LQ; i < NF && i < (q + 1) * LQ; ++i) load(buf, 1, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    dma_wait<(NBUF - 2) * NDMA>();
    lds_barrier();
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      if (q == 0) __builtin_amdgcn_s_setprio(1);
      acc[q / IN][q % IN] = mfma(fa[1][q / IN], fb[1][q % IN], acc[q / IN][q % IN]);
#pragma unroll
      for (int i = q * LQ; i < NF && i < (q + 1) * LQ; ++i) load(next, 0, i);
#pragma unroll
      for (int i = q * DQ; i < NDMA && i < (q + 1) * DQ; ++i) issue(buf, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    buf = next;
  }
  dma_wait();
  __syncthreads();
  leave<T, IM, IN>(g, acc, reinterpret_cast<float *>(smem) + w * 32 * (WN + 4), m0 + wm, n0 + wn,
                   split, lane);
}

// Small products: a 64 x 64 tile whose reduction steps the four waves deal out among themselves (wave
// w: steps w, w + 4, ..), each through two tile pairs of its own, without a barrier until their sums
// meet in LDS.  A product of few tiles is bound by the latency of its chain of steps: with the tile
// cut into 32 x 32 per wave (one product between two LDS round trips and a barrier) a step took 0.45
// us, here a wave's step is eight products behind one round trip and four run at once.  (Rings of
// four fit a CU once: 1 024 x 2 048 outputs, 128 / 1 024 steps 9.9 / 14.6 us against 6.9 / 12.1.)
// 1 999 x 1 301 x 775 f16: 20.6 us, 195 TFLOP/s, 2.6 rounds of workgroups of 13 steps.
template <typename T, bool TA, bool TB>
__global__ __launch_bounds__(256) void linear_stream_kernel(GemmArgs g) {
  typedef typename Matrix<T>::E E;
  typedef DmaPanel<E, TA, 64, 64> PA;
  typedef DmaPanel<E, TB, 64, 64> PB;
  typedef typename Elem<E>::Vec Vec;
  constexpr int TILE = PA::BYTES + PB::BYTES, NDMA = PA::N + PB::N, CP = 64 + 4;
  constexpr int PASSES = sizeof(T) == 4 ? 6 : 1, SUMS = 4 * 64 * CP * 4;
  __shared__ __attribute__((aligned(1024))) char smem[8 * TILE > SUMS ? 8 * TILE : SUMS];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int m0, n0, split;
  place<64, 64>(g, m0, n0, split);
  const int kbeg = split * g.chunk, kend = min(g.k, kbeg + g.chunk);
  const int nk = kend > kbeg ? (kend - kbeg + kStep - 1) / kStep : 0, steps = nk * PASSES;
  const E *ap = (const E *)g.a + (TA ? (long long)m0 : m0 * g.lda);
  const E *bp = (const E *)g.b + (TB ? (long long)n0 : n0 * g.ldb);
  PA pa;
  PB pb;
  pa.init(g.lda, m0, g.m, lane);
  pb.init(g.ldb, n0, g.n, lane);
  const int ab = PA::base(lane), bb = PB::base(lane);
  char *ring = smem + w * 2 * TILE;

  f32x16_t acc[2][2] = {};
  int ik = w, pass = 0;                            // the next step to be asked for
  while (nk && ik >= nk && pass < PASSES) {
    ik -= nk;
    ++pass;
  }
  auto issue = [&](int buf) {
    char *la = ring + buf * TILE;
    const int k0 = kbeg + ik * kStep, left = pass < PASSES ? kend - k0 : 0;
    const i32x4_t ra =
        PA::rsrc(ap + (PASSES > 1 ? (kPlanesA >> (4 * pass) & 15) * g.aplane : 0), g.lda, k0);
    const i32x4_t rb =
        PB::rsrc(bp + (PASSES > 1 ? (kPlanesB >> (4 * pass) & 15) * g.bplane : 0), g.ldb, k0);
#pragma unroll
    for (int i = 0; i < PA::N; ++i) pa.issue(ra, i, left, la, lane, 0);
#pragma unroll
    for (int i = 0; i < PB::N; ++i) pb.issue(rb, i, left, la + PA::BYTES, lane, 0);
    ik += 4;
    while (ik >= nk && pass < PASSES) {
      ik -= nk;
      ++pass;
    }
  };
  if (w < steps)
    for (int t = 0; t < 2; ++t) issue(t);
  int buf = 0;
  for (int step = w; step < steps; step += 4) {
    dma_wait<NDMA>();
    const char *la = ring + buf * TILE, *lb = la + PA::BYTES;
    Vec fa[2][2], fb[2][2];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        fa[ks][i] = PA::frag(la, ab, 32 * i, ks);
        fb[ks][i] = PB::frag(lb, bb, 32 * i, ks);
      }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    issue(buf);                                    // two steps on, into the pair just read
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = mfma(fa[ks][i], fb[ks][j], acc[i][j]);
    buf ^= 1;
  }
  dma_wait();
  __syncthreads();
  float *own = reinterpret_cast<float *>(smem) + w * 64 * CP;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        own[(32 * i + (v & 3) + 8 * (v >> 2) + 4 * (lane >> 5)) * CP + 32 * j + (lane & 31)] =
            acc[i][j][v];
  __syncthreads();
  constexpr int V = Elem<T>::kVec, PR = 64 / V, NQ = 64 * PR / 256;
  const int col = (tid % PR) * V, gc = n0 + col;
  if (gc >= g.n) return;
  const bool whole = g.nsplit == 1;
  typename Elem<T>::Vec bias = {}, res[NQ];
  if (whole) bias = bias_at<T>(g, gc);
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int gr = m0 + tid / PR + 256 / PR * q;
    res[q] = typename Elem<T>::Vec{};
    if (whole && gr < g.m) res[q] = res_at<T>(g, gr, gc);
  }
#pragma unroll
  for (int q = 0; q < NQ; ++q) {
    const int row = tid / PR + 256 / PR * q, gr = m0 + row;
    if (gr >= g.m) continue;
    float s[V] = {};
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int u = 0; u < V; u += 4) {
        const f32x4_t t = *reinterpret_cast<const f32x4_t *>(
            reinterpret_cast<const float *>(smem) + (k * 64 + row) * CP + col + u);
#pragma unroll
        for (int x = 0; x < 4; ++x) s[u + x] += t[x];
      }
    if (whole) {
      epilogue<T>(g, gr, gc, s, bias, res[q]);
    } else {
      float *dst = g.part + ((long long)split * g.m + gr) * g.n;
#pragma unroll
      for (int u = 0; u < V; u += 4)
        store_row(dst, gc + u, g.n, f32x4_t{s[u], s[u + 1], s[u + 2], s[u + 3]});
    }
  }
}

// Few rows of x (up to 16 MT): a workgroup's eight waves share 16 rows of W and split the reduction
// (wave w: the steps of 32 numbered w, w + 8, ..), W goes from memory into the matrix instructions,
// the eight sums meet in LDS.  Bound by the bytes of W: eight loads of 1 KB in flight a wave (1 row x
// 4 096 x 4 096 bf16: 9.4 us; its bytes are 6.8 at a large copy's rate).
// COLS: the roles the other way round -- few outputs (up to 16 MT), 16 rows of x a workgroup, x read
// once where it is.
template <typename T, int MT, bool COLS>
__global__ __launch_bounds__(512) void linear_rows_kernel(GemmArgs g) {
  constexpr int P = Op<T>::P, U = sizeof(T) == 4 ? 4 : 8;
  __shared__ float part[8][MT][16][20];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l15 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  f32x4_t acc[MT] = {};
  const int many = COLS ? g.m : g.n, few = COLS ? g.n : g.m;
  const long long ldm = COLS ? g.lda : g.ldb, ldf = COLS ? g.ldb : g.lda;
  const T *wrow = (const T *)(COLS ? g.a : g.b) + min(n0 + l15, many - 1) * ldm;
  const T *xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xrow[t] = (const T *)(COLS ? g.b : g.a) + min(16 * t + l15, few - 1) * ldf;
  // U steps of 32 at a time, their loads together
  for (int s0 = w * U * 32; s0 < g.k; s0 += 8 * U * 32) {
    typename Elem<T>::Vec wv[U][sizeof(T) / 2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int h = 0; h < (int)sizeof(T) / 2; ++h)
        wv[u][h] = load_row(wrow, s0 + 32 * u + 8 * q + 4 * h, g.k);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      typename Op<T>::Frag fw[P], fx[P];
      pack(wv[u], fw);
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        typename Elem<T>::Vec xv[sizeof(T) / 2];
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h)
          xv[h] = load_row(xrow[t], s0 + 32 * u + 8 * q + 4 * h, g.k);
        pack(xv, fx);
        if constexpr (P == 3) {
          acc[t] = mfma16(fw[2], fx[0], acc[t]);
          acc[t] = mfma16(fw[0], fx[2], acc[t]);
          acc[t] = mfma16(fw[1], fx[1], acc[t]);
          acc[t] = mfma16(fw[1], fx[0], acc[t]);
          acc[t] = mfma16(fw[0], fx[1], acc[t]);
        }
        acc[t] = mfma16(fw[0], fx[0], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)                     // [of the few][of the 16]
    *reinterpret_cast<f32x4_t *>(&part[w][t][l15][4 * q]) = acc[t];
  __syncthreads();
  // 16 outputs of a row in pieces of V columns
  constexpr int V = Elem<T>::kVec;
  if constexpr (COLS) {
    constexpr int PC = MT * 16 / V;
    for (int e = tid; e < 16 * PC; e += 512) {
      const int row = e / PC, col = (e % PC) * V;
      if (n0 + row >= g.m || col >= g.n) continue;
      float s[V] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int u = 0; u < V; ++u) s[u] += part[k][col >> 4][(col & 15) + u][row];
      epilogue<T>(g, n0 + row, col, s, bias_at<T>(g, col), res_at<T>(g, n0 + row, col));
    }
    return;
  }
  constexpr int PR = 16 / V;
  for (int e = tid; e < MT * 16 * PR; e += 512) {
    const int row = e / PR, col = (e % PR) * V;
    if (row >= g.m || n0 + col >= g.n) continue;
    float s[V] = {};
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int u = 0; u < V; ++u) s[u] += part[k][row >> 4][row & 15][col + u];
    epilogue<T>(g, row, n0 + col, s, bias_at<T>(g, n0 + col), res_at<T>(g, row, n0 + col));
  }
}

// Rows of up to two operands (blockIdx.y) -> rows of ldd elements on 16-byte boundaries, zeros behind
// them; f32: three bf16 planes of such rows
struct PackArgs {
  struct One {
    long long rows, ld, plane;
    int cols, ldd;
    const void *src;
    void *dst;
  } op[2];
};
template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(PackArgs a) {
  typedef typename Op<T>::Frag Frag;
  constexpr int V = Elem<T>::kVec, H = 8 / V;
  const PackArgs::One o = a.op[blockIdx.y];
  const int units = o.ldd / 8;
  const long long total = o.rows * units;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total;
       e += (long long)gridDim.x * 256) {
    const long long row = e / units;
    const int col = (int)(e - row * units) * 8;
    typename Elem<T>::Vec v[H];
#pragma unroll
    for (int h = 0; h < H; ++h) v[h] = load_row((const T *)o.src + row * o.ld, col + h * V, o.cols);
    Frag p[Op<T>::P];
    pack(v, p);
#pragma unroll
    for (int i = 0; i < Op<T>::P; ++i)
      *reinterpret_cast<Frag *>((typename Matrix<T>::E *)o.dst + i * o.plane + row * o.ldd + col) = p[i];
  }
}

// adds the shares of the reduction in order, then the epilogue (bound by memory: four shares of 4 096
// x 1 024 sums 13.5 us, 5.6 TB/s)
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(GemmArgs g) {
  constexpr int V = Elem<T>::kVec;
  const int per_row = (g.n + V - 1) / V;
  const long long pieces = (long long)g.m * per_row;
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < pieces;
       e += (long long)gridDim.x * 256) {
    const long long row = e / per_row;
    const int col = (int)(e - row * per_row) * V;
    float s[V] = {};
    for (int t = 0; t < g.nsplit; ++t) {
      const float *p = g.part + ((long long)t * g.m + row) * g.n;
#pragma unroll
      for (int u = 0; u < V; u += 4) {
        const f32x4_t q = load_row(p, col + u, g.n);
#pragma unroll
        for (int i = 0; i < 4; ++i) s[u + i] += q[i];
      }
    }
    epilogue<T>(g, row, col, s, bias_at<T>(g, col), res_at<T>(g, row, col));
  }
}

// the largest finite |dy| of each workgroup's rows (16 384 x 4 096: 38 us, 3.5 TB/s)
constexpr int kMostBlocks = 1024;
template <typename T>
__global__ __launch_bounds__(256) void linear_most_kernel(long long m, int n, const T *dy,
                                                          long long lddy, float *most) {
  constexpr int V = Elem<T>::kVec;
  __shared__ float red[4];
  const int per_row = (n + V - 1) / V, at = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  const int rows = step / per_row, pieces = step - rows * per_row;   // from one piece to the next
  long long row = at / per_row;
  int piece = at - (int)row * per_row;
  float big = 0.f;
  while (row < m) {
    typename Elem<T>::Vec g[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {                  // (four loads in flight; past the end: the last row)
      g[i] = load_row(dy + min(row, m - 1) * lddy, piece * V, n);
      row += rows;
      piece += pieces;
      if (piece >= per_row) {
        piece -= per_row;
        ++row;
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float a = fabsf((float)g[i][j]);
        big = a < INFINITY ? fmaxf(big, a) : big;
      }
  }
  for (int i = 32; i > 0; i >>= 1) big = fmaxf(big, __shfl_xor(big, i));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = big;
  __syncthreads();
  if (threadIdx.x == 0) most[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// dz = dy slope (ReLU: dy where it is on) into rows of ldz elements, zeros behind them (f32: into
// its three planes), and the column sums of dz over this workgroup's rows: 32 threads along the
// columns (8 each), 8 rows at a time.  dz NULL: the sums only.  (Bound by memory: 16 384 x 4 096 bf16
// 74 us, 5.4 TB/s.  In the products' own staging it would be recomputed per tile, 4 to 64 times.)
// most (float16, `count` of them, then the place of the factor that undoes it, or NULL): dz is written
// as 2^up dz, |dz| <= 1.13 |dy| < 2^(e + 1) as below 1.13 2^14.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(long long m, int n, const T *dy,
                                                        long long lddy, const typename Slope<T>::S *slope,
                                                        int act,
                                                        typename Matrix<T>::E *dz, int ldz,
                                                        long long plane, float *part, float *most,
                                                        int count) {
  constexpr int V = Elem<T>::kVec, H = 8 / V;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[8][32 * 8];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, col = (blockIdx.x * 32 + cl) * 8;
  float up = 1.f;
  if (kHalf<T> && most) {
    float big = 0.f;
    for (int i = threadIdx.x; i < count; i += 256) big = fmaxf(big, most[i]);
    for (int i = 32; i > 0; i >>= 1) big = fmaxf(big, __shfl_xor(big, i));
    if ((threadIdx.x & 63) == 0) red[0][threadIdx.x >> 6] = big;
    __syncthreads();
    big = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    __syncthreads();
    const int e = 14 - __builtin_amdgcn_frexp_expf(big);
    up = __builtin_ldexpf(1.f, e);
    if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0)
      most[count] = __builtin_ldexpf(1.f, -e);
  }
  float sum[8] = {};
  if (col < n)
    for (long long row = (long long)blockIdx.y * 8 + rl; row < m; row += (long long)gridDim.y * 8) {
      Vec g[H];
      typename Elem<typename Slope<T>::S>::Vec d[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        g[h] = load_row(dy + row * lddy, col + h * V, n);
        if (act != kActNone) d[h] = load_row(slope + row * n, col + h * V, n);
      }
#pragma unroll
      for (int h = 0; h < H; ++h)
#pragma unroll
        for (int j = 0; j < V; ++j) {
          float z = (float)g[h][j];
          if (act != kActNone) z = Slope<T>::times(g[h][j], d[h][j], act);
          sum[h * V + j] += z;
          g[h][j] = (T)(kHalf<T> ? z * up : z);
        }
      if (dz) {
        typename Op<T>::Frag f[Op<T>::P];
        pack(g, f);
#pragma unroll
        for (int p = 0; p < Op<T>::P; ++p)
          *reinterpret_cast<typename Op<T>::Frag *>(dz + p * plane + row * ldz + col) = f[p];
      }
    }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) red[rl][cl * 8 + j] = sum[j];
  __syncthreads();
  const int c = threadIdx.x;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) t += red[k][c];
  if (blockIdx.x * 256 + c < n) part[(long long)blockIdx.y * n + blockIdx.x * 256 + c] = t;
}

// dbias = sum of the workgroups' rows, in order
template <typename T>
__global__ __launch_bounds__(1024) void linear_dbias_kernel(const float *part, int blocks, int n,
                                                            T *db) {
  const int c = blockIdx.x * 32 + (threadIdx.x & 31);
  const float t = column_sum(part, blocks, n, c);
  if (threadIdx.x < 32 && c < n) db[c] = (T)t;
}

// --------------------------------------------------------------------------------------- host
struct Plan {
  int bm, bn, mt, nt, nsplit, chunk;
};

// Tile and shares of the reduction by estimated time: workgroups a CU gets x (64-step pieces x what
// one costs + what a workgroup costs besides), not below one workgroup's own latency, plus the
// partial sums' way through memory.  The figures are us, measured for bf16 with each tile in turn: a
// full chip at 16 384 x 4 096 x 1 024 and 16 384 x 1 024 x 4 096, one workgroup or two per CU at 1 024 x
// (32 .. 2 048) x 2 048.  f32 runs six passes over k.
Plan plan_gemm(int m, int n, int k, int passes) {
  static const struct { int bm, bn, threads; double step, fixed, alone; } kTile[4] = {
      {256, 256, 512, 1.65, 11.0, 1.06}, {256, 128, 512, 1.02, 6.7, 0.62},
      {128, 128, 256, 0.65, 5.5, 0.8}, {64, 64, 256, 0.22, 2.0, 0.2}};
  Plan best{};
  double least = 1e30;
  for (const auto &t : kTile) {
    const int mt = cdiv(m, t.bm), nt = cdiv(n, t.bn);
    const long long tiles = (long long)mt * nt;
    if (tiles * t.threads >= 1ll << 32) continue;  // (a grid's thread numbers; check(): not all tiles)
    for (int s = 1; s <= 32 && (s == 1 || (k / s * passes >= 128 && tiles * s <= 2048)); ++s) {
      const int chunk = std::max(64, cdiv(cdiv(k, s), 64) * 64), real = std::max(1, cdiv(k, chunk));
      if (real != s) continue;
      const double steps = chunk / 64 * passes;
      double us = std::max((double)((tiles * s + 255) / 256) * (steps * t.step + t.fixed),
                           steps * t.alone + t.fixed + 1.5);
      if (s > 1) us += 3.0 + (2.0 * s + 1.0) * m * n * 4.0 / 5e6;
      if (us < least) {
        least = us;
        best = Plan{t.bm, t.bn, mt, nt, s, chunk};
      }
    }
  }
  return best;
}
int passes_of(int dtype) { return dtype == BTR_F32 ? 6 : 1; }
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
size_t split_bytes(int m, int n, int k, int dtype) {
  const Plan p = plan_gemm(m, n, k, passes_of(dtype));
  return p.nsplit > 1 ? align256((size_t)p.nsplit * m * n * sizeof(float)) : 0;
}
int up8(int v) { return (v + 7) & ~7; }
// rows a DMA may read where they are: 16 bits, whole 16-byte units on 16-byte boundaries, a tile's
// offsets below 2^31
bool dma_rows(int dtype, const void *p, long long ld, int len) {
  return dtype != BTR_F32 && ((uintptr_t)p & 15) == 0 && len % 8 == 0 && ld % 8 == 0 &&
         ld <= (1 << 22);
}
// one plane of packed rows in elements, and the bytes of all
long long plane_of(long long rows, int len) { return (long long)(align256((size_t)rows * up8(len) * 2) / 2); }
size_t packed_bytes(int dtype, long long rows, int len) {
  return (size_t)plane_of(rows, len) * 2 * (dtype == BTR_F32 ? 3 : 1);
}
size_t pack_bytes(int dtype, const void *p, long long ld, long long rows, int len) {
  return dma_rows(dtype, p, ld, len) ? 0 : packed_bytes(dtype, rows, len);
}
constexpr int kFewRows = 16;       // linear_rows_kernel up to here, whatever the rest
// workgroups along the rows of the dz / dbias pass
int dz_blocks(long long m, int n) {
  const long long cols = cdiv(n, 256);
  return (int)std::max<long long>(1, std::min<long long>((m + 31) / 32, (1024 + cols - 1) / cols));
}

// operands as the DMA kernel wants them: where they are, or packed / split into ws (which moves on),
// one launch for both
struct Rows {
  const void *p;
  long long ld, plane, rows;
  int len;
};
template <typename T>
void pack_rows(Rows *r, int count, char *&ws, hipStream_t hs) {
  constexpr int dtype = sizeof(T) == 4 ? BTR_F32 : BTR_BF16;
  PackArgs a{};
  long long most = 0;
  int n = 0;
  for (int i = 0; i < count; ++i) {
    if (dma_rows(dtype, r[i].p, r[i].ld, r[i].len)) continue;
    const int ldd = up8(r[i].len);
    const long long plane = plane_of(r[i].rows, r[i].len);
    a.op[n++] = PackArgs::One{r[i].rows, r[i].ld, plane, r[i].len, ldd, r[i].p, ws};
    most = std::max(most, r[i].rows * (ldd / 8));
    r[i].p = ws;
    r[i].ld = ldd;
    r[i].plane = plane;
    ws += packed_bytes(dtype, r[i].rows, r[i].len);
  }
  if (n)
    hipLaunchKernelGGL((linear_pack_kernel<T>),
                       dim3((unsigned)std::min<long long>(4096, (most + 255) / 256), n), dim3(256), 0,
                       hs, a);
}

template <typename T, bool TA, bool TB>
void launch_gemm(GemmArgs g, Rows a, Rows b, void *ws, hipStream_t hs) {
  const Plan p = plan_gemm(g.m, g.n, g.k, sizeof(T) == 4 ? 6 : 1);
  g.a = a.p; g.lda = a.ld; g.aplane = a.plane;
  g.b = b.p; g.ldb = b.ld; g.bplane = b.plane;
  g.mt = p.mt; g.nt = p.nt; g.nsplit = p.nsplit; g.chunk = p.chunk; g.part = (float *)ws;
  const dim3 grid((unsigned)((long long)p.mt * p.nt * p.nsplit));
  if (p.bm == 256 && p.bn == 256)
    hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 256, 256, 2, 4, 4, 2>), grid, dim3(512), 0, hs, g);
  else if (p.bm == 256)
    hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 256, 128, 4, 2, 3, 4>), grid, dim3(512), 0, hs, g);
  else if (p.bm == 128)
    hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 128, 128, 2, 2, 4, 2>), grid, dim3(256), 0, hs, g);
  else
    hipLaunchKernelGGL((linear_stream_kernel<T, TA, TB>), grid, dim3(256), 0, hs, g);
  if (p.nsplit > 1) {
    const long long pieces = (long long)g.m * cdiv(g.n, Elem<T>::kVec);
    hipLaunchKernelGGL((linear_join_kernel<T>),
                       dim3((unsigned)std::min<long long>(4096, (pieces + 255) / 256)), dim3(256), 0,
                       hs, g);
  }
}

int check(const char *what, const btr_linear_t *p) {
  BTR_REQUIRE(p, "%s: null description", what);
  BTR_REQUIRE(p->dtype >= BTR_F32 && p->dtype <= BTR_F16, "%s: unknown element type %d", what,
              p->dtype);
  BTR_REQUIRE(p->act >= BTR_ACT_NONE && p->act <= BTR_ACT_GELU, "%s: unknown activation %d", what,
              p->act);
  const int m = p->m, n = p->n, k = p->k;
  BTR_REQUIRE(m >= 0 && n >= 1 && k >= 1 && m <= (1 << 30) && n <= (1 << 22) && k <= (1 << 22) &&
                  ((long long)cdiv(m, 256) * cdiv(n, 256) <= (1 << 22)) &&
                  ((long long)cdiv(m, 256) * cdiv(k, 256) <= (1 << 22)) &&
                  ((long long)cdiv(n, 256) * cdiv(k, 256) <= (1 << 22)),
              "%s: (%d, %d) x (%d, %d)", what, m, k, n, k);
  BTR_REQUIRE(m == 0 || (p->x && p->weight && p->ldx >= k && p->ldw >= k &&
                         (!p->residual || p->ldr >= n)),
              "%s: null pointer or a row stride below the row", what);
  return BTR_OK;
}

// Does linear_rows_kernel take a forward product with `few` rows (or outputs) against `many` outputs
// (or rows)?  f32: up to 64, where the tiled kernels would first write three planes of the long operand
// (rows x reduction x outputs, 32 x 4 096 x 4 096: 64 -> 33 us, 64 x 4 096 x 4 096: 68 -> 50, 30 000 x
// 2 048 x 64: 274 -> 165; of what was timed only 30 000 x 128 x 64 loses, 28 -> 33).  16 bits: up to 32
// while a round of workgroups covers the long side and the reduction is short (4 096 x 2 048 x 32 bf16:
// 10.6 -> 9.5, 1 024 x 288 x 23 off 16-byte boundaries 9.2 -> 6.1; beyond: 30 000 x 128 x 23 8 -> 33,
// 2 048 x 4 096 x 32 12 -> 15).
bool few_of(int dtype, int few, int many, int k) {
  return dtype == BTR_F32 ? few <= 64 : few <= 32 && many <= 4096 && k <= 2048;
}
bool few_rows(const btr_linear_t &p) { return p.m <= kFewRows || few_of(p.dtype, p.m, p.n, p.k); }
bool few_columns(const btr_linear_t &p) { return few_of(p.dtype, p.n, p.m, p.k); }
template <typename T, bool COLS>
void launch_rows(const GemmArgs &g, int few, int many, hipStream_t hs) {
  const dim3 grid(cdiv(many, 16));
  if (few <= 16) {
    hipLaunchKernelGGL((linear_rows_kernel<T, 1, COLS>), grid, dim3(512), 0, hs, g);
  } else if (few <= 32) {
    hipLaunchKernelGGL((linear_rows_kernel<T, 2, COLS>), grid, dim3(512), 0, hs, g);
  } else {
    if constexpr (sizeof(T) == 4)
      hipLaunchKernelGGL((linear_rows_kernel<T, 4, COLS>), grid, dim3(512), 0, hs, g);
  }
}
// few outputs: as many rows a launch as a grid of 32-bit thread numbers has room for
template <typename T>
void launch_columns(GemmArgs g, hipStream_t hs) {
  constexpr int kRows = 1 << 26;                   // 2^31 threads
  const int m = g.m, n = g.n;
  for (int row = 0; row < m; row += kRows) {       // (m <= 2^30: no overflow)
    GemmArgs part = g;
    part.m = std::min(kRows, m - row);
    part.a = (const T *)g.a + row * g.lda;
    part.c = (T *)g.c + (long long)row * n;
    if (g.res) part.res = (const T *)g.res + row * g.ldres;
    if (g.slope) part.slope = (typename Slope<T>::S *)g.slope + (long long)row * n;
    launch_rows<T, true>(part, n, part.m, hs);
  }
}
size_t fwd_bytes(const btr_linear_t &p) {
  if (few_rows(p) || few_columns(p)) return 0;
  return pack_bytes(p.dtype, p.x, p.ldx, p.m, p.k) + pack_bytes(p.dtype, p.weight, p.ldw, p.n, p.k) +
         split_bytes(p.m, p.n, p.k, p.dtype);
}

template <typename T>
void forward(const btr_linear_t &p, void *y, void *slope, void *workspace, hipStream_t hs) {
  GemmArgs g{};
  g.m = p.m; g.n = p.n; g.k = p.k;
  g.bias = p.bias; g.res = p.residual; g.ldres = p.ldr; g.act = p.act;
  g.c = y; g.slope = slope; g.nsplit = 1;
  if (few_rows(p) || few_columns(p)) {
    g.a = p.x; g.lda = p.ldx; g.b = p.weight; g.ldb = p.ldw;
    if (few_rows(p))
      launch_rows<T, false>(g, p.m, p.n, hs);
    else
      launch_columns<T>(g, hs);
    return;
  }
  char *ws = (char *)workspace;
  Rows op[2] = {{p.x, p.ldx, 0, p.m, p.k}, {p.weight, p.ldw, 0, p.n, p.k}};
  pack_rows<T>(op, 2, ws, hs);
  launch_gemm<T, false, false>(g, op[0], op[1], ws, hs);
}

// dz is written unless dy itself can be read as it is
bool writes_dz(const btr_linear_t &p, const void *dy, long long lddy) {
  return p.act != BTR_ACT_NONE || !dma_rows(p.dtype, dy, lddy, p.n);
}
// float16 dz with slopes below 1: scaled.  The floats that takes: the workgroups' largest |dy|, the factor
bool scales_dz(const btr_linear_t &p) { return p.dtype == BTR_F16 && p.act == BTR_ACT_GELU; }
size_t most_bytes(const btr_linear_t &p) {
  return scales_dz(p) ? align256((kMostBlocks + 1) * sizeof(float)) : 0;
}
size_t bwd_bytes(const btr_linear_t &p, const void *dy, long long lddy) {
  const int m = p.m, n = p.n, k = p.k;
  if (m == 0) return 0;
  size_t v = align256((size_t)dz_blocks(m, n) * n * sizeof(float)) + most_bytes(p);
  if (writes_dz(p, dy, lddy)) v += packed_bytes(p.dtype, m, n);
  v += pack_bytes(p.dtype, p.x, p.ldx, m, k) + pack_bytes(p.dtype, p.weight, p.ldw, n, k);
  return v + std::max(split_bytes(m, k, n, p.dtype), split_bytes(n, k, m, p.dtype));
}

template <typename T>
void backward(const btr_linear_t &p, const void *slope, const void *dy, long long lddy, void *dx,
              void *dweight, void *dbias, void *workspace, hipStream_t hs) {
  typedef typename Matrix<T>::E E;
  const int m = p.m, n = p.n, k = p.k;
  char *ws = (char *)workspace;
  float *part = (float *)ws;
  const int blocks = m > 0 ? dz_blocks(m, n) : 0;
  Rows dz{dy, lddy, 0, m, n};                      // what the two products read
  float *most = nullptr;
  if (m > 0) {
    ws += align256((size_t)blocks * n * sizeof(float));
    if constexpr (kHalf<T>) {
      if (scales_dz(p) && (dx || dweight)) {
        most = (float *)ws;
        hipLaunchKernelGGL((linear_most_kernel<T>), dim3(kMostBlocks), dim3(256), 0, hs, (long long)m,
                           n, (const T *)dy, lddy, most);
      }
    }
    ws += most_bytes(p);
    E *out = nullptr;
    if (writes_dz(p, dy, lddy) && (dx || dweight)) {
      out = (E *)ws;
      dz = Rows{ws, up8(n), plane_of(m, n), m, n};
      ws += packed_bytes(p.dtype, m, n);
    }
    if (out || dbias)
      hipLaunchKernelGGL((linear_dz_kernel<T>), dim3(cdiv(n, 256), blocks), dim3(256), 0, hs,
                         (long long)m, n, (const T *)dy, lddy,
                         (const typename Slope<T>::S *)slope, p.act, out, up8(n),
                         dz.plane, dbias ? part : nullptr, most, kMostBlocks);
  }
  if (dbias)   // (no rows: zeros)
    hipLaunchKernelGGL((linear_dbias_kernel<T>), dim3(cdiv(n, 32)), dim3(1024), 0, hs, part, blocks, n,
                       (T *)dbias);
  const float *unscale = most ? most + kMostBlocks : nullptr;
  Rows op[2] = {{p.weight, p.ldw, 0, n, k}, {p.x, p.ldx, 0, m, k}};
  if (m > 0 && (dx || dweight))
    pack_rows<T>(op + (dx ? 0 : 1), (dx ? 1 : 0) + (dweight ? 1 : 0), ws, hs);
  if (dx && m > 0) {
    GemmArgs g{};
    g.m = m; g.n = k; g.k = n; g.c = dx; g.unscale = unscale;
    launch_gemm<T, false, true>(g, dz, op[0], ws, hs);
  }
  if (dweight) {
    GemmArgs g{};
    g.m = n; g.n = k; g.k = m; g.c = dweight; g.unscale = unscale;   // (no rows: writes zeros)
    launch_gemm<T, true, true>(g, dz, op[1], ws, hs);
  }
}

}  // namespace
}  // namespace btr

using namespace btr;

extern "C" size_t btr_linear_fwd_workspace_bytes(const btr_linear_t *p) {
  return check("linear_fwd", p) == BTR_OK ? fwd_bytes(*p) : 0;
}

extern "C" int btr_linear_fwd(const btr_linear_t *p, void *y, void *slope, void *workspace,
                              size_t workspace_bytes, btr_stream_t stream) {
  const int rc = check("linear_fwd", p);
  if (rc != BTR_OK) return rc;
  if (p->m == 0) return BTR_OK;
  BTR_REQUIRE(y, "linear_fwd: null pointer");
  const size_t need = fwd_bytes(*p);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "linear_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  BTR_REQUIRE(aligned16(workspace), "linear_fwd: workspace off a 16-byte boundary");
  BTR_DISPATCH_DTYPE(p->dtype, forward<T>(*p, y, slope, workspace, as_stream(stream)));
  return check_launch("linear_fwd");
}

extern "C" size_t btr_linear_bwd_workspace_bytes(const btr_linear_t *p, const void *dy,
                                                 long long lddy) {
  return check("linear_bwd", p) == BTR_OK ? bwd_bytes(*p, dy, lddy) : 0;
}

extern "C" int btr_linear_bwd(const btr_linear_t *p, const void *slope, const void *dy,
                              long long lddy, void *dx, void *dweight, void *dbias,
                              void *workspace, size_t workspace_bytes, btr_stream_t stream) {
  const int rc = check("linear_bwd", p);
  if (rc != BTR_OK) return rc;
  BTR_REQUIRE(p->m == 0 || (dy && lddy >= p->n && (p->act == BTR_ACT_NONE || slope)),
              "linear_bwd: null pointer or a row stride below the row");
  const size_t need = bwd_bytes(*p, dy, lddy);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "linear_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  BTR_REQUIRE(aligned16(workspace), "linear_bwd: workspace off a 16-byte boundary");
  BTR_DISPATCH_DTYPE(p->dtype, backward<T>(*p, slope, dy, lddy, dx, dweight, dbias, workspace,
                                           as_stream(stream)));
  return check_launch("linear_bwd");
}
