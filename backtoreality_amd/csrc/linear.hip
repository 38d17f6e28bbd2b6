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
// transposed in memory.  16-bit operands go to LDS by DMA (linear_dma_kernel); rows that do not lie
// on 16-byte boundaries in whole 16-byte units are first copied to rows that do, in the workspace.
// f32 operands pass through registers, where they are split (linear_gemm_kernel).  Few rows
// (single tokens) read W once, straight into the matrix instructions (linear_rows_kernel).
//
// Numbers: every product accumulates in f32 and the epilogue works on the f32 sums; y is rounded
// once.  f32 operands are split into three bf16 terms (8 + 8 + 8 bits: exact up to the 24th) and
// multiplied as the six products above 2^-24, which the bf16 matrix pipe does 2.7 times faster
// than the f32 instructions do one; an infinite f32 element makes the sums it enters NaN.  What the
// backward needs of the activation is its slope act'(z), taken from the f32 sum in the forward's
// epilogue and kept in the type of x (half an ulp; 0 and 1 of ReLU are exact); dz is rounded to the
// type of x as well before the two products that read it.
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
  void *c, *slope;           // contiguous (m, n); slope: act' of the sums, or NULL
  float *part;               // split reduction: (nsplit, m, n) partial sums
  int nsplit, chunk;         // shares of k, their length
  int mt, nt;                // tiles
};

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

__device__ __forceinline__ f32x16_t mfma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// f = h + m + l; an h that left the range of bf16 keeps no rest
__device__ __forceinline__ void split3(f32x4_t f, bf16x4_t (&p)[3]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __bf16 h = (__bf16)f[i];
    float r = f[i] - (float)h;
    if (!(__builtin_fabsf((float)h) < INFINITY)) r = 0.f;
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
  split3(v[0], a);
  split3(v[1], b);
#pragma unroll
  for (int p = 0; p < 3; ++p)
    f[p] = __builtin_shufflevector(a[p], b[p], 0, 1, 2, 3, 4, 5, 6, 7);
}

// f32: R rows of the operand (its m or n axis) x BK of the reduction, in LDS as three bf16 planes.  TR false: [R][BK], read
// as rows; true: [BK][R], read transposed.  Row pitches: an odd number of 16-byte units (sixteen
// rows at one column: distinct banks) / 64 mod 256 bytes (four rows x 64 bytes: distinct banks).
template <bool TR, int R, int BK>
struct Panel {
  static constexpr int P = 3, V = 4;
  static constexpr int ROWS = TR ? BK : R, COLS = TR ? R : BK;
  static constexpr int PITCH = TR ? (R * 2 / 256) * 256 + (R * 2 % 256 <= 64 ? 64 : R * 2 % 256 <= 192 ? 192 : 320)
                                  : COLS * 2 + 16;
  static constexpr int PLANE = ROWS * PITCH, BYTES = P * PLANE;
  static constexpr int PER_ROW = COLS / V, N = ROWS * PER_ROW / 256;
  static_assert(ROWS * PER_ROW % 256 == 0, "whole vectors per thread");
  static_assert(!TR || (PITCH >= R * 2 && (PITCH % 256 == 64 || PITCH % 256 == 192)), "pitch");
  f32x4_t r[N];

  // r0: first index of the operand's m / n axis, k0: of the reduction; beyond rmax / kmax zeros
  __device__ __forceinline__ void fetch(const float *src, long long ld, int r0, int rmax, int k0,
                                        int kmax, int tid) {
    const int row0 = TR ? k0 : r0, col0 = TR ? r0 : k0, rows = TR ? kmax : rmax,
              cols = TR ? rmax : kmax;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i, row = row0 + e / PER_ROW, col = col0 + (e % PER_ROW) * V;
      r[i] = f32x4_t{};
      if (row < rows && col < cols) r[i] = load_row(src + row * ld, col, cols);
    }
  }
  __device__ __forceinline__ void store(char *lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i;
      char *p = lds + (e / PER_ROW) * PITCH + (e % PER_ROW) * V * 2;
      bf16x4_t q[3];
      split3(r[i], q);
#pragma unroll
      for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x4_t *>(p + j * PLANE) = q[j];
    }
  }
  // fragment of the 32 rows at r0 and the 16 reduction steps at ks
  __device__ static __forceinline__ bf16x8_t frag(const char *lds, int plane, int r0,
                                                              int ks, int lane) {
    const char *t = lds + plane * PLANE;
    if constexpr (!TR) {
      return *reinterpret_cast<const bf16x8_t *>(
          t + (r0 + (lane & 31)) * PITCH + (ks + 8 * (lane >> 5)) * 2);
    } else {
      // lane p of a group of 16 addresses row p / 4, columns 4 (p % 4) .. + 3 of a [4][16] block and
      // receives column p, rows 0 .. 3
      const int p = lane & 15;
      const char *q = t + (ks + 8 * (lane >> 5) + (p >> 2)) * PITCH +
                      (r0 + 16 * ((lane >> 4) & 1) + 4 * (p & 3)) * 2;
      union {
        s16x4_t s[2];
        bf16x8_t f;
      } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q);
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 4 * PITCH));
      return u.f;
    }
  }
};

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
// act(z), and act'(z) into slope
template <bool F32>
__device__ __forceinline__ float activate(float z, int act, float &slope) {
  slope = 1.f;
  if (act == kActRelu) {
    slope = z > 0.f ? 1.f : 0.f;
    return z > 0.f ? z : z != z ? z : 0.f;
  }
  if (act == kActGelu) return gelu<F32>(z, slope);
  return z;
}

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
  typename Elem<T>::Vec slope, y;
#pragma unroll
  for (int j = 0; j < V; ++j) {
    float d;
    y[j] = (T)(activate<sizeof(T) == 4>(s[j] + (float)bias[j], g.act, d) + (float)res[j]);
    slope[j] = (T)d;
  }
  if (g.slope) store_row((T *)g.slope + row * g.n, col, g.n, slope);
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

// f32: BM x BN tile by four waves (2 x 2), 32 reduction steps at a time, the next in registers
template <bool TA, bool TB, int BM, int BN>
__global__ __launch_bounds__(256) void linear_gemm_kernel(GemmArgs g) {
  constexpr int BK = 32, WM = BM / 2, WN = BN / 2, IM = WM / 32, IN = WN / 32;
  typedef Panel<TA, BM, BK> PA;
  typedef Panel<TB, BN, BK> PB;
  constexpr int SLAB = 4 * 32 * (WN + 4) * 4, TILE = PA::BYTES + PB::BYTES;
  __shared__ __attribute__((aligned(16))) char smem[TILE > SLAB ? TILE : SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  int m0, n0, split;
  place<BM, BN>(g, m0, n0, split);
  const int kbeg = split * g.chunk, kend = min(g.k, kbeg + g.chunk);
  const int wm = (w >> 1) * WM, wn = (w & 1) * WN;

  f32x16_t acc[IM][IN] = {};
  PA pa;
  PB pb;
  char *la = smem, *lb = smem + PA::BYTES;
  if (kbeg < kend) {
    pa.fetch((const float *)g.a, g.lda, m0, g.m, kbeg, kend, tid);
    pb.fetch((const float *)g.b, g.ldb, n0, g.n, kbeg, kend, tid);
  }
  for (int k0 = kbeg; k0 < kend; k0 += BK) {
    lds_barrier();                                 // the previous step's reads are done
    pa.store(la, tid);
    pb.store(lb, tid);
    if (k0 + BK < kend) {
      pa.fetch((const float *)g.a, g.lda, m0, g.m, k0 + BK, kend, tid);
      pb.fetch((const float *)g.b, g.ldb, n0, g.n, k0 + BK, kend, tid);
    }
    lds_barrier();
#pragma unroll
    for (int ks = 0; ks < BK; ks += 16) {
      bf16x8_t fa[IM][3], fb[IN][3];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
#pragma unroll
        for (int i = 0; i < IM; ++i) fa[i][p] = PA::frag(la, p, wm + 32 * i, ks, lane);
#pragma unroll
        for (int j = 0; j < IN; ++j) fb[j][p] = PB::frag(lb, p, wn + 32 * j, ks, lane);
      }
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) {             // smallest terms first
          acc[i][j] = mfma(fa[i][2], fb[j][0], acc[i][j]);
          acc[i][j] = mfma(fa[i][0], fb[j][2], acc[i][j]);
          acc[i][j] = mfma(fa[i][1], fb[j][1], acc[i][j]);
          acc[i][j] = mfma(fa[i][1], fb[j][0], acc[i][j]);
          acc[i][j] = mfma(fa[i][0], fb[j][1], acc[i][j]);
          acc[i][j] = mfma(fa[i][0], fb[j][0], acc[i][j]);
        }
    }
  }
  __syncthreads();
  leave<float, IM, IN>(g, acc, reinterpret_cast<float *>(smem) + w * 32 * (WN + 4), m0 + wm, n0 + wn,
                       split, lane);
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
template <typename T, bool TA, bool TB, int BM, int BN, int GM, int GN, int NBUF,
          int OCC>
__global__ __launch_bounds__(64 * GM * GN, OCC) void linear_dma_kernel(GemmArgs g) {
  constexpr int THREADS = 64 * GM * GN, WM = BM / GM, WN = BN / GN, IM = WM / 32, IN = WN / 32;
  typedef DmaPanel<T, TA, BM, THREADS> PA;
  typedef DmaPanel<T, TB, BN, THREADS> PB;
  typedef typename Elem<T>::Vec Vec;
  constexpr int TILE = PA::BYTES + PB::BYTES, SLAB = GM * GN * 32 * (WN + 4) * 4;
  constexpr int NDMA = PA::N + PB::N;              // instructions a wave issues per step
  constexpr int NF = IM + IN, NP = IM * IN;        // fragments and products of a group
  constexpr int LQ = (NF + NP - 1) / NP, DQ = (NDMA + NP - 1) / NP;   // between two products, at most
  __shared__ __attribute__((aligned(1024))) char smem[NBUF * TILE > SLAB ? NBUF * TILE : SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  int m0, n0, split;
  place<BM, BN>(g, m0, n0, split);
  const int kbeg = split * g.chunk, kend = min(g.k, kbeg + g.chunk);
  const int wm = w / GN * WM, wn = w % GN * WN;
  const T *ap = (const T *)g.a + (TA ? (long long)m0 : m0 * g.lda);
  const T *bp = (const T *)g.b + (TB ? (long long)n0 : n0 * g.ldb);
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
  auto issue = [&](int k0, int buf, int i) {       // DMA instruction i of a step
    char *la = smem + buf * TILE;
    if (i == 0) ra = PA::rsrc(ap, g.lda, k0);
    if (i == PA::N) rb = PB::rsrc(bp, g.ldb, k0);
    if (i < PA::N) pa.issue(ra, i, kend - k0, la, tid, w);
    else pb.issue(rb, i - PA::N, kend - k0, la + PA::BYTES, tid, w);
  };
  if (kbeg < kend) {
#pragma unroll
    for (int t = 0; t < NBUF - 1; ++t)
#pragma unroll
      for (int i = 0; i < NDMA; ++i) issue(kbeg + t * kStep, t, i);
    dma_wait<(NBUF - 2) * NDMA>();
    lds_barrier();
#pragma unroll
    for (int i = 0; i < NDMA; ++i) issue(kbeg + (NBUF - 1) * kStep, NBUF - 1, i);
#pragma unroll
    for (int i = 0; i < NF; ++i) load(0, 0, i);
  }
  int buf = 0;
  for (int k0 = kbeg; k0 < kend; k0 += kStep) {
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
      for (int i = q * DQ; i < NDMA && i < (q + 1) * DQ; ++i) issue(k0 + NBUF * kStep, buf, i);
      __builtin_amdgcn_sched_barrier(0);
    }
    buf = next;
  }
  dma_wait();
  __syncthreads();
  leave<T, IM, IN>(g, acc, reinterpret_cast<float *>(smem) + w * 32 * (WN + 4), m0 + wm, n0 + wn,
                   split, lane);
}

// Few rows of x (up to 16 MT): a workgroup's eight waves share 16 rows of W and split the reduction
// (wave w: the steps of 32 numbered w, w + 8, ..), W goes from memory into the matrix instructions,
// the eight sums meet in LDS.  Bound by the bytes of W: eight loads of 1 KB in flight a wave.
template <typename T, int MT>
__global__ __launch_bounds__(512) void linear_rows_kernel(GemmArgs g) {
  constexpr int P = Op<T>::P, U = sizeof(T) == 4 ? 4 : 8;
  __shared__ float part[8][MT][16][20];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l15 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16;
  f32x4_t acc[MT] = {};
  const T *wrow = (const T *)g.b + min(n0 + l15, g.n - 1) * g.ldb;
  const T *xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xrow[t] = (const T *)g.a + min(16 * t + l15, g.m - 1) * g.lda;
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
  for (int t = 0; t < MT; ++t)                     // [row of x][row of W]
    *reinterpret_cast<f32x4_t *>(&part[w][t][l15][4 * q]) = acc[t];
  __syncthreads();
  // 16 outputs of a row in pieces of V columns
  constexpr int V = Elem<T>::kVec, PR = 16 / V;
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

// 16-bit rows -> rows of ldd elements on 16-byte boundaries, zeros behind them
template <typename T>
__global__ __launch_bounds__(256) void linear_pack_kernel(long long rows, int cols, const T *src,
                                                          long long ld, T *dst, int ldd) {
  const long long total = rows * (ldd / 8);
  for (long long e = (long long)blockIdx.x * 256 + threadIdx.x; e < total;
       e += (long long)gridDim.x * 256) {
    const long long row = e / (ldd / 8);
    const int col = (int)(e - row * (ldd / 8)) * 8;
    *reinterpret_cast<typename Elem<T>::Vec *>(dst + row * ldd + col) =
        load_row(src + row * ld, col, cols);
  }
}

// adds the shares of the reduction in order, then the epilogue
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

// dz = dy slope (ReLU: dy where slope > 0) into rows of ldz elements, zeros behind them, and the
// column sums of dz over this workgroup's rows: 32 threads along the columns (a vector each), 8 rows
// at a time.  dz NULL: the sums only.
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(long long m, int n, const T *dy,
                                                        long long lddy, const T *slope, int act,
                                                        T *dz, int ldz, float *part) {
  constexpr int V = Elem<T>::kVec;
  __shared__ float red[8][32 * V];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, col = (blockIdx.x * 32 + cl) * V;
  float sum[V] = {};
  if (col < n)
    for (long long row = (long long)blockIdx.y * 8 + rl; row < m; row += (long long)gridDim.y * 8) {
      typename Elem<T>::Vec g = load_row(dy + row * lddy, col, n);
      if (act != kActNone) {
        const typename Elem<T>::Vec d = load_row(slope + row * n, col, n);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (act == kActRelu)                     // (a select: an infinite dy stays out of it)
            g[j] = (float)d[j] > 0.f ? g[j] : (T)0.f;
          else
            g[j] = (T)((float)g[j] * (float)d[j]);
        }
      }
      if (dz) store_row(dz + row * ldz, col, ldz, g);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += (float)g[j];
    }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) red[rl][cl * V + j] = sum[j];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * V; c += 256) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][c];
    if (blockIdx.x * 32 * V + c < n) part[(long long)blockIdx.y * n + blockIdx.x * 32 * V + c] = t;
  }
}

// dbias = sum of the workgroups' rows, in order: 32 columns x 8 row groups a workgroup
template <typename T>
__global__ __launch_bounds__(256) void linear_dbias_kernel(const float *part, int blocks, int n,
                                                           T *db) {
  __shared__ float s[8][32];
  const int cl = threadIdx.x & 31, rg = threadIdx.x >> 5, c = blockIdx.x * 32 + cl;
  float acc = 0.f;
  if (c < n)
    for (int r = rg; r < blocks; r += 8) acc += part[(long long)r * n + c];
  s[rg][cl] = acc;
  __syncthreads();
  if (rg == 0 && c < n) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += s[k][cl];
    db[c] = (T)t;
  }
}

// --------------------------------------------------------------------------------------- host
struct Plan {
  int bm, bn, mt, nt, nsplit, chunk;
};

// Tile and shares of the reduction by estimated time: workgroups a CU gets x (64-step pieces x what
// one costs + what a workgroup costs besides), not below one workgroup's own latency, plus the
// partial sums' way through memory.  The figures are us, measured for bf16 at 16 384 x 4 096 x 1 024
// and 16 384 x 1 024 x 4 096 with each tile in turn.  (f32 has the two small tiles.)
Plan plan_gemm(int m, int n, int k, bool dma) {
  static const struct { int bm, bn; double step, fixed, alone; } kTile[4] = {
      {256, 256, 1.65, 11.0, 1.65}, {256, 128, 1.02, 6.7, 1.02}, {128, 128, 0.6, 3.4, 0.75},
      {64, 64, 0.26, 1.3, 0.45}};
  Plan best{};
  double least = 1e30;
  for (int i = dma ? 0 : 2; i < 4; ++i) {
    const auto &t = kTile[i];
    const int mt = cdiv(m, t.bm), nt = cdiv(n, t.bn);
    const long long tiles = (long long)mt * nt;
    for (int s = 1; s <= 32 && (s == 1 || (k / s >= 128 && tiles * s <= 2048)); ++s) {
      const int chunk = std::max(64, cdiv(cdiv(k, s), 64) * 64), real = std::max(1, cdiv(k, chunk));
      if (real != s) continue;
      const double steps = chunk / 64;
      double us = std::max((double)((tiles * s + 255) / 256) * (steps * t.step + t.fixed),
                           steps * t.alone + t.fixed);
      if (s > 1) us += 4.0 + (2.0 * s + 1.0) * m * n * 4.0 / 4e6;
      if (us < least) {
        least = us;
        best = Plan{t.bm, t.bn, mt, nt, s, chunk};
      }
    }
  }
  return best;
}
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
size_t split_bytes(int m, int n, int k, bool dma) {
  const Plan p = plan_gemm(m, n, k, dma);
  return p.nsplit > 1 ? align256((size_t)p.nsplit * m * n * sizeof(float)) : 0;
}
int up8(int v) { return (v + 7) & ~7; }
// rows a DMA may read where they are: whole 16-byte units on 16-byte boundaries, a tile's offsets
// below 2^31
bool dma_rows(const void *p, long long ld, int len) {
  return ((uintptr_t)p & 15) == 0 && len % 8 == 0 && ld % 8 == 0 && ld <= (1 << 22);
}
size_t pack_bytes(const void *p, long long ld, long long rows, int len) {
  return dma_rows(p, ld, len) ? 0 : align256((size_t)rows * up8(len) * 2);
}
constexpr int kFewRows = 16;       // linear_rows_kernel up to here
// workgroups along the rows of the dz / dbias pass
int dz_blocks(long long m, int n) {
  const long long cols = cdiv(n, 128);
  return (int)std::max<long long>(1, std::min<long long>((m + 31) / 32, (2048 + cols - 1) / cols));
}

// an operand as the DMA kernels want it: where it is, or packed into ws (which moves on)
template <typename T>
void pack_rows(const void *&p, long long &ld, long long rows, int len, char *&ws, hipStream_t hs) {
  if (dma_rows(p, ld, len)) return;
  const int ldd = up8(len);
  const long long units = rows * (ldd / 8);
  hipLaunchKernelGGL((linear_pack_kernel<T>),
                     dim3((unsigned)std::min<long long>(4096, (units + 255) / 256)), dim3(256), 0, hs,
                     rows, len, (const T *)p, ld, (T *)ws, ldd);
  p = ws;
  ld = ldd;
  ws += align256((size_t)rows * ldd * 2);
}

template <typename T, bool TA, bool TB>
void launch_gemm(GemmArgs g, void *ws, hipStream_t hs) {
  constexpr bool DMA = sizeof(T) == 2;
  const Plan p = plan_gemm(g.m, g.n, g.k, DMA);
  g.mt = p.mt; g.nt = p.nt; g.nsplit = p.nsplit; g.chunk = p.chunk; g.part = (float *)ws;
  const dim3 grid((unsigned)((long long)p.mt * p.nt * p.nsplit));
  if constexpr (DMA) {
    if (p.bm == 256 && p.bn == 128)
      hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 256, 128, 4, 2, 3, 4>), grid, dim3(512), 0, hs, g);
    else if (p.bm == 256)
      hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 256, 256, 2, 4, 4, 2>), grid, dim3(512), 0, hs, g);
    else if (p.bm == 128)
      hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 128, 128, 2, 2, 4, 2>), grid, dim3(256), 0, hs, g);
    else
      hipLaunchKernelGGL((linear_dma_kernel<T, TA, TB, 64, 64, 2, 2, 4, 2>), grid, dim3(256), 0, hs, g);
  } else {
    if (p.bm == 128)
      hipLaunchKernelGGL((linear_gemm_kernel<TA, TB, 128, 128>), grid, dim3(256), 0, hs, g);
    else
      hipLaunchKernelGGL((linear_gemm_kernel<TA, TB, 64, 64>), grid, dim3(256), 0, hs, g);
  }
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
  BTR_REQUIRE(m >= 0 && n >= 1 && k >= 1 && m <= (1 << 30) && n <= (1 << 30) && k <= (1 << 30) &&
                  ((long long)cdiv(m, 64) * cdiv(n, 64) <= (1 << 30)) &&
                  ((long long)cdiv(m, 64) * cdiv(k, 64) <= (1 << 30)) &&
                  ((long long)cdiv(n, 64) * cdiv(k, 64) <= (1 << 30)),
              "%s: (%d, %d) x (%d, %d)", what, m, k, n, k);
  BTR_REQUIRE(m == 0 || (p->x && p->weight && p->ldx >= k && p->ldw >= k &&
                         (!p->residual || p->ldr >= n)),
              "%s: null pointer or a row stride below the row", what);
  return BTR_OK;
}

size_t fwd_bytes(const btr_linear_t &p) {
  if (p.m <= kFewRows) return 0;
  if (p.dtype == BTR_F32) return split_bytes(p.m, p.n, p.k, false);
  return pack_bytes(p.x, p.ldx, p.m, p.k) + pack_bytes(p.weight, p.ldw, p.n, p.k) +
         split_bytes(p.m, p.n, p.k, true);
}

template <typename T>
void forward(const btr_linear_t &p, void *y, void *slope, void *workspace, hipStream_t hs) {
  GemmArgs g{};
  g.m = p.m; g.n = p.n; g.k = p.k;
  g.a = p.x; g.lda = p.ldx; g.b = p.weight; g.ldb = p.ldw;
  g.bias = p.bias; g.res = p.residual; g.ldres = p.ldr; g.act = p.act;
  g.c = y; g.slope = slope;
  if (p.m <= kFewRows) {
    hipLaunchKernelGGL((linear_rows_kernel<T, 1>), dim3(cdiv(p.n, 16)), dim3(512), 0, hs, g);
    return;
  }
  char *ws = (char *)workspace;
  if constexpr (sizeof(T) == 2) {
    pack_rows<T>(g.a, g.lda, p.m, p.k, ws, hs);
    pack_rows<T>(g.b, g.ldb, p.n, p.k, ws, hs);
  }
  launch_gemm<T, false, false>(g, ws, hs);
}

// dz is written unless dy itself can be read as it is
bool writes_dz(const btr_linear_t &p, const void *dy, long long lddy) {
  return p.act != BTR_ACT_NONE || (p.dtype != BTR_F32 && !dma_rows(dy, lddy, p.n));
}
size_t bwd_bytes(const btr_linear_t &p, const void *dy, long long lddy) {
  const int m = p.m, n = p.n, k = p.k;
  if (m == 0) return 0;
  const bool f32 = p.dtype == BTR_F32;
  size_t v = align256((size_t)dz_blocks(m, n) * n * sizeof(float));
  if (writes_dz(p, dy, lddy)) v += align256((size_t)m * (f32 ? n * 4ll : up8(n) * 2ll));
  if (!f32) v += pack_bytes(p.x, p.ldx, m, k) + pack_bytes(p.weight, p.ldw, n, k);
  return v + std::max(split_bytes(m, k, n, !f32), split_bytes(n, k, m, !f32));
}

template <typename T>
void backward(const btr_linear_t &p, const void *slope, const void *dy, long long lddy, void *dx,
              void *dweight, void *dbias, void *workspace, hipStream_t hs) {
  const int m = p.m, n = p.n, k = p.k;
  char *ws = (char *)workspace;
  float *part = (float *)ws;
  const int blocks = m > 0 ? dz_blocks(m, n) : 0;
  const void *gz = dy;                             // what the two products read
  long long ldg = lddy;
  if (m > 0) {
    ws += align256((size_t)blocks * n * sizeof(float));
    void *dz = nullptr;
    const int ldz = sizeof(T) == 4 ? n : up8(n);
    if (writes_dz(p, dy, lddy)) {
      dz = ws;
      ws += align256((size_t)m * ldz * sizeof(T));
      gz = dz;
      ldg = ldz;
    }
    if (dz || dbias)
      hipLaunchKernelGGL((linear_dz_kernel<T>), dim3(cdiv(n, 32 * Elem<T>::kVec), blocks), dim3(256),
                         0, hs, (long long)m, n, (const T *)dy, lddy, (const T *)slope, p.act,
                         (T *)dz, ldz, dbias ? part : nullptr);
  }
  if (dbias)   // (no rows: zeros)
    hipLaunchKernelGGL((linear_dbias_kernel<T>), dim3(cdiv(n, 32)), dim3(256), 0, hs, part, blocks, n,
                       (T *)dbias);
  const void *x = p.x, *wt = p.weight;
  long long ldx = p.ldx, ldw = p.ldw;
  if constexpr (sizeof(T) == 2) {
    if (m > 0 && dweight) pack_rows<T>(x, ldx, m, k, ws, hs);
    if (m > 0 && dx) pack_rows<T>(wt, ldw, n, k, ws, hs);
  }
  if (dx && m > 0) {
    GemmArgs g{};
    g.m = m; g.n = k; g.k = n;
    g.a = gz; g.lda = ldg; g.b = wt; g.ldb = ldw; g.c = dx;
    launch_gemm<T, false, true>(g, ws, hs);
  }
  if (dweight) {
    GemmArgs g{};
    g.m = n; g.n = k; g.k = m;                     // (no rows: an empty reduction writes zeros)
    g.a = gz; g.lda = ldg; g.b = x; g.ldb = ldx; g.c = dweight;
    launch_gemm<T, true, true>(g, ws, hs);
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
  BTR_DISPATCH_DTYPE(p->dtype, backward<T>(*p, slope, dy, lddy, dx, dweight, dbias, workspace,
                                           as_stream(stream)));
  return check_launch("linear_bwd");
}
