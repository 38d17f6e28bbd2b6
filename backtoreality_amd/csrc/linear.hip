// linear.hip -- a linear layer with its epilogue, forward and backward:
//
//   z = x W^T + bias,  y = act(z) [+ residual],   act = identity, ReLU, GELU (z Phi(z), erf form)
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  dbias = colsum(dz),  dresidual = dy
//
// x (m, k), W (n, k) as in torch.nn.Linear; float32, bfloat16, float16; any sizes and row strides.
// (reference: linear1 / linear2 and the projections of detection/GroupFree3D/models/
// transformer.py:36-76; csrc/sa_mlp.hip has the float32 GEMMs with BatchNorm around them.)
//
// One tile kernel serves the three products; what differs is whether the reduction runs along a
// row of the operand (x, W forward, dz for dx) or across its rows (W for dx; dz and x for dW).  Both
// are staged the way memory has them, 16 bytes a lane along the rows; the second kind is read out
// of LDS with gfx950's transpose read, so nothing is ever transposed in memory.
//
// Numbers: every product accumulates in f32 and the epilogue works on the f32 sums; y is rounded
// once.  f32 operands are split into three bf16 terms (8 + 8 + 8 bits: exact up to the 24th) and
// multiplied as the six products above 2^-24, which the bf16 matrix pipe does 2.7 times faster
// than the f32 instructions do one; an infinite f32 element makes the sums it enters NaN.  z is kept
// for the backward in the type of x (act' sees z with half an ulp of error), dz likewise is rounded
// to the type of x before the two products that read it.
#include <algorithm>

#include "decoder_ops.hpp"

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
  void *c, *z;               // contiguous (m, n); z: the sums before the activation, or NULL
  float *part;               // split reduction: (nsplit, m, n) partial sums
  int nsplit, chunk;         // shares of k, their length
  int mt, nt;                // tiles
};

typedef __attribute__((address_space(3))) s16x4_t *lds_s16x4;

// what the matrix instructions eat: T itself, or three bf16 planes of f32
template <typename T>
struct Op {
  static constexpr int P = 1, V = 8;
  typedef typename Elem<T>::Vec Frag;
  typedef T E;
};
template <>
struct Op<float> {
  static constexpr int P = 3, V = 4;
  typedef bf16x8_t Frag;
  typedef __bf16 E;
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

// R rows of the operand (its m or n axis) x BK of the reduction, in LDS.  TR false: [R][BK], read
// as rows; true: [BK][R], read transposed.  Row pitches: an odd number of 16-byte units (sixteen
// rows at one column: distinct banks) / 64 mod 256 bytes (four rows x 64 bytes: distinct banks).
template <typename T, bool TR, int R, int BK>
struct Panel {
  static constexpr int P = Op<T>::P, V = Op<T>::V;
  static constexpr int ROWS = TR ? BK : R, COLS = TR ? R : BK;
  static constexpr int PITCH = TR ? (R * 2 / 256) * 256 + (R * 2 % 256 <= 64 ? 64 : R * 2 % 256 <= 192 ? 192 : 320)
                                  : COLS * 2 + 16;
  static constexpr int PLANE = ROWS * PITCH, BYTES = P * PLANE;
  static constexpr int PER_ROW = COLS / V, N = ROWS * PER_ROW / 256;
  static_assert(ROWS * PER_ROW % 256 == 0, "whole vectors per thread");
  static_assert(!TR || (PITCH >= R * 2 && (PITCH % 256 == 64 || PITCH % 256 == 192)), "pitch");
  typename Elem<T>::Vec r[N];

  // r0: first index of the operand's m / n axis, k0: of the reduction; beyond rmax / kmax zeros
  __device__ __forceinline__ void fetch(const T *src, long long ld, int r0, int rmax, int k0,
                                        int kmax, int tid) {
    const int row0 = TR ? k0 : r0, col0 = TR ? r0 : k0, rows = TR ? kmax : rmax,
              cols = TR ? rmax : kmax;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i, row = row0 + e / PER_ROW, col = col0 + (e % PER_ROW) * V;
      r[i] = typename Elem<T>::Vec{};
      if (row < rows && col < cols) r[i] = load_row(src + row * ld, col, cols);
    }
  }
  __device__ __forceinline__ void store(char *lds, int tid) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int e = tid + 256 * i;
      char *p = lds + (e / PER_ROW) * PITCH + (e % PER_ROW) * V * 2;
      if constexpr (P == 1) {
        *reinterpret_cast<typename Elem<T>::Vec *>(p) = r[i];
      } else {
        bf16x4_t q[3];
        split3(r[i], q);
#pragma unroll
        for (int j = 0; j < 3; ++j) *reinterpret_cast<bf16x4_t *>(p + j * PLANE) = q[j];
      }
    }
  }
  // fragment of the 32 rows at r0 and the 16 reduction steps at ks
  __device__ static __forceinline__ typename Op<T>::Frag frag(const char *lds, int plane, int r0,
                                                              int ks, int lane) {
    const char *t = lds + plane * PLANE;
    if constexpr (!TR) {
      return *reinterpret_cast<const typename Op<T>::Frag *>(
          t + (r0 + (lane & 31)) * PITCH + (ks + 8 * (lane >> 5)) * 2);
    } else {
      // lane p of a group of 16 addresses row p / 4, columns 4 (p % 4) .. + 3 of a [4][16] block and
      // receives column p, rows 0 .. 3
      const int p = lane & 15;
      const char *q = t + (ks + 8 * (lane >> 5) + (p >> 2)) * PITCH +
                      (r0 + 16 * ((lane >> 4) & 1) + 4 * (p & 3)) * 2;
      union {
        s16x4_t s[2];
        typename Op<T>::Frag f;
      } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)q);
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(q + 4 * PITCH));
      return u.f;
    }
  }
};

__device__ __forceinline__ float gelu_cdf(float z) {   // Phi(z); the tail without cancellation
  return 0.5f * erfcf(-z * 0.70710678118654752f);
}
__device__ __forceinline__ float activate(float z, int act) {
  if (act == kActRelu) return z > 0.f ? z : z != z ? z : 0.f;
  if (act == kActGelu) return z == -INFINITY ? 0.f : z * gelu_cdf(z);
  return z;
}
__device__ __forceinline__ float activate_grad(float z, int act) {
  if (act == kActRelu) return z > 0.f ? 1.f : 0.f;
  if (act == kActGelu) {
    if (__builtin_fabsf(z) > 30.f) return z > 0.f ? 1.f : 0.f;   // (beyond f32's smallest density)
    return gelu_cdf(z) + z * 0.39894228040143268f * __builtin_amdgcn_exp2f(-0.72134752044448170f * z * z);
  }
  return 1.f;
}

// V consecutive columns of one row: bias, activation, residual, one rounding
template <typename T>
__device__ __forceinline__ void epilogue(const GemmArgs &g, long long row, int col,
                                         const float (&s)[Elem<T>::kVec]) {
  constexpr int V = Elem<T>::kVec;
  typename Elem<T>::Vec bias = {}, res = {}, z, y;
  if (g.bias) bias = load_row((const T *)g.bias, col, g.n);
  if (g.res) res = load_row((const T *)g.res + row * g.ldres, col, g.n);
#pragma unroll
  for (int j = 0; j < V; ++j) {
    const float t = s[j] + (float)bias[j];
    z[j] = (T)t;
    y[j] = (T)(activate(t, g.act) + (float)res[j]);
  }
  if (g.z) store_row((T *)g.z + row * g.n, col, g.n, z);
  store_row((T *)g.c + row * g.n, col, g.n, y);
}

// BM x BN tile by four waves (2 x 2), BK reduction steps at a time, the next in registers
template <typename T, bool TA, bool TB, int BM, int BN>
__global__ __launch_bounds__(256) void linear_gemm_kernel(GemmArgs g) {
  constexpr int BK = sizeof(T) == 4 ? 32 : 64, P = Op<T>::P, V = Elem<T>::kVec;
  constexpr int WM = BM / 2, WN = BN / 2, IM = WM / 32, IN = WN / 32;
  typedef Panel<T, TA, BM, BK> PA;
  typedef Panel<T, TB, BN, BK> PB;
  constexpr int CP = WN + 4;                       // floats per row of the epilogue's slab
  constexpr int SLAB = 4 * 32 * CP * 4, TILE = PA::BYTES + PB::BYTES;
  __shared__ __attribute__((aligned(16))) char smem[TILE > SLAB ? TILE : SLAB];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  // workgroups land on the eight XCDs in turn: each XCD gets a contiguous eighth of the tiles, and
  // walks them in columns of eight row tiles, so that what its L2 holds is read several times
  const int total = gridDim.x, id = blockIdx.x, per = total / 8;
  int t = id < per * 8 ? (id & 7) * per + (id >> 3) : id;
  const int split = t / (g.mt * g.nt);
  t -= split * (g.mt * g.nt);
  const int band = t / (8 * g.nt), in = t - band * 8 * g.nt, bh = min(8, g.mt - band * 8);
  const int m0 = (band * 8 + in % bh) * BM, n0 = (in / bh) * BN;
  const int kbeg = split * g.chunk, kend = min(g.k, kbeg + g.chunk);
  const int wm = (w >> 1) * WM, wn = (w & 1) * WN;

  f32x16_t acc[IM][IN] = {};
  PA pa;
  PB pb;
  char *la = smem, *lb = smem + PA::BYTES;
  if (kbeg < kend) {
    pa.fetch((const T *)g.a, g.lda, m0, g.m, kbeg, kend, tid);
    pb.fetch((const T *)g.b, g.ldb, n0, g.n, kbeg, kend, tid);
  }
  for (int k0 = kbeg; k0 < kend; k0 += BK) {
    lds_barrier();                                 // the previous step's reads are done
    pa.store(la, tid);
    pb.store(lb, tid);
    if (k0 + BK < kend) {
      pa.fetch((const T *)g.a, g.lda, m0, g.m, k0 + BK, kend, tid);
      pb.fetch((const T *)g.b, g.ldb, n0, g.n, k0 + BK, kend, tid);
    }
    lds_barrier();
#pragma unroll
    for (int ks = 0; ks < BK; ks += 16) {
      typename Op<T>::Frag fa[IM][P], fb[IN][P];
#pragma unroll
      for (int p = 0; p < P; ++p) {
#pragma unroll
        for (int i = 0; i < IM; ++i) fa[i][p] = PA::frag(la, p, wm + 32 * i, ks, lane);
#pragma unroll
        for (int j = 0; j < IN; ++j) fb[j][p] = PB::frag(lb, p, wn + 32 * j, ks, lane);
      }
#pragma unroll
      for (int i = 0; i < IM; ++i)
#pragma unroll
        for (int j = 0; j < IN; ++j) {
          if constexpr (P == 3) {                  // smallest terms first
            acc[i][j] = mfma(fa[i][2], fb[j][0], acc[i][j]);
            acc[i][j] = mfma(fa[i][0], fb[j][2], acc[i][j]);
            acc[i][j] = mfma(fa[i][1], fb[j][1], acc[i][j]);
            acc[i][j] = mfma(fa[i][1], fb[j][0], acc[i][j]);
            acc[i][j] = mfma(fa[i][0], fb[j][1], acc[i][j]);
          }
          acc[i][j] = mfma(fa[i][0], fb[j][0], acc[i][j]);
        }
    }
  }
  // the tile leaves through LDS, 32 rows of a wave at a time, as 16-byte row pieces
  float *slab = reinterpret_cast<float *>(smem) + w * 32 * CP;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < IM; ++i) {
#pragma unroll
    for (int j = 0; j < IN; ++j)
#pragma unroll
      for (int v = 0; v < 16; ++v)
        slab[((v & 3) + 8 * (v >> 2) + 4 * (lane >> 5)) * CP + 32 * j + (lane & 31)] = acc[i][j][v];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    constexpr int PR = WN / V;                     // pieces per row
#pragma unroll
    for (int q = 0; q < 32 * PR / 64; ++q) {
      const int e = lane + 64 * q, row = e / PR, col = (e % PR) * V;
      const int gr = m0 + wm + 32 * i + row, gc = n0 + wn + col;
      float s[V];
#pragma unroll
      for (int u = 0; u < V; ++u) s[u] = slab[row * CP + col + u];
      if (gr < g.m && gc < g.n) {
        if (g.nsplit > 1) {
          float *dst = g.part + ((long long)split * g.m + gr) * g.n;
#pragma unroll
          for (int u = 0; u < V; u += 4)
            store_row(dst, gc + u, g.n, f32x4_t{s[u], s[u + 1], s[u + 2], s[u + 3]});
        } else {
          epilogue<T>(g, gr, gc, s);
        }
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
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
    epilogue<T>(g, row, col, s);
  }
}

// dz = dy act'(z) and the column sums of dz over this workgroup's rows: 32 threads along the
// columns (a vector each), 8 rows at a time
template <typename T>
__global__ __launch_bounds__(256) void linear_dz_kernel(long long m, int n, const T *dy,
                                                        long long lddy, const T *z, int act, T *dz,
                                                        float *part) {
  constexpr int V = Elem<T>::kVec;
  __shared__ float red[8][32 * V];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5, col = (blockIdx.x * 32 + cl) * V;
  float sum[V] = {};
  if (col < n)
    for (long long row = (long long)blockIdx.y * 8 + rl; row < m; row += (long long)gridDim.y * 8) {
      typename Elem<T>::Vec g = load_row(dy + row * lddy, col, n);
      if (act != kActNone) {
        const typename Elem<T>::Vec zz = load_row(z + row * n, col, n);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          if (act == kActRelu)                     // (a select: an infinite dy stays out of it)
            g[j] = (float)zz[j] > 0.f ? g[j] : (T)0.f;
          else
            g[j] = (T)((float)g[j] * activate_grad((float)zz[j], act));
        }
        store_row(dz + row * n, col, n, g);
      }
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
  int bm, mt, nt, nsplit, chunk;
};

// 128 x 128 tiles where they give every CU one; else 64 x 64, and while those leave CUs idle the
// reduction is cut into shares of at least 256 steps
Plan plan_gemm(int m, int n, int k) {
  Plan p;
  p.bm = (long long)cdiv(m, 128) * cdiv(n, 128) >= 256 ? 128 : 64;
  p.mt = cdiv(m, p.bm);
  p.nt = cdiv(n, p.bm);
  const long long tiles = (long long)p.mt * p.nt;
  long long s = 1;
  if (tiles < 256) s = std::max<long long>(1, std::min<long long>((512 + tiles - 1) / tiles, k / 256));
  p.chunk = std::max(64, cdiv(cdiv(k, s), 64) * 64);
  p.nsplit = std::max(1, cdiv(k, p.chunk));
  return p;
}
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }
size_t split_bytes(int m, int n, int k) {
  const Plan p = plan_gemm(m, n, k);
  return p.nsplit > 1 ? align256((size_t)p.nsplit * m * n * sizeof(float)) : 0;
}
// workgroups along the rows of the dz / dbias pass
int dz_blocks(long long m, int n) {
  const long long cols = cdiv(n, 128);
  return (int)std::max<long long>(1, std::min<long long>((m + 31) / 32, (2048 + cols - 1) / cols));
}

template <typename T, bool TA, bool TB>
void launch_gemm(GemmArgs g, float *ws, hipStream_t hs) {
  const Plan p = plan_gemm(g.m, g.n, g.k);
  g.mt = p.mt; g.nt = p.nt; g.nsplit = p.nsplit; g.chunk = p.chunk; g.part = ws;
  const dim3 grid((unsigned)((long long)p.mt * p.nt * p.nsplit));
  if (p.bm == 128)
    hipLaunchKernelGGL((linear_gemm_kernel<T, TA, TB, 128, 128>), grid, dim3(256), 0, hs, g);
  else
    hipLaunchKernelGGL((linear_gemm_kernel<T, TA, TB, 64, 64>), grid, dim3(256), 0, hs, g);
  if (p.nsplit > 1) {
    const long long pieces = (long long)g.m * cdiv(g.n, Elem<T>::kVec);
    hipLaunchKernelGGL((linear_join_kernel<T>),
                       dim3((unsigned)std::min<long long>(4096, (pieces + 255) / 256)), dim3(256), 0,
                       hs, g);
  }
}

int check(const char *what, int dtype, int m, int n, int k, int act) {
  BTR_REQUIRE(dtype >= BTR_F32 && dtype <= BTR_F16, "%s: unknown element type %d", what, dtype);
  BTR_REQUIRE(act >= BTR_ACT_NONE && act <= BTR_ACT_GELU, "%s: unknown activation %d", what, act);
  BTR_REQUIRE(m >= 0 && n >= 1 && k >= 1 && m <= (1 << 30) && n <= (1 << 30) && k <= (1 << 30) &&
                  ((long long)cdiv(m, 64) * cdiv(n, 64) <= (1 << 30)) &&
                  ((long long)cdiv(m, 64) * cdiv(k, 64) <= (1 << 30)) &&
                  ((long long)cdiv(n, 64) * cdiv(k, 64) <= (1 << 30)),
              "%s: (%d, %d) x (%d, %d)", what, m, k, n, k);
  return BTR_OK;
}

}  // namespace
}  // namespace btr

using namespace btr;

extern "C" size_t btr_linear_fwd_workspace_bytes(int m, int n, int k) {
  if (check("linear_fwd", BTR_F32, m, n, k, 0) != BTR_OK || m == 0) return 0;
  return split_bytes(m, n, k);
}

extern "C" int btr_linear_fwd(int dtype, int m, int n, int k, const void *x, long long ldx,
                              const void *weight, long long ldw, const void *bias, int act,
                              const void *residual, long long ldr, void *y, void *z,
                              void *workspace, size_t workspace_bytes, btr_stream_t stream) {
  const int rc = check("linear_fwd", dtype, m, n, k, act);
  if (rc != BTR_OK) return rc;
  if (m == 0) return BTR_OK;
  BTR_REQUIRE(x && weight && y && ldx >= k && ldw >= k && (!residual || ldr >= n),
              "linear_fwd: null pointer or a row stride below the row");
  const size_t need = btr_linear_fwd_workspace_bytes(m, n, k);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "linear_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  GemmArgs g{};
  g.m = m; g.n = n; g.k = k;
  g.a = x; g.lda = ldx; g.b = weight; g.ldb = ldw;
  g.bias = bias; g.res = residual; g.ldres = ldr; g.act = act;
  g.c = y; g.z = z;
  BTR_DISPATCH_DTYPE(dtype, (launch_gemm<T, false, false>(g, (float *)workspace, as_stream(stream))));
  return check_launch("linear_fwd");
}

extern "C" size_t btr_linear_bwd_workspace_bytes(int dtype, int m, int n, int k) {
  if (check("linear_bwd", dtype, m, n, k, 0) != BTR_OK || m == 0) return 0;
  const size_t elem = dtype == BTR_F32 ? 4 : 2;
  return align256((size_t)m * n * elem) + align256((size_t)dz_blocks(m, n) * n * sizeof(float)) +
         std::max(split_bytes(m, k, n), split_bytes(n, k, m));
}

extern "C" int btr_linear_bwd(int dtype, int m, int n, int k, const void *x, long long ldx,
                              const void *weight, long long ldw, int act, const void *z,
                              const void *dy, long long lddy, void *dx, void *dweight,
                              void *dbias, void *workspace, size_t workspace_bytes,
                              btr_stream_t stream) {
  const int rc = check("linear_bwd", dtype, m, n, k, act);
  if (rc != BTR_OK) return rc;
  hipStream_t hs = as_stream(stream);
  BTR_REQUIRE(m == 0 || (dy && lddy >= n && (act == BTR_ACT_NONE || z) &&
                         (!dx || (weight && ldw >= k)) && (!dweight || (x && ldx >= k))),
              "linear_bwd: null pointer or a row stride below the row");
  const size_t need = btr_linear_bwd_workspace_bytes(dtype, m, n, k);
  BTR_REQUIRE(workspace_bytes >= need && (need == 0 || workspace),
              "linear_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
  const size_t elem = dtype == BTR_F32 ? 4 : 2;
  char *ws = (char *)workspace;
  void *dz = ws;
  float *part = (float *)(ws + align256((size_t)m * n * elem));
  float *share = (float *)((char *)part + align256((size_t)dz_blocks(m, n) * n * sizeof(float)));
  const void *gz = dy;                             // what the two products read
  long long ldg = lddy;
  if (m > 0 && (act != BTR_ACT_NONE || dbias)) {
    const int blocks = dz_blocks(m, n);
    BTR_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL(
        (linear_dz_kernel<T>), dim3(cdiv(n, 32 * Elem<T>::kVec), blocks), dim3(256), 0, hs,
        (long long)m, n, (const T *)dy, lddy, (const T *)z, act, (T *)dz, dbias ? part : nullptr));
    if (act != BTR_ACT_NONE) {
      gz = dz;
      ldg = n;
    }
  }
  if (dbias)   // (no rows: zeros)
    BTR_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL((linear_dbias_kernel<T>), dim3(cdiv(n, 32)),
                                                 dim3(256), 0, hs, part,
                                                 m > 0 ? dz_blocks(m, n) : 0, n, (T *)dbias));
  if (dx && m > 0) {
    GemmArgs g{};
    g.m = m; g.n = k; g.k = n;
    g.a = gz; g.lda = ldg; g.b = weight; g.ldb = ldw; g.c = dx;
    BTR_DISPATCH_DTYPE(dtype, (launch_gemm<T, false, true>(g, share, hs)));
  }
  if (dweight) {
    GemmArgs g{};
    g.m = n; g.n = k; g.k = m;                     // (no rows: an empty reduction writes zeros)
    g.a = gz; g.lda = ldg; g.b = x; g.ldb = ldx; g.c = dweight;
    BTR_DISPATCH_DTYPE(dtype, (launch_gemm<T, true, true>(g, share, hs)));
  }
  return check_launch("linear_bwd");
}
