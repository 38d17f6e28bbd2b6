// layer_norm.hip -- layer norm over the rows of a matrix, with the residual addition in front of it:
//
//   s = x [+ residual],  mean, rstd = 1 / sqrt(var(s) + eps) over the row,  xh = (s - mean) * rstd
//   y = xh * weight + bias
//   backward, t = dy * weight:
//   ds = rstd * (t - mean_row(t) - xh * mean_row(t * xh))        (the gradient of x AND residual)
//   dweight = sum_rows(dy * xh),  dbias = sum_rows(dy)
//
// (reference: the three nn.LayerNorm of detection/GroupFree3D/models/transformer.py:36-76 behind
// their residual additions; csrc/decoder.hip has the float32, dropout-carrying form that lives
// inside the whole-layer call.)
//
// Bound by HBM: forward reads x (and the residual) once and writes y; the backward reads x, residual
// and dy once and writes ds.  s is never stored: the backward adds x and the residual again, which
// moves the same bytes as writing s in the forward and reading it, and keeps s unrounded.  A row
// stays in the registers of one wave (up to 1 024 columns: no barrier at all), of a workgroup of four
// waves or of sixteen (up to 8 192; wider rows are read again per pass, out of L2); statistics are two
// passes over registers (mean, then the sum of squared deviations), in f32.  dweight / dbias: every
// thread keeps the f32 sums of its columns over the rows its workgroup visits, a second launch adds
// the workgroups' partial rows in a fixed order: no atomics, equal results from run to run.
// 32 768 x 2 048 bf16 with residual: forward 73 - 76 us, backward 108 - 112, both 5.0 TB/s, as a large
// copy, and 5 for the parameter sums.  1 024 x 288 f32 (a decoder layer's): 4.5, 6.8 and 3.0 us, a
// launch and one trip to memory each.  5 003 x 1 155 f16 off every boundary: 11.2 us, 2.1 TB/s.
#include <algorithm>

#include "decoder_ops.hpp"

namespace btr {
namespace {

struct LnArgs {
  long long rows;
  int width;
  const void *x, *res, *dy;
  long long ldx, ldr, lddy;
  const void *w, *b;
  float eps;
  void *out;        // y, or ds
  float *stats;     // (rows, 2): mean, rstd
  float *part;      // (blocks, 2 * width): dweight sums, dbias sums
};

// sums of NS values over the G threads that share a row, in every one of them.  G > 64: through
// LDS, one barrier; `slot` alternates so that the next reduction does not wait for this one's reads
template <int G, int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], float *lds, int &slot) {
#pragma unroll
  for (int i = 0; i < NS; ++i) v[i] = wave_sum_f32(v[i]);
  if (G == 64) return;
  constexpr int NW = G / 64;
  float *s = lds + slot * (NW * 2);
  slot ^= 1;
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
#pragma unroll
    for (int i = 0; i < NS; ++i) s[2 * w + i] = v[i];
  }
  lds_barrier();
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < NW; ++k) t += s[2 * k + i];
    v[i] = t;
  }
}

// G threads per row, NV 16-byte vectors per thread
template <typename T, int G, int NV>
__global__ __launch_bounds__(G == 64 ? 256 : G) void layer_norm_fwd_kernel(LnArgs a) {
  constexpr int V = Elem<T>::kVec, RPB = G == 64 ? 4 : 1;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[G / 64 * 4];
  const int lane = threadIdx.x % G;
  const long long row0 = (long long)blockIdx.x * RPB + threadIdx.x / G;
  const float inv_n = 1.f / (float)a.width;
  Vec w[NV], b[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e0 = (lane + G * i) * V;
    if (a.w) w[i] = load_row((const T *)a.w, e0, a.width);
    if (a.b) b[i] = load_row((const T *)a.b, e0, a.width);
  }
  int slot = 0;
  for (long long row = row0; row < a.rows; row += (long long)gridDim.x * RPB) {
    float s[NV][V], sum[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (lane + G * i) * V;
      const Vec x = load_row((const T *)a.x + row * a.ldx, e0, a.width);
      Vec r = {};
      if (a.res) r = load_row((const T *)a.res + row * a.ldr, e0, a.width);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[i][j] = (float)x[j] + (float)r[j];
        sum[0] += s[i][j];                       // (zero beyond the row)
      }
    }
    row_sum<G, 1>(sum, red, slot);
    const float mean = sum[0] * inv_n;
    float sq[1] = {0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s[i][j] -= mean;
        if ((lane + G * i) * V + j < a.width) sq[0] = fmaf(s[i][j], s[i][j], sq[0]);
      }
    row_sum<G, 1>(sq, red, slot);
    const float rstd = 1.f / sqrtf(fmaf(sq[0], inv_n, a.eps));
    if (a.stats && lane == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec y;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float v = s[i][j] * rstd;
        if (a.w) v *= (float)w[i][j];
        if (a.b) v += (float)b[i][j];
        y[j] = (T)v;
      }
      store_row((T *)a.out + row * a.width, (lane + G * i) * V, a.width, y);
    }
  }
}

template <typename T, int G, int NV>
__global__ __launch_bounds__(G == 64 ? 256 : G) void layer_norm_bwd_kernel(LnArgs a) {
  constexpr int V = Elem<T>::kVec, RPB = G == 64 ? 4 : 1;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[G / 64 * 4];
  extern __shared__ float cols[];                // G == 64: 2 * width sums of the four waves
  const int lane = threadIdx.x % G;
  const long long row0 = (long long)blockIdx.x * RPB + threadIdx.x / G;
  const float inv_n = 1.f / (float)a.width;
  Vec w[NV];
  float dw[NV][V], db[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (a.w) w[i] = load_row((const T *)a.w, (lane + G * i) * V, a.width);
#pragma unroll
    for (int j = 0; j < V; ++j) dw[i][j] = db[i][j] = 0.f;
  }
  int slot = 0;
  for (long long row = row0; row < a.rows; row += (long long)gridDim.x * RPB) {
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    Vec xv[NV], rv[NV], gv[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int e0 = (lane + G * i) * V;
      xv[i] = load_row((const T *)a.x + row * a.ldx, e0, a.width);
      if (a.res) rv[i] = load_row((const T *)a.res + row * a.ldr, e0, a.width);
      gv[i] = load_row((const T *)a.dy + row * a.lddy, e0, a.width);
    }
    float xh[NV][V], c[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float s = (float)xv[i][j];
        if (a.res) s += (float)rv[i][j];
        s = (s - mean) * rstd;
        xh[i][j] = (lane + G * i) * V + j < a.width ? s : 0.f;
        const float g = (float)gv[i][j];
        dw[i][j] = fmaf(g, xh[i][j], dw[i][j]);
        db[i][j] += g;
        const float t = a.w ? g * (float)w[i][j] : g;
        c[0] += t;
        c[1] = fmaf(t, xh[i][j], c[1]);
      }
    row_sum<G, 2>(c, red, slot);
    c[0] *= inv_n;
    c[1] *= inv_n;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      Vec o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float g = (float)gv[i][j];
        const float t = a.w ? g * (float)w[i][j] : g;
        o[j] = (T)(rstd * (t - c[0] - xh[i][j] * c[1]));
      }
      store_row((T *)a.out + row * a.width, (lane + G * i) * V, a.width, o);
    }
  }
  if (!a.part) return;
  float *part = a.part + (long long)blockIdx.x * 2 * a.width;
  if (G == 64) {   // the four waves hold the same columns: add them in wave order
    for (int k = 0; k < 4; ++k) {
      if ((int)(threadIdx.x >> 6) == k) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const int e = (lane + G * i) * V + j;
            if (e < a.width) {
              cols[e] = dw[i][j] + (k ? cols[e] : 0.f);
              cols[a.width + e] = db[i][j] + (k ? cols[a.width + e] : 0.f);
            }
          }
      }
      __syncthreads();
    }
    for (int e = threadIdx.x; e < 2 * a.width; e += 256) part[e] = cols[e];
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const int e = (lane + G * i) * V + j;
        if (e < a.width) {
          part[e] = dw[i][j];
          part[a.width + e] = db[i][j];
        }
      }
  }
}

// column sums of part (blocks, 2 * width) -> dweight, dbias
template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_params_kernel(const float *part, int blocks,
                                                                 int width, T *dw, T *db) {
  for (long long c0 = blockIdx.x * 32ll; c0 < 2ll * width; c0 += gridDim.x * 32ll) {
    const long long c = c0 + (threadIdx.x & 31);
    const float t = column_sum(part, blocks, 2ll * width, c);
    if (threadIdx.x < 32 && c < 2ll * width) {
      if (c < width) {
        if (dw) dw[c] = (T)t;
      } else if (db) {
        db[c - width] = (T)t;
      }
    }
    __syncthreads();                             // (its LDS is used again)
  }
}

// ---- rows wider than a workgroup's registers hold (8 192): the row is read once per pass, the
// later passes out of L2; the parameter sums are a launch of their own (their columns do not fit
// the registers either)
template <typename T>
__device__ __forceinline__ void wide_s(const LnArgs &a, long long row, int e0,
                                       float (&s)[Elem<T>::kVec]) {
  const typename Elem<T>::Vec x = load_row((const T *)a.x + row * a.ldx, e0, a.width);
  typename Elem<T>::Vec r = {};
  if (a.res) r = load_row((const T *)a.res + row * a.ldr, e0, a.width);
#pragma unroll
  for (int j = 0; j < Elem<T>::kVec; ++j) s[j] = (float)x[j] + (float)r[j];
}

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_fwd_wide_kernel(LnArgs a) {
  constexpr int V = Elem<T>::kVec;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[1024 / 64 * 4];
  const float inv_n = 1.f / (float)a.width;
  int slot = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float sum[1] = {0.f}, sq[1] = {0.f}, s[V];
    for (int e0 = threadIdx.x * V; e0 < a.width; e0 += 1024 * V) {
      wide_s<T>(a, row, e0, s);
#pragma unroll
      for (int j = 0; j < V; ++j) sum[0] += s[j];
    }
    row_sum<1024, 1>(sum, red, slot);
    const float mean = sum[0] * inv_n;
    for (int e0 = threadIdx.x * V; e0 < a.width; e0 += 1024 * V) {
      wide_s<T>(a, row, e0, s);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (e0 + j < a.width) sq[0] = fmaf(s[j] - mean, s[j] - mean, sq[0]);
    }
    row_sum<1024, 1>(sq, red, slot);
    const float rstd = 1.f / sqrtf(fmaf(sq[0], inv_n, a.eps));
    if (a.stats && threadIdx.x == 0) {
      a.stats[2 * row] = mean;
      a.stats[2 * row + 1] = rstd;
    }
    for (int e0 = threadIdx.x * V; e0 < a.width; e0 += 1024 * V) {
      wide_s<T>(a, row, e0, s);
      Vec w, b, y;
      if (a.w) w = load_row((const T *)a.w, e0, a.width);
      if (a.b) b = load_row((const T *)a.b, e0, a.width);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        float v = (s[j] - mean) * rstd;
        if (a.w) v *= (float)w[j];
        if (a.b) v += (float)b[j];
        y[j] = (T)v;
      }
      store_row((T *)a.out + row * a.width, e0, a.width, y);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void layer_norm_bwd_wide_kernel(LnArgs a) {
  constexpr int V = Elem<T>::kVec;
  typedef typename Elem<T>::Vec Vec;
  __shared__ float red[1024 / 64 * 4];
  const float inv_n = 1.f / (float)a.width;
  int slot = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    float c[2] = {0.f, 0.f}, s[V];
    for (int pass = 0; pass < 2; ++pass) {
      for (int e0 = threadIdx.x * V; e0 < a.width; e0 += 1024 * V) {
        wide_s<T>(a, row, e0, s);
        const Vec g = load_row((const T *)a.dy + row * a.lddy, e0, a.width);
        Vec w, o;
        if (a.w) w = load_row((const T *)a.w, e0, a.width);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float xh = e0 + j < a.width ? (s[j] - mean) * rstd : 0.f;
          const float t = a.w ? (float)g[j] * (float)w[j] : (float)g[j];
          if (pass == 0) {
            c[0] += t;
            c[1] = fmaf(t, xh, c[1]);
          } else {
            o[j] = (T)(rstd * (t - c[0] - xh * c[1]));
          }
        }
        if (pass) store_row((T *)a.out + row * a.width, e0, a.width, o);
      }
      if (pass == 0) {
        row_sum<1024, 2>(c, red, slot);
        c[0] *= inv_n;
        c[1] *= inv_n;
      }
    }
  }
}

// partial parameter sums: thread = one vector of columns, blockIdx.y = a strided share of the rows
template <typename T>
__global__ __launch_bounds__(256) void layer_norm_cols_wide_kernel(LnArgs a) {
  constexpr int V = Elem<T>::kVec;
  const int e0 = (blockIdx.x * 256 + threadIdx.x) * V;
  if (e0 >= a.width) return;
  float dw[V] = {}, db[V] = {}, s[V];
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float mean = a.stats[2 * row], rstd = a.stats[2 * row + 1];
    wide_s<T>(a, row, e0, s);
    const typename Elem<T>::Vec g = load_row((const T *)a.dy + row * a.lddy, e0, a.width);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      dw[j] = fmaf((float)g[j], (s[j] - mean) * rstd, dw[j]);
      db[j] += (float)g[j];
    }
  }
  float *part = a.part + (long long)blockIdx.y * 2 * a.width;
#pragma unroll
  for (int j = 0; j < V; ++j)
    if (e0 + j < a.width) {
      part[e0 + j] = dw[j];
      part[a.width + e0 + j] = db[j];
    }
}

constexpr int kWide = 8192;   // register-resident up to here

// rows of the partial sums: the backward's workgroups (wide rows: the row shares)
int ln_bwd_blocks(long long rows, int width) {
  const long long per = width <= 1024 ? 4 : 1, most = width <= kWide ? 1024 : 64;
  return (int)std::max<long long>(1, std::min<long long>(most, (rows + per - 1) / per));
}

// Threads per row and vectors per thread: at most 16 elements a thread (a float and two sums of
// each live in the backward's registers) except where one wave still holds the row.
template <typename T>
int launch(const LnArgs &a, bool bwd, hipStream_t hs) {
  constexpr int V = Elem<T>::kVec;
  const int cap = bwd ? ln_bwd_blocks(a.rows, a.width) : 2048;
#define BTR_LN(G, NV)                                                                           \
  do {                                                                                          \
    const int rpb = (G) == 64 ? 4 : 1, thr = (G) == 64 ? 256 : (G);                             \
    const int grid = (int)std::min<long long>(cap, (a.rows + rpb - 1) / rpb);                   \
    if (bwd)                                                                                    \
      hipLaunchKernelGGL((layer_norm_bwd_kernel<T, G, NV>), dim3(grid), dim3(thr),              \
                         (G) == 64 ? 2 * a.width * sizeof(float) : 0, hs, a);                   \
    else                                                                                        \
      hipLaunchKernelGGL((layer_norm_fwd_kernel<T, G, NV>), dim3(grid), dim3(thr), 0, hs, a);   \
    return grid;                                                                                \
  } while (0)
  if (a.width <= 64 * V) BTR_LN(64, 1);
  if (a.width <= 128 * V) BTR_LN(64, 2);
  if (V == 4) {
    if (a.width <= 1024) BTR_LN(64, 8 / V * 2);
    if (a.width <= 2048) BTR_LN(256, 8 / V);
    if (a.width <= 4096) BTR_LN(256, 8 / V * 2);
    if (a.width <= kWide) BTR_LN(1024, 8 / V);
  } else {
    if (a.width <= 2048) BTR_LN(256, 1);
    if (a.width <= 4096) BTR_LN(256, 2);
    if (a.width <= kWide) BTR_LN(1024, 8 / V);
  }
#undef BTR_LN
  const int grid = (int)std::min<long long>(2048, a.rows);
  if (!bwd) {
    hipLaunchKernelGGL((layer_norm_fwd_wide_kernel<T>), dim3(grid), dim3(1024), 0, hs, a);
    return grid;
  }
  hipLaunchKernelGGL((layer_norm_bwd_wide_kernel<T>), dim3(grid), dim3(1024), 0, hs, a);
  if (a.part)
    hipLaunchKernelGGL((layer_norm_cols_wide_kernel<T>), dim3(cdiv(a.width, 256 * V), cap),
                       dim3(256), 0, hs, a);
  return cap;
}

int check(const char *what, int dtype, long long rows, int width, const void *x, long long ldx,
          const void *res, long long ldr) {
  BTR_REQUIRE(dtype >= BTR_F32 && dtype <= BTR_F16, "%s: unknown element type %d", what, dtype);
  BTR_REQUIRE(rows >= 0 && width >= 1 && width <= (1 << 28), "%s: rows %lld, width %d",
              what, rows, width);
  BTR_REQUIRE(rows == 0 || (x && ldx >= width && (!res || ldr >= width)),
              "%s: null pointer or a row stride below the width", what);
  return BTR_OK;
}

}  // namespace
}  // namespace btr

using namespace btr;

extern "C" int btr_layer_norm_fwd(int dtype, long long rows, int width, const void *x,
                                  long long ldx, const void *residual, long long ldr,
                                  const void *weight, const void *bias, float eps, void *y,
                                  float *stats, btr_stream_t stream) {
  const int rc = check("layer_norm_fwd", dtype, rows, width, x, ldx, residual, ldr);
  if (rc != BTR_OK) return rc;
  if (rows == 0) return BTR_OK;
  BTR_REQUIRE(y, "layer_norm_fwd: null pointer");
  const LnArgs a{rows, width, x, residual, nullptr, ldx, ldr, 0, weight, bias, eps, y, stats,
                 nullptr};
  BTR_DISPATCH_DTYPE(dtype, launch<T>(a, false, as_stream(stream)));
  return check_launch("layer_norm_fwd");
}

extern "C" size_t btr_layer_norm_bwd_workspace_bytes(long long rows, int width) {
  if (rows <= 0 || width <= 0) return 0;
  return (size_t)ln_bwd_blocks(rows, width) * 2 * width * sizeof(float);
}

extern "C" int btr_layer_norm_bwd(int dtype, long long rows, int width, const void *x,
                                  long long ldx, const void *residual, long long ldr,
                                  const void *dy, long long lddy, const void *weight,
                                  const float *stats, void *dx, void *dweight, void *dbias,
                                  void *workspace, size_t workspace_bytes, btr_stream_t stream) {
  const int rc = check("layer_norm_bwd", dtype, rows, width, x, ldx, residual, ldr);
  if (rc != BTR_OK) return rc;
  const bool params = dweight || dbias;
  BTR_REQUIRE(rows == 0 || (dy && lddy >= width && stats && dx),
              "layer_norm_bwd: null pointer or a row stride below the width");
  BTR_REQUIRE(rows == 0 || !params ||
                  (workspace && workspace_bytes >= btr_layer_norm_bwd_workspace_bytes(rows, width)),
              "layer_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes,
              btr_layer_norm_bwd_workspace_bytes(rows, width));
  hipStream_t hs = as_stream(stream);
  int blocks = 0;
  if (rows > 0) {
    const LnArgs a{rows, width, x, residual, dy, ldx, ldr, lddy, weight, nullptr, 0.f, dx,
                   const_cast<float *>(stats), params ? (float *)workspace : nullptr};
    BTR_DISPATCH_DTYPE(dtype, blocks = launch<T>(a, true, hs));
  }
  if (params)   // (no rows: zeros)
    BTR_DISPATCH_DTYPE(dtype, hipLaunchKernelGGL(
        (layer_norm_params_kernel<T>), dim3(std::min(1 << 20, cdiv(2ll * width, 32))), dim3(1024), 0, hs,
        (const float *)workspace, blocks, width, (T *)dweight, (T *)dbias));
  return check_launch("layer_norm_bwd");
}
