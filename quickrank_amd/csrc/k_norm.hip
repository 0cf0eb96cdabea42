// k_norm.hip -- layer norm over the rows of a matrix, forward and backward.
//
//   mu = sum_j x_j / C,  r = 1 / sqrt(sum_j (x_j - mu)^2 / C + eps),  y_j = (x_j - mu) r w_j + b_j
//   xh_j = (x_j - mu) r,  g_j = dy_j w_j
//   dx_j = r (g_j - mean(g) - xh_j mean(g xh)),  dw_j = sum_rows dy_j xh_j,  db_j = sum_rows dy_j
//
// Statistics and sums are held in 32 bits; outputs are rounded once.
#include "qr_dense.h"

namespace {

__device__ __forceinline__ float wave_sum_f(float v) {
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// one wave per row
template <class T, class P>
__global__ __launch_bounds__(256) void k_norm(const size_t rows, const int cols, const T *__restrict__ x, const size_t ldx,
                                              const P *__restrict__ w, const P *__restrict__ b, const float eps, T *__restrict__ y,
                                              const size_t ldy, float *__restrict__ mean, float *__restrict__ rstd) {
  const int lane = threadIdx.x & 63;
  for (size_t r = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (size_t)gridDim.x * 4) {
    const T *xr = x + r * ldx;
    float s = 0.f;
    for (int j = lane; j < cols; j += 64) s += (float)xr[j];
    const float mu = wave_sum_f(s) / (float)cols;
    float q = 0.f;
    for (int j = lane; j < cols; j += 64) {
      const float d = (float)xr[j] - mu;
      q = fmaf(d, d, q);
    }
    const float rs = 1.f / sqrtf(wave_sum_f(q) / (float)cols + eps);
    for (int j = lane; j < cols; j += 64) {
      const float h = ((float)xr[j] - mu) * rs;
      y[r * ldy + j] = (T)fmaf(h, w ? (float)w[j] : 1.f, b ? (float)b[j] : 0.f);
    }
    if (lane == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <class T, class P>
__global__ __launch_bounds__(256) void k_norm_dx(const size_t rows, const int cols, const T *dy, const size_t lddy, const T *x,
                                                 const size_t ldx, const P *__restrict__ w, const float *__restrict__ mean,
                                                 const float *__restrict__ rstd, T *dx, const size_t lddx) {
  const int lane = threadIdx.x & 63;
  for (size_t r = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (size_t)gridDim.x * 4) {
    const float mu = mean[r], rs = rstd[r];
    float a = 0.f, c = 0.f;
    for (int j = lane; j < cols; j += 64) {
      const float g = (float)dy[r * lddy + j] * (w ? (float)w[j] : 1.f), h = ((float)x[r * ldx + j] - mu) * rs;
      a += g;
      c = fmaf(g, h, c);
    }
    a = wave_sum_f(a) / (float)cols;
    c = wave_sum_f(c) / (float)cols;
    for (int j = lane; j < cols; j += 64) {
      const float g = (float)dy[r * lddy + j] * (w ? (float)w[j] : 1.f), h = ((float)x[r * ldx + j] - mu) * rs;
      dx[r * lddx + j] = (T)(rs * (g - a - h * c));
    }
  }
}

constexpr int PARTS = 256;  // shares of the rows whose column sums are joined in a second launch

template <class T>
__global__ __launch_bounds__(256) void k_norm_cols(const size_t rows, const int cols, const T *__restrict__ dy, const size_t lddy,
                                                   const T *__restrict__ x, const size_t ldx, const float *__restrict__ mean,
                                                   const float *__restrict__ rstd, float *__restrict__ part) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= cols) return;
  const size_t r0 = rows * blockIdx.y / PARTS, r1 = rows * (blockIdx.y + 1) / PARTS;
  float sw = 0.f, sb = 0.f;
  for (size_t r = r0; r < r1; ++r) {
    const float d = (float)dy[r * lddy + j];
    sw = fmaf(d, ((float)x[r * ldx + j] - mean[r]) * rstd[r], sw);
    sb += d;
  }
  part[(size_t)blockIdx.y * 2 * cols + j] = sw;
  part[(size_t)blockIdx.y * 2 * cols + cols + j] = sb;
}

template <class P>
__global__ __launch_bounds__(256) void k_norm_join(const int cols, const int parts, const float *__restrict__ part, P *__restrict__ dw, P *__restrict__ db) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= cols) return;
  float sw = 0.f, sb = 0.f;
  for (int p = 0; p < parts; ++p) {
    sw += part[(size_t)p * 2 * cols + j];
    sb += part[(size_t)p * 2 * cols + cols + j];
  }
  if (dw) dw[j] = (P)sw;
  if (db) db[j] = (P)sb;
}

}  // namespace

extern "C" int qr_layer_norm_async(int device, void *stream, int type, int param_type, size_t rows, size_t cols, const void *x,
                                   size_t ldx, const void *weight, const void *bias, float eps, void *y, size_t ldy, float *mean,
                                   float *rstd) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "layer norm: unknown element type");
  QR_DENSE_ARG(param_type == type || param_type == QR_F32, "layer norm: weight and bias have the rows' type or f32");
  QR_DENSE_ARG(cols > 0, "layer norm: rows of no columns");
  QR_DENSE_ARG(eps >= 0.f && eps < INFINITY, "layer norm: eps is a finite number of at least 0");
  QR_DENSE_ARG(qr_dense_fits(rows, cols, ldx) && qr_dense_fits(rows, cols, ldy), "layer norm: sizes out of range");
  QR_DENSE_ARG(rows < 2 || ldy >= cols, "layer norm: the stride of y is shorter than a row");
  if (!rows) return QR_OK;
  QR_DENSE_ARG(x && y, "layer norm: x or y is NULL");
  QR_DENSE_DEVICE(device);
  const unsigned grid = (unsigned)((rows + 3) / 4 < 4096 ? (rows + 3) / 4 : 4096);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      k_norm<T, P><<<grid, 256, 0, (hipStream_t)stream>>>(rows, (int)cols, (const T *)x, ldx, (const P *)weight, (const P *)bias, eps,
                                                         (T *)y, ldy, mean, rstd);
    };
    if (param_type == QR_F32) go(float{});
    else go(T{});
  });
  return qr_dense_launched("layer norm");
}

extern "C" int qr_layer_norm_backward_workspace(size_t rows, size_t cols, size_t *bytes) {
  QR_DENSE_ARG(bytes && cols > 0 && cols < ((size_t)1 << 31), "layer norm backward: bad size");
  *bytes = rows ? (size_t)PARTS * 2 * cols * 4 : 0;
  return QR_OK;
}

extern "C" int qr_layer_norm_backward_async(int device, void *stream, int type, int param_type, size_t rows, size_t cols,
                                            const void *dy, size_t lddy, const void *x, size_t ldx, const void *weight,
                                            const float *mean, const float *rstd, void *dx, size_t lddx, void *dweight, void *dbias,
                                            void *workspace, size_t workspace_bytes) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "layer norm backward: unknown element type");
  QR_DENSE_ARG(param_type == type || param_type == QR_F32, "layer norm backward: weight and bias have the rows' type or f32");
  QR_DENSE_ARG(cols > 0, "layer norm backward: rows of no columns");
  QR_DENSE_ARG(qr_dense_fits(rows, cols, ldx) && qr_dense_fits(rows, cols, lddy) && qr_dense_fits(rows, cols, lddx),
               "layer norm backward: sizes out of range");
  QR_DENSE_ARG(!dx || rows < 2 || lddx >= cols, "layer norm backward: the stride of dx is shorter than a row");
  QR_DENSE_ARG(!rows || (dy && x && mean && rstd), "layer norm backward: dy, x, mean or rstd is NULL");
  const bool sums = dweight || dbias;
  size_t need = 0;
  (void)qr_layer_norm_backward_workspace(rows, cols, &need);
  QR_DENSE_ARG(!sums || !rows || (workspace && workspace_bytes >= need), "layer norm backward: the workspace is too small");
  QR_DENSE_DEVICE(device);
  const hipStream_t s = (hipStream_t)stream;
  const unsigned grid = (unsigned)((rows + 3) / 4 < 4096 ? (rows + 3) / 4 : 4096), cb = (unsigned)((cols + 255) / 256);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      // (the column sums first: dx may be written over dy or x)
      if (sums) {
        if (rows)
          k_norm_cols<T><<<dim3(cb, PARTS), 256, 0, s>>>(rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, mean, rstd,
                                                        (float *)workspace);
        k_norm_join<P><<<cb, 256, 0, s>>>((int)cols, rows ? PARTS : 0, (const float *)workspace, (P *)dweight, (P *)dbias);
      }
      if (dx && rows)
        k_norm_dx<T, P><<<grid, 256, 0, s>>>(rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)weight, mean, rstd,
                                            (T *)dx, lddx);
    };
    if (param_type == QR_F32) go(float{});
    else go(T{});
  });
  return qr_dense_launched("layer norm backward");
}
