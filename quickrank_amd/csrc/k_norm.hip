// k_norm.hip -- layer norm over the rows of a matrix, forward and backward.
//
//   mu = sum_j x_j / C,  r = 1 / sqrt(sum_j (x_j - mu)^2 / C + eps),  y_j = (x_j - mu) r w_j + b_j
//   xh_j = (x_j - mu) r,  g_j = dy_j w_j
//   dx_j = r (g_j - mean(g) - xh_j mean(g xh)),  dw_j = sum_rows dy_j xh_j,  db_j = sum_rows dy_j
//
// Statistics and sums are held in 32 bits; outputs are rounded once.  Bound by memory: a row is read once, kept
// in the registers of G lanes (16 for short rows, a wave, or a workgroup of four) as pieces of 16 bytes, and the
// variance is taken from the mean, not from the squares.  The backward pass reads a row of dy and of x once for
// dx and for the two column sums: a lane owns the same columns of every row its workgroup takes, adds them up in
// registers, and the workgroups' sums are joined by a second launch in a fixed order.
//
// Measured, where a copy of the same bytes reaches 4.9 to 5.4 TB/s: forward 1000000 x 136 f32 208 us (5.3 TB/s); backward
// with its join 65536 x 2048 bf16 160 + 10 us (4.7), 71291 x 1001 f16 89 + 6 us (4.5); 100 x 136 f32 4.0 us, a launch.
#include <algorithm>
#include <type_traits>

#include "qr_dense.h"

namespace {

template <int CTRL>
__device__ __forceinline__ float dpp(const float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_of(const float v, const int l) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
// sums over groups of G lanes, in a fixed order: every lane gets its group's (G > 64: the workgroup's, through `lds`)
template <int G>
__device__ __forceinline__ float wave_part(float v) {
  v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
  v += dpp<0x141>(v);  // row_half_mirror
  v += dpp<0x140>(v);  // row_mirror
  if constexpr (G >= 64) v = (lane_of(v, 0) + lane_of(v, 16)) + (lane_of(v, 32) + lane_of(v, 48));
  return v;
}
template <int G>
__device__ __forceinline__ void group_sum(float &a, float &b, float *lds) {
  a = wave_part<G>(a);
  b = wave_part<G>(b);
  if constexpr (G > 64) {
    constexpr int W = G / 64;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) {
      lds[threadIdx.x >> 6] = a;
      lds[W + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = lds[0], b = lds[W];
#pragma unroll
    for (int j = 1; j < W; ++j) {
      a += lds[j];
      b += lds[W + j];
    }
  }
}
template <int G>
__device__ __forceinline__ float group_sum(float a, float *lds) {
  float none = 0.f;
  if constexpr (G > 64) group_sum<G>(a, none, lds);
  else a = wave_part<G>(a);
  return a;
}

// The pieces of a row that lane l of G holds: l, l + G, ...; the last piece of a row is moved back to end with the
// row, so that every load and store is a whole one, and its first `dup` elements belong to the piece before it.
template <class T, int G>
struct Pieces {
  static constexpr int V = 16 / sizeof(T);
  int cols, last;  // columns; the last piece
  __device__ __forceinline__ Pieces(int c) : cols(c), last((c - 1) / V) {}
  // the pieces l + G i of all lanes lie inside the row, none of them the last
  __device__ __forceinline__ bool inner(int i) const { return G * (i + 1) <= last; }
  __device__ __forceinline__ bool any(int i, int l) const { return l + G * i <= last; }
  __device__ __forceinline__ int at(int i, int l) const { return l + G * i < last ? (l + G * i) * V : cols - V; }
  __device__ __forceinline__ int dup(int i, int l) const { return (l + G * i) * V - at(i, l); }
};

template <class T>
struct Raw {
  T v[16 / sizeof(T)];
};
template <class T>
__device__ __forceinline__ Raw<T> load(const T *p) {
  Raw<T> r;
  __builtin_memcpy(&r, p, 16);
  return r;
}
template <class P, int V>
__device__ __forceinline__ void load_params(const P *p, const int at, const float none, float (&v)[V]) {
  if (p) {
    P t[V];
    __builtin_memcpy(t, p + at, sizeof t);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (float)t[e];
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = none;
  }
}

// One row a group of lanes, read and written once: bound by memory.  (Sixteen lanes up to 1 KB: a wave has loads of four
// rows under way, and a row's sum is four lane exchanges.)
template <class T, class P, int G, int N>
__global__ __launch_bounds__(256) void k_norm(const size_t rows, const int cols, const T *x, const size_t ldx, const P *__restrict__ w,
                                              const P *__restrict__ b, const float eps, T *y, const size_t ldy,
                                              float *__restrict__ mean, float *__restrict__ rstd) {
  constexpr int V = Pieces<T, G>::V;
  __shared__ float lds[8];
  const Pieces<T, G> S(cols);
  const int l = threadIdx.x % G;
  const size_t mine = (size_t)blockIdx.x * (256 / G) + threadIdx.x / G, r = mine < rows ? mine : rows - 1;
  Raw<T> raw[N];
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (S.inner(i) || S.any(i, l)) raw[i] = load(x + r * ldx + S.at(i, l));
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (S.inner(i)) {
#pragma unroll
      for (int e = 0; e < V; ++e) s += (float)raw[i].v[e];
    } else if (S.any(i, l)) {
      const int dup = S.dup(i, l);
#pragma unroll
      for (int e = 0; e < V; ++e) s += e >= dup ? (float)raw[i].v[e] : 0.f;
    }
  }
  const float mu = group_sum<G>(s, lds) / (float)cols;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (S.inner(i)) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (float)raw[i].v[e] - mu;
        s = fmaf(d, d, s);
      }
    } else if (S.any(i, l)) {
      const int dup = S.dup(i, l);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = e >= dup ? (float)raw[i].v[e] - mu : 0.f;
        s = fmaf(d, d, s);
      }
    }
  }
  const float rs = 1.f / sqrtf(group_sum<G>(s, lds) / (float)cols + eps);
  if (mine >= rows) return;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (S.inner(i) || S.any(i, l)) {
      const int at = S.at(i, l);
      float vw[V], vb[V];
      load_params<P, V>(w, at, 1.f, vw);
      load_params<P, V>(b, at, 0.f, vb);
      Raw<T> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = (T)fmaf(((float)raw[i].v[e] - mu) * rs, vw[e], vb[e]);
      __builtin_memcpy(y + r * ldy + at, &o, 16);
    }
  }
  if (l == 0) {
    if (mean) mean[r] = mu;
    if (rstd) rstd[r] = rs;
  }
}

// Rows one after the other, the next one's pieces under way: bound by memory.  A lane's column sums stay in registers for
// all of its workgroup's rows, so the workgroups are few (parts_of) and their sums small beside the rows.
// part: [workgroup][2][cols] column sums of the rows a workgroup took, or NULL; of a single workgroup they go straight to
// dw and db
template <class T, class P, int G, int N>
__global__ __launch_bounds__(G > 256 ? G : 256) void k_norm_grad(const size_t rows, const int cols, const T *dy, const size_t lddy, const T *x,
                                                   const size_t ldx, const P *__restrict__ w, const float *__restrict__ mean,
                                                   const float *__restrict__ rstd, T *dx, const size_t lddx, float *__restrict__ part,
                                                   P *__restrict__ dw, P *__restrict__ db) {
  constexpr int V = Pieces<T, G>::V, RPB = G > 256 ? 1 : 256 / G;
  __shared__ float lds[32];
  const Pieces<T, G> S(cols);
  const int l = threadIdx.x % G, grp = threadIdx.x / G;
  const float inv = 1.f / (float)cols;
  float sw[N][V], sb[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int e = 0; e < V; ++e) sw[i][e] = sb[i][e] = 0.f;

  // a row's pieces are on their way while the row before is worked on; a group without a row works on zeros
  Raw<T> nx[N], nd[N];
  auto fetch = [&](const size_t first) {  // -> the row's mean and rstd
    const size_t r = first + grp;
    const bool live = r < rows;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      nx[i] = nd[i] = Raw<T>{};
      if (live && (S.inner(i) || S.any(i, l))) {
        nx[i] = load(x + r * ldx + S.at(i, l));
        nd[i] = load(dy + r * lddy + S.at(i, l));
      }
    }
    return live ? float2{mean[r], rstd[r]} : float2{0.f, 0.f};
  };
  size_t first = (size_t)blockIdx.x * RPB;
  float2 stat = {0.f, 0.f};
  if (first < rows) stat = fetch(first);
  for (; first < rows; first += (size_t)gridDim.x * RPB) {
    float h[N][V], g[N][V], sg = 0.f, sh = 0.f;
    const float mu = stat.x, rs = stat.y;
    const size_t r = first + grp;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!S.inner(i) && !S.any(i, l)) continue;
      const int dup = S.dup(i, l);
      float vw[V];
      load_params<P, V>(w, S.at(i, l), 1.f, vw);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (float)nd[i].v[e];
        h[i][e] = ((float)nx[i].v[e] - mu) * rs;
        g[i][e] = d * vw[e];
        const float once = e >= dup ? g[i][e] : 0.f;
        sg += once;
        sh = fmaf(once, h[i][e], sh);
        // (what a moved-back piece adds up in its first `dup` columns is not read)
        sw[i][e] = fmaf(d, h[i][e], sw[i][e]);
        sb[i][e] += d;
      }
    }
    if (first + (size_t)gridDim.x * RPB < rows) stat = fetch(first + (size_t)gridDim.x * RPB);
    if (!dx) continue;
    group_sum<G>(sg, sh, lds);
    const float a = -rs * (sg * inv), c = -rs * (sh * inv);
    if (r >= rows) continue;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!S.inner(i) && !S.any(i, l)) continue;
      Raw<T> o;
#pragma unroll
      for (int e = 0; e < V; ++e) o.v[e] = (T)fmaf(h[i][e], c, fmaf(g[i][e], rs, a));
      __builtin_memcpy(dx + r * lddx + S.at(i, l), &o, 16);
    }
  }
  if (!part) return;
  const bool direct = gridDim.x == 1;
  auto keep = [&](const int j, const float vw, const float vb) {
    if (direct) {
      if (dw) dw[j] = (P)vw;
      if (db) db[j] = (P)vb;
    } else {
      part[(size_t)blockIdx.x * 2 * cols + j] = vw;
      part[((size_t)blockIdx.x * 2 + 1) * cols + j] = vb;
    }
  };
  // a wave's groups are added by their lanes, the four waves' sums through LDS (each column has one owner in a group)
  extern __shared__ float sum[];
  float *const own = sum + (threadIdx.x >> 6) * 2 * cols;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (!S.inner(i) && !S.any(i, l)) continue;
    const int at = S.at(i, l), dup = S.dup(i, l);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float vw = sw[i][e], vb = sb[i][e];
      if constexpr (G < 64) {
        vw += __shfl_xor(vw, 16), vb += __shfl_xor(vb, 16);
        vw += __shfl_xor(vw, 32), vb += __shfl_xor(vb, 32);
      }
      if (e < dup || (threadIdx.x & 63) >= G) continue;
      if constexpr (RPB == 1) keep(at + e, vw, vb);
      else own[at + e] = vw, own[cols + at + e] = vb;
    }
  }
  if constexpr (RPB > 1) {
    __syncthreads();
    for (int j = threadIdx.x; j < cols; j += 256) {
      const float *const v = sum + j, *const u = v + cols;
      keep(j, (v[0] + v[2 * cols]) + (v[4 * cols] + v[6 * cols]), (u[0] + u[2 * cols]) + (u[4 * cols] + u[6 * cols]));
    }
  }
}

// Partial sums joined in a fixed order: 1024 / Q columns by Q shares
template <class P, int Q>
__global__ __launch_bounds__(1024) void k_norm_join(const int cols, const int parts, const float *__restrict__ part, P *__restrict__ dw,
                                                    P *__restrict__ db) {
  constexpr int W = 1024 / Q;
  __shared__ float lds[Q][W + 1];
  const int c = threadIdx.x % W, q = threadIdx.x / W;
  const size_t j = (size_t)blockIdx.x * W + c, n = 2 * (size_t)cols;
  float s = 0.f;
  if (j < n)
#pragma unroll 4
    for (int p = q; p < parts; p += Q) s += part[p * n + j];
  lds[q][c] = s;
  __syncthreads();
  if constexpr (Q == 64) {
    if (threadIdx.x < 256) {
      // four shares a thread, then the four quarters of a column's sixteen
      const int h = threadIdx.x >> 4;
      s = (lds[4 * h][c] + lds[4 * h + 1][c]) + (lds[4 * h + 2][c] + lds[4 * h + 3][c]);
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
    }
    __syncthreads();
    if (threadIdx.x < 256 && (threadIdx.x & 63) < 16) lds[threadIdx.x >> 6][c] = s;
    __syncthreads();
  }
  if (threadIdx.x < W && j < n) {
    s = (lds[0][c] + lds[1][c]) + (lds[2][c] + lds[3][c]);
    if (j < (size_t)cols) {
      if (dw) dw[j] = (P)s;
    } else if (db) {
      db[j - cols] = (P)s;
    }
  }
}
// 64 shares, or four where there are few parts (the whole gradient of 5 x 12089 bf16 18.2 us, by 64 shares 20.8)
template <class P>
void norm_join(QrDenseStream &s, size_t cols, size_t parts, const float *part, void *dw, void *db) {
  if (parts >= 64) s.launch(k_norm_join<P, 64>, (unsigned)((2 * cols + 15) / 16), 1024, 0, (int)cols, (int)parts, part, (P *)dw, (P *)db);
  else s.launch(k_norm_join<P, 4>, (unsigned)((2 * cols + 255) / 256), 1024, 0, (int)cols, (int)parts, part, (P *)dw, (P *)db);
}

// ---- rows that no workgroup's registers hold (and rows of less than 16 bytes): read again for every step ----------

// the sum over a workgroup of 1024, in every thread
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float lds[32];
  return group_sum<1024>(v, lds);
}

template <class T, class P>
__global__ __launch_bounds__(1024) void k_norm_any(const size_t rows, const int cols, const T *x, const size_t ldx,
                                                  const P *__restrict__ w, const P *__restrict__ b, const float eps, T *y,
                                                  const size_t ldy, float *__restrict__ mean, float *__restrict__ rstd) {
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const T *xr = x + r * ldx;
    float s = 0.f;
    for (int j = threadIdx.x; j < cols; j += 1024) s += (float)xr[j];
    const float mu = block_sum(s) / (float)cols;
    s = 0.f;
    for (int j = threadIdx.x; j < cols; j += 1024) {
      const float d = (float)xr[j] - mu;
      s = fmaf(d, d, s);
    }
    const float rs = 1.f / sqrtf(block_sum(s) / (float)cols + eps);
    for (int j = threadIdx.x; j < cols; j += 1024)
      y[r * ldy + j] = (T)fmaf(((float)xr[j] - mu) * rs, w ? (float)w[j] : 1.f, b ? (float)b[j] : 0.f);
    if (threadIdx.x == 0) {
      if (mean) mean[r] = mu;
      if (rstd) rstd[r] = rs;
    }
  }
}

template <class T, class P>
__global__ __launch_bounds__(1024) void k_norm_grad_any(const size_t rows, const int cols, const T *dy, const size_t lddy, const T *x,
                                                       const size_t ldx, const P *__restrict__ w, const float *__restrict__ mean,
                                                       const float *__restrict__ rstd, T *dx, const size_t lddx) {
  for (size_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float mu = mean[r], rs = rstd[r];
    float a = 0.f, c = 0.f;
    for (int j = threadIdx.x; j < cols; j += 1024) {
      const float g = (float)dy[r * lddy + j] * (w ? (float)w[j] : 1.f), h = ((float)x[r * ldx + j] - mu) * rs;
      a += g;
      c = fmaf(g, h, c);
    }
    a = block_sum(a) / (float)cols;
    c = block_sum(c) / (float)cols;
    for (int j = threadIdx.x; j < cols; j += 1024) {
      const float g = (float)dy[r * lddy + j] * (w ? (float)w[j] : 1.f), h = ((float)x[r * ldx + j] - mu) * rs;
      dx[r * lddx + j] = (T)(rs * (g - a - h * c));
    }
  }
}

template <class T>
__global__ __launch_bounds__(256) void k_norm_cols(const size_t rows, const int cols, const T *__restrict__ dy, const size_t lddy,
                                                   const T *__restrict__ x, const size_t ldx, const float *__restrict__ mean,
                                                   const float *__restrict__ rstd, float *__restrict__ part) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= cols) return;
  const size_t r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float sw = 0.f, sb = 0.f;
  for (size_t r = r0; r < r1; ++r) {
    const float d = (float)dy[r * lddy + j];
    sw = fmaf(d, ((float)x[r * ldx + j] - mean[r]) * rstd[r], sw);
    sb += d;
  }
  part[(size_t)blockIdx.y * 2 * cols + j] = sw;
  part[(size_t)blockIdx.y * 2 * cols + cols + j] = sb;
}

// The lanes and pieces a row is kept in: f(G, N), or false where no workgroup's registers hold a row.  Forward, the
// fewest lanes of 16, 64 and 256 that hold it in four (16: rows of up to 1 KB) or eight pieces each.  Backward, where
// a piece also has column sums, at most two pieces but for rows of 1 KB and less.
template <bool BACK, class F>
bool by_row(size_t cols, size_t e, F &&f) {
  using std::integral_constant;
  const size_t v = 16 / e, n = (cols + v - 1) / v;
  if (cols < v || n > 2048) return false;
  if (n <= 16) f(integral_constant<int, 16>{}, integral_constant<int, 1>{});
  else if (n <= 32) f(integral_constant<int, 16>{}, integral_constant<int, 2>{});
  else if (n <= 48) f(integral_constant<int, 16>{}, integral_constant<int, 3>{});
  else if constexpr (BACK) {
    if (n <= 64) f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    else if (n <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (n <= 256) f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    else if (n <= 512) f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    else if (n <= 1024) f(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
    else f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
  } else {
    if (n <= 64) f(integral_constant<int, 16>{}, integral_constant<int, 4>{});
    else if (n <= 128) f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    else if (n <= 256) f(integral_constant<int, 64>{}, integral_constant<int, 4>{});
    else if (n <= 512) f(integral_constant<int, 64>{}, integral_constant<int, 8>{});
    else if (n <= 1024) f(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    else f(integral_constant<int, 256>{}, integral_constant<int, 8>{});
  }
  return true;
}

// Workgroups of a backward pass, whose column sums are joined: as many as the registers let the chip hold at a time
// (six of 256 threads a compute unit with one piece a lane, four with more, two of 1024).  65536 x 2048 bf16 by 768 /
// 1024 / 1536 / 2048 workgroups: 200 / 188 / 183 / 218 us; 71291 x 1001 f16 (two pieces): 114 / 111 / 127 / 123 us.
size_t parts_of(size_t rows, int lanes, int pieces) {
  const size_t most = lanes > 256 ? 512 : pieces > 1 ? 1024 : 1536;
  return rows < most ? rows : most;
}
// ... of rows that no registers hold: as many as give 2^21 threads a share of a column, up to 512
size_t parts_any(size_t rows, size_t cols) {
  const size_t most = std::max<size_t>(std::min<size_t>(((size_t)1 << 21) / cols, 512), 1);
  return rows < most ? rows : most;
}
// columns that the registers of a workgroup hold at most, of any type
constexpr size_t COLS_HELD = 16384;
// Up to this many rows a workgroup takes at a time, one workgroup takes them all and no join follows: a second launch
// costs more than the rows one after the other.
constexpr size_t ALONE = 4;

constexpr size_t COLS_MOST = (size_t)1 << 24;

}  // namespace

extern "C" int qr_layer_norm_async(int device, void *stream, int type, int param_type, size_t rows, size_t cols, const void *x,
                                   size_t ldx, const void *weight, const void *bias, float eps, void *y, size_t ldy, float *mean,
                                   float *rstd) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "layer norm: unknown element type");
  QR_DENSE_ARG(param_type == type || param_type == QR_F32, "layer norm: weight and bias have the rows' type or f32");
  QR_DENSE_ARG(cols > 0, "layer norm: rows of no columns");
  if (cols > COLS_MOST) return qr_dense_fail(QR_ERR_UNSUPPORTED, "layer norm: rows of more than 2^24 columns");
  QR_DENSE_ARG(eps >= 0.f && eps < INFINITY, "layer norm: eps is a finite number of at least 0");
  QR_DENSE_ARG(qr_dense_fits(rows, cols, ldx) && qr_dense_fits(rows, cols, ldy), "layer norm: sizes out of range");
  QR_DENSE_ARG(rows < 2 || ldy >= cols, "layer norm: the stride of y is shorter than a row");
  if (!rows) return QR_OK;
  QR_DENSE_ARG(x && y, "layer norm: x or y is NULL");
  const QrDenseMatrix mx{x, rows, cols, ldx}, my{y, rows, cols, ldy};
  QR_DENSE_ARG(qr_dense_in_place(my, mx) || !qr_dense_share(my, mx, qr_dense_size(type)), "layer norm: y lies over x, but not row for row");
  QR_DENSE_DEVICE(device);
  QrDenseStream s(stream);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      const bool fits = by_row<false>(cols, sizeof(T), [&](auto G, auto N) {
        constexpr size_t RPB = 256 / G(), MOST = RPB << 23;  // (a launch has fewer than 2^32 threads)
        for (size_t r = 0; r < rows; r += MOST) {
          const size_t n = std::min(rows - r, MOST);
          s.launch(k_norm<T, P, G(), N()>, (unsigned)((n + RPB - 1) / RPB), 256, 0,
                   n, (int)cols, (const T *)x + r * ldx, ldx, (const P *)weight, (const P *)bias, eps, (T *)y + r * ldy, ldy,
                   mean ? mean + r : nullptr, rstd ? rstd + r : nullptr);
        }
      });
      if (!fits)
        s.launch(k_norm_any<T, P>, (unsigned)(rows < 65536 ? rows : 65536), 1024, 0, rows, (int)cols, (const T *)x, ldx, (const P *)weight,
                 (const P *)bias, eps, (T *)y, ldy, mean, rstd);
    };
    if (param_type == QR_F32) go(float{});
    else go(T{});
  });
  return qr_dense_launched(s, "layer norm");
}

extern "C" int qr_layer_norm_backward_workspace(size_t rows, size_t cols, size_t *bytes) {
  QR_DENSE_ARG(bytes && cols > 0 && cols <= COLS_MOST, "layer norm backward: bad size");
  *bytes = (cols <= COLS_HELD ? parts_of(rows, 1, 1) : parts_any(rows, cols)) * 2 * cols * 4;
  return QR_OK;
}

extern "C" int qr_layer_norm_backward_async(int device, void *stream, int type, int param_type, size_t rows, size_t cols,
                                            const void *dy, size_t lddy, const void *x, size_t ldx, const void *weight,
                                            const float *mean, const float *rstd, void *dx, size_t lddx, void *dweight, void *dbias,
                                            void *workspace, size_t workspace_bytes) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "layer norm backward: unknown element type");
  QR_DENSE_ARG(param_type == type || param_type == QR_F32, "layer norm backward: weight and bias have the rows' type or f32");
  QR_DENSE_ARG(cols > 0, "layer norm backward: rows of no columns");
  if (cols > COLS_MOST) return qr_dense_fail(QR_ERR_UNSUPPORTED, "layer norm backward: rows of more than 2^24 columns");
  QR_DENSE_ARG(qr_dense_fits(rows, cols, ldx) && qr_dense_fits(rows, cols, lddy) && qr_dense_fits(rows, cols, lddx),
               "layer norm backward: sizes out of range");
  QR_DENSE_ARG(!dx || rows < 2 || lddx >= cols, "layer norm backward: the stride of dx is shorter than a row");
  QR_DENSE_ARG(!rows || (dy && x && mean && rstd), "layer norm backward: dy, x, mean or rstd is NULL");
  const bool sums = dweight || dbias;
  size_t need = 0;
  (void)qr_layer_norm_backward_workspace(rows, cols, &need);
  QR_DENSE_ARG(!sums || !rows || (workspace && workspace_bytes >= need), "layer norm backward: the workspace is too small");
  const QrDenseMatrix mdx{dx, rows, cols, lddx}, in[2] = {{dy, rows, cols, lddy}, {x, rows, cols, ldx}};
  for (int i = 0; i < 2; ++i)
    QR_DENSE_ARG(qr_dense_in_place(mdx, in[i]) || !qr_dense_share(mdx, in[i], qr_dense_size(type)),
                 "layer norm backward: dx lies over dy or x, but not row for row");
  if (!rows && !sums) return QR_OK;
  QR_DENSE_DEVICE(device);
  QrDenseStream s(stream);
  const unsigned any = (unsigned)parts_any(rows, cols);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto p) {
      using P = decltype(p);
      float *const part = sums ? (float *)workspace : nullptr;
      const bool fits = !rows || by_row<true>(cols, sizeof(T), [&](auto G, auto N) {
        constexpr size_t RPB = G() > 256 ? 1 : 256 / G();
        const size_t want = (rows + RPB - 1) / RPB, parts = parts_of(rows, G(), N());
        const unsigned grid = want <= ALONE ? 1 : (unsigned)(want < parts ? want : parts);
        s.launch(k_norm_grad<T, P, G(), N()>, grid, G() > 256 ? G() : 256, RPB > 1 && sums ? 8 * cols * 4 : 0,
                 rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)weight, mean, rstd, (T *)dx, lddx, part, (P *)dweight, (P *)dbias);
        if (sums && grid > 1) norm_join<P>(s, cols, grid, part, dweight, dbias);
      });
      if (fits && rows) return;
      // (the column sums first: dx may be written over dy or x)
      if (rows && sums)
        s.launch(k_norm_cols<T>, dim3((unsigned)((cols + 255) / 256), any), 256, 0, rows, (int)cols, (const T *)dy, lddy, (const T *)x,
                 ldx, mean, rstd, part);
      if (sums)
        norm_join<P>(s, cols, any, part, dweight, dbias);
      if (rows && dx)
        s.launch(k_norm_grad_any<T, P>, (unsigned)(rows < 65536 ? rows : 65536), 1024, 0,
                 rows, (int)cols, (const T *)dy, lddy, (const T *)x, ldx, (const P *)weight, mean, rstd, (T *)dx, lddx);
    };
    if (param_type == QR_F32) go(float{});
    else go(T{});
  });
  return qr_dense_launched(s, "layer norm backward");
}
