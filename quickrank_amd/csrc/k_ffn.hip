// k_ffn.hip -- the gated feed-forward unit h = act(x Wg^T) * (x Wu^T) and its backward pass.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Products accumulate in 32 bits.
#include "qr_dense.h"

namespace {

// the activation and its derivative
__device__ __forceinline__ void act_of(const int act, const float g, float &a, float &d) {
  if (act == QR_ACT_RELU) {
    a = g > 0.f ? g : (g != g ? g : 0.f);
    d = g > 0.f ? 1.f : 0.f;
  } else if (act == QR_ACT_GELU) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    d = fmaf(g * 0.39894228040143268f, expf(-0.5f * g * g), cdf);
  } else if (act == QR_ACT_GELU_TANH) {
    const float c = 0.79788456080286536f, t = tanhf(c * (g + 0.044715f * g * g * g));
    a = 0.5f * g * (1.f + t);
    d = 0.5f * (1.f + t) + 0.5f * g * (1.f - t * t) * c * (1.f + 3.f * 0.044715f * g * g);
  } else {
    const float s = 1.f / (1.f + expf(-g));
    a = act == QR_ACT_SIGMOID ? s : g * s;
    d = act == QR_ACT_SIGMOID ? s * (1.f - s) : s * (1.f + g * (1.f - s));
  }
}

// A matrix whose element (row, k) is p[row * sr + k * sk]
template <class T>
struct Mat {
  const T *p;
  size_t sr, sk;
};

// 16 x 16 outputs per workgroup, one per thread, through LDS; D pairs of operands: two sums (gate and up: PAIR)
// or one sum over both pairs.
template <class T, bool PAIR, class Epi>
__global__ __launch_bounds__(256) void k_simple(const size_t m, const size_t n, const size_t k, const Mat<T> a0, const Mat<T> b0,
                                                const Mat<T> a1, const Mat<T> b1, const bool two, const Epi epi) {
  __shared__ float la[16][17], lb[16][17];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const size_t r0 = (size_t)blockIdx.y * 16, c0 = (size_t)blockIdx.x * 16, r = r0 + ty, c = c0 + tx;
  float acc[2] = {0.f, 0.f};
  for (int h = 0; h < (two ? 2 : 1); ++h) {
    const Mat<T> A = h ? a1 : a0, B = h ? b1 : b0;
    for (size_t q = 0; q < k; q += 16) {
      la[ty][tx] = r < m && q + tx < k ? (float)A.p[r * A.sr + (q + tx) * A.sk] : 0.f;
      lb[ty][tx] = c0 + ty < n && q + tx < k ? (float)B.p[(c0 + ty) * B.sr + (q + tx) * B.sk] : 0.f;
      __syncthreads();
      float s = acc[PAIR ? h : 0];
      for (int i = 0; i < 16; ++i) s = fmaf(la[ty][i], lb[tx][i], s);
      acc[PAIR ? h : 0] = s;
      __syncthreads();
    }
  }
  if (r < m && c < n) epi(r, c, acc[0], acc[1]);
}

template <class T>
struct EpiGated {
  T *h, *g, *u;
  size_t ldh, n;
  int act;
  __device__ void operator()(size_t r, size_t c, float vg, float vu) const {
    float a, d;
    act_of(act, vg, a, d);
    h[r * ldh + c] = (T)(a * vu);
    if (g) g[r * n + c] = (T)vg, u[r * n + c] = (T)vu;
  }
};
template <class T>
struct EpiStore {
  T *o;
  size_t ld;
  __device__ void operator()(size_t r, size_t c, float v, float) const { o[r * ld + c] = (T)v; }
};

template <class T>
__global__ __launch_bounds__(256) void k_gate_grad(const size_t m, const size_t n, const int act, const T *__restrict__ dh,
                                                   const size_t lddh, const T *__restrict__ g, const T *__restrict__ u,
                                                   T *__restrict__ dg, T *__restrict__ du) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < m * n; i += (size_t)gridDim.x * 256) {
    const size_t r = i / n, c = i - r * n;
    float a, d;
    act_of(act, (float)g[i], a, d);
    const float v = (float)dh[r * lddh + c];
    dg[i] = (T)(v * (float)u[i] * d);
    du[i] = (T)(v * a);
  }
}

bool act_ok(int act) { return act >= QR_ACT_SILU && act <= QR_ACT_SIGMOID; }

}  // namespace

extern "C" int qr_gated_ffn_async(int device, void *stream, int type, int act, size_t m, size_t k, size_t n, const void *x, size_t ldx,
                                  const void *w_gate, const void *w_up, size_t ldw, void *h, size_t ldh, void *gate, void *up) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "gated ffn: unknown element type");
  QR_DENSE_ARG(act_ok(act), "gated ffn: unknown activation");
  QR_DENSE_ARG(k > 0 && n > 0, "gated ffn: no columns");
  QR_DENSE_ARG(qr_dense_fits(m, k, ldx) && qr_dense_fits(n, k, ldw) && qr_dense_fits(m, n, ldh), "gated ffn: sizes out of range");
  QR_DENSE_ARG(m < 2 || ldh >= n, "gated ffn: the stride of h is shorter than a row");
  QR_DENSE_ARG(!gate == !up, "gated ffn: gate and up are kept both or neither");
  if (!m) return QR_OK;
  QR_DENSE_ARG(x && w_gate && w_up && h, "gated ffn: x, a weight or h is NULL");
  const size_t e = qr_dense_size(type);
  const void *out[3] = {h, gate, up};
  const size_t bytes[3] = {qr_dense_span(m, n, ldh, e), m * n * e, m * n * e};
  for (int i = 0; i < 3; ++i) {
    QR_DENSE_ARG(!qr_dense_overlap(out[i], bytes[i], x, qr_dense_span(m, k, ldx, e)) &&
                     !qr_dense_overlap(out[i], bytes[i], w_gate, qr_dense_span(n, k, ldw, e)) &&
                     !qr_dense_overlap(out[i], bytes[i], w_up, qr_dense_span(n, k, ldw, e)),
                 "gated ffn: an output lies over an input");
    for (int j = 0; j < i; ++j) QR_DENSE_ARG(!qr_dense_overlap(out[i], bytes[i], out[j], bytes[j]), "gated ffn: outputs overlap");
  }
  QR_DENSE_DEVICE(device);
  const dim3 grid((unsigned)((n + 15) / 16), (unsigned)((m + 15) / 16));
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    const Mat<T> a{(const T *)x, ldx, 1}, b0{(const T *)w_gate, ldw, 1}, b1{(const T *)w_up, ldw, 1};
    k_simple<T, true><<<grid, 256, 0, (hipStream_t)stream>>>(m, n, k, a, b0, a, b1, true,
                                                             EpiGated<T>{(T *)h, (T *)gate, (T *)up, ldh, n, act});
  });
  return qr_dense_launched("gated ffn");
}

extern "C" int qr_gated_ffn_backward_workspace(int type, size_t m, size_t k, size_t n, size_t *bytes) {
  QR_DENSE_ARG(bytes && qr_dense_type_ok(type) && k > 0 && n > 0 && qr_dense_fits(m, n, n) && qr_dense_fits(n, k, k),
               "gated ffn backward: bad size");
  *bytes = 2 * m * n * qr_dense_size(type);
  return QR_OK;
}

extern "C" int qr_gated_ffn_backward_async(int device, void *stream, int type, int act, size_t m, size_t k, size_t n, const void *dh,
                                           size_t lddh, const void *x, size_t ldx, const void *w_gate, const void *w_up, size_t ldw,
                                           const void *gate, const void *up, void *dx, size_t lddx, void *dw_gate, void *dw_up,
                                           void *workspace, size_t workspace_bytes) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "gated ffn backward: unknown element type");
  QR_DENSE_ARG(act_ok(act), "gated ffn backward: unknown activation");
  QR_DENSE_ARG(k > 0 && n > 0, "gated ffn backward: no columns");
  QR_DENSE_ARG(qr_dense_fits(m, k, ldx) && qr_dense_fits(n, k, ldw) && qr_dense_fits(m, n, lddh) && qr_dense_fits(m, k, lddx),
               "gated ffn backward: sizes out of range");
  QR_DENSE_ARG(!dx || m < 2 || lddx >= k, "gated ffn backward: the stride of dx is shorter than a row");
  QR_DENSE_ARG(!m || (dh && x && w_gate && w_up && gate && up), "gated ffn backward: an input is NULL");
  QR_DENSE_ARG(!dw_gate == !dw_up, "gated ffn backward: the weights' gradients are asked for both or neither");
  size_t need = 0;
  if (int rc = qr_gated_ffn_backward_workspace(type, m, k, n, &need)) return rc;
  QR_DENSE_ARG(!need || (workspace && workspace_bytes >= need), "gated ffn backward: the workspace is too small");
  const size_t e = qr_dense_size(type);
  const void *out[4] = {dx, dw_gate, dw_up, workspace}, *in[6] = {dh, x, w_gate, w_up, gate, up};
  const size_t ob[4] = {qr_dense_span(m, k, lddx, e), n * k * e, n * k * e, need};
  const size_t ib[6] = {qr_dense_span(m, n, lddh, e), qr_dense_span(m, k, ldx, e), qr_dense_span(n, k, ldw, e),
                        qr_dense_span(n, k, ldw, e), m * n * e, m * n * e};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 6; ++j) QR_DENSE_ARG(!qr_dense_overlap(out[i], ob[i], in[j], ib[j]), "gated ffn backward: an output lies over an input");
    for (int j = 0; j < i; ++j) QR_DENSE_ARG(!qr_dense_overlap(out[i], ob[i], out[j], ob[j]), "gated ffn backward: outputs overlap");
  }
  QR_DENSE_DEVICE(device);
  const hipStream_t s = (hipStream_t)stream;
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    T *dg = (T *)workspace, *du = dg + m * n;
    if (m)
      k_gate_grad<T><<<(unsigned)((m * n + 255) / 256 < 65536 ? (m * n + 255) / 256 : 65536), 256, 0, s>>>(
          m, n, act, (const T *)dh, lddh, (const T *)gate, (const T *)up, dg, du);
    if (dx && m)
      k_simple<T, false><<<dim3((unsigned)((k + 15) / 16), (unsigned)((m + 15) / 16)), 256, 0, s>>>(
          m, k, n, Mat<T>{dg, n, 1}, Mat<T>{(const T *)w_gate, 1, ldw}, Mat<T>{du, n, 1}, Mat<T>{(const T *)w_up, 1, ldw}, true,
          EpiStore<T>{(T *)dx, lddx});
    for (int i = 0; i < 2 && dw_gate; ++i)
      k_simple<T, false><<<dim3((unsigned)((k + 15) / 16), (unsigned)((n + 15) / 16)), 256, 0, s>>>(
          n, k, m, Mat<T>{i ? du : dg, 1, n}, Mat<T>{(const T *)x, 1, ldx}, Mat<T>{}, Mat<T>{}, false,
          EpiStore<T>{(T *)(i ? dw_up : dw_gate), k});
  });
  return qr_dense_launched("gated ffn backward");
}
