// k_drop.hip -- dropout whose mask is a function of (seed, offset, element) and is never stored.
//
//   word w of a call = mix(mix(seed) + G (offset + w + 1)),  mix = the finalizer of the --subsample draw's
//   keys (k_sample.hip), G its increment; element i (row * cols + column) owns bits 16 (i % 4) .. + 15 of
//   word i / 4 and is dropped iff they are below t = floor(65536 p + 0.5)
//   y = residual + (kept ? x * 65536 / (65536 - t) : 0)
//
// The scale is that of the probability the 16 bits can express, so the expectation is x exactly.
// The backward pass is the same call on dy.
//
// Bound by memory: some thirty integer instructions a word of four elements hide behind it.  65536 x 2048 bf16 with a
// residual 151 us (5.3 TB/s), 99991 x 1145 f16 without 83 us (5.5), where a copy reaches 4.9 to 5.4; 100 x 512 f32 2.7 us.
#include "qr_dense.h"

namespace {

__host__ __device__ __forceinline__ uint64_t mix64(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
constexpr uint64_t WEYL = 0x9E3779B97F4A7C15ull;

template <class T>
struct Raw {
  T v[16 / sizeof(T)];
};

template <class T>
__device__ __forceinline__ T dropped(const T x, const float r, const uint32_t bits, const uint32_t t, const float scale) {
  return (T)((bits >= t ? (float)x * scale : 0.f) + r);
}

// rows without gaps: a thread takes pieces of 16 bytes of the whole, U of them under way at a time (their loads' latency
// is what a wave would wait for)
template <class T, bool RES, int U>
__global__ __launch_bounds__(256) void k_drop_flat(const size_t n, const T *x, const T *res, T *y, const uint32_t t, const float scale,
                                                   const uint64_t key, const uint64_t offset, const uint64_t *__restrict__ counter) {
  constexpr int V = 16 / sizeof(T), W = V / 4;
  const size_t pieces = (n + V - 1) / V, step = (size_t)gridDim.x * 256;
  const uint64_t first = key + WEYL * (offset + (counter ? *counter : 0) + 1);
  for (size_t p0 = (size_t)blockIdx.x * 256 + threadIdx.x; p0 < pieces; p0 += step * U) {
    Raw<T> vx[U], vr[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t at = (p0 + u * step) * V;
      if (at + V <= n) {
        __builtin_memcpy(&vx[u], x + at, 16);
        if (RES) __builtin_memcpy(&vr[u], res + at, 16);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t p = p0 + u * step, at = p * V;
      if (at >= n) continue;
      uint64_t bits[W];
#pragma unroll
      for (int w = 0; w < W; ++w) bits[w] = mix64(first + WEYL * (p * W + w));
      if (at + V <= n) {
        Raw<T> o;
#pragma unroll
        for (int e = 0; e < V; ++e)
          o.v[e] = dropped(vx[u].v[e], RES ? (float)vr[u].v[e] : 0.f, (uint32_t)(bits[e / 4] >> (16 * (e % 4))) & 0xFFFF, t, scale);
        __builtin_memcpy(y + at, &o, 16);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (at + e < n)
            y[at + e] = dropped(x[at + e], RES ? (float)res[at + e] : 0.f, (uint32_t)(bits[e / 4] >> (16 * (e % 4))) & 0xFFFF, t, scale);
      }
    }
  }
}

// rows of a stride: one thread per word, four elements that may lie in several rows
template <class T>
__global__ __launch_bounds__(256) void k_drop_rows(const size_t rows, const size_t cols, const T *x, const size_t ldx, const T *res,
                                                   const size_t ldr, T *y, const size_t ldy, const uint32_t t, const float scale,
                                                   const uint64_t key, const uint64_t offset, const uint64_t *__restrict__ counter) {
  const size_t n = rows * cols, words = (n + 3) / 4;
  const uint64_t first = offset + (counter ? *counter : 0) + 1;
  for (size_t w = (size_t)blockIdx.x * 256 + threadIdx.x; w < words; w += (size_t)gridDim.x * 256) {
    const uint64_t bits = mix64(key + WEYL * (first + w));
    size_t r = w * 4 / cols, j = w * 4 - r * cols;
    for (int e = 0; e < 4 && w * 4 + e < n; ++e) {
      y[r * ldy + j] = dropped(x[r * ldx + j], res ? (float)res[r * ldr + j] : 0.f, (uint32_t)(bits >> (16 * e)) & 0xFFFF, t, scale);
      if (++j == cols) j = 0, ++r;
    }
  }
}

}  // namespace

extern "C" int qr_dropout_async(int device, void *stream, int type, size_t rows, size_t cols, const void *x, size_t ldx,
                                const void *residual, size_t ldr, void *y, size_t ldy, double p, uint64_t seed, uint64_t offset,
                                const uint64_t *counter) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "dropout: unknown element type");
  QR_DENSE_ARG(p >= 0.0 && p <= 1.0, "dropout: p is a number of 0 to 1");
  QR_DENSE_ARG(qr_dense_spans(rows, cols, ldx) && qr_dense_spans(rows, cols, ldy) && qr_dense_spans(rows, cols, residual ? ldr : 0),
               "dropout: sizes out of range");
  QR_DENSE_ARG(rows < 2 || ldy >= cols, "dropout: the stride of y is shorter than a row");
  if (!rows || !cols) return QR_OK;
  QR_DENSE_ARG(x && y, "dropout: x or y is NULL");
  const QrDenseMatrix my{y, rows, cols, ldy}, in[2] = {{x, rows, cols, ldx}, {residual, rows, cols, ldr}};
  for (int i = 0; i < 2; ++i)
    QR_DENSE_ARG(qr_dense_in_place(my, in[i]) || !qr_dense_share(my, in[i], qr_dense_size(type)),
                 "dropout: y lies over x or the residual, but not row for row");
  QR_DENSE_DEVICE(device);
  const uint32_t t = (uint32_t)(p * 65536.0 + 0.5);
  const float scale = t < 65536 ? 65536.f / (float)(65536 - t) : 0.f;
  const size_t n = rows * cols;
  const bool flat = rows == 1 || (ldx == cols && ldy == cols && (!residual || ldr == cols));
  const auto grid = [](size_t threads) { return (unsigned)((threads + 255) / 256 < 8192 ? (threads + 255) / 256 : 8192); };
  QrDenseStream s(stream);
  qr_dense_dispatch(type, [&](auto tt) {
    using T = decltype(tt);
    const unsigned pieces = grid((n + 16 / sizeof(T) - 1) / (16 / sizeof(T)));
    if (flat && residual)
      s.launch(k_drop_flat<T, true, 2>, pieces, 256, 0, n, (const T *)x, (const T *)residual, (T *)y, t, scale, mix64(seed), offset, counter);
    else if (flat)
      s.launch(k_drop_flat<T, false, 4>, pieces, 256, 0, n, (const T *)x, nullptr, (T *)y, t, scale, mix64(seed), offset, counter);
    else
      s.launch(k_drop_rows<T>, grid((n + 3) / 4), 256, 0, rows, cols, (const T *)x, ldx, (const T *)residual, ldr, (T *)y, ldy, t, scale,
               mix64(seed), offset, counter);
  });
  return qr_dense_launched(s, "dropout");
}
