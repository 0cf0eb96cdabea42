// k_drop.hip -- dropout whose mask is a function of (seed, offset, element) and is never stored.
//
//   word w of a call = mix(mix(seed) + G (offset + w + 1)),  mix = the finalizer of the --subsample draw's
//   keys (k_sample.hip), G its increment; element i (row * cols + column) owns bits 16 (i % 4) .. + 15 of
//   word i / 4 and is dropped iff they are below t = floor(65536 p + 0.5)
//   y = residual + (kept ? x * 65536 / (65536 - t) : 0)
//
// The scale is that of the probability the 16 bits can express, so the expectation is x exactly.
// The backward pass is the same call on dy.
#include "qr_dense.h"

namespace {

__host__ __device__ __forceinline__ uint64_t mix64(uint64_t z) {
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  return z ^ (z >> 31);
}
constexpr uint64_t WEYL = 0x9E3779B97F4A7C15ull;

// one thread per word: four elements, which may lie in several rows
template <class T>
__global__ __launch_bounds__(256) void k_drop(const size_t rows, const size_t cols, const T *x, const size_t ldx, const T *res,
                                              const size_t ldr, T *y, const size_t ldy, const uint32_t t, const float scale,
                                              const uint64_t key, const uint64_t offset, const uint64_t *__restrict__ counter) {
  const size_t n = rows * cols, words = (n + 3) / 4;
  const uint64_t first = offset + (counter ? *counter : 0) + 1;
  for (size_t w = (size_t)blockIdx.x * 256 + threadIdx.x; w < words; w += (size_t)gridDim.x * 256) {
    const uint64_t bits = mix64(key + WEYL * (first + w));
    size_t r = w * 4 / cols, j = w * 4 - r * cols;
    for (int e = 0; e < 4 && w * 4 + e < n; ++e) {
      const bool keep = (uint32_t)((bits >> (16 * e)) & 0xFFFF) >= t;
      float v = keep ? (float)x[r * ldx + j] * scale : 0.f;
      if (res) v += (float)res[r * ldr + j];
      y[r * ldy + j] = (T)v;
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
  QR_DENSE_ARG(qr_dense_fits(rows, cols, ldx) && qr_dense_fits(rows, cols, ldy) && qr_dense_fits(rows, cols, residual ? ldr : 0),
               "dropout: sizes out of range");
  QR_DENSE_ARG(rows < 2 || ldy >= cols, "dropout: the stride of y is shorter than a row");
  if (!rows || !cols) return QR_OK;
  QR_DENSE_ARG(x && y, "dropout: x or y is NULL");
  QR_DENSE_DEVICE(device);
  const uint32_t t = (uint32_t)(p * 65536.0 + 0.5);
  const float scale = t < 65536 ? 65536.f / (float)(65536 - t) : 0.f;
  const size_t words = (rows * cols + 3) / 4;
  const unsigned grid = (unsigned)((words + 255) / 256 < 65536 ? (words + 255) / 256 : 65536);
  qr_dense_dispatch(type, [&](auto tt) {
    using T = decltype(tt);
    k_drop<T><<<grid, 256, 0, (hipStream_t)stream>>>(rows, cols, (const T *)x, ldx, (const T *)residual, ldr, (T *)y, ldy, t, scale,
                                                     mix64(seed), offset, counter);
  });
  return qr_dense_launched("dropout");
}
