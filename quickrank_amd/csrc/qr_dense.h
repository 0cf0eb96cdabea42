// qr_dense.h -- what the dense operators (k_norm.hip, k_drop.hip, k_ffn.hip) share: element types,
// argument checks and the host side of a stateless launch.
//
// Unlike the calls that take a qr_ctx, these hold no state between calls: device, stream and
// workspace come with each call, so calls of several threads and captured graphs have nothing in
// common but what their caller shares.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <string>
#include <tuple>

#include "../../include/qr_hip.h"

// the calling thread's message, read with qr_last_error(NULL); never throws (qr_api.hip)
int qr_dense_fail(int code, const char *what) noexcept;

#define QR_DENSE_ARG(cond, msg) \
  do {                          \
    if (!(cond)) return qr_dense_fail(QR_ERR_ARG, msg); \
  } while (0)

// Makes the call's device current for as long as it lives and puts the caller's back.
struct QrDeviceGuard {
  int old = -1;
  hipError_t err = hipSuccess;
  explicit QrDeviceGuard(int device) {
    int cur = -1;
    err = hipGetDevice(&cur);
    if (err == hipSuccess && cur != device) {
      err = hipSetDevice(device);
      if (err == hipSuccess) old = cur;
    }
  }
  ~QrDeviceGuard() {
    if (old >= 0) (void)hipSetDevice(old);
  }
};

#define QR_DENSE_DEVICE(device)                                                              \
  QrDeviceGuard _guard(device);                                                              \
  if (_guard.err != hipSuccess) {                                                            \
    (void)hipGetLastError();                                                                 \
    return qr_dense_fail(_guard.err == hipErrorNoDevice ? QR_ERR_NO_DEVICE : QR_ERR_ARG,     \
                         "the device cannot be made current (this library has no CPU fallback)"); \
  }

// The call's stream.  A launch's outcome is what it returns, not the thread's last error, which an earlier call of somebody
// else's may have left; behind one that failed nothing more is launched.
struct QrDenseStream {
  hipStream_t stream;
  hipError_t err = hipSuccess;
  explicit QrDenseStream(void *s) : stream((hipStream_t)s) {}
  template <class... P, class... A>
  void launch(void (*kernel)(P...), dim3 grid, unsigned block, size_t lds, const A &...a) {
    if (err != hipSuccess) return;
    std::tuple<P...> v(static_cast<P>(a)...);
    std::apply(
        [&](P &...p) {
          void *args[] = {(void *)&p...};
          err = hipLaunchKernel((const void *)kernel, grid, dim3(block), args, lds, stream);
        },
        v);
  }
};

inline int qr_dense_launched(const QrDenseStream &s, const char *what) noexcept {
  if (s.err == hipSuccess) return QR_OK;
  (void)hipGetLastError();  // (reported here)
  return qr_dense_fail(QR_ERR_HIP, hipGetErrorString(s.err) ? hipGetErrorString(s.err) : what);
}

inline bool qr_dense_type_ok(int t) { return t == QR_F32 || t == QR_BF16 || t == QR_F16; }
inline size_t qr_dense_size(int t) { return t == QR_F32 ? 4 : 2; }
// bytes from the first to behind the last element of a [rows][cols] matrix of stride ld
inline size_t qr_dense_span(size_t rows, size_t cols, size_t ld, size_t e) {
  return rows && cols ? ((rows - 1) * ld + cols) * e : 0;
}
inline bool qr_dense_overlap(const void *p, size_t np, const void *q, size_t nq) {
  const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
  return p && q && np && nq && a < b + nq && b < a + np;
}
// A matrix of a call.
struct QrDenseMatrix {
  const void *p;
  size_t rows, cols, ld;
};
// Whether two matrices of elements of e bytes may share any.  Exact for rows of one stride, of which one matrix may have the
// first columns and the other the rest; those of two strides do if their memory from end to end overlaps.
inline bool qr_dense_share(const QrDenseMatrix &a, const QrDenseMatrix &b, size_t e) {
  if (!qr_dense_overlap(a.p, qr_dense_span(a.rows, a.cols, a.ld, e), b.p, qr_dense_span(b.rows, b.cols, b.ld, e))) return false;
  const uintptr_t p = (uintptr_t)a.p, q = (uintptr_t)b.p;
  if (a.ld != b.ld || a.cols > a.ld || b.cols > a.ld || (p > q ? p - q : q - p) % e) return true;
  const size_t away = (p > q ? p - q : q - p) / e % a.ld, d = p > q && away ? a.ld - away : away;  // b's first column among a's
  return d < a.cols || d + b.cols > a.ld;
}
// ... of an output that may also be the input itself, row for row
inline bool qr_dense_in_place(const QrDenseMatrix &out, const QrDenseMatrix &in) {
  return out.p == in.p && (out.rows < 2 || out.ld == in.ld);
}
// rows * cols elements of stride ld stay far below 2^63 bytes
inline bool qr_dense_spans(size_t rows, size_t cols, size_t ld) {
  const size_t most = (size_t)1 << 58;
  return rows == 0 || (ld < most && cols < most && rows < most / ((ld > cols ? ld : cols) + 1));
}
// ... and a row's elements below 2^31
inline bool qr_dense_fits(size_t rows, size_t cols, size_t ld) { return cols < ((size_t)1 << 31) && qr_dense_spans(rows, cols, ld); }

// `T` of a type code for a generic lambda: qr_dense_dispatch(type, [&](auto t) { using T = decltype(t); ... })
template <class F>
inline void qr_dense_dispatch(int type, F &&f) {
  if (type == QR_F32) f(float{});
  else if (type == QR_BF16) f(__bf16{});
  else f(_Float16{});
}
