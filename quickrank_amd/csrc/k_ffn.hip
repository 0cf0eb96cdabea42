// k_ffn.hip -- the gated feed-forward unit h = act(x Wg^T) * (x Wu^T) and its backward pass.
//
//   g = x Wg^T, u = x Wu^T, h = act(g) u
//   dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// All five products run through one matrix-core kernel (k_gemm) that accumulates in 32 bits.  Both operands
// are staged through LDS in tiles of 128 bytes of the summed dimension, either as rows (that dimension is
// contiguous in memory) or as columns (it is the strided one: the 16-bit types are then transposed by the LDS
// read itself).  The forward pass interleaves blocks of 16 rows of Wg and of Wu in its second operand's tile,
// so that one lane ends with g and u of the same outputs and the activation, the product and the rounding
// need no second kernel.
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

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
#define QR_LDS __attribute__((address_space(3)))
#define QR_GLB __attribute__((address_space(1)))

// 16 bytes of the summed dimension a lane holds of one operand, against 16 rows of either: lane l has row l % 16
// and the (l / 16)-th 16 bytes.  acc[v] of lane l is (row 4 (l / 16) + v of a, row l % 16 of b).
template <class T>
__device__ __forceinline__ f4 mma(const i4 a, const i4 b, f4 c) {
  if constexpr (sizeof(T) == 4) {
    const f4 x = __builtin_bit_cast(f4, a), y = __builtin_bit_cast(f4, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
  }
}

// ---- LDS tiles -----------------------------------------------------------------------------------------
// A tile holds R rows (outputs) of KT = 128 / sizeof(T) summed elements in 128 R bytes, moved in pieces of 16.
//
// Rows layout: row r at 128 r, its piece c at position c ^ (r & 7): the 16 lanes that read the same piece of 16
// consecutive rows touch every bank once.
// Columns layout: summed element k at k R sizeof(T), its pieces XORed with col_swz(k) so that the lanes of one
// read, which lie in 8 (16-bit) or 4 (f32) such lines, touch every bank once.
template <class T, int R>
__device__ __forceinline__ int col_swz(const int k) {
  if constexpr (sizeof(T) == 4) return ((k >> 2) & 3) << 2;              // segments of 16 floats
  else if constexpr (R >= 128) return ((k & 3) | (((k >> 3) & 1) << 2)) << 1;  // segments of 16 elements = 32 bytes
  else return (((k >> 1) & 1) | (((k >> 3) & 1) << 1)) << 1;              // two lines of 128 bytes share the banks
}

// the piece q (of R * 8) of a tile in LDS order -> where it comes from
template <class T, int R, bool KS>
__device__ __forceinline__ void piece_of(const int q, int &r, int &k) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (!KS) {
    r = q >> 3;
    k = ((q & 7) ^ (r & 7)) * E;
  } else {
    constexpr int PER = R / E;
    k = q / PER;
    r = ((q % PER) ^ col_swz<T, R>(k)) * E;
  }
}

// one operand fragment: 16 rows from row16 * 16 on, the step-th half of the tile's summed dimension
template <class T, int R, bool KS>
__device__ __forceinline__ i4 frag(const char *lds, const int row16, const int step) {
  const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
  if constexpr (!KS) {
    return *(const i4 *)(lds + (row16 * 16 + i) * 128 + (((step * 4 + g) ^ (i & 7)) << 4));
  } else if constexpr (sizeof(T) == 2) {
    const int k = step * 32 + 8 * g + (i >> 2);
    const char *p = lds + k * (R * 2) + (((row16 * 2) ^ col_swz<T, R>(k)) << 4) + (i & 3) * 8;
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QR_LDS s4 *)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QR_LDS s4 *)(p + 4 * R * 2));
    i4 v;
    __builtin_memcpy(&v, &lo, 8);
    __builtin_memcpy((char *)&v + 8, &hi, 8);
    return v;
  } else {
    const int k = step * 16 + 4 * g;
    const char *p = lds + k * (R * 4) + (((row16 * 4) ^ col_swz<T, R>(k)) << 4) + i * 4;
    i4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *(const int *)(p + e * R * 4);
    return v;
  }
}

// 16 bytes of a matrix of rows of stride ld, from (line, at) on; elements beyond `lines` or `len` as zeros
template <class T>
__device__ __forceinline__ i4 fetch16(const T *p, const size_t ld, const size_t line, const size_t lines, const size_t at, const size_t len) {
  constexpr int E = 16 / sizeof(T);
  i4 v = {0, 0, 0, 0};
  if (line < lines && at < len) {
    const T *s = p + line * ld + at;
    if (at + E <= len) {
      __builtin_memcpy(&v, s, 16);
    } else {
      T t[E] = {};
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at + e < len) t[e] = s[e];
      __builtin_memcpy(&v, t, 16);
    }
  }
  return v;
}

// eight results of one row, rounded; the row's base need not be aligned
template <class T>
__device__ __forceinline__ void store8(T *p, const float (&v)[8], const size_t at, const size_t len) {
  if (at + 8 <= len) {
    T t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (T)v[e];
    __builtin_memcpy(p + at, t, sizeof t);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at + e < len) p[at + e] = (T)v[e];
  }
}

// ---- the product -----------------------------------------------------------------------------------------
enum Kind { FWD, DX, DW };

template <class T>
struct GemmArgs {
  const T *a[2], *b[2];  // FWD: x | Wg, Wu.  DX: dg, du | Wg, Wu.  DW: dg, du | x.  Rows at 16-byte boundaries
  size_t lda, ldb;
  size_t rows, cols, k;  // outputs (FWD: of h; DW: of one dW) and the length of one sum (DX: of each of its two)
  T *o[3];               // FWD: h, g, u.  DX: dx.  DW: dWg, dWu
  float *part;           // DW: partial sums [split][2][rows][cols] where the sum is split
  size_t ldo;
  int act;
  unsigned row_tiles, col_tiles, splits, steps;  // steps: k tiles of one split
};

// TM x TN sums (FWD: TM x TN / 2 of each product) by WM x WN waves.  Whole tiles go from memory to LDS without
// passing registers; the last, partial one of a sum goes through them, zero-filled.
template <class T, Kind KIND, int TM, int TN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, 2) void k_gemm(const GemmArgs<T> P) {
  constexpr bool AKS = KIND == DW, BKS = KIND != FWD;
  constexpr int NT = WM * WN * 64, KT = 128 / sizeof(T), E = 16 / sizeof(T);
  constexpr int MI = TM / WM / 16, NI = TN / WN / 16, PA = TM * 8 / NT, PB = TN * 8 / NT;
  constexpr int COLS = KIND == FWD ? TN / 2 : TN;
  __shared__ __align__(128) char l0[(TM + TN) * 128];
  __shared__ __align__(128) char l1[(TM + TN) * 128];

  // consecutive workgroups go to the eight XCDs in turn: each XCD gets a run of tiles, and a run covers bands of
  // eight tile rows column by column, so that its L2 sees the same rows and columns again
  const unsigned tiles = P.row_tiles * P.col_tiles * (KIND == DW ? 2 * P.splits : 1);
  const unsigned per = (tiles + 7) / 8, id = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (id >= tiles) return;
  unsigned t2 = id, z = 0, split = 0;
  if constexpr (KIND == DW) {
    split = id / (P.row_tiles * P.col_tiles * 2);
    t2 = id % (P.row_tiles * P.col_tiles * 2);
    z = t2 / (P.row_tiles * P.col_tiles);
    t2 %= P.row_tiles * P.col_tiles;
  }
  const unsigned band = t2 / (8 * P.col_tiles), in = t2 % (8 * P.col_tiles);
  const unsigned high = P.row_tiles - band * 8 < 8 ? P.row_tiles - band * 8 : 8;
  const size_t r0 = (size_t)(band * 8 + in % high) * TM, c0 = (size_t)(in / high) * COLS;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const T *const a0 = KIND == DW ? P.a[z] : P.a[0];

  // a row of the second operand's tile: the output column it makes, and (FWD) of which product
  auto b_row = [&](int r, size_t &row, bool &up) {
    up = KIND == FWD && ((r >> 4) & 1);
    row = KIND == FWD ? c0 + (r >> 5) * 16 + (r & 15) : c0 + r;
  };
  // where this thread's pieces come from: bytes from the operand's first element of a tile.  Rows behind the
  // matrix are replaced by its last piece of rows: their sums are not stored
  int64_t offa[PA], offb[PB];
#pragma unroll
  for (int j = 0; j < PA; ++j) {
    int r, k;
    piece_of<T, TM, AKS>(j * NT + tid, r, k);
    const size_t most = AKS ? (P.rows - 1) / E * E : P.rows - 1, row = r0 + r < most ? r0 + r : most;
    offa[j] = (int64_t)((AKS ? k * P.lda + row : row * P.lda + k) * sizeof(T));
  }
#pragma unroll
  for (int j = 0; j < PB; ++j) {
    int r, k;
    size_t row;
    bool up;
    piece_of<T, TN, BKS>(j * NT + tid, r, k);
    b_row(r, row, up);
    const size_t most = BKS ? (P.cols - 1) / E * E : P.cols - 1;
    row = row < most ? row : most;
    offb[j] = (int64_t)((BKS ? k * P.ldb + row : row * P.ldb + k) * sizeof(T)) +
              (up ? (const char *)P.b[1] - (const char *)P.b[0] : 0);
  }

  const unsigned kt_all = (unsigned)((P.k + KT - 1) / KT);  // tiles of one sum
  unsigned first = 0, last = KIND == DX ? 2 * kt_all : kt_all;
  if constexpr (KIND == DW) {
    first = split * P.steps;
    last = first + P.steps < last ? first + P.steps : last;
  }
  const unsigned odd = P.k % KT ? kt_all - 1 : kt_all;  // the partial tile of a sum

  auto load = [&](unsigned t, char *to) {
    const bool second = KIND == DX && t >= kt_all;
    const unsigned kt = second ? t - kt_all : t;
    if (kt != odd) {
      const char *pa = (const char *)(second ? P.a[1] : a0) + (AKS ? (size_t)kt * KT * P.lda : (size_t)kt * KT) * sizeof(T);
      const char *pb = (const char *)(second ? P.b[1] : P.b[0]) + (BKS ? (size_t)kt * KT * P.ldb : (size_t)kt * KT) * sizeof(T);
#pragma unroll
      for (int j = 0; j < PA; ++j)
        __builtin_amdgcn_global_load_lds((const QR_GLB void *)(pa + offa[j]), (QR_LDS void *)(to + (j * NT + wave * 64) * 16), 16, 0, 0);
#pragma unroll
      for (int j = 0; j < PB; ++j)
        __builtin_amdgcn_global_load_lds((const QR_GLB void *)(pb + offb[j]), (QR_LDS void *)(to + (TM * 8 + j * NT + wave * 64) * 16),
                                         16, 0, 0);
    } else {
      const size_t kb = (size_t)kt * KT;
#pragma unroll 1
      for (int q = tid; q < TM * 8; q += NT) {
        int r, k;
        piece_of<T, TM, AKS>(q, r, k);
        const T *p = second ? P.a[1] : a0;
        *(i4 *)(to + q * 16) = AKS ? fetch16(p, P.lda, kb + k, P.k, r0 + r, P.rows) : fetch16(p, P.lda, r0 + r, P.rows, kb + k, P.k);
      }
#pragma unroll 1
      for (int q = tid; q < TN * 8; q += NT) {
        int r, k;
        size_t row;
        bool up;
        piece_of<T, TN, BKS>(q, r, k);
        b_row(r, row, up);
        const T *p = second || up ? P.b[1] : P.b[0];
        *(i4 *)(to + (TM * 8 + q) * 16) = BKS ? fetch16(p, P.ldb, kb + k, P.k, row, P.cols) : fetch16(p, P.ldb, row, P.cols, kb + k, P.k);
      }
    }
  };

  f4 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f4{0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const char *from) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      i4 fa[MI], fb[NI];
#pragma unroll
      for (int n = 0; n < NI; ++n) fb[n] = frag<T, TN, BKS>(from + TM * 128, wn * NI + n, s);
#pragma unroll
      for (int m = 0; m < MI; ++m) fa[m] = frag<T, TM, AKS>(from, wm * MI + m, s);
#pragma unroll
      for (int m = 0; m < MI; ++m)
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[m][n] = mma<T>(fb[n], fa[m], acc[m][n]);
    }
  };

  // tile t lies in one half of the LDS while t + 1 arrives in the other; one barrier a tile
  if (first < last) {
    load(first, l0);
    __syncthreads();
    for (unsigned t = first; t < last; t += 2) {
      if (t + 1 < last) load(t + 1, l1);
      compute(l0);
      __syncthreads();
      if (t + 1 < last) {
        if (t + 2 < last) load(t + 2, l0);
        compute(l1);
        __syncthreads();
      }
    }
  }

  // Results pass through the wave's own share of the LDS, so that a lane ends with eight neighbours of a row: one
  // wide store, and one copy of the activation's code.  Pieces of four are XORed with the row against bank conflicts.
  constexpr int WTN = NI * 16, PIECES = WTN / 4, SHARE = (TM + TN) * 256 / (WM * WN);
  constexpr int MB = SHARE / (16 * WTN * 4) < MI ? SHARE / (16 * WTN * 4) : MI;  // blocks of 16 rows at a time
  constexpr int HALF = WM * WN / 2;
  static_assert(MI % MB == 0, "blocks fit the waves' shares");
  char *const own = (wave < HALF ? l0 + wave * SHARE : l1 + (wave - HALF) * SHARE);
  const int l = tid & 63;
#pragma unroll
  for (int m0 = 0; m0 < MI; m0 += MB) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
        *(f4 *)(own + ((m * 16 + (l & 15)) * PIECES + ((n * 4 + (l >> 4)) ^ (l & 15 & (PIECES - 1)))) * 16) = acc[m0 + m][n];
    __builtin_amdgcn_wave_barrier();
    constexpr int SEGS = (KIND == FWD ? WTN / 2 : WTN) / 8;  // eight outputs a lane
#pragma unroll 1
    for (int q = l; q < MB * 16 * SEGS; q += 64) {
      const int r = q / SEGS, s = q % SEGS;
      const size_t row = r0 + (wm * MI + m0) * 16 + r, col = c0 + wn * (SEGS * 8) + s * 8;
      auto take = [&](int piece, float (&v)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f4 x = *(const f4 *)(own + (r * PIECES + ((piece + h) ^ (r & 15 & (PIECES - 1)))) * 16);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[h * 4 + e] = x[e];
        }
      };
      if (row >= P.rows || col >= P.cols) continue;
      float v[8];
      if constexpr (KIND == FWD) {
        float u[8], h[8];
        take((s >> 1) * 8 + (s & 1) * 2, v);
        take((s >> 1) * 8 + 4 + (s & 1) * 2, u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float a, d;
          act_of(P.act, v[e], a, d);
          h[e] = a * u[e];
        }
        store8(P.o[0] + row * P.ldo, h, col, P.cols);
        if (P.o[1]) {
          store8(P.o[1] + row * P.cols, v, col, P.cols);
          store8(P.o[2] + row * P.cols, u, col, P.cols);
        }
      } else {
        take(s * 2, v);
        if (KIND == DW && P.part) store8(P.part + ((size_t)(split * 2 + z) * P.rows + row) * P.cols, v, col, P.cols);
        else store8(P.o[KIND == DW ? z : 0] + row * P.ldo, v, col, P.cols);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// the partial sums of the weights' gradients, joined in the order of the splits
template <class T>
__global__ __launch_bounds__(256) void k_join(const float *__restrict__ part, const size_t n, const unsigned splits, T *__restrict__ o0,
                                              T *__restrict__ o1) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < 2 * n; i += (size_t)gridDim.x * 256) {
    float s = 0.f;
    for (unsigned p = 0; p < splits; ++p) s += part[p * 2 * n + i];
    if (i < n) o0[i] = (T)s;
    else o1[i - n] = (T)s;
  }
}

// dg, du in rows of stride ld, their padding zeroed
template <class T>
__global__ __launch_bounds__(256) void k_gate_grad(const size_t m, const size_t n, const int act, const T *__restrict__ dh,
                                                   const size_t lddh, const T *__restrict__ g, const T *__restrict__ u,
                                                   T *__restrict__ dg, T *__restrict__ du, const size_t ld) {
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < m * ld; i += (size_t)gridDim.x * 256) {
    const size_t r = i / ld, c = i - r * ld;
    float vg = 0.f, vu = 0.f;
    if (c < n) {
      float a, d;
      act_of(act, (float)g[r * n + c], a, d);
      const float v = (float)dh[r * lddh + c];
      vg = v * (float)u[r * n + c] * d;
      vu = v * a;
    }
    dg[i] = (T)vg;
    du[i] = (T)vu;
  }
}

// a matrix whose rows do not start at 16-byte boundaries, copied to one whose rows do; the padding zeroed
template <class T>
__global__ __launch_bounds__(256) void k_pack(const size_t rows, const size_t cols, const T *__restrict__ p, const size_t ld,
                                              T *__restrict__ q, const size_t to) {
  constexpr int E = 16 / sizeof(T);
  const size_t per = to / E;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < rows * per; i += (size_t)gridDim.x * 256) {
    const size_t r = i / per, c = (i - r * per) * E;
    *(i4 *)(q + r * to + c) = fetch16(p, ld, r, rows, c, cols);
  }
}

bool act_ok(int act) { return act >= QR_ACT_SILU && act <= QR_ACT_SIGMOID; }
unsigned tiles_of(size_t n, size_t t) { return (unsigned)((n + t - 1) / t); }

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
size_t padded(size_t cols, size_t e) { return (cols + 16 / e - 1) / (16 / e) * (16 / e); }
size_t pack_bytes(size_t rows, size_t cols, size_t e) { return round256(rows * padded(cols, e) * e); }
unsigned blocks(size_t n) { return (unsigned)((n + 255) / 256 < 65536 ? (n + 255) / 256 : 65536); }

// whether the product kernel can read a matrix where it lies: rows at 16-byte boundaries and, where the columns are
// what it moves in pieces (the columns layout), none cut by the row's end
bool in_place(const void *p, size_t ld, size_t cols, size_t e, bool columns) {
  return ((uintptr_t)p & 15) == 0 && (ld * e) % 16 == 0 && (!columns || (cols * e) % 16 == 0);
}

template <class T>
void pack(hipStream_t s, size_t rows, size_t cols, const T *&p, size_t ld, char *&ws) {
  const size_t to = padded(cols, sizeof(T));
  if (rows) k_pack<T><<<blocks(rows * to * sizeof(T) / 16), 256, 0, s>>>(rows, cols, p, ld, (T *)ws, to);
  p = (const T *)ws;
  ws += pack_bytes(rows, cols, sizeof(T));
}

template <class T, Kind KIND, int TM, int TN, int WM, int WN>
void launch_gemm(hipStream_t s, GemmArgs<T> P) {
  P.row_tiles = tiles_of(P.rows, TM);
  P.col_tiles = tiles_of(P.cols, KIND == FWD ? TN / 2 : TN);
  const unsigned tiles = P.row_tiles * P.col_tiles * (KIND == DW ? 2 * P.splits : 1);
  k_gemm<T, KIND, TM, TN, WM, WN><<<(tiles + 7) / 8 * 8, WM * WN * 64, 0, s>>>(P);
}

constexpr unsigned CUS = 256;

// Outputs a workgroup takes: the largest square that still gives every compute unit a tile.
int tile_of(size_t e, size_t rows, size_t cols, size_t times) {
  if (e == 2 && (size_t)tiles_of(rows, 256) * tiles_of(cols, 256) * times >= CUS) return 256;
  if ((size_t)tiles_of(rows, 128) * tiles_of(cols, 128) * times >= CUS) return 128;
  return 64;
}

template <class T, Kind KIND>
void gemm(hipStream_t s, int tile, const GemmArgs<T> &P) {
  if constexpr (sizeof(T) == 2)
    if (tile == 256) return launch_gemm<T, KIND, 256, 256, 2, 4>(s, P);
  if (tile == 128) return launch_gemm<T, KIND, 128, 128, 2, 2>(s, P);
  launch_gemm<T, KIND, 64, 64, 2, 2>(s, P);
}

// The weights' gradients sum over all m rows: with few outputs the sum is split so that the launch fills the
// compute units, in shares of at least 512 rows.
void plan_dw(size_t e, size_t m, size_t k, size_t n, int &tile, unsigned &splits, unsigned &steps) {
  const size_t kt = 128 / e, tiles = (m + kt - 1) / kt;
  const size_t most = m / 512 ? m / 512 : 1;
  tile = tile_of(e, n, k, 2 * most);
  const size_t out = 2 * (size_t)tiles_of(n, tile) * tiles_of(k, tile);
  size_t want = (2 * CUS + out - 1) / out;
  want = want < most ? want : most;
  if (!want) want = 1;
  steps = (unsigned)((tiles + want - 1) / want);
  if (!steps) steps = 1;
  splits = (unsigned)((tiles + steps - 1) / steps);
  if (!splits) splits = 1;
}

}  // namespace

extern "C" int qr_gated_ffn_workspace(int type, size_t m, size_t k, size_t n, size_t *bytes) {
  QR_DENSE_ARG(bytes && qr_dense_type_ok(type) && k > 0 && n > 0 && qr_dense_fits(m, k, k) && qr_dense_fits(n, k, k),
               "gated ffn: bad size");
  const size_t e = qr_dense_size(type);
  *bytes = m ? pack_bytes(m, k, e) + 2 * pack_bytes(n, k, e) + 256 : 0;
  return QR_OK;
}

extern "C" int qr_gated_ffn_async(int device, void *stream, int type, int act, size_t m, size_t k, size_t n, const void *x, size_t ldx,
                                  const void *w_gate, const void *w_up, size_t ldw, void *h, size_t ldh, void *gate, void *up,
                                  void *workspace, size_t workspace_bytes) {
  QR_DENSE_ARG(qr_dense_type_ok(type), "gated ffn: unknown element type");
  QR_DENSE_ARG(act_ok(act), "gated ffn: unknown activation");
  QR_DENSE_ARG(k > 0 && n > 0, "gated ffn: no columns");
  QR_DENSE_ARG(qr_dense_fits(m, k, ldx) && qr_dense_fits(n, k, ldw) && qr_dense_fits(m, n, ldh), "gated ffn: sizes out of range");
  QR_DENSE_ARG(m < 2 || ldh >= n, "gated ffn: the stride of h is shorter than a row");
  QR_DENSE_ARG(!gate == !up, "gated ffn: gate and up are kept both or neither");
  if (!m) return QR_OK;
  QR_DENSE_ARG(x && w_gate && w_up && h, "gated ffn: x, a weight or h is NULL");
  const size_t e = qr_dense_size(type);
  const bool px = !in_place(x, ldx, k, e, false), pw = !in_place(w_gate, ldw, k, e, false) || !in_place(w_up, ldw, k, e, false);
  size_t need = 0;
  if (px || pw)
    if (int rc = qr_gated_ffn_workspace(type, m, k, n, &need)) return rc;
  QR_DENSE_ARG(!need || (workspace && workspace_bytes >= need),
               "gated ffn: rows that do not start at 16-byte boundaries need the workspace");
  const void *out[4] = {h, gate, up, workspace};
  const size_t bytes[4] = {qr_dense_span(m, n, ldh, e), m * n * e, m * n * e, need};
  for (int i = 0; i < 4; ++i) {
    QR_DENSE_ARG(!qr_dense_overlap(out[i], bytes[i], x, qr_dense_span(m, k, ldx, e)) &&
                     !qr_dense_overlap(out[i], bytes[i], w_gate, qr_dense_span(n, k, ldw, e)) &&
                     !qr_dense_overlap(out[i], bytes[i], w_up, qr_dense_span(n, k, ldw, e)),
                 "gated ffn: an output lies over an input");
    for (int j = 0; j < i; ++j) QR_DENSE_ARG(!qr_dense_overlap(out[i], bytes[i], out[j], bytes[j]), "gated ffn: outputs overlap");
  }
  QR_DENSE_DEVICE(device);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    const hipStream_t s = (hipStream_t)stream;
    char *ws = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    GemmArgs<T> P{};
    P.a[0] = (const T *)x, P.b[0] = (const T *)w_gate, P.b[1] = (const T *)w_up;
    P.lda = ldx, P.ldb = ldw, P.rows = m, P.cols = n, P.k = k;
    P.o[0] = (T *)h, P.o[1] = (T *)gate, P.o[2] = (T *)up, P.ldo = ldh, P.act = act;
    if (px) pack(s, m, k, P.a[0], ldx, ws), P.lda = padded(k, e);
    if (pw) pack(s, n, k, P.b[0], ldw, ws), pack(s, n, k, P.b[1], ldw, ws), P.ldb = padded(k, e);
    gemm<T, FWD>(s, tile_of(e, m, 2 * n, 1), P);
  });
  return qr_dense_launched("gated ffn");
}

extern "C" int qr_gated_ffn_backward_workspace(int type, size_t m, size_t k, size_t n, size_t *bytes) {
  QR_DENSE_ARG(bytes && qr_dense_type_ok(type) && k > 0 && n > 0 && qr_dense_fits(m, n, n) && qr_dense_fits(m, k, k) && qr_dense_fits(n, k, k),
               "gated ffn backward: bad size");
  const size_t e = qr_dense_size(type);
  int tile;
  unsigned splits, steps;
  plan_dw(e, m, k, n, tile, splits, steps);
  // dg, du, the partial sums, copies of x and the weights where their rows are not aligned
  *bytes = m ? 2 * pack_bytes(m, n, e) + round256(splits > 1 ? (size_t)splits * 2 * n * k * 4 : 0) + pack_bytes(m, k, e) +
                   2 * pack_bytes(n, k, e) + 256
             : 0;
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
    char *ws = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    const size_t ld = padded(n, e);
    T *const dg = (T *)ws, *const du = (T *)(ws + pack_bytes(m, n, e));
    ws += 2 * pack_bytes(m, n, e);
    if (m)
      k_gate_grad<T><<<blocks(m * ld), 256, 0, s>>>(m, n, act, (const T *)dh, lddh, (const T *)gate, (const T *)up, dg, du, ld);
    if (dx && m) {
      GemmArgs<T> P{};
      P.a[0] = dg, P.a[1] = du, P.b[0] = (const T *)w_gate, P.b[1] = (const T *)w_up;
      P.lda = ld, P.ldb = ldw, P.rows = m, P.cols = k, P.k = n, P.o[0] = (T *)dx, P.ldo = lddx;
      if (!in_place(w_gate, ldw, k, e, true) || !in_place(w_up, ldw, k, e, true))
        pack(s, n, k, P.b[0], ldw, ws), pack(s, n, k, P.b[1], ldw, ws), P.ldb = padded(k, e);
      gemm<T, DX>(s, tile_of(e, m, k, 1), P);
    }
    if (dw_gate) {
      GemmArgs<T> P{};
      int tile;
      plan_dw(e, m, k, n, tile, P.splits, P.steps);
      P.a[0] = dg, P.a[1] = du, P.b[0] = (const T *)x, P.lda = ld, P.ldb = ldx, P.rows = n, P.cols = k, P.k = m;
      P.o[0] = (T *)dw_gate, P.o[1] = (T *)dw_up, P.ldo = k;
      if (m && !in_place(x, ldx, k, e, true)) pack(s, m, k, P.b[0], ldx, ws), P.ldb = padded(k, e);
      if (P.splits > 1) P.part = (float *)ws;
      gemm<T, DW>(s, tile, P);
      if (P.splits > 1)
        k_join<T><<<blocks(2 * n * k), 256, 0, s>>>(P.part, n * k, P.splits, (T *)dw_gate, (T *)dw_up);
    }
  });
  return qr_dense_launched("gated ffn backward");
}
