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
#include <algorithm>
#include <type_traits>

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
  } else {
    // gelu_tanh is g sigmoid(2 c (g + 0.044715 g^3)), c = sqrt(2 / pi).  The hardware's exp2 and reciprocal are good to
    // one step of f32, the product in exp2's argument to |g| steps
    const float c2 = 1.5957691216057308f, z = act == QR_ACT_GELU_TANH ? c2 * fmaf(0.044715f * g * g, g, g) : g;
    const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
    // s' / z'.  Where it is 0 (far from zero, in f32) the derivative is s, though z' may be infinite
    const float t = s * (1.f - s);
    a = act == QR_ACT_SIGMOID ? s : g * s;
    d = act == QR_ACT_SIGMOID ? t
                              : t == 0.f ? s : fmaf(g * (act == QR_ACT_GELU_TANH ? c2 * fmaf(3.f * 0.044715f * g, g, 1.f) : 1.f), t, s);
  }
}

// f(activation) as a constant
template <class F>
__host__ __device__ __forceinline__ void by_act(const int act, F &&f) {
  if (act == QR_ACT_SILU) f(std::integral_constant<int, QR_ACT_SILU>{});
  else if (act == QR_ACT_GELU) f(std::integral_constant<int, QR_ACT_GELU>{});
  else if (act == QR_ACT_GELU_TANH) f(std::integral_constant<int, QR_ACT_GELU_TANH>{});
  else if (act == QR_ACT_RELU) f(std::integral_constant<int, QR_ACT_RELU>{});
  else f(std::integral_constant<int, QR_ACT_SIGMOID>{});
}

typedef float f4 __attribute__((ext_vector_type(4)));
typedef int i4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
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

// f32 operands of the product kernel as three bf16 each: 24 bits of mantissa are 8 + 8 + 8, so high + mid + low IS the
// number (down to 2^-110; one that is infinite, or 2^128 - 2^119 and more, has NaN parts).  Each part is the nearest to what
// is left, so that the next is small and of either sign: of the nine products the six largest are taken, each exact in f32;
// those left out are at most 2 x 2^-24 of the product, 0.09 x 2^-24 by the root of their mean square, and lean to no side.
// (Parts cut off instead leave out 7 x 2^-24 at most and 0.63 x 2^-24 on average, always toward zero; 1 to 4 % less time.)
// Six bf16 matrix instructions take 96 cycles for 16 x 16 x 32 where the f32 ones take 256, at 5.5 vector instructions an
// element of each fragment.
struct Split {
  b8 part[3];
};
__device__ __forceinline__ Split three_parts(const i4 u, const i4 v) {
  const f4 fu = __builtin_bit_cast(f4, u), fv = __builtin_bit_cast(f4, v);
  float x[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = fu[e], x[4 + e] = fv[e];
  Split s;
#pragma unroll
  for (int p = 0; p < 3; ++p) {
    i4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (p < 2) {  // two numbers at a time; what rounding leaves of each is exact
        const b2 near = __builtin_convertvector(f2{x[2 * e], x[2 * e + 1]}, b2);
        const uint32_t both = __builtin_bit_cast(uint32_t, near);
        w[e] = (int)both;
        x[2 * e] -= __builtin_bit_cast(float, both << 16);
        x[2 * e + 1] -= __builtin_bit_cast(float, both & 0xFFFF0000u);
      } else {  // (eight bits each: their upper halves)
        w[e] = (int)__builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, x[2 * e + 1]), __builtin_bit_cast(uint32_t, x[2 * e]), 0x07060302u);
      }
    }
    s.part[p] = __builtin_bit_cast(b8, w);
  }
  return s;
}

// ---- LDS tiles -----------------------------------------------------------------------------------------
// A stage holds R rows (outputs) of KT = 128 / sizeof(T) summed elements in 128 R bytes, moved in pieces of 16.  A row's
// 128 bytes are a whole line of the L2, whose requests, not its bytes, were the bound with rows of 64 (1159 against 1344
// TFLOP/s at 8192 x 8192 x 4096 bf16).
//
// Rows layout: row r at 128 r, its piece c at position c ^ (r & 7).  A 16-byte read of a wave is served in four parts,
// lanes 0-3 12-15 20-27, 4-11 16-19 28-31 and the same 32 higher; the lanes of each touch every bank once.
// Columns layout: summed element k at k R sizeof(T), blocks of 16 elements permuted within the line (col_at) so that the
// lanes of one read, which lie in 8 (16-bit) or 4 (f32) such lines, touch every bank once (but for widths of f32 that are
// no power of two).
// the position of block `b` of 16 elements in the line of summed element k
template <class T, int R>
__device__ __forceinline__ int col_at(const int b, const int k) {
  if constexpr (sizeof(T) == 4) {
    const int f = (k >> 2) & 3;
    if constexpr ((R & (R - 1)) == 0) return b ^ f;
    else return b + f >= R / 16 ? b + f - R / 16 : b + f;
  } else if constexpr (R >= 128) {
    return b ^ ((k & 3) | (((k >> 3) & 1) << 2));
  } else {
    return b ^ (((k >> 1) & 1) | (((k >> 3) & 1) << 1));  // two lines of 128 bytes share the banks
  }
}

// the piece q (of R * 8) of a stage in LDS order -> where it comes from
template <class T, int R, bool KS>
__device__ __forceinline__ void piece_of(const int q, int &r, int &k) {
  constexpr int E = 16 / sizeof(T);
  if constexpr (!KS) {
    r = q >> 3;
    k = ((q & 7) ^ (r & 7)) * E;
  } else {
    constexpr int PER = R / E, B = 16 / E;  // pieces of a line, of a block
    k = q / PER;
    const int at = (q % PER) / B;
    int b = col_at<T, R>(at, k);  // (exclusive or undoes itself)
    if constexpr ((R & (R - 1)) != 0) {
      b = at - ((k >> 2) & 3);
      b = b < 0 ? b + R / 16 : b;
    }
    r = b * 16 + (q % B) * E;
  }
}

// One operand fragment: 16 rows of one half (0, 1) of a stage, the c-th block of 16 behind the wave's first, `block` (a
// multiple of the blocks a wave has).  `at` is the address frag_base gave; a block's number and the half are XORed in where
// they can be.
template <class T, int R, bool KS>
__device__ __forceinline__ uint32_t frag_base(const uint32_t stage, const int block) {
  const int l = threadIdx.x & 63, g = l >> 4, i = l & 15;
  if constexpr (!KS) {
    return stage + (block * 16 + i) * 128 + ((g ^ (i & 7)) << 4);
  } else if constexpr (sizeof(T) == 2) {
    const int k = 8 * g + (i >> 2);
    return stage + k * (R * 2) + (col_at<T, R>(block, k) << 5) + (i & 3) * 8;
  } else {
    return stage + 4 * g * (R * 4) + i * 4;
  }
}
template <class T, int R, bool KS>
__device__ __forceinline__ i4 frag(const uint32_t at, const int block, const int c, const int half) {
  if constexpr (!KS) {
    return *(QR_LDS const i4 *)((at ^ (half << 6)) + c * 2048);
  } else if constexpr (sizeof(T) == 2) {
    const uint32_t p = (at ^ (c << 5)) + half * (32 * R * 2);
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QR_LDS s4 *)p);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((QR_LDS s4 *)(p + 4 * R * 2));
    return __builtin_bit_cast(i4, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
  } else {
    const uint32_t p = at + (col_at<T, R>(block + c, 4 * ((threadIdx.x & 63) >> 4)) << 6) + half * (16 * R * 4);
    i4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = *(QR_LDS const int *)(p + e * R * 4);
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

// V neighbouring results of one row, rounded; the row's base need not be aligned.  `stream`: past the caches
template <class T, int V>
__device__ __forceinline__ void store(const bool stream, T *p, const float (&v)[V], const size_t at, const size_t len) {
  typedef int words __attribute__((ext_vector_type(V / 2)));
  if (at + V <= len) {
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = (T)v[e];
    if constexpr (sizeof(T) == 2)
      if (stream) {
        __builtin_nontemporal_store(__builtin_bit_cast(words, t), (words *)(p + at));
        return;
      }
    __builtin_memcpy(p + at, t, sizeof t);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (at + e < len) p[at + e] = (T)v[e];
  }
}

// ---- the product -----------------------------------------------------------------------------------------
enum Kind { FWD, DX, DW };

template <class T>
struct GemmArgs {
  const T *a[2], *b[2];  // FWD: x | Wg, Wu.  DX: dg, du | Wg, Wu.  DW: dg, du | x.  Rows at 16-byte boundaries
  size_t lda, ldb;
  size_t rows, cols, k;  // outputs (FWD: of h; DW: of one dW), length of one sum (DX: of each of its two, whole stages)
  T *o[3];               // FWD: h, g, u.  DX: dx.  DW: dWg, dWu
  float *part;           // partial sums, DX [split][rows][cols], DW [split][2][rows][cols], where the sums are split
  const float *back;     // f16 DX, DW: what the sums are multiplied by (dg and du are held times its reciprocal), or NULL
  size_t ldo;
  int act;
  bool stream;           // results go past the caches
  unsigned row_tiles, col_tiles, splits, steps;  // steps: k tiles of one split
};

// Memory to LDS and its order.  The loads are written by hand so that the compiler does not wait for them in front of
// LDS reads of other stages; every wait they need is wait_all, and all waves' parts are there behind the barrier after it.
// 64 lanes bring 16 bytes each, from `base` + their `off`, to consecutive LDS addresses from `to` on.
// (The wait states are those between a vector instruction's write of a scalar register and the load that reads it.)
__device__ __forceinline__ void dma16(const char *base, const uint32_t off, const uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(to)), "v"(off),
               "s"(base)
               : "m0");
}
// none of this wave's loads and LDS operations is under way
__device__ __forceinline__ void wait_all() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { asm volatile("s_barrier" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_offset(const char *p) { return (uint32_t)(uintptr_t)(QR_LDS const char *)p; }

// TM x TN sums (FWD: TM x TN / 2 of each product) by 2 x WN waves.  While the matrix cores work on one stage the next is
// on its way.  WN = 2: the first operand's to the other half of its LDS buffer without passing registers, the second's in
// registers, from where it is written to its single buffer behind a barrier.  (Both double-buffered, two workgroups of 256
// x 128 would not fit a compute unit, 160 KB; they do, and one's matrix instructions run under the other's waits, first
// loads and epilogue.)  WN = 4, 256 x 256: one workgroup fills the compute unit; both operands are double-buffered and
// pass no registers, and the next stage is sent for in the first half of this one.  The last, partial stage of a sum is
// zero-filled.  RAG (FWD, WN = 2): rows at any alignment, both operands through registers.
//
// What bounds it, 16-bit types: at 256 x 128 the way from L2 to the compute units (48 bytes a cycle and unit at the full
// matrix rate, of 64), at 256 x 256 (32 bytes) the matrix cores at the clock that the card holds under them, 1.9 GHz (76 %
// of the cycles).  1490 TF at 8192 x 8192 x (2 x 4096) bf16, where a large library product reaches 1300; 1240 TF at 32768 x
// 1024 x (2 x 4096), whose 16 stages leave a fifth of a tile's time to its first loads and its results (1040 TF with g and u
// stored too: 805 MB whose writing overlaps little).
// f32: the six products and the splits before them, whose times add up: 190 TF at 4096 x 1024 x (2 x 4096), the matrix cores
// busy for 50 % of the cycles (37 and 46 % in the gradients of 136 columns, padded to 160).
template <class T, Kind KIND, int TM, int TN, int WN, bool RAG>
__global__ __launch_bounds__(128 * WN, 2) void k_gemm(const GemmArgs<T> P) {
  constexpr bool AKS = KIND == DW, BKS = KIND != FWD, BD = WN > 2;
  constexpr int WM = 2, NT = 128 * WN, KT = 128 / sizeof(T), E = 16 / sizeof(T);
  constexpr int MI = TM / WM / 16, NI = TN / WN / 16, PA = TM * 8 / NT, PB = TN * 8 / NT;
  constexpr int COLS = KIND == FWD ? TN / 2 : TN;
  constexpr bool DIRECT = KIND == FWD && sizeof(T) == 2;  // results are stored from the registers of the sums
  constexpr uint32_t ABUF = TM * 128, BBUF = BD ? TN * 128 : 0, LDS_BYTES = 2 * ABUF + TN * 128 + BBUF;
  __shared__ __align__(1024) char lds[LDS_BYTES];

  // consecutive workgroups go to the eight XCDs in turn: each XCD gets a run of tiles, and a run covers bands of
  // eight tile rows column by column, so that its L2 sees the same rows and columns again
  constexpr unsigned OUTS = KIND == DW ? 2 : 1;
  const unsigned one = P.row_tiles * P.col_tiles, tiles = one * OUTS * (KIND == FWD ? 1 : P.splits);
  const unsigned per = (tiles + 7) / 8, id = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (id >= tiles) return;
  const unsigned split = KIND == FWD ? 0 : id / (one * OUTS), z = KIND == DW ? id / one % 2 : 0, t2 = KIND == FWD ? id : id % one;
  const unsigned band = t2 / (8 * P.col_tiles), in = t2 % (8 * P.col_tiles);
  const unsigned high = P.row_tiles - band * 8 < 8 ? P.row_tiles - band * 8 : 8;
  const size_t r0 = (size_t)(band * 8 + in % high) * TM, c0 = (size_t)(in / high) * COLS;

  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;

  // a row of the second operand's tile: the output column it makes, and (FWD) of which product
  auto b_row = [&](int r, size_t &row, bool &up) {
    up = KIND == FWD && ((r >> 4) & 1);
    row = c0 + r;
    // (of a wave's two pairs of blocks, 16-bit types: by fours in turn, so that a lane's sums of both are eight neighbours)
    if (KIND == FWD) row = c0 + (DIRECT && NI == 4 ? (r >> 6) * 32 + ((r >> 2) & 3) * 8 + ((r >> 5) & 1) * 4 + (r & 3) : (r >> 5) * 16 + (r & 15));
  };
  const unsigned kt_all = (unsigned)((P.k + KT - 1) / KT);  // stages of one sum
  unsigned first = 0, last = KIND == DX ? 2 * kt_all : kt_all;
  const bool odd = KIND != DX && P.k % KT;  // (DX: both sums are whole stages)
  unsigned whole = odd ? last - 1 : last;   // stages that are whole
  if constexpr (KIND != FWD) {
    first = split * P.steps;
    last = first + P.steps < last ? first + P.steps : last;
    whole = whole < last ? whole : last;
  }

  // Where this thread's pieces of a stage come from: bytes from the operand's next stage of the tile (a wave's pieces of
  // the forward pass's second operand are all of one weight; 256 rows stay below 2^31 bytes).  Rows behind the matrix are
  // replaced by its last piece of rows: their sums are not stored
  uint32_t offa[PA], offb[PB];
#pragma unroll
  for (int j = 0; j < PA; ++j) {
    int r, k;
    piece_of<T, TM, AKS>(j * NT + tid, r, k);
    const uint32_t most = (uint32_t)((AKS ? (P.rows - 1) / E * E : P.rows - 1) - r0 < TM - 1 ? (AKS ? (P.rows - 1) / E * E : P.rows - 1) - r0 : TM - 1);
    const uint32_t row = (uint32_t)r < most ? r : most;
    offa[j] = (AKS ? k * (uint32_t)P.lda + row : row * (uint32_t)P.lda + k) * sizeof(T);
  }
#pragma unroll
  for (int j = 0; j < PB; ++j) {
    int r, k;
    size_t row;
    bool up;
    piece_of<T, TN, BKS>(j * NT + tid, r, k);
    b_row(r, row, up);
    const size_t most = BKS ? (P.cols - 1) / E * E : P.cols - 1;
    const uint32_t rel = (uint32_t)((row < most ? row : most) - c0);
    offb[j] = (BKS ? k * (uint32_t)P.ldb + rel : rel * (uint32_t)P.ldb + k) * sizeof(T);
  }
  const unsigned second = KIND == DX && first >= kt_all ? 1 : 0;
  const size_t k0 = (size_t)(first - (second ? kt_all : 0)) * KT;
  const char *sa = (const char *)(P.a[KIND == DW ? z : second] + (AKS ? k0 * P.lda + r0 : r0 * P.lda + k0));
  const char *sb = (const char *)(P.b[KIND == FWD ? (wave >> 1) & 1 : second] + (BKS ? k0 * P.ldb + c0 : c0 * P.ldb + k0));
  // stages are loaded in order
  auto next_a = [&](const unsigned t) {
    sa += (AKS ? KT * P.lda : (size_t)KT) * sizeof(T);
    if (KIND == DX && t + 1 == kt_all) sa = (const char *)(P.a[1] + r0 * P.lda);
  };
  auto next_b = [&](const unsigned t) {
    sb += (BKS ? KT * P.ldb : (size_t)KT) * sizeof(T);
    if (KIND == DX && t + 1 == kt_all) sb = (const char *)(P.b[1] + c0);
  };
  i4 va[RAG ? PA : 1], vb[PB];
  auto load_a = [&](const int d, const uint32_t to) { dma16(sa, offa[d], to + (d * NT + wave * 64) * 16); };
  auto dma_b = [&](const int d, const uint32_t to) { dma16(sb, offb[d], to + (d * NT + wave * 64) * 16); };
  // A piece of a row at any alignment (RAG); in the partial stage one that lies across the sum's end is put together
  auto ragged = [&](const char *p, const unsigned t, const int d) {
    i4 v;
    if (t < whole) {
      typedef int loose __attribute__((ext_vector_type(4), aligned(2)));
      v = *(const QR_GLB loose *)(const QR_GLB char *)p;
    } else {
      int r, k;
      piece_of<T, TM, false>(d * NT + tid, r, k);
      v = fetch16((const T *)p - k, 0, 0, 1, k, P.k - (size_t)t * KT);
    }
    return v;
  };
  // The partial stage's: pieces inside the sum (none lies across its end) come as a whole stage's do, the others are zero
  auto inside = [&](const auto tile, const bool columns, const unsigned t, const int d) {
    int r, k;
    if (columns) piece_of<T, tile(), true>(d * NT + tid, r, k);
    else piece_of<T, tile(), false>(d * NT + tid, r, k);
    return (size_t)t * KT + k < P.k;
  };
  constexpr std::integral_constant<int, TM> tile_a;
  constexpr std::integral_constant<int, TN> tile_b;
  auto part_a = [&](const unsigned t, const uint32_t to) {
#pragma unroll
    for (int d = 0; d < PA; ++d) {
      if (inside(tile_a, AKS, t, d)) load_a(d, to);
      else *(QR_LDS i4 *)(to + (d * NT + tid) * 16) = i4{0, 0, 0, 0};
    }
  };
  auto part_b = [&](const unsigned t, const uint32_t to) {
#pragma unroll
    for (int d = 0; d < PB; ++d) {
      if (inside(tile_b, BKS, t, d)) dma_b(d, to);
      else *(QR_LDS i4 *)(to + (d * NT + tid) * 16) = i4{0, 0, 0, 0};
    }
  };
  auto load_b = [&](const unsigned t) {
#pragma unroll
    for (int d = 0; d < PB; ++d) {
      if constexpr (RAG) {
        vb[d] = ragged(sb + offb[d], t, d);
      } else {
        vb[d] = i4{0, 0, 0, 0};
        if (KIND == DX || t < whole || inside(tile_b, BKS, t, d)) vb[d] = *(const QR_GLB i4 *)((const QR_GLB char *)sb + offb[d]);
      }
    }
    next_b(t);
  };
  auto keep_b = [&]() {
#pragma unroll
    for (int d = 0; d < PB; ++d) *(i4 *)(lds + 2 * ABUF + (d * NT + tid) * 16) = vb[d];
  };
  auto ragged_a = [&](const unsigned t) {
#pragma unroll
    for (int d = 0; d < PA; ++d) va[d] = ragged(sa + offa[d], t, d);
    next_a(t);
  };
  auto keep_a = [&](const uint32_t to) {
#pragma unroll
    for (int d = 0; d < PA; ++d) *(i4 *)(lds + to + (d * NT + tid) * 16) = va[d];
  };

  f4 acc[MI][NI];
#pragma unroll
  for (int m = 0; m < MI; ++m)
#pragma unroll
    for (int n = 0; n < NI; ++n) acc[m][n] = f4{0.f, 0.f, 0.f, 0.f};
  const uint32_t base_a = frag_base<T, TM, AKS>(lds_offset(lds), wm * MI);
  const uint32_t base_b = frag_base<T, TN, BKS>(lds_offset(lds) + 2 * ABUF, wn * NI);
  auto read_a = [&](const uint32_t ra, const int m, const int half) { return frag<T, TM, AKS>(ra, wm * MI, m, half); };
  // 16-bit types: a stage's 2 x MI rows of blocks, the first operand's fragments read D ahead of their use.
  // f32: its MI rows of blocks, split into three parts, one ahead.  In the steady state the next stage's loads are spread
  // over the rows.
  auto compute = [&](auto steady, const uint32_t ra, const uint32_t rb, const uint32_t to, const uint32_t to_b) {
    constexpr bool STEADY = decltype(steady)::value;
    auto read_b = [&](const int n, const int half) { return frag<T, TN, BKS>(rb, wn * NI, n, half); };
    if constexpr (sizeof(T) == 4) {
      Split fb[NI];
      i4 next[2] = {read_a(ra, 0, 0), read_a(ra, 0, 1)};
#pragma unroll
      for (int n = 0; n < NI; ++n) fb[n] = three_parts(read_b(n, 0), read_b(n, 1));
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const Split fa = three_parts(next[0], next[1]);
        if (m + 1 < MI) next[0] = read_a(ra, m + 1, 0), next[1] = read_a(ra, m + 1, 1);
        if constexpr (STEADY)
#pragma unroll
          for (int d = m * PA / MI; d < (m + 1) * PA / MI && !RAG; ++d) load_a(d, to);
        constexpr int HI[6] = {1, 0, 2, 0, 1, 0}, LO[6] = {1, 2, 0, 1, 0, 0};  // the smallest first
#pragma unroll
        for (int p = 0; p < 6; ++p)
#pragma unroll
          for (int n = 0; n < NI; ++n)
            acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[n].part[HI[p]], fa.part[LO[p]], acc[m][n], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      constexpr int D = MI > 3 ? 3 : MI - 1, ROWS = BD ? MI : 2 * MI;  // rows over which the loads are spread
      i4 fa[D + 1], fb[2][NI];
#pragma unroll
      for (int n = 0; n < NI; ++n) fb[0][n] = read_b(n, 0);
#pragma unroll
      for (int m = 0; m < D; ++m) fa[m] = read_a(ra, m, 0);
#pragma unroll
      for (int q = 0; q < 2 * MI; ++q) {
        if (q + D < 2 * MI) fa[(q + D) % (D + 1)] = read_a(ra, (q + D) % MI, (q + D) / MI);
        if (q < MI)
#pragma unroll
          for (int n = q * NI / MI; n < (q + 1) * NI / MI; ++n) fb[1][n] = read_b(n, 1);
        if constexpr (STEADY)
#pragma unroll
          for (int d = q * PA / ROWS; d < (q + 1) * PA / ROWS && d < PA && !RAG; ++d) load_a(d, to);
        if constexpr (STEADY && BD)
#pragma unroll
          for (int d = q * PB / ROWS; d < (q + 1) * PB / ROWS && d < PB; ++d) dma_b(d, to_b);
#pragma unroll
        for (int n = 0; n < NI; ++n) acc[q % MI][n] = mma<T>(fb[q / MI][n], fa[q % (D + 1)], acc[q % MI][n]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  const uint32_t at_a = lds_offset(lds), at_b = at_a + 2 * ABUF;
  if (first < last) {
    if (RAG) {
      ragged_a(first);
      keep_a(0);
    } else if (KIND == DX || first < whole) {
#pragma unroll
      for (int d = 0; d < PA; ++d) load_a(d, at_a);
      next_a(first);
    } else {
      part_a(first, at_a);
    }
    if (!BD) {
      load_b(first);
      keep_b();
    } else if (KIND == DX || first < whole) {
#pragma unroll
      for (int d = 0; d < PB; ++d) dma_b(d, at_b);
      next_b(first);
    } else {
      part_b(first, at_b);
    }
    uint32_t cur = 0, cur_b = 0;
    unsigned t = first;
    for (; t + 1 < whole; ++t, cur ^= ABUF, cur_b ^= BBUF) {
      wait_all();
      barrier();  // stage t is there, and every wave is done with stage t - 1 where there are two buffers
      if (RAG) ragged_a(t + 1);
      if (!BD) load_b(t + 1);
      compute(std::true_type{}, base_a + cur, base_b + cur_b, at_a + (cur ^ ABUF), at_b + (cur_b ^ BBUF));
      if (RAG) keep_a(cur ^ ABUF);
      else next_a(t + 1);
      if (BD) {
        next_b(t + 1);
      } else {
        barrier();  // every wave is done with the second operand's stage t
        keep_b();
      }
    }
    for (; t < last; ++t, cur ^= ABUF, cur_b ^= BBUF) {
      wait_all();
      barrier();
      if (t + 1 < last) {
        if (RAG) ragged_a(t + 1);
        else part_a(t + 1, at_a + (cur ^ ABUF));
        if (BD) part_b(t + 1, at_b + (cur_b ^ BBUF));
        else load_b(t + 1);
      }
      compute(std::false_type{}, base_a + cur, base_b + cur_b, 0, 0);
      if (!BD || t + 1 == last) barrier();
      if (!BD && t + 1 < last) {
        if (RAG) keep_a(cur ^ ABUF);
        keep_b();
      }
    }
  }

  const int l = tid & 63;
  const bool stream = sizeof(T) == 2 && P.stream;
  if constexpr (DIRECT) {
    // A lane has g and u of V neighbours of a row, for each block of 16 rows; four lanes make 64 bytes of a row.  (Through
    // LDS 466 us where this takes 438, 32768 x 1024 x 4096 bf16; f32 results, twice as wide, come out faster through LDS:
    // 158 against 205 us, 100000 x 32 x 512 with g and u.)
    constexpr int V = NI * 2;
    auto finish = [&](auto act) {
#pragma unroll
      for (int m = 0; m < MI; ++m) {
        const size_t row = r0 + (wm * MI + m) * 16 + (l & 15), col = c0 + wn * (NI * 8) + (l >> 4) * V;
        if (row >= P.rows || col >= P.cols) continue;
        float g[V], u[V], h[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
          float a, d;
          g[e] = acc[m][e / 4 * 2][e % 4], u[e] = acc[m][e / 4 * 2 + 1][e % 4];
          act_of(act(), g[e], a, d);
          h[e] = a * u[e];
        }
        store(stream, P.o[0] + row * P.ldo, h, col, P.cols);
        if (P.o[1]) {
          store(stream, P.o[1] + row * P.cols, g, col, P.cols);
          store(stream, P.o[2] + row * P.cols, u, col, P.cols);
        }
      }
    };
    by_act(P.act, finish);
    return;
  }
  // Results pass through the wave's own share of the LDS, so that a lane ends with eight neighbours of a row: one
  // wide store.  Pieces of four are moved by the row against bank conflicts.
  constexpr int WTN = NI * 16, PIECES = WTN / 4, SHARE = LDS_BYTES / (WM * WN) / (16 * WTN * 4) * (16 * WTN * 4);
  constexpr int FIT = SHARE / (16 * WTN * 4), MB = FIT >= MI ? MI : FIT >= MI / 2 ? MI / 2 : MI / 4;  // blocks of 16 rows at a time
  static_assert(MB > 0 && MB <= FIT && MI % MB == 0 && (BD || PA % MI == 0), "blocks fit the waves' shares");
  char *const own = lds + wave * SHARE;
  auto at = [&](const int row, const int piece) -> f4 * {
    const int r = row & 15, c = (PIECES & (PIECES - 1)) == 0 ? piece ^ (r & (PIECES - 1)) : (piece + r) % PIECES;
    return (f4 *)(own + (row * PIECES + c) * 16);
  };
#pragma unroll
  for (int m0 = 0; m0 < MI; m0 += MB) {
#pragma unroll
    for (int m = 0; m < MB; ++m)
#pragma unroll
      for (int n = 0; n < NI; ++n)
        *at(m * 16 + (l & 15), n * 4 + (l >> 4)) = acc[m0 + m][n];
    __builtin_amdgcn_wave_barrier();
    constexpr int SEGS = (KIND == FWD ? WTN / 2 : WTN) / 8;  // eight outputs a lane
#pragma unroll 1
    for (int q = l; q < MB * 16 * SEGS; q += 64) {
      const int r = q / SEGS, s = q % SEGS;
      const size_t row = r0 + (wm * MI + m0) * 16 + r, col = c0 + wn * (SEGS * 8) + s * 8;
      if (row >= P.rows || col >= P.cols) continue;
      auto take = [&](int piece, float (&v)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f4 x = *at(r, piece + h);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[h * 4 + e] = x[e];
        }
      };
      float v[8];
      if constexpr (KIND == FWD) {
        float u[8], h[8];
        take((s >> 1) * 8 + (s & 1) * 2, v);
        take((s >> 1) * 8 + 4 + (s & 1) * 2, u);
        by_act(P.act, [&](auto act) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            float a, d;
            act_of(act(), v[e], a, d);
            h[e] = a * u[e];
          }
        });
        store(stream, P.o[0] + row * P.ldo, h, col, P.cols);
        if (P.o[1]) {
          store(stream, P.o[1] + row * P.cols, v, col, P.cols);
          store(stream, P.o[2] + row * P.cols, u, col, P.cols);
        }
      } else {
        take(s * 2, v);
        if constexpr (__is_same(T, _Float16)) {
          const float back = P.back ? *P.back : 1.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= back;
        }
        if (P.part) store(stream, P.part + ((size_t)(split * OUTS + z) * P.rows + row) * P.cols, v, col, P.cols);
        else store(stream, P.o[z] + row * P.ldo, v, col, P.cols);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// The forward pass of few rows: bound by reading the weights once and by latency, so no tile is staged.  A workgroup
// makes 16 columns of h for 16 MB rows; its eight waves share the sum over k in steps of 128 bytes, read straight into
// fragments (any alignment: a lane takes 32 consecutive bytes of a row, in x and in the weights alike), and are joined in
// LDS in a fixed order.  One row of k 1024, n 4096 bf16 (16.8 MB of weights) 5.3 us, 3.2 TB/s; 100 x 136 x 512 f32 4.0 us.
template <class T, int MB>
__global__ __launch_bounds__(512) void k_few(const GemmArgs<T> P) {
  constexpr int W = 8, KT = 128 / sizeof(T), E = 16 / sizeof(T);
  __shared__ f4 part[W][MB][2][64];
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = tid & 63, g = l >> 4, i = l & 15;
  const size_t c0 = (size_t)blockIdx.x * 16, r0 = (size_t)blockIdx.y * (16 * MB);
  const size_t col = c0 + i < P.cols ? c0 + i : P.cols - 1;
  size_t row[MB];
#pragma unroll
  for (int b = 0; b < MB; ++b) row[b] = r0 + 16 * b + i < P.rows ? r0 + 16 * b + i : P.rows - 1;
  f4 acc[MB][2];
#pragma unroll
  for (int b = 0; b < MB; ++b) acc[b][0] = acc[b][1] = f4{0.f, 0.f, 0.f, 0.f};
  auto work = [&](const i4(&vw)[2][2], const i4(&vx)[MB][2]) {
#pragma unroll
    for (int b = 0; b < MB; ++b)
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int h = 0; h < 2; ++h) acc[b][p] = mma<T>(vw[p][h], vx[b][h], acc[b][p]);
  };
  size_t k = (size_t)w * KT;
#pragma unroll 2
  for (; k + KT <= P.k; k += W * KT) {
    i4 vw[2][2], vx[MB][2];
    const size_t at = k + 2 * g * E;
#pragma unroll
    for (int p = 0; p < 2; ++p) __builtin_memcpy(vw[p], P.b[p] + col * P.ldb + at, 32);
#pragma unroll
    for (int b = 0; b < MB; ++b) __builtin_memcpy(vx[b], P.a[0] + row[b] * P.lda + at, 32);
    work(vw, vx);
  }
  if (k < P.k) {
    i4 vw[2][2], vx[MB][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const size_t at = k + (2 * g + h) * E;
#pragma unroll
      for (int p = 0; p < 2; ++p) vw[p][h] = fetch16(P.b[p], P.ldb, col, P.cols, at, P.k);
#pragma unroll
      for (int b = 0; b < MB; ++b) vx[b][h] = fetch16(P.a[0], P.lda, row[b], P.rows, at, P.k);
    }
    work(vw, vx);
  }
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int p = 0; p < 2; ++p) part[w][b][p][l] = acc[b][p];
  __syncthreads();
  if (tid >= MB * 64) return;
  f4 sum[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    sum[p] = part[0][w][p][l];
#pragma unroll
    for (int q = 1; q < W; ++q) sum[p] += part[q][w][p][l];
  }
  const size_t r = r0 + 16 * w + i, c = c0 + 4 * g;
  if (r >= P.rows || c >= P.cols) return;
  float a[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float d;
    act_of(P.act, sum[0][e], a[e], d);
    a[e] *= sum[1][e];
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < P.cols) {
      P.o[0][r * P.ldo + c + e] = (T)a[e];
      if (P.o[1]) P.o[1][r * P.cols + c + e] = (T)sum[0][e], P.o[2][r * P.cols + c + e] = (T)sum[1][e];
    }
}

constexpr unsigned CUS = 256;

// Partial sums joined in a fixed order: `outs` matrices of [rows][cols], rows of stride ldo.  V = 4: four neighbours of a
// row a thread (cols a multiple of four); P shares of the splits, of threads of their own
template <class T, int V, int P>
__global__ __launch_bounds__(256) void k_join(const float *__restrict__ part, const size_t rows, const size_t cols, const unsigned outs,
                                              const unsigned splits, T *__restrict__ o0, T *__restrict__ o1, const size_t ldo) {
  constexpr int W = 256 / P;
  const size_t n = rows * cols;
  const unsigned w = threadIdx.x % W, q = threadIdx.x / W;
  __shared__ float lds[P][W][V];
  for (size_t i0 = (size_t)blockIdx.x * W * V; i0 < outs * n; i0 += (size_t)gridDim.x * W * V) {
    const size_t i = i0 + (size_t)w * V;
    float s[V] = {}, v[V];
    if (i < outs * n)
#pragma unroll 4
      for (unsigned p = q; p < splits; p += P) {
        __builtin_memcpy(v, part + p * outs * n + i, sizeof v);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += v[e];
      }
    if constexpr (P > 1) {
      __builtin_memcpy(lds[q][w], s, sizeof s);
      __syncthreads();
      if (q == 0)
#pragma unroll
        for (int p = 1; p < P; ++p)
#pragma unroll
          for (int e = 0; e < V; ++e) s[e] += lds[p][w][e];
      __syncthreads();
    }
    if (q || i >= outs * n) continue;
    const size_t j = i < n ? i : i - n, r = n <= 0xFFFFFFFFu ? (uint32_t)j / (uint32_t)cols : j / cols;
    T t[V];
#pragma unroll
    for (int e = 0; e < V; ++e) t[e] = (T)s[e];
    __builtin_memcpy((i < n ? o0 : o1) + r * ldo + (j - r * cols), t, sizeof t);
  }
}
// 16 shares where there are at least as many splits and one thread an output would not fill the chip's waves
template <class T>
void join(QrDenseStream &s, const float *part, size_t rows, size_t cols, unsigned outs, unsigned splits, T *o0, T *o1, size_t ldo) {
  const auto go = [&](auto v, auto p) {
    constexpr int V = decltype(v)::value, P = decltype(p)::value;
    const size_t groups = (outs * rows * cols / V + 256 / P - 1) / (256 / P);
    s.launch(k_join<T, V, P>, (unsigned)std::min<size_t>(groups, 65536), 256, 0, part, rows, cols, outs, splits, o0, o1, ldo);
  };
  using one = std::integral_constant<int, 1>;
  using four = std::integral_constant<int, 4>;
  using sixteen = std::integral_constant<int, 16>;
  const bool shares = splits >= 16 && outs * rows * cols < CUS * 2048;
  if (cols % 4 == 0) shares ? go(four{}, sixteen{}) : go(four{}, one{});
  else shares ? go(one{}, sixteen{}) : go(one{}, one{});
}

// Matrices whose rows do not start or end at 16-byte boundaries, copied to ones whose rows do; the padding, and rows up to
// rows_to, zeroed.  Each has workgroups of its own.  Bound by memory: 101549 x 609 f16 49 us (5.0 TB/s)
template <class T>
struct Packs {
  struct {
    const T *p;
    T *q;
    size_t rows, cols, ld, to, rows_to;
    unsigned groups;
  } m[3] = {};
  unsigned n = 0, groups = 0;
};
template <class T>
__device__ __forceinline__ void pack_group(const Packs<T> &packs, unsigned group) {
  constexpr int E = 16 / sizeof(T);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    const auto &m = packs.m[j];
    if (group < m.groups) {
      const size_t per = m.to / E;
      for (size_t i = (size_t)group * 256 + threadIdx.x; i < m.rows_to * per; i += (size_t)m.groups * 256) {
        const size_t r = i / per, c = (i - r * per) * E;
        *(i4 *)(m.q + r * m.to + c) = fetch16(m.p, m.ld, r, m.rows, c, m.cols);
      }
      return;
    }
    group -= m.groups;
  }
}
template <class T>
__global__ __launch_bounds__(256) void k_pack(const Packs<T> packs) {
  pack_group(packs, blockIdx.x);
}

// Eight neighbours of dg and du, from column c of row r on; behind the row's end zeros
template <class T, int ACT>
__device__ __forceinline__ void gate_piece(const size_t n, const T *__restrict__ dh, const size_t lddh, const T *__restrict__ g,
                                           const T *__restrict__ u, const size_t r, const size_t c, float (&dg)[8], float (&du)[8]) {
  T vh[8] = {}, vg[8] = {}, vu[8] = {};
  if (c + 8 <= n) {
    __builtin_memcpy(vh, dh + r * lddh + c, sizeof vh);
    __builtin_memcpy(vg, g + r * n + c, sizeof vg);
    __builtin_memcpy(vu, u + r * n + c, sizeof vu);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < n) vh[e] = dh[r * lddh + c + e], vg[e] = g[r * n + c + e], vu[e] = u[r * n + c + e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float a, d;
    act_of(ACT, (float)vg[e], a, d);
    const float v = (float)vh[e];
    dg[e] = v * (float)vu[e] * d;
    du[e] = v * a;
  }
}

// f16 has five bits of exponent: gradients of the products below 2^-14 would lose bits and those above 65504 become infinite,
// though dx and dW are well inside.  So dg and du are held times a power of two that brings the largest finite one of both to
// 2^14 .. 2^15 (one scale, for dx adds up products of both), and the products' sums are multiplied by its reciprocal: an
// element keeps f16's 11 bits, or 2^-39 of the call's largest.  The largest is found first, by a launch that reads what the
// gate gradient reads, the part of a workgroup to a place of its own; every workgroup of the gate gradient takes the largest of
// those.  Bound by memory: with it 16384 x 1024 x 4096 takes 666 us (without 578), 100000 x 136 x 512 310 (253), 300 x 136 x
// 512 27 (25).  (Read backwards by the gate gradient, for what the caches still hold, or by twice the workgroups: the same.)
constexpr unsigned MAXIMA = 1024;  // workgroups of that launch at most
__device__ __forceinline__ float block_max(float v) {  // of 256 threads, none of them negative, in every thread
  __shared__ float lds[4];
#pragma unroll
  for (int s = 1; s < 64; s *= 2) v = fmaxf(v, __shfl_xor(v, s));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  return fmaxf(fmaxf(lds[0], lds[1]), fmaxf(lds[2], lds[3]));
}
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_gate_max(const size_t m, const size_t n, const T *__restrict__ dh, const size_t lddh,
                                                  const T *__restrict__ g, const T *__restrict__ u, float *__restrict__ maxima) {
  const size_t per = (n + 7) / 8;
  float most = 0.f;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < m * per; i += (size_t)gridDim.x * 256) {
    const size_t r = i / per;
    float dg[8], du[8];
    gate_piece<T, ACT>(n, dh, lddh, g, u, r, (i - r * per) * 8, dg, du);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf(dg[e]), b = fabsf(du[e]);
      most = a < INFINITY ? fmaxf(most, a) : most;  // (false for NaN)
      most = b < INFINITY ? fmaxf(most, b) : most;
    }
  }
  most = block_max(most);
  if (threadIdx.x == 0) maxima[blockIdx.x] = most;
}

// dg, du in rows of stride ld, their padding zeroed; eight elements a thread.  Bound by memory: five matrices, 16384 x 4096
// bf16 111 us, 100000 x 512 f32 168 us (6.1 TB/s, some of it from the caches).  They are rounded to T so that the products
// take them as they are: an f32 dx or dW is as exact as without, a 16-bit one is off by 2^1/2 times its own rounding (what
// adds up is the rounding of each of many terms).  In 32 bits they would be twice the bytes and three products for one.
// Matrices to be copied for the products are copied by the launch's first workgroups.  (The padding is at least as long as what
// a row's last eight reach over.)
template <class T, int ACT>
__global__ __launch_bounds__(256) void k_gate_grad(const size_t m, const size_t n, const T *__restrict__ dh, const size_t lddh,
                                                   const T *__restrict__ g, const T *__restrict__ u, T *__restrict__ dg,
                                                   T *__restrict__ du, const size_t ld, const Packs<T> packs,
                                                   const float *__restrict__ maxima, const unsigned parts, float *__restrict__ back) {
  if (blockIdx.x < packs.groups) return pack_group(packs, blockIdx.x);
  const size_t per = ld / 8;
  const unsigned group = blockIdx.x - packs.groups, groups = gridDim.x - packs.groups;
  float scale = 1.f;
  if constexpr (__is_same(T, _Float16)) {
    float most = 0.f;
    for (unsigned p = threadIdx.x; p < parts; p += 256) most = fmaxf(most, maxima[p]);
    // 2^(14 - the exponent), between 2^-100 and 2^100
    const int e = 268 - (int)(__builtin_bit_cast(uint32_t, block_max(most)) >> 23), bits = e < 27 ? 27 : e > 227 ? 227 : e;
    scale = __builtin_bit_cast(float, bits << 23);
    if (group == 0 && threadIdx.x == 0) *back = __builtin_bit_cast(float, (254 - bits) << 23);
  }
  for (size_t i = (size_t)group * 256 + threadIdx.x; i < m * per; i += (size_t)groups * 256) {
    const size_t r = i / per, c = (i - r * per) * 8;
    float vg[8], vu[8];
    T og[8], ou[8];
    gate_piece<T, ACT>(n, dh, lddh, g, u, r, c, vg, vu);
#pragma unroll
    for (int e = 0; e < 8; ++e) og[e] = (T)(vg[e] * scale), ou[e] = (T)(vu[e] * scale);
    __builtin_memcpy(dg + r * ld + c, og, sizeof og);
    __builtin_memcpy(du + r * ld + c, ou, sizeof ou);
  }
}
// maxima, back: f16 only, MAXIMA floats and one
template <class T>
void gate_grad(QrDenseStream &s, size_t m, size_t n, int act, const void *dh, size_t lddh, const void *g, const void *u, T *dg, T *du,
               size_t ld, const Packs<T> &packs, float *maxima, float *back) {
  const auto groups = [](size_t threads, size_t most) { return (unsigned)std::min((threads + 255) / 256, most); };
  constexpr bool scaled = __is_same(T, _Float16);
  const unsigned grid = groups(m * (ld / 8), scaled ? 4096 : 65536), parts = scaled ? groups(m * ((n + 7) / 8), MAXIMA) : 0;
  const auto go = [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    if constexpr (scaled) s.launch(k_gate_max<T, ACT>, parts, 256, 0, m, n, (const T *)dh, lddh, (const T *)g, (const T *)u, maxima);
    s.launch(k_gate_grad<T, ACT>, packs.groups + grid, 256, 0, m, n, (const T *)dh, lddh, (const T *)g, (const T *)u, dg, du, ld, packs, maxima,
             parts, back);
  };
  by_act(act, go);
}

bool act_ok(int act) { return act >= QR_ACT_SILU && act <= QR_ACT_SIGMOID; }
unsigned tiles_of(size_t n, size_t t) { return (unsigned)((n + t - 1) / t); }

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }
size_t padded(size_t cols, size_t e) { return (cols + 16 / e - 1) / (16 / e) * (16 / e); }
// the length of one of DX's two sums, in whole stages
size_t stages_of(size_t n, size_t e) { return (n + 128 / e - 1) / (128 / e) * (128 / e); }
size_t pack_bytes(size_t rows, size_t cols, size_t e) { return round256(rows * padded(cols, e) * e); }
// f16: the workgroups' largest gradients and what the products are multiplied by
size_t scale_bytes(int type) { return type == QR_F16 ? round256((MAXIMA + 1) * 4) : 0; }
unsigned blocks(size_t n) { return (unsigned)((n + 255) / 256 < 65536 ? (n + 255) / 256 : 65536); }

// longest row the product kernel takes: a tile's 256 rows lie within 2^31 bytes
constexpr size_t ROW_BYTES = (size_t)1 << 22;
// most rows and most outputs of a row: a launch has fewer than 2^32 threads
constexpr size_t ROWS_MOST = (size_t)1 << 30, OUTS_MOST = (size_t)1 << 28;
// ... and most tiles of 128 x 128 sums (dx: 128 x 64, its narrowest), of 256 threads
constexpr size_t TILES_MOST = ((size_t)1 << 24) - 1;

// whether the product kernel can read a matrix where it lies: rows of whole pieces of 16 bytes at 16-byte boundaries
bool in_place(const void *p, size_t ld, size_t cols, size_t e) {
  return ((uintptr_t)p & 15) == 0 && (ld * e) % 16 == 0 && ld * e <= ROW_BYTES && (cols * e) % 16 == 0;
}

// notes that `p` is to be copied, and makes it and its stride those of the copy
template <class T>
void pack(Packs<T> &packs, size_t rows, size_t cols, const T *&p, size_t &ld, char *&ws, size_t rows_to) {
  const size_t to = padded(cols, sizeof(T));
  const unsigned groups = blocks(rows_to * to * sizeof(T) / 16);
  packs.m[packs.n++] = {p, (T *)ws, rows, cols, ld, to, rows_to, groups};
  packs.groups += groups;
  p = (const T *)ws;
  ld = to;
  ws += pack_bytes(rows_to, cols, sizeof(T));
}
// Whether results go past the caches, so that they do not push the operands out.  Only in whole parts of 64 bytes, what
// the memory writes at once (65536 x 256 x 1000 bf16, both products kept: 356 us past the caches, 174 through them).  Where
// the three results are kept, the caches' 256 MB take some of them up: past the caches where the sums are long, or not short
// and the results larger than that.  Past / through, 16384 x 32 x 4096 121 / 102 us, 32768 x 256 x 1024 69 / 58, 16384 x 256
// x 4096 125 / 149, 32768 x 1024 x 4096 542 / 596; one result, 32768 x 32 x 1024 33 / 35, 8192 x 8192 x 4096 740 / 799.
template <class T>
bool streams(const GemmArgs<T> &P, const size_t outs) {
  bool whole = (P.ldo * sizeof(T)) % 64 == 0 && (P.cols * sizeof(T)) % 64 == 0;
  for (size_t i = 0; i < outs; ++i) whole &= ((uintptr_t)P.o[i] & 63) == 0;
  const size_t sum = P.k * sizeof(T), bytes = outs * P.rows * P.cols * sizeof(T);
  return whole && (outs < 3 || sum >= 1024 || (sum >= 256 && bytes > ((size_t)256 << 20)));
}

template <class T, Kind KIND, int TM, int TN, int WN = 2, bool RAG = false>
void launch_gemm(QrDenseStream &s, GemmArgs<T> P) {
  P.row_tiles = tiles_of(P.rows, TM);
  P.stream = streams(P, KIND == FWD ? (P.o[1] ? 3 : 1) : KIND == DW ? 2 : 1);
  P.col_tiles = tiles_of(P.cols, KIND == FWD ? TN / 2 : TN);
  const unsigned tiles = P.row_tiles * P.col_tiles * (KIND == FWD ? 1 : (KIND == DW ? 2 : 1) * P.splits);
  s.launch(k_gemm<T, KIND, TM, TN, WN, RAG>, (tiles + 7) / 8 * 8, 128 * WN, 0, P);
}



// Whether the forward pass takes the few-rows kernel: where tiles of 64 x 64 sums would leave half the compute units (16-bit
// types: three quarters) without one, and up to 64 (32) rows.  Few rows / tiles in us, back to back in a graph: k 1024, n
// 4096 bf16 1 row 5.3 / 7.4, 32 7.0 / 7.7, 64 9.5 / 8.0, 200 25 / 10; k 2048, n 1024 bf16 100 rows 10.4 / 12.1, 200 14.4 /
// 12.4; k 136, n 512 f32 100 rows 4.0 / 7.0, 512 6.5 / 7.1, 1000 9.0 / 7.6.
bool few(size_t e, size_t m, size_t n) {
  const size_t rows = e == 2 ? 32 : 64, tiles = e == 2 ? CUS / 4 : CUS / 2;
  return n < ((size_t)1 << 26) && (m <= rows || (size_t)tiles_of(m, 64) * tiles_of(2 * n, 64) <= tiles);
}

template <class T>
void launch_few(QrDenseStream &s, const GemmArgs<T> &P) {
  const unsigned cols = tiles_of(P.cols, 16);
  // the most rows a workgroup that still leave every compute unit one (16-bit types: 64 rows never do)
  if constexpr (sizeof(T) == 4)
    if (P.rows > 32 && (size_t)cols * tiles_of(P.rows, 64) >= CUS) return s.launch(k_few<T, 4>, dim3(cols, tiles_of(P.rows, 64)), 512, 0, P);
  if (P.rows > 16 && (size_t)cols * tiles_of(P.rows, 32) >= CUS) s.launch(k_few<T, 2>, dim3(cols, tiles_of(P.rows, 32)), 512, 0, P);
  else s.launch(k_few<T, 1>, dim3(cols, tiles_of(P.rows, 16)), 512, 0, P);
}

struct Tile {
  int rows, cols;
};

// Sums a workgroup takes: 256 x 128 (16-bit types) or 128 x 128 where that gives every compute unit a tile, else 64 x 64.
// Gradients may be narrow (features), and a width of 128 would pad 136 columns to 256: there the width is the one whose
// tiles cost least.  16-bit types, 64 against 128: the columns.  f32, 64, 96, 128 or 160: by a wave's cycles per stage, of
// its matrix instructions (4 rows of blocks of 6 x 16 each) or of the splitting of its 4 + width / 32 blocks (44 x 4 each).
Tile tile_of(size_t e, size_t rows, size_t cols, size_t times, bool narrow) {
  size_t w = 128, least = ~(size_t)0;
  for (size_t v = 64; v <= 160 && narrow; v += 32) {
    if (e == 2 && v % 64) continue;
    const size_t b = v / 32, mat = 4 * b * 96, vec = (4 + b) * 176;
    const size_t cost = tiles_of(cols, v) * (e == 2 ? v : mat > vec ? mat : vec);
    if (cost <= least && v <= (e == 2 ? 128 : 160)) least = cost, w = v;
  }
  const bool tall = tiles_of(rows, 256) * 14 <= tiles_of(rows, 128) * 8;
  if (e == 2 && w == 128 && tall && (size_t)tiles_of(rows, 256) * tiles_of(cols, 128) * times >= CUS) return {256, 128};
  if (rows > 64 && (size_t)tiles_of(rows, 128) * tiles_of(cols, w) * times >= CUS) return {128, (int)w};
  return {64, 64};
}

template <class T, Kind KIND>
void gemm(QrDenseStream &s, const Tile t, const GemmArgs<T> &P) {
  if constexpr (sizeof(T) == 2)
    if (t.rows == 256) return t.cols == 256 ? launch_gemm<T, KIND, 256, 256, 4>(s, P) : launch_gemm<T, KIND, 256, 128>(s, P);
  if (t.rows == 128 && t.cols == 128) return launch_gemm<T, KIND, 128, 128>(s, P);
  if constexpr (KIND != FWD) {
    if (t.rows == 128 && t.cols == 64) return launch_gemm<T, KIND, 128, 64>(s, P);
    if constexpr (sizeof(T) == 4) {
      if (t.rows == 128 && t.cols == 96) return launch_gemm<T, KIND, 128, 96>(s, P);
      if (t.rows == 128 && t.cols == 160) return launch_gemm<T, KIND, 128, 160>(s, P);
    }
  }
  launch_gemm<T, KIND, 64, 64>(s, P);
}

// 256 x 256 sums a workgroup instead of 256 x 128, one workgroup a compute unit instead of two: a third less to load for
// each product, but a tile's first loads and its results' way out have nothing beside them.  In hundredths of a stage's
// time (1.39 us with every compute unit at work), fitted to times measured between 2 and 64 stages: a full round of the
// large tiles takes 100 a stage and `edge`, one of the small 118 a stage and `edge` less 110 (290 where three matrices are
// stored); a part of a round takes 3 / 4 of one, a small tile alone on its compute unit 1 / 2.  `large`, `small`: the
// launches' workgroups and stages.  Measured: 8192 x 8192 x (2 x 4096) 740 us against 845, 32768 x 1024 x (2 x 4096) 445
// against 476 (with g and u stored 532 against 549), their gradients for half the rows 564 against 604; but 8192 x 4096 x
// (2 x 1152), 288 large tiles, 176 against 161.
struct Launch {
  size_t groups, stages;
};
bool larger(const Launch large, const Launch small, const bool saves) {
  const size_t rounds = large.groups / CUS, rest = small.groups % (2 * CUS);
  const size_t edge = saves ? (rounds < 8 ? 890 : 780) : 530;  // (over many rounds the workgroups' stores come apart)
  const size_t of_large = rounds * 4 + (large.groups % CUS ? 3 : 0);
  const size_t of_small = small.groups / (2 * CUS) * 4 + (rest ? rest > CUS ? 4 : 2 : 0);
  return of_large * (large.stages * 100 + edge) < of_small * (small.stages * 118 + edge - (saves ? rounds < 8 ? 290 : 230 : 110));
}

Tile tile_forward(size_t e, size_t m, size_t k, size_t n, bool saves) {
  const Tile t = tile_of(e, m, 2 * n, 1, false);
  const size_t rows = tiles_of(m, 256), stages = (k * e + 127) / 128;
  if (t.rows < 256 || !larger({rows * tiles_of(2 * n, 256), stages}, {rows * tiles_of(2 * n, 128), stages}, saves)) return t;
  return {256, 256};
}

// How the gradients' products are made: `outs` matrices of rows x cols, sums of `stages` stages.  With few outputs the
// sums are split so that the launch gives every compute unit two workgroups (not one more: a third makes it work half as
// long again), in shares of at least eight stages.
struct Plan {
  Tile tile;
  unsigned splits, steps;
};
Plan plan(size_t e, size_t rows, size_t cols, size_t outs, size_t stages) {
  const size_t most = std::max<size_t>(stages / 8, 1);
  auto with = [&](const Tile t, const size_t groups) {
    const size_t one = std::max<size_t>(outs * tiles_of(rows, t.rows) * tiles_of(cols, t.cols), 1);  // (no rows)
    const size_t want = std::min(std::max<size_t>(groups / one, 1), most);
    Plan p{t, 1, (unsigned)std::max<size_t>((stages + want - 1) / want, 1)};
    p.splits = (unsigned)std::max<size_t>((stages + p.steps - 1) / p.steps, 1);
    return std::pair<Plan, Launch>(p, {one * p.splits, p.steps});
  };
  const auto small = with(tile_of(e, rows, cols, outs * most, true), 2 * CUS), large = with({256, 256}, CUS);
  return small.first.tile.rows == 256 && larger(large.second, small.second, false) ? large.first : small.first;
}
Plan plan_dx(size_t e, size_t m, size_t k, size_t n) { return plan(e, m, k, 1, 2 * stages_of(n, e) * e / 128); }
Plan plan_dw(size_t e, size_t m, size_t k, size_t n) { return plan(e, n, k, 2, (m * e + 127) / 128); }
size_t part_bytes(const Plan &p, size_t rows, size_t cols, size_t outs) {
  return p.splits > 1 ? round256(p.splits * outs * rows * cols * 4) : 0;
}

// Whether the forward pass reads rows off 16-byte boundaries as they lie, through registers, instead of copying them first:
// where few tiles read a row again, or few tiles are made and a launch is what counts.  As they lie / copied, us a call:
// 100000 x 601 x 64 bf16 45 / 64, 20000 x 1023 x 64 24 / 30, 1000 x 601 x 500 11 / 14, f32 100000 x 601 x 200 360 / 425;
// but 4000 x 1023 x 4000 bf16 124 / 66, 100000 x 65 x 200 48 / 42, f32 20000 x 65 x 4000 240 / 222.
bool as_they_lie(size_t e, size_t m, size_t n) {
  const size_t cols = tiles_of(2 * n, 128);
  return cols <= (e == 2 ? 2 : 8) || (size_t)tiles_of(m, 128) * cols <= 2 * CUS;
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
  const bool px = !few(e, m, n) && !in_place(x, ldx, k, e), pw = !few(e, m, n) && (!in_place(w_gate, ldw, k, e) || !in_place(w_up, ldw, k, e));
  const bool direct = (px || pw) && ldx * e <= ROW_BYTES && ldw * e <= ROW_BYTES && as_they_lie(e, m, n);
  size_t need = 0;
  if (px || pw)  // (asked for by the rows alone, whichever way they are then read)
    if (int rc = qr_gated_ffn_workspace(type, m, k, n, &need)) return rc;
  QR_DENSE_ARG(!need || (workspace && workspace_bytes >= need),
               "gated ffn: rows that start or end off 16-byte boundaries or lie more than 4 MB apart need the workspace");
  if (m > ROWS_MOST || n > OUTS_MOST) return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn: more than 2^30 rows or 2^28 outputs");
  if (!few(e, m, n) && (size_t)tiles_of(m, 128) * tiles_of(2 * n, 128) > TILES_MOST)
    return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn: 2^24 tiles of 128 x 64 outputs or more");
  if (!few(e, m, n) && k * e > ROW_BYTES) return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn: rows longer than 4 MB");
  // (the workspace as one row)
  const QrDenseMatrix out[4] = {{h, m, n, ldh}, {gate, m, n, n}, {up, m, n, n}, {workspace, 1, need / e, need / e}},
                      in[3] = {{x, m, k, ldx}, {w_gate, n, k, ldw}, {w_up, n, k, ldw}};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 3; ++j) QR_DENSE_ARG(!qr_dense_share(out[i], in[j], e), "gated ffn: an output lies over an input");
    for (int j = 0; j < i; ++j) QR_DENSE_ARG(!qr_dense_share(out[i], out[j], e), "gated ffn: outputs overlap");
  }
  QR_DENSE_DEVICE(device);
  QrDenseStream s(stream);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    char *ws = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    GemmArgs<T> P{};
    P.a[0] = (const T *)x, P.b[0] = (const T *)w_gate, P.b[1] = (const T *)w_up;
    P.lda = ldx, P.ldb = ldw, P.rows = m, P.cols = n, P.k = k;
    P.o[0] = (T *)h, P.o[1] = (T *)gate, P.o[2] = (T *)up, P.ldo = ldh, P.act = act;
    Packs<T> packs;
    if (direct) {
      const Tile t = tile_of(e, m, 2 * n, 1, false);
      return t.rows > 64 ? launch_gemm<T, FWD, 128, 128, 2, true>(s, P) : launch_gemm<T, FWD, 64, 64, 2, true>(s, P);
    }
    if (px) pack(packs, m, k, P.a[0], P.lda, ws, m);
    if (pw) {
      size_t ld = ldw;
      pack(packs, n, k, P.b[0], ld, ws, n), pack(packs, n, k, P.b[1], P.ldb, ws, n);
    }
    if (packs.groups) s.launch(k_pack<T>, packs.groups, 256, 0, packs);
    if (few(e, m, n)) launch_few(s, P);
    else gemm<T, FWD>(s, tile_forward(e, m, k, n, gate != nullptr), P);
  });
  return qr_dense_launched(s, "gated ffn");
}

extern "C" int qr_gated_ffn_backward_workspace(int type, size_t m, size_t k, size_t n, size_t *bytes) {
  QR_DENSE_ARG(bytes && qr_dense_type_ok(type) && k > 0 && n > 0 && qr_dense_fits(m, n, n) && qr_dense_fits(m, k, k) && qr_dense_fits(n, k, k),
               "gated ffn backward: bad size");
  const size_t e = qr_dense_size(type);
  // the scale, dg, du, the partial sums (dx is made before the weights' gradients), copies of x and the weights where their
  // rows are not aligned
  *bytes = m ? scale_bytes(type) + 2 * pack_bytes(m, stages_of(n, e), e) +
                   std::max(part_bytes(plan_dx(e, m, k, n), m, k, 1), part_bytes(plan_dw(e, m, k, n), n, k, 2)) + pack_bytes(m, k, e) +
                   2 * pack_bytes(stages_of(n, e), k, e) + 256
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
  if (m > ROWS_MOST) return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn backward: more than 2^30 rows");
  if (k * e > ROW_BYTES || stages_of(n, e) * e > ROW_BYTES)
    return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn backward: rows longer than 4 MB");
  if (dx && (size_t)tiles_of(m, 128) * tiles_of(k, 64) > TILES_MOST)
    return qr_dense_fail(QR_ERR_UNSUPPORTED, "gated ffn backward: 2^24 tiles of 128 x 64 elements of dx or more");
  const QrDenseMatrix out[4] = {{dx, m, k, lddx}, {dw_gate, n, k, k}, {dw_up, n, k, k}, {workspace, 1, need / e, need / e}},
                      in[6] = {{dh, m, n, lddh}, {x, m, k, ldx}, {w_gate, n, k, ldw}, {w_up, n, k, ldw}, {gate, m, n, n}, {up, m, n, n}};
  for (int i = 0; i < 4; ++i) {
    for (int j = 0; j < 6; ++j) QR_DENSE_ARG(!qr_dense_share(out[i], in[j], e), "gated ffn backward: an output lies over an input");
    for (int j = 0; j < i; ++j) QR_DENSE_ARG(!qr_dense_share(out[i], out[j], e), "gated ffn backward: outputs overlap");
  }
  QR_DENSE_DEVICE(device);
  QrDenseStream s(stream);
  qr_dense_dispatch(type, [&](auto t) {
    using T = decltype(t);
    char *ws = (char *)(((uintptr_t)workspace + 255) & ~(uintptr_t)255);
    const size_t ld = stages_of(n, e);
    float *const maxima = (float *)ws, *const back = maxima + MAXIMA;
    if (m) ws += scale_bytes(type);
    T *const dg = (T *)ws, *const du = (T *)(ws + pack_bytes(m, ld, e));
    ws += 2 * pack_bytes(m, ld, e);
    const Plan px = plan_dx(e, m, k, n), pw = plan_dw(e, m, k, n);
    float *const part = (float *)ws;
    if (m) ws += std::max(part_bytes(px, m, k, 1), part_bytes(pw, n, k, 2));
    GemmArgs<T> X{}, W{};
    X.a[0] = dg, X.a[1] = du, X.b[0] = (const T *)w_gate, X.b[1] = (const T *)w_up;
    X.lda = ld, X.ldb = ldw, X.rows = m, X.cols = k, X.k = ld, X.o[0] = (T *)dx, X.ldo = lddx;
    W.a[0] = dg, W.a[1] = du, W.b[0] = (const T *)x;
    W.lda = ld, W.ldb = ldx, W.rows = n, W.cols = k, W.k = m, W.o[0] = (T *)dw_gate, W.o[1] = (T *)dw_up, W.ldo = k;
    Packs<T> packs;
    if (dx && m && (ld != n || !in_place(w_gate, ldw, k, e) || !in_place(w_up, ldw, k, e))) {
      size_t to = ldw;
      pack(packs, n, k, X.b[0], to, ws, ld), pack(packs, n, k, X.b[1], X.ldb, ws, ld);
    }
    if (dw_gate && m && !in_place(x, ldx, k, e)) pack(packs, m, k, W.b[0], W.ldb, ws, m);
    if (m) gate_grad<T>(s, m, n, act, dh, lddh, gate, up, dg, du, ld, packs, maxima, back);
    X.back = W.back = m && scale_bytes(type) ? back : nullptr;
    if (dx && m) {
      X.splits = px.splits, X.steps = px.steps, X.part = px.splits > 1 ? part : nullptr;
      gemm<T, DX>(s, px.tile, X);
      if (X.part) join(s, part, m, k, 1, px.splits, (T *)dx, (T *)dx, lddx);
    }
    if (dw_gate) {
      W.splits = pw.splits, W.steps = pw.steps, W.part = pw.splits > 1 ? part : nullptr;
      gemm<T, DW>(s, pw.tile, W);
      if (W.part) join(s, part, n, k, 2, pw.splits, (T *)dw_gate, (T *)dw_up, k);
    }
  });
  return qr_dense_launched(s, "gated ffn backward");
}
