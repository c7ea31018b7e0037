// nn_gemm.h -- the matrix products of the gated block on the matrix cores: C[m][n] = sum over k of A(m, k) B(n, k), with
// both operands staged through registers into LDS as rows of 16-byte chunks along k, and the accumulators handed to an
// epilogue.
//
// Types. bf16 and int8 go through the matrix cores as they are (fp32 and whole-number sums). fp32 values are split on
// their way into LDS into three bf16 numbers, x = hi + mid + lo (each the rounded rest of the one before: 24 bits in
// all), and a product is the six products of those whose sizes add up to more than 2^-24 of the largest:
// hi hi + hi mid + mid hi + mid mid + hi lo + lo hi (Henry, Tang and Heinecke, "Leveraging the bfloat16 artificial
// intelligence datatype for higher-precision computations", 2019). The bf16 matrix rate is sixteen times the fp32
// one, so six products beat one. Where a sum comes out infinite or NaN (an operand was, or was too large to round to
// bf16: a rest of an infinity is NaN), that output is summed again in plain fp32, so it is what the formula gives.
//
// LDS. A chunk (row, c) lies in the row's slot c ^ swizzle(row): the eight rows of a phase of a 16-byte read, and the
// rows four apart that a transposing store writes, fall into different banks.
#pragma once
#include "nn_common.h"

namespace g1nn {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef signed char i8;

// How a type goes through the matrix cores: planes in LDS, bytes of a plane's row, elements per 16-byte chunk.
template <typename T>
struct Form;
template <>
struct Form<float> {
  static constexpr int kPlanes = 3, kRowBytes = 64, kPer = 8;
  typedef f32x16 Acc;
};
template <>
struct Form<bf16> {
  static constexpr int kPlanes = 1, kRowBytes = 128, kPer = 8;
  typedef f32x16 Acc;
};
template <>
struct Form<i8> {
  static constexpr int kPlanes = 1, kRowBytes = 128, kPer = 16;
  typedef i32x16 Acc;
};

template <typename T>
constexpr int kSlots = Form<T>::kRowBytes / 16;          // chunks of a row
template <typename T>
constexpr int kDepth = kSlots<T> * Form<T>::kPer;        // k of a tile

template <typename T>
__device__ __forceinline__ int lds_at(int rows, int plane, int row, int c) {
  const int s = kSlots<T> == 8 ? (row ^ (row >> 3)) & 7 : ((row >> 1) ^ (row >> 3)) & 3;
  return ((plane * rows + row) * kSlots<T> + (c ^ s)) * 16;
}

// N values as N/2 words of two bf16 numbers each, x = hi + mid + lo, each rounded to nearest: 11 operations a pair.
template <int N>
__device__ __forceinline__ void split(const float (&x)[N], unsigned (&hi)[N / 2], unsigned (&mid)[N / 2], unsigned (&lo)[N / 2]) {
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    f32x2 v = {x[2 * i], x[2 * i + 1]};
    hi[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
    v[0] -= __uint_as_float(hi[i] << 16);
    v[1] -= __uint_as_float(hi[i] & 0xffff0000u);
    mid[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
    v[0] -= __uint_as_float(mid[i] << 16);
    v[1] -= __uint_as_float(mid[i] & 0xffff0000u);
    lo[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
  }
}

// ---- operands: where the rows of a tile lie ---------------------------------------------------------------------
// Along: a row's k are contiguous. row(r) is the start of the tile's row r; rows past the end repeat the last one, and
// what they give is never stored.
template <typename T>
struct Along {
  static constexpr bool kAlong = true;
  const T* p;
  long stride;
  int row0, rows;
  __device__ const T* row(int r) const {
    const int i = row0 + r;
    return p + (long)(i < rows ? i : rows - 1) * stride;
  }
  __device__ T at(int r, int k) const { return row(r)[k]; }
};

// Both projections' weights in one tile: 32 rows of the gate, then the 32 of the other projection for the same
// outputs, so that a lane's accumulators hold both values of an output.
template <typename T>
struct Paired {
  static constexpr bool kAlong = true;
  const T *g, *u;
  long gs, us;
  int f0, F;
  __device__ const T* row(int r) const {
    const int i = f0 + (r >> 6) * 32 + (r & 31), c = i < F ? i : F - 1;
    return (r & 32) ? u + (long)c * us : g + (long)c * gs;
  }
  __device__ T at(int r, int k) const { return row(r)[k]; }
};

// Across: k counts the rows of memory, and the tile's rows are its columns [col0, cols). tile(k0) is the start of the
// memory row k0, from which the tile's rows follow `step(k0)` apart, and whole(k0, n) says whether all n exist.
template <typename T>
struct Across {
  static constexpr bool kAlong = false;
  const T* p;
  long stride;
  int col0, cols;
  __device__ const T* tile(long k0) const { return p + k0 * stride; }
  __device__ long step(long) const { return stride; }
  __device__ bool whole(long, int) const { return true; }
  __device__ bool has(long) const { return true; }
  __device__ T at(int r, long k) const { return p[k * stride + col0 + r]; }
};

// Across the rows of both weights one after the other, each padded to `half` rows (a multiple of every tile's depth) of
// which F exist.
template <typename T>
struct AcrossPair {
  static constexpr bool kAlong = false;
  const T *g, *u;
  long gs, us;
  int half, F;
  int col0, cols;
  __device__ const T* tile(long k0) const { return k0 < half ? g + k0 * gs : u + (k0 - half) * us; }
  __device__ long step(long k0) const { return k0 < half ? gs : us; }
  __device__ bool whole(long k0, int n) const { return (k0 < half ? k0 : k0 - half) + n <= F; }
  __device__ bool has(long k) const { return (k < half ? k : k - half) < F; }
  __device__ T at(int r, long k) const { return has(k) ? tile(k)[col0 + r] : (T)0.0f; }
};

// ---- staging: global memory -> registers -> LDS -----------------------------------------------------------------
// WIDE: every chunk's elements lie within the operand and can be read in one aligned access (the host has checked
// addresses, strides and lengths); otherwise they are read one by one.
template <typename T, typename Op, int ROWS, int THREADS, bool WIDE, bool ALONG = Op::kAlong>
struct Stage;

template <typename T, typename Op, int ROWS, int THREADS, bool WIDE>
struct Stage<T, Op, ROWS, THREADS, WIDE, true> {
  static constexpr int kPer = Form<T>::kPer, kUnits = ROWS * kSlots<T> / THREADS, kAcc = sizeof(T) == 4 ? 2 : 1;
  static_assert(ROWS * kSlots<T> % THREADS == 0, "whole units");
  union Chunk {
    i32x4 w[kAcc];
    T e[kPer];
  };
  const T* at[kUnits];
  Chunk v[kUnits];

  __device__ __forceinline__ void init(const Op& o) {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const int u = threadIdx.x + i * THREADS;
      at[i] = o.row(u / kSlots<T>) + u % kSlots<T> * kPer;
    }
  }
  __device__ __forceinline__ void load(const Op&, long k0, long end) {
    if (WIDE && k0 + kDepth<T> <= end) {
#pragma unroll
      for (int i = 0; i < kUnits; i++)
#pragma unroll
        for (int a = 0; a < kAcc; a++) v[i].w[a] = reinterpret_cast<const i32x4*>(at[i] + k0)[a];
      return;
    }
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const T* p = at[i] + k0;
      const long k = k0 + (threadIdx.x + i * THREADS) % kSlots<T> * kPer;
      if (WIDE) {
#pragma unroll
        for (int a = 0; a < kAcc; a++)
          v[i].w[a] = k + a * (16 / (int)sizeof(T)) < end ? reinterpret_cast<const i32x4*>(p)[a] : i32x4{0, 0, 0, 0};
      } else {
#pragma unroll
        for (int e = 0; e < kPer; e++) v[i].e[e] = k + e < end ? p[e] : (T)0;
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const int u = threadIdx.x + i * THREADS, row = u / kSlots<T>, c = u % kSlots<T>;
      if constexpr (sizeof(T) == 4) {
        unsigned h[3][4];
        split(v[i].e, h[0], h[1], h[2]);
#pragma unroll
        for (int p = 0; p < 3; p++)
          *reinterpret_cast<u32x4*>(lds + lds_at<T>(ROWS, p, row, c)) = u32x4{h[p][0], h[p][1], h[p][2], h[p][3]};
      } else {
        *reinterpret_cast<i32x4*>(lds + lds_at<T>(ROWS, 0, row, c)) = v[i].w[0];
      }
    }
  }
};

// Transposing: a unit is four columns of kLines consecutive memory rows (a chunk, or half of one in fp32).
template <typename T, typename Op, int ROWS, int THREADS, bool WIDE>
struct Stage<T, Op, ROWS, THREADS, WIDE, false> {
  static constexpr int kLines = sizeof(T) == 4 ? 4 : 8, kQuads = ROWS / 4;
  static constexpr int kUnits = kQuads * (kDepth<T> / kLines) / THREADS;
  static_assert(kQuads * (kDepth<T> / kLines) % THREADS == 0, "whole units");
  typedef T Quad __attribute__((ext_vector_type(4)));
  Quad v[kUnits][kLines];

  __device__ __forceinline__ void init(const Op&) {}
  __device__ __forceinline__ void load(const Op& o, long k0, long end) {
    const T* p = o.tile(k0);
    const long step = o.step(k0);
    if (WIDE && k0 + kDepth<T> <= end && o.whole(k0, kDepth<T>)) {
      // offsets from a common start, in 32 bits: the host takes strides up to 2^22 elements
#pragma unroll
      for (int i = 0; i < kUnits; i++) {
        const int u = threadIdx.x + i * THREADS, c = o.col0 + u % kQuads * 4;
        // columns past the end: any one, whose values go nowhere
        const unsigned at = (unsigned)(u / kQuads * kLines) * (unsigned)step + (unsigned)(c < o.cols ? c : 0);
#pragma unroll
        for (int l = 0; l < kLines; l++) v[i][l] = *reinterpret_cast<const Quad*>(p + l * step + at);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const int u = threadIdx.x + i * THREADS, c = o.col0 + u % kQuads * 4;
#pragma unroll
      for (int l = 0; l < kLines; l++) {
        const int k = u / kQuads * kLines + l;
        const bool ok = k0 + k < end && o.has(k0 + k);
        const T* q = p + k * step + c;
#pragma unroll
        for (int e = 0; e < 4; e++) v[i][l][e] = ok && c + e < o.cols ? q[e] : (T)0.0f;
      }
    }
  }
  __device__ __forceinline__ void store(char* lds) const {
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
      const int u = threadIdx.x + i * THREADS, row = u % kQuads * 4, part = u / kQuads;
#pragma unroll
      for (int e = 0; e < 4; e++) {
        if constexpr (sizeof(T) == 4) {
          const float x[4] = {v[i][0][e], v[i][1][e], v[i][2][e], v[i][3][e]};
          unsigned h[3][2];
          split(x, h[0], h[1], h[2]);
#pragma unroll
          for (int p = 0; p < 3; p++)
            *reinterpret_cast<u32x2*>(lds + lds_at<T>(ROWS, p, row + e, part >> 1) + (part & 1) * 8) = u32x2{h[p][0], h[p][1]};
        } else {
          bf16x8 h;
#pragma unroll
          for (int l = 0; l < 8; l++) h[l] = v[i][l][e];
          *reinterpret_cast<bf16x8*>(lds + lds_at<T>(ROWS, 0, row + e, part)) = h;
        }
      }
    }
  }
};

// ---- the product --------------------------------------------------------------------------------------------------
template <typename T>
struct Mma;
template <>
struct Mma<bf16> {
  typedef bf16x8 Op;
  static __device__ __forceinline__ f32x16 go(Op a, Op b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mma<float> : Mma<bf16> {};
template <>
struct Mma<i8> {
  typedef i32x4 Op;
  static __device__ __forceinline__ i32x16 go(Op a, Op b, i32x16 c) {
    return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
  }
};

// A block's tile is BM x BN, on WM x WN waves of IM x JN accumulators of 32 x 32.
template <int BM_, int BN_, int WM_, int WN_>
struct Shape {
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_;
  static constexpr int kThreads = WM * WN * 64, IM = BM / WM / 32, JN = BN / WN / 32;
};

template <typename T, typename S>
constexpr int kLdsBytes = Form<T>::kPlanes * (S::BM + S::BN) * Form<T>::kRowBytes;

// The accumulators over k in [k0, end). One LDS buffer: the next tile's global loads are in flight while this one is
// multiplied, and the two or three blocks of a CU cover each other's barriers and stores.
template <typename T, typename S, bool WIDE, typename OpA, typename OpB>
__device__ __forceinline__ void multiply(const OpA& A, const OpB& B, long k0, long end, char* lds,
                                         typename Form<T>::Acc (&acc)[S::IM][S::JN]) {
  constexpr int P = Form<T>::kPlanes;
  typedef typename Mma<T>::Op Op;
  char* la = lds;
  char* lb = lds + P * S::BM * Form<T>::kRowBytes;
  Stage<T, OpA, S::BM, S::kThreads, WIDE> sa;
  Stage<T, OpB, S::BN, S::kThreads, WIDE> sb;
  sa.init(A);
  sb.init(B);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int ra = wave / S::WN * S::IM * 32 + (lane & 31), rb = wave % S::WN * S::JN * 32 + (lane & 31);
  if (k0 < end) {
    sa.load(A, k0, end);
    sb.load(B, k0, end);
  }
  for (; k0 < end; k0 += kDepth<T>) {
    __syncthreads();
    sa.store(la);
    sb.store(lb);
    __syncthreads();
    if (k0 + kDepth<T> < end) {
      sa.load(A, k0 + kDepth<T>, end);
      sb.load(B, k0 + kDepth<T>, end);
    }
#pragma unroll
    for (int s = 0; s < kSlots<T> / 2; s++) {
      const int c = s * 2 + (lane >> 5);
      Op a[P][S::IM], b[P][S::JN];
#pragma unroll
      for (int p = 0; p < P; p++) {
#pragma unroll
        for (int i = 0; i < S::IM; i++) a[p][i] = *reinterpret_cast<const Op*>(la + lds_at<T>(S::BM, p, ra + i * 32, c));
#pragma unroll
        for (int j = 0; j < S::JN; j++) b[p][j] = *reinterpret_cast<const Op*>(lb + lds_at<T>(S::BN, p, rb + j * 32, c));
      }
      // the planes' products, the smallest first
      constexpr int pa[6] = {2, 0, 1, 1, 0, 0}, pb[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
      for (int q = P == 3 ? 0 : 5; q < 6; q++)
#pragma unroll
        for (int i = 0; i < S::IM; i++)
#pragma unroll
          for (int j = 0; j < S::JN; j++) acc[i][j] = Mma<T>::go(a[pa[q]][i], b[pb[q]][j], acc[i][j]);
    }
  }
}

// One output again, in plain fp32
template <typename OpA, typename OpB>
__device__ __attribute__((noinline)) float again(const OpA& A, int ra, const OpB& B, int rb, long k0, long end) {
  float v = 0;
  for (long k = k0; k < end; k++) v = __builtin_fmaf((float)A.at(ra, k), (float)B.at(rb, k), v);
  return v;
}

// row of C (within the block's tile) that register r of accumulator i holds
template <typename S>
__device__ __forceinline__ int c_row(int i, int r) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  return wave / S::WN * S::IM * 32 + i * 32 + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}
// and the column of accumulator j
template <typename S>
__device__ __forceinline__ int c_col(int j) {
  return (int)(threadIdx.x >> 6) % S::WN * S::JN * 32 + j * 32 + (threadIdx.x & 31);
}

// The fp32 outputs that came out infinite or NaN, again: those of rows below `rows` and of columns that are stored
// (a column is one of them where stored(column)).
template <typename S, typename OpA, typename OpB, typename C>
__device__ __forceinline__ void mend(const OpA& A, const OpB& B, long k0, long end, int rows, C stored,
                                     f32x16 (&acc)[S::IM][S::JN]) {
  float z = 0;   // stays zero unless one of them is: a multiplication each
#pragma unroll
  for (int i = 0; i < S::IM; i++)
#pragma unroll
    for (int j = 0; j < S::JN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) z = __builtin_fmaf(acc[i][j][r], 0.0f, z);
  if (z == 0) return;
#pragma unroll
  for (int i = 0; i < S::IM; i++)
#pragma unroll
    for (int j = 0; j < S::JN; j++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int row = c_row<S>(i, r), col = c_col<S>(j);
        if (acc[i][j][r] * 0.0f != 0 && row < rows && stored(col)) acc[i][j][r] = again(A, row, B, col, k0, end);
      }
}

// Blocks to tiles (rows of tiles `tm`, `tn` in each): block b runs on XCD b mod 8, and a row of tiles stays on one
// XCD, so that its part of A is read from memory by one L2 only.
__device__ __forceinline__ bool tile_of(int b, int tm, int tn, int& m, int& n) {
  const int i = b >> 3;
  m = i / tn * 8 + (b & 7);
  n = i % tn;
  return m < tm;
}
inline unsigned tile_grid(long tm, long tn) { return (unsigned)((tm + 7) / 8 * 8 * tn); }

}  // namespace g1nn
