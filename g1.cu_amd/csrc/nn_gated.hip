// nn_gated.hip -- the gated block: y = act(x Wg^T + bg) * (x Wu^T + bu), its gradients, and the same on 8-bit rows and
// weights.
//
//   g = x Wg^T + bg;  u = x Wu^T + bu;  y = act(g) u
//   dg = dy u act'(g);  du = dy act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dbg, dbu = column sums
//
// Forward: one product whose tile holds both projections of its outputs; activation and product in the epilogue.
// Backward: the same product again with an epilogue that reads dy and writes d = [dg | du] (it costs 4 K operations a
// value and saves writing and reading g and u), then dx = d [Wg; Wu], then [dWg; dWu] = d^T x with the rows split
// over the blocks, and a join of those parts and of the column sums in a fixed order. d is held in the tensors' type.
#include <initializer_list>

#include "../../include/g1nn.h"
#include "nn_gemm.h"

namespace g1nn {

constexpr int kActs = 4;

// act(g), and act'(g) where it is asked for
template <bool D>
__device__ __forceinline__ float activation(int act, float g, float& d) {
  if (act == 0 || act == 2) {
    const float p = 1.0f / (1.0f + expf(-g));
    if (act == 2) {
      if (D) d = p * (1.0f - p);
      return p;
    }
    if (D) d = p * (1.0f + g * (1.0f - p));
    return g * p;
  }
  if (act == 1) {
    // 0.5 g (1 + tanh z) with z = sqrt(2/pi) (g + 0.044715 g^3)
    const float z = 0.7978845608028654f * (g + 0.044715f * g * g * g), t = tanhf(z);
    if (D) d = 0.5f * (1.0f + t) + 0.5f * g * (1.0f - t * t) * 0.7978845608028654f * (1.0f + 0.134145f * g * g);
    return 0.5f * g * (1.0f + t);
  }
  const float e = g > 0 ? g : expm1f(g);
  if (D) d = g > 0 ? 1.0f : e + 1.0f;
  return e;
}

struct GatedArgs {
  int M, K, F;
  const void *x, *wg, *wu, *bg, *bu, *dy;
  long xs, wgs, wus, dys;
  int act;
  void* y;
  // backward
  int half;                 // F rounded up to 64: d is [M][2 half]
  void* d;
  float* sums;              // column sums of d by rows of waves, or null
  void *dx, *dwg, *dwu, *dbg, *dbu;
  float* parts;             // [splits][2 half][K]
  int splits, chunk;        // rows of a split
  int sum_rows;
  // 8-bit rows and weights
  const float *s, *sg, *su;
};

using Large = Shape<128, 128, 2, 2>;
using Small = Shape<64, 64, 2, 1>;

// y, or d and its column sums
template <typename T, typename O, typename S, bool WIDE, bool GRAD>
__global__ __launch_bounds__(S::kThreads) void k_gated(GatedArgs a) {
  __shared__ __align__(16) char lds[kLdsBytes<T, S>];
  const int cover = GRAD ? a.half : a.F, tm = (a.M + S::BM - 1) / S::BM, tn = (cover + S::BN / 2 - 1) / (S::BN / 2);
  int m, n;
  if (!tile_of(blockIdx.x, tm, tn, m, n)) return;
  const Along<T> A{(const T*)a.x, a.xs, m * S::BM, a.M};
  const Paired<T> B{(const T*)a.wg, (const T*)a.wu, a.wgs, a.wus, n * (S::BN / 2), a.F};
  typename Form<T>::Acc acc[S::IM][S::JN] = {};
  multiply<T, S, WIDE>(A, B, 0, a.K, lds, acc);
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int j = 0; j < S::JN; j += 2) {
    const int col = c_col<S>(j), f = B.f0 + (col >> 6) * 32 + (lane & 31);
    const bool in = f < a.F;
    float bg = 0, bu = 0, sg = 0, su = 0;
    if constexpr (sizeof(T) == 1) {
      if (in) {
        bg = a.bg ? ((const float*)a.bg)[f] : 0;
        bu = a.bu ? ((const float*)a.bu)[f] : 0;
        sg = a.sg[f];
        su = a.su[f];
      }
    } else if (in) {
      bg = a.bg ? (float)((const T*)a.bg)[f] : 0;
      bu = a.bu ? (float)((const T*)a.bu)[f] : 0;
    }
    float sum_g = 0, sum_u = 0;
#pragma unroll
    for (int i = 0; i < S::IM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int tr = c_row<S>(i, r), row = m * S::BM + tr;
        if (row >= a.M) continue;
        float g, u;
        if constexpr (sizeof(T) == 1) {
          const float s = a.s[row];
          g = (float)acc[i][j][r] * (s * sg) + bg;
          u = (float)acc[i][j + 1][r] * (s * su) + bu;
        } else {
          g = acc[i][j][r];
          u = acc[i][j + 1][r];
          if (sizeof(T) == 4 && in) {
            if (!is_finite(g)) g = again(A, tr, B, col, 0, a.K);
            if (!is_finite(u)) u = again(A, tr, B, col + 32, 0, a.K);
          }
          g += bg;
          u += bu;
        }
        float d;
        const float v = activation<GRAD>(a.act, g, d);
        if constexpr (!GRAD) {
          if (in) ((O*)a.y)[(long)row * a.F + f] = (O)(v * u);
        } else {
          float dg = 0, du = 0;
          if (in) {
            const float dy = (float)((const T*)a.dy)[(long)row * a.dys + f];
            dg = dy * u * d;
            du = dy * v;
          }
          T* to = (T*)a.d + (long)row * (2 * a.half);
          if (f < a.half) {
            to[f] = (T)dg;
            to[a.half + f] = (T)du;
          }
          sum_g += dg;
          sum_u += du;
        }
      }
    if constexpr (GRAD) {
      if (a.sums) {
        sum_g += __shfl_xor(sum_g, 32);
        sum_u += __shfl_xor(sum_u, 32);
        float* to = a.sums + ((long)m * S::WM + (threadIdx.x >> 6) / S::WN) * (2 * a.half);
        if (lane < 32 && f < a.half) {
          to[f] = sum_g;
          to[a.half + f] = sum_u;
        }
      }
    }
  }
}

// dx = d [Wg; Wu]
template <typename T, typename S, bool WIDE>
__global__ __launch_bounds__(S::kThreads) void k_gated_dx(GatedArgs a) {
  __shared__ __align__(16) char lds[kLdsBytes<T, S>];
  const int tm = (a.M + S::BM - 1) / S::BM, tn = (a.K + S::BN - 1) / S::BN;
  int m, n;
  if (!tile_of(blockIdx.x, tm, tn, m, n)) return;
  const Along<T> A{(const T*)a.d, 2l * a.half, m * S::BM, a.M};
  const AcrossPair<T> B{(const T*)a.wg, (const T*)a.wu, a.wgs, a.wus, a.half, a.F, n * S::BN, a.K};
  typename Form<T>::Acc acc[S::IM][S::JN] = {};
  multiply<T, S, WIDE>(A, B, 0, 2 * a.half, lds, acc);
#pragma unroll
  for (int j = 0; j < S::JN; j++)
#pragma unroll
    for (int i = 0; i < S::IM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int tr = c_row<S>(i, r), row = m * S::BM + tr, tc = c_col<S>(j), col = n * S::BN + tc;
        if (row >= a.M || col >= a.K) continue;
        float v = acc[i][j][r];
        if (sizeof(T) == 4 && !is_finite(v)) v = again(A, tr, B, tc, 0, 2 * a.half);
        ((T*)a.dx)[(long)row * a.K + col] = (T)v;
      }
}

// parts of [dWg; dWu] = d^T x: split s takes the rows [s chunk, (s + 1) chunk). Blocks of one split run on one XCD, which
// then reads those rows of d and x from memory once.
template <typename T, typename S, bool WIDE>
__global__ __launch_bounds__(S::kThreads) void k_gated_dw(GatedArgs a) {
  __shared__ __align__(16) char lds[kLdsBytes<T, S>];
  const int tm = (2 * a.half + S::BM - 1) / S::BM, tn = (a.K + S::BN - 1) / S::BN;
  int split, t;
  if (!tile_of(blockIdx.x, a.splits, tm * tn, split, t)) return;
  const int m = t / tn, n = t % tn;
  const Across<T> A{(const T*)a.d, 2l * a.half, m * S::BM, 2 * a.half};
  const Across<T> B{(const T*)a.x, a.xs, n * S::BN, a.K};
  const long k0 = (long)split * a.chunk, end = k0 + a.chunk < a.M ? k0 + a.chunk : a.M;
  typename Form<T>::Acc acc[S::IM][S::JN] = {};
  multiply<T, S, WIDE>(A, B, k0, end, lds, acc);
  float* to = a.parts + (long)split * (2 * a.half) * a.K;
#pragma unroll
  for (int j = 0; j < S::JN; j++)
#pragma unroll
    for (int i = 0; i < S::IM; i++)
#pragma unroll
      for (int r = 0; r < 16; r++) {
        const int tr = c_row<S>(i, r), row = m * S::BM + tr, tc = c_col<S>(j), col = n * S::BN + tc;
        if (row >= 2 * a.half || col >= a.K) continue;
        float v = acc[i][j][r];
        if (sizeof(T) == 4 && !is_finite(v)) v = again(A, tr, B, tc, k0, end);
        to[(long)row * a.K + col] = v;
      }
}

// The parts joined: blocks [0, wide) take 256 weights each, the others 32 biases each.
template <typename T>
__global__ __launch_bounds__(256) void k_gated_join(GatedArgs a, int wide) {
  if ((int)blockIdx.x < wide) {
    const long n = (long)a.F * a.K, i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * n) return;
    const bool up = i >= n;
    const long at = up ? i - n : i, from = at + (up ? (long)a.half * a.K : 0), step = 2l * a.half * a.K;
    T* to = (T*)(up ? a.dwu : a.dwg);
    if (!to) return;
    float v = 0;
    for (int s = 0; s < a.splits; s++) v += a.parts[s * step + from];
    to[at] = (T)v;
    return;
  }
  __shared__ float part[8][32];
  const int c = threadIdx.x & 31, o = threadIdx.x >> 5, i = (blockIdx.x - wide) * 32 + c;
  const bool up = i >= a.half;
  const int f = up ? i - a.half : i;
  T* to = (T*)(up ? a.dbu : a.dbg);
  float v = 0;
  if (to && f < a.F)
    for (int p = o; p < a.sum_rows; p += 8) v += a.sums[(long)p * (2 * a.half) + i];
  part[o][c] = v;
  __syncthreads();
  if (o == 0 && to && f < a.F) {
    for (int p = 1; p < 8; p++) v += part[p][c];
    to[f] = (T)v;
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------
// Tiles of 128 x 128 where they give every CU one; else of 64 x 64, four times as many.
inline bool large(long m, long n) { return ((m + 127) / 128) * ((n + 127) / 128) >= 256; }

template <typename T, typename O, typename S, bool GRAD>
int run_gated(const GatedArgs& a, bool wide, hipStream_t st) {
  const dim3 grid(tile_grid((a.M + S::BM - 1) / S::BM, ((GRAD ? a.half : a.F) + S::BN / 2 - 1) / (S::BN / 2)));
  if (wide) return launch(k_gated<T, O, S, true, GRAD>, grid, dim3(S::kThreads), st, a);
  return launch(k_gated<T, O, S, false, GRAD>, grid, dim3(S::kThreads), st, a);
}

template <typename T, typename O, bool GRAD>
int run_gated(const GatedArgs& a, bool wide, hipStream_t st) {
  if (large(a.M, 2l * a.F)) return run_gated<T, O, Large, GRAD>(a, wide, st);
  return run_gated<T, O, Small, GRAD>(a, wide, st);
}

template <typename T, typename S>
int run_dx(const GatedArgs& a, bool wide, hipStream_t st) {
  const dim3 grid(tile_grid((a.M + S::BM - 1) / S::BM, (a.K + S::BN - 1) / S::BN));
  if (wide) return launch(k_gated_dx<T, S, true>, grid, dim3(S::kThreads), st, a);
  return launch(k_gated_dx<T, S, false>, grid, dim3(S::kThreads), st, a);
}

template <typename T, typename S>
int run_dw(const GatedArgs& a, bool wide, hipStream_t st) {
  const dim3 grid(tile_grid(a.splits, ((2 * a.half + S::BM - 1) / S::BM) * (long)((a.K + S::BN - 1) / S::BN)));
  if (wide) return launch(k_gated_dw<T, S, true>, grid, dim3(S::kThreads), st, a);
  return launch(k_gated_dw<T, S, false>, grid, dim3(S::kThreads), st, a);
}

// How [dWg; dWu] is split over the rows: as many parts as give two blocks to each CU, of 256 rows at least.
struct Split {
  int half, splits, chunk;
  bool large;
  Split(long M, int K, int F) {
    half = (F + 63) / 64 * 64;
    const long t128 = ((2l * half + 127) / 128) * ((K + 127) / 128), t64 = (2l * half / 64) * ((K + 63) / 64);
    large = t128 * ((M + 255) / 256) >= 512;
    const long tiles = large ? t128 : t64, most = (M + 255) / 256;
    long s = (512 + tiles - 1) / tiles;
    s = s < most ? s : most;
    s = s < 1 ? 1 : s;
    chunk = (int)((((M + s - 1) / s) + 63) / 64 * 64);
    chunk = chunk < 64 ? 64 : chunk;
    splits = (int)((M + chunk - 1) / chunk);
  }
};

inline long round16(long n) { return (n + 15) / 16 * 16; }

struct Workspace {
  long d, sums, parts, bytes;
  Workspace(int type, long M, int K, const Split& s) {
    d = 0;
    sums = d + round16(M * 2 * s.half * (type == 0 ? 4 : 2));
    // rows of column sums: ceil(M / BM) WM of them, two for every 128 rows with large tiles, four with small ones
    parts = sums + round16((M + 127) / 128 * 4 * 2 * s.half * 4);
    bytes = parts + (long)s.splits * 2 * s.half * K * 4;
  }
};

inline bool bad_gated(int type, long M, int K, int F, int act) {
  if (type != 0 && type != 1) return refuse("type is 0 (fp32) or 1 (bf16)");
  if (M < 0 || M > (1l << 30)) return refuse("0 to 2^30 rows are supported");
  if (K < 1 || K > (1 << 17) || F < 1 || F > (1 << 17)) return refuse("widths of 1 to 131072 are supported");
  if (act < 0 || act >= kActs) return refuse("unknown activation");
  return false;
}

inline bool bad_place(int type, std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (!aligned(p, type == 0 ? 4 : 2)) return refuse("an address is not aligned to its elements");
  return false;
}

// Whether rows of n elements can be read in accesses of `bytes`.
inline bool even(const void* p, long stride, long n, int size, int bytes) {
  return aligned(p, bytes) && stride * size % bytes == 0 && n * size % bytes == 0;
}

template <typename T>
int gated_backward(GatedArgs a, const Split& s, hipStream_t st) {
  const int size = sizeof(T);
  const bool xw = even(a.x, a.xs, a.K, size, 16);
  const bool wide = xw && even(a.wg, a.wgs, a.K, size, 16) && even(a.wu, a.wus, a.K, size, 16);
  const bool weights = a.dwg || a.dwu, biases = a.dbg || a.dbu;
  if (!biases) a.sums = nullptr;
  const bool big = large(a.M, 2l * a.F);
  a.sum_rows = big ? (a.M + Large::BM - 1) / Large::BM * Large::WM : (a.M + Small::BM - 1) / Small::BM * Small::WM;
  if (a.M > 0) {
    int rc = run_gated<T, T, true>(a, wide, st);
    if (rc) return rc;
    if (a.dx) {
      rc = large(a.M, a.K) ? run_dx<T, Large>(a, wide, st) : run_dx<T, Small>(a, wide, st);
      if (rc) return rc;
    }
    if (weights) {
      rc = s.large ? run_dw<T, Large>(a, xw, st) : run_dw<T, Small>(a, xw, st);
      if (rc) return rc;
    }
  } else {
    a.splits = a.sum_rows = 0;
  }
  if (!weights && !biases) return 0;
  const long nw = weights ? (2l * a.F * a.K + 255) / 256 : 0, nb = biases ? 2 * a.half / 32 : 0;
  return launch(k_gated_join<T>, dim3((unsigned)(nw + nb)), dim3(256), st, a, (int)nw);
}

}  // namespace g1nn

using namespace g1nn;

extern "C" int g1_nn_gated(int type, long M, int K, int F, const void* x, long xs, const void* wg, long wgs,
                           const void* wu, long wus, const void* bg, const void* bu, int act, void* y, void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M == 0) return 0;
  if (!x || !wg || !wu || !y) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {x, wg, wu, bg, bu, y})) return -1;
  GatedArgs a{};
  a.M = (int)M, a.K = K, a.F = F, a.x = x, a.wg = wg, a.wu = wu, a.bg = bg, a.bu = bu;
  a.xs = xs, a.wgs = wgs, a.wus = wus, a.act = act, a.y = y;
  const int size = type == 0 ? 4 : 2;
  const bool wide = even(x, xs, K, size, 16) && even(wg, wgs, K, size, 16) && even(wu, wus, K, size, 16);
  if (type == 0) return run_gated<float, float, false>(a, wide, (hipStream_t)stream);
  return run_gated<bf16, bf16, false>(a, wide, (hipStream_t)stream);
}

extern "C" long g1_nn_gated_backward_workspace(int type, long M, int K, int F) {
  return Workspace(type, M, K, Split(M, K, F)).bytes;
}

extern "C" int g1_nn_gated_backward(int type, long M, int K, int F, const void* x, long xs, const void* wg, long wgs,
                                    const void* wu, long wus, const void* bg, const void* bu, int act, const void* dy,
                                    long dys, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, void* ws,
                                    void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M > 0 && (!x || !wg || !wu || !dy || !ws)) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {x, wg, wu, bg, bu, dy, dx, dwg, dwu, dbg, dbu})) return -1;
  if (!aligned(ws, 16)) return refuse("the workspace is not aligned to 16 bytes") ? -1 : 0;
  const Split s(M, K, F);
  const Workspace w(type, M, K, s);
  GatedArgs a{};
  a.M = (int)M, a.K = K, a.F = F, a.x = x, a.wg = wg, a.wu = wu, a.bg = bg, a.bu = bu, a.dy = dy;
  a.xs = xs, a.wgs = wgs, a.wus = wus, a.dys = dys, a.act = act;
  a.half = s.half, a.splits = s.splits, a.chunk = s.chunk;
  a.d = (char*)ws + w.d, a.sums = (float*)((char*)ws + w.sums), a.parts = (float*)((char*)ws + w.parts);
  a.dx = dx, a.dwg = dwg, a.dwu = dwu, a.dbg = dbg, a.dbu = dbu;
  if (type == 0) return gated_backward<float>(a, s, (hipStream_t)stream);
  return gated_backward<bf16>(a, s, (hipStream_t)stream);
}

extern "C" int g1_nn_gated_q8(int type, long M, int K, int F, const signed char* q, long qs, const float* s,
                              const signed char* qg, const float* sg, const signed char* qu, const float* su,
                              const float* bg, const float* bu, int act, void* y, void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M == 0) return 0;
  if (!q || !s || !qg || !sg || !qu || !su || !y) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {y}) || bad_place(0, {s, sg, su, bg, bu})) return -1;
  GatedArgs a{};
  a.M = (int)M, a.K = K, a.F = F, a.x = q, a.wg = qg, a.wu = qu, a.bg = bg, a.bu = bu;
  a.xs = qs, a.wgs = a.wus = K, a.act = act, a.y = y, a.s = s, a.sg = sg, a.su = su;
  const bool wide = even(q, qs, K, 1, 16) && even(qg, K, K, 1, 16) && even(qu, K, K, 1, 16);
  if (type == 0) return run_gated<i8, float, false>(a, wide, (hipStream_t)stream);
  return run_gated<i8, bf16, false>(a, wide, (hipStream_t)stream);
}
