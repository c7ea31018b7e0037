// nn_gated.hip -- the gated block: y = act(x Wg^T + bg) * (x Wu^T + bu), its gradients, and the same on 8-bit rows and
// weights.
//
//   g = x Wg^T + bg;  u = x Wu^T + bu;  y = act(g) u
//   dg = dy u act'(g);  du = dy act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x;  dbg, dbu = column sums
//
// The backward pass computes g and u again: per value that costs 4 K operations, and saves writing and reading both.
#include <initializer_list>

#include "../../include/g1nn.h"
#include "nn_common.h"

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
  long M;
  int K, F;
  const void *x, *wg, *wu, *bg, *bu, *dy;
  long xs, wgs, wus, dys;
  int act;
  void* y;
  float* d;        // backward: [M][2F] dg and du
};

constexpr int kT = 16;

// one value of y (or of dg and du) to a thread
template <typename T, bool GRAD>
__global__ __launch_bounds__(kT * kT) void k_gated(GatedArgs a) {
  __shared__ float xs[kT][kT + 1], gs[kT][kT + 1], us[kT][kT + 1];
  const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
  const long m = (long)blockIdx.x * kT + ty;
  const int f0 = blockIdx.y * kT;
  float g = 0, u = 0;
  for (int k0 = 0; k0 < a.K; k0 += kT) {
    const int k = k0 + tx, f = f0 + ty;
    xs[ty][tx] = m < a.M && k < a.K ? (float)((const T*)a.x)[m * a.xs + k] : 0;
    gs[ty][tx] = f < a.F && k < a.K ? (float)((const T*)a.wg)[f * a.wgs + k] : 0;
    us[ty][tx] = f < a.F && k < a.K ? (float)((const T*)a.wu)[f * a.wus + k] : 0;
    __syncthreads();
    for (int i = 0; i < kT; i++) {
      g = __builtin_fmaf(xs[ty][i], gs[tx][i], g);
      u = __builtin_fmaf(xs[ty][i], us[tx][i], u);
    }
    __syncthreads();
  }
  const int f = f0 + tx;
  if (m >= a.M || f >= a.F) return;
  if (a.bg) g += (float)((const T*)a.bg)[f];
  if (a.bu) u += (float)((const T*)a.bu)[f];
  float d;
  const float v = activation<GRAD>(a.act, g, d);
  if (!GRAD) {
    ((T*)a.y)[m * a.F + f] = (T)(v * u);
    return;
  }
  const float dy = (float)((const T*)a.dy)[m * a.dys + f];
  a.d[m * 2 * a.F + f] = dy * u * d;
  a.d[m * 2 * a.F + a.F + f] = dy * v;
}

// dx = dg Wg + du Wu
template <typename T>
__global__ __launch_bounds__(kT * kT) void k_gated_dx(GatedArgs a, T* dx) {
  __shared__ float ds[kT][kT + 1], ws[kT][kT + 1];
  const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
  const long m = (long)blockIdx.x * kT + ty;
  const int k = blockIdx.y * kT + tx;
  float v = 0;
  for (int half = 0; half < 2; half++) {
    const T* w = (const T*)(half ? a.wu : a.wg);
    const long stride = half ? a.wus : a.wgs;
    for (int f0 = 0; f0 < a.F; f0 += kT) {
      ds[ty][tx] = m < a.M && f0 + tx < a.F ? a.d[m * 2 * a.F + half * (long)a.F + f0 + tx] : 0;
      ws[ty][tx] = f0 + ty < a.F && k < a.K ? (float)w[(f0 + ty) * stride + k] : 0;
      __syncthreads();
      for (int i = 0; i < kT; i++) v = __builtin_fmaf(ds[ty][i], ws[i][tx], v);
      __syncthreads();
    }
  }
  if (m < a.M && k < a.K) dx[m * a.K + k] = (T)v;
}

// dW [F][K] = d^T x, and the column sums of d (by the blocks of the first 16 columns of x)
template <typename T>
__global__ __launch_bounds__(kT * kT) void k_gated_dw(GatedArgs a, T* dwg, T* dwu, T* dbg, T* dbu) {
  __shared__ float ds[kT][kT + 1], xs[kT][kT + 1];
  const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
  const int f0 = blockIdx.x * kT, k = blockIdx.y * kT + tx, half = blockIdx.z;
  float v = 0, b = 0;
  for (long m0 = 0; m0 < a.M; m0 += kT) {
    ds[ty][tx] = m0 + ty < a.M && f0 + tx < a.F ? a.d[(m0 + ty) * 2 * a.F + half * (long)a.F + f0 + tx] : 0;
    xs[ty][tx] = m0 + ty < a.M && k < a.K ? (float)((const T*)a.x)[(m0 + ty) * a.xs + k] : 0;
    __syncthreads();
    for (int i = 0; i < kT; i++) {
      v = __builtin_fmaf(ds[i][ty], xs[i][tx], v);
      b += ds[i][ty];
    }
    __syncthreads();
  }
  const int f = f0 + ty;
  T* dw = half ? dwu : dwg;
  T* db = half ? dbu : dbg;
  if (dw && f < a.F && k < a.K) dw[(long)f * a.K + k] = (T)v;
  if (db && f < a.F && k == 0) db[f] = (T)b;
}

struct GatedQ8Args {
  long M;
  int K, F;
  const signed char *q, *qg, *qu;
  const float *s, *sg, *su, *bg, *bu;
  long qs;
  int act;
  void* y;
};

template <typename T>
__global__ __launch_bounds__(kT * kT) void k_gated_q8(GatedQ8Args a) {
  __shared__ int xs[kT][kT + 1], gs[kT][kT + 1], us[kT][kT + 1];
  const int tx = threadIdx.x % kT, ty = threadIdx.x / kT;
  const long m = (long)blockIdx.x * kT + ty;
  const int f0 = blockIdx.y * kT;
  int g = 0, u = 0;
  for (int k0 = 0; k0 < a.K; k0 += kT) {
    const int k = k0 + tx, f = f0 + ty;
    xs[ty][tx] = m < a.M && k < a.K ? a.q[m * a.qs + k] : 0;
    gs[ty][tx] = f < a.F && k < a.K ? a.qg[(long)f * a.K + k] : 0;
    us[ty][tx] = f < a.F && k < a.K ? a.qu[(long)f * a.K + k] : 0;
    __syncthreads();
    for (int i = 0; i < kT; i++) {
      g += xs[ty][i] * gs[tx][i];
      u += xs[ty][i] * us[tx][i];
    }
    __syncthreads();
  }
  const int f = f0 + tx;
  if (m >= a.M || f >= a.F) return;
  float d;
  const float gate = (float)g * (a.s[m] * a.sg[f]) + (a.bg ? a.bg[f] : 0.0f);
  const float up = (float)u * (a.s[m] * a.su[f]) + (a.bu ? a.bu[f] : 0.0f);
  ((T*)a.y)[m * a.F + f] = (T)(activation<false>(a.act, gate, d) * up);
}

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

inline dim3 tiles(long m, long n, int z = 1) { return dim3((m + kT - 1) / kT, (n + kT - 1) / kT, z); }

}  // namespace g1nn

using namespace g1nn;

extern "C" int g1_nn_gated(int type, long M, int K, int F, const void* x, long xs, const void* wg, long wgs,
                           const void* wu, long wus, const void* bg, const void* bu, int act, void* y, void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M == 0) return 0;
  if (!x || !wg || !wu || !y) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {x, wg, wu, bg, bu, y})) return -1;
  const GatedArgs a{M, K, F, x, wg, wu, bg, bu, nullptr, xs, wgs, wus, 0, act, y, nullptr};
  const hipStream_t st = (hipStream_t)stream;
  if (type == 0) return launch(k_gated<float, false>, tiles(M, F), dim3(kT * kT), st, a);
  return launch(k_gated<bf16, false>, tiles(M, F), dim3(kT * kT), st, a);
}

extern "C" long g1_nn_gated_backward_workspace(int type, long M, int K, int F) {
  (void)type;
  (void)K;
  return M * 2 * F * (long)sizeof(float);
}

template <typename T>
static int gated_backward(const GatedArgs& a, T* dx, T* dwg, T* dwu, T* dbg, T* dbu, hipStream_t st) {
  if (a.M > 0) {
    if (launch(k_gated<T, true>, tiles(a.M, a.F), dim3(kT * kT), st, a)) return -2;
    if (dx && launch(k_gated_dx<T>, tiles(a.M, a.K), dim3(kT * kT), st, a, dx)) return -2;
  }
  if (dwg || dwu || dbg || dbu)
    return launch(k_gated_dw<T>, tiles(a.F, a.K, 2), dim3(kT * kT), st, a, dwg, dwu, dbg, dbu);
  return 0;
}

extern "C" int g1_nn_gated_backward(int type, long M, int K, int F, const void* x, long xs, const void* wg, long wgs,
                                    const void* wu, long wus, const void* bg, const void* bu, int act, const void* dy,
                                    long dys, void* dx, void* dwg, void* dwu, void* dbg, void* dbu, void* ws,
                                    void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M > 0 && (!x || !wg || !wu || !dy || !ws)) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {x, wg, wu, bg, bu, dy, dx, dwg, dwu, dbg, dbu})) return -1;
  if (!aligned(ws, 16)) return refuse("the workspace is not aligned to 16 bytes") ? -1 : 0;
  const GatedArgs a{M, K, F, x, wg, wu, bg, bu, dy, xs, wgs, wus, dys, act, nullptr, (float*)ws};
  const hipStream_t st = (hipStream_t)stream;
  if (type == 0)
    return gated_backward<float>(a, (float*)dx, (float*)dwg, (float*)dwu, (float*)dbg, (float*)dbu, st);
  return gated_backward<bf16>(a, (bf16*)dx, (bf16*)dwg, (bf16*)dwu, (bf16*)dbg, (bf16*)dbu, st);
}

extern "C" int g1_nn_gated_q8(int type, long M, int K, int F, const signed char* q, long qs, const float* s,
                              const signed char* qg, const float* sg, const signed char* qu, const float* su,
                              const float* bg, const float* bu, int act, void* y, void* stream) {
  if (bad_gated(type, M, K, F, act)) return -1;
  if (M == 0) return 0;
  if (!q || !s || !qg || !sg || !qu || !su || !y) return refuse("a null pointer") ? -1 : 0;
  if (bad_place(type, {y}) || bad_place(0, {s, sg, su, bg, bu})) return -1;
  const GatedQ8Args a{M, K, F, q, qg, qu, s, sg, su, bg, bu, qs, act, y};
  const hipStream_t st = (hipStream_t)stream;
  if (type == 0) return launch(k_gated_q8<float>, tiles(M, F), dim3(kT * kT), st, a);
  return launch(k_gated_q8<bf16>, tiles(M, F), dim3(kT * kT), st, a);
}
