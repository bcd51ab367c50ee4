// The norms around a block, its gate and its residual scale, joined with the residual add, forward and backward, for
// gfx950. Per row of D elements, f the block's output, g its gate's (before the activation act):
//   rf = 1 / sqrt(mean(f^2) + eps),  n = f rf w_branch          (the norm after the block)
//   xn = x + scale act(g) n                                     (the residual stream)
//   rx = 1 / sqrt(mean(xn^2) + eps), y = xn rx w                (the norm before the next block)
// Backward, with dy the gradient of y and dres that of xn from its other use:
//   hx = xn rx, u = dy w:    dxn = rx (u - hx mean(u hx)) + dres (= dx)
//   hf = f rf, v = dxn scale act(g) w_branch:  df = rf (v - hf mean(v hf)),  dg = dxn scale n act'(g)
//   dw = sum over rows of dy hx;  q = sum over rows of dxn act(g) hf:  dw_branch = scale q,  dscale = w_branch q
//
// Bound by memory: of each element the forward moves x, f, g, xn and y (14 bytes with bfloat16 f, g and y), the backward
// xn, f, g, dy, dres, dx, df and dg (22). A row belongs to one wave up to 1024 columns, to 256 threads up to 4096, else
// to 1024: never more than four vectors of four values to a thread, which stay in registers between the two sums of a
// row, so that every operand is read once. All vectors but the last lie in the row whatever its size, and carry no
// masks. Sums over rows: a thread's, a partial row of the workgroup, and a second kernel that adds the partial rows in
// order, so that they are the same in every run.
// Measured (N 16376, D 1024, bfloat16): forward 41 us (5.7 TB/s), backward 70 us (5.2 TB/s) and 5 for the partial rows.
// Results written past the nearest caches make the backward alone 4 us faster, and what reads them next 10 slower.

#include <algorithm>

#include "mg_vec.h"

namespace mg {
namespace blocknorm {

constexpr int kNone = 0, kSigmoid = 1, kSilu = 2;
constexpr int kMaxD = 16384;
constexpr int threads_of(int tpr) { return tpr < 256 ? 256 : tpr; }

// The sum over the threads of a row; every thread gets it
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float* red) {
  a = wave_sum(a);
  if constexpr (TPR > 64) {
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = a;
    __syncthreads();
    a = 0.0f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) a += red[i];
  }
  return a;
}

template <int TPR>
__device__ __forceinline__ int64_t first_row() {
  return static_cast<int64_t>(blockIdx.x) * (threads_of(TPR) / TPR) +
         (TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
}

// act(g); slope: act'(g). A gate of -inf shuts: silu's 0 there, not -inf 0. 1 - sigma is made from the power, since the
// rounded sigma of an open gate has lost its digits; where the power is infinite, it is 1 (the minimum of a NaN and 1).
__device__ __forceinline__ float act_of(int act, float g, float& slope) {
  const float e = exp2_raw(g * -kLog2e), s = __builtin_amdgcn_rcpf(1.0f + e), rest = fminf(e * s, 1.0f);
  if (act == kSigmoid) {
    slope = s * rest;
    return s;
  }
  const float v = s == 0.0f ? 0.0f : g * s;
  slope = s + v * rest;
  return v;
}

// load4 in the form of memory, to be widened where it is used: a branch that converts waits for all loads before it
template <typename T>
struct raw4 {
  typedef T vec __attribute__((ext_vector_type(4)));
  typedef T vecu __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  vec x;
  __device__ __forceinline__ void load(const void* base, int64_t at, int left) {
    const T* p = static_cast<const T*>(base) + at;
    x = vec{0, 0, 0, 0};
    if (left >= 4) {
      x = *reinterpret_cast<const vecu*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < 3; ++j)
        if (j < left) x[j] = p[j];
    }
  }
  __device__ __forceinline__ f4 wide() const {
    f4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2) r.v[j] = bf16_to_f32(x[j]);
      else r.v[j] = x[j];
    }
    return r;
  }
};

struct Fwd {
  const float* x;
  const void *f, *g;
  const float *wf, *w, *scale;
  float* xn;
  void* y;
  float *rf, *rx;
  int64_t N;
  int D, act;
  float eps;
};

template <typename Tf, typename Ty, int TPR, int STEPS>
__global__ __launch_bounds__(threads_of(TPR)) void fwd_kernel(Fwd a) {
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.D);
  const auto left = [&](int i, int c) { return i + 1 < STEPS ? 4 : a.D - c; };
  for (int64_t row = first_row<TPR>(); row < a.N; row += static_cast<int64_t>(gridDim.x) * (threads_of(TPR) / TPR)) {
    const int64_t base = row * a.D;
    raw4<Tf> raw_f[STEPS], raw_g[STEPS];
    f4 x[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      raw_f[i].load(a.f, base + c, left(i, c));
      if (a.act) raw_g[i].load(a.g, base + c, left(i, c));
      x[i] = load4(a.x + base + c, left(i, c));
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const f4 f = raw_f[i].wide();
#pragma unroll
      for (int j = 0; j < 4; ++j) s += f.v[j] * f.v[j];
    }
    const float rf = 1.0f / sqrtf(row_sum<TPR>(s, red) * inv + a.eps);
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      const f4 wf = load4(a.wf + c, left(i, c)), f = raw_f[i].wide();
      f4 scale = io4<float>::fill(1.0f), g;
      if (a.scale) scale = load4(a.scale + c, left(i, c));
      if (a.act) g = raw_g[i].wide();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v = f.v[j] * rf * wf.v[j], slope;
        if (a.act) v *= act_of(a.act, g.v[j], slope);
        x[i].v[j] = __builtin_fmaf(scale.v[j], v, x[i].v[j]);
        s += x[i].v[j] * x[i].v[j];  // (0 past the row)
      }
      store4(a.xn + base + c, x[i], left(i, c));
    }
    const float rx = 1.0f / sqrtf(row_sum<TPR>(s, red) * inv + a.eps);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      f4 w = load4(a.w + c, left(i, c));
#pragma unroll
      for (int j = 0; j < 4; ++j) w.v[j] *= x[i].v[j] * rx;
      store4(static_cast<Ty*>(a.y) + base + c, w, left(i, c));
    }
    if (t == 0 && a.rf) a.rf[row] = rf, a.rx[row] = rx;
  }
}

struct Bwd {
  const float* xn;
  const void *f, *g;
  const float *wf, *w, *scale, *rf, *rx;
  const void* dy;
  const float* dres;
  float* dx;
  void *df, *dg;
  float* part;  // [workgroups][2][D]
  int64_t N;
  int D, act;
};

// A thread's sums over its rows, of each of its columns two: in registers, or at its own places in LDS
template <int THREADS, int STEPS, bool LDS>
struct Sums {
  f4 r[LDS ? 1 : STEPS][2];
  f4 (*l)[2][THREADS];
  __device__ __forceinline__ f4& at(int i, int k) {
    if constexpr (LDS) return l[i][k][threadIdx.x];
    else return r[i][k];
  }
};

template <typename Tf, typename Ty, int TPR, int STEPS>
__global__ __launch_bounds__(threads_of(TPR)) void bwd_kernel(Bwd a) {
  constexpr int kRows = threads_of(TPR) / TPR;
  __shared__ float red[TPR > 64 ? TPR / 64 : 1];
  __shared__ f4 s_sum[2][TPR == 64 ? kRows : 1][TPR == 64 ? 64 : 1];
  // 1024 threads have 128 registers each: with three vectors of every operand the sums do not fit beside them (N 1024
  // D 16384: 207 us with 84 registers spilled, 116 from LDS; one wave to a row is no faster from LDS)
  constexpr bool kLds = TPR == 1024 && (STEPS >= 3);
  __shared__ f4 s_acc[kLds ? STEPS : 1][2][kLds ? threads_of(TPR) : 1];
  Sums<kLds ? threads_of(TPR) : 1, STEPS, kLds> sums;
  sums.l = s_acc;
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.D);
  const auto left = [&](int i, int c) { return i + 1 < STEPS ? 4 : a.D - c; };
#pragma unroll
  for (int i = 0; i < STEPS; ++i) sums.at(i, 0) = sums.at(i, 1) = io4<float>::fill(0.0f);
  for (int64_t row = first_row<TPR>(); row < a.N; row += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t base = row * a.D;
    const float rf = a.rf[row], rx = a.rx[row];
    raw4<Ty> raw_dy[STEPS];
    raw4<Tf> raw_f[STEPS], raw_g[STEPS];
    f4 hx[STEPS], u[STEPS], d[STEPS], hf[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      hx[i] = load4(a.xn + base + c, left(i, c));
      raw_dy[i].load(a.dy, base + c, left(i, c));
      d[i] = io4<float>::fill(0.0f);
      if (a.dres) d[i] = load4(a.dres + base + c, left(i, c));
      raw_f[i].load(a.f, base + c, left(i, c));
      if (a.act) raw_g[i].load(a.g, base + c, left(i, c));
    }
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      const f4 w = load4(a.w + c, left(i, c));
      f4 sum = sums.at(i, 0);
      u[i] = raw_dy[i].wide();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hx[i].v[j] *= rx;
        sum.v[j] += u[i].v[j] * hx[i].v[j];
        u[i].v[j] *= w.v[j];
        s += u[i].v[j] * hx[i].v[j];
      }
      sums.at(i, 0) = sum;
    }
    const float mx = row_sum<TPR>(s, red) * inv;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      const f4 wf = load4(a.wf + c, left(i, c));
      f4 scale = io4<float>::fill(1.0f);
      if (a.scale) scale = load4(a.scale + c, left(i, c));
      f4 sum = sums.at(i, 1), g;
      hf[i] = raw_f[i].wide();
      if (a.act) g = raw_g[i].wide();
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float dxn = d[i].v[j] + rx * (u[i].v[j] - hx[i].v[j] * mx);
        d[i].v[j] = dxn;
        hf[i].v[j] *= rf;
        float act = 1.0f, slope = 0.0f;
        if (a.act) act = act_of(a.act, g.v[j], slope);
        sum.v[j] += dxn * (act * hf[i].v[j]);
        const float b = dxn * scale.v[j] * wf.v[j];
        if (a.act) g.v[j] = b * hf[i].v[j] * slope;
        u[i].v[j] = b * act;
        s += u[i].v[j] * hf[i].v[j];
      }
      sums.at(i, 1) = sum;
      if (a.dx) store4(a.dx + base + c, d[i], left(i, c));
      if (a.dg) store4(static_cast<Tf*>(a.dg) + base + c, g, left(i, c));
    }
    const float mf = row_sum<TPR>(s, red) * inv;
    if (a.df) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int c = 4 * (t + TPR * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[i].v[j] = rf * (u[i].v[j] - hf[i].v[j] * mf);
        store4(static_cast<Tf*>(a.df) + base + c, u[i], left(i, c));
      }
    }
  }
  if (!a.part) return;
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.D;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = 4 * (t + TPR * i);
    if constexpr (TPR > 64) {
      store4(part + c, sums.at(i, 0), left(i, c));
      store4(part + a.D + c, sums.at(i, 1), left(i, c));
    } else {
      const int wave = threadIdx.x / 64;
      __syncthreads();
      s_sum[0][wave][t] = sums.at(i, 0);
      s_sum[1][wave][t] = sums.at(i, 1);
      __syncthreads();
      if (wave < 2) {
        f4 x = s_sum[wave][0][t];
#pragma unroll
        for (int q = 1; q < kRows; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) x.v[j] += s_sum[wave][q][t].v[j];
        store4(part + wave * a.D + c, x, left(i, c));
      }
    }
  }
}

// [P][2 D] partial rows to the weights' gradients: 16 columns per workgroup, four to a thread, 64 threads' rows of each
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ part, int P, int D, const float* __restrict__ wf,
                                                        const float* __restrict__ scale, float* __restrict__ dw,
                                                        float* __restrict__ dwf, float* __restrict__ dscale) {
  __shared__ float s[64][17];
  const int n = 2 * D, c = 16 * blockIdx.x + 4 * (threadIdx.x % 4), g = threadIdx.x / 4;
  f4 x = io4<float>::fill(0.0f);
#pragma unroll 4
  for (int p = g; p < P; p += 64) {
    const f4 y = load4(part + static_cast<int64_t>(p) * n + c, n - c);
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] += y.v[j];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) s[g][4 * (threadIdx.x % 4) + j] = x.v[j];
  __syncthreads();
  const int col = threadIdx.x / 16, q = threadIdx.x % 16, e = 16 * blockIdx.x + col;
  float sum = (s[q][col] + s[q + 16][col]) + (s[q + 32][col] + s[q + 48][col]);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 16);
  if (q != 0 || e >= n) return;
  if (e < D) {
    if (dw) dw[e] = sum;
  } else {
    const int d = e - D;
    if (dwf) dwf[d] = sum * (scale ? scale[d] : 1.0f);
    if (dscale) dscale[d] = sum * wf[d];
  }
}

inline int rows_per_wg(int D) { return D <= 1024 ? 4 : 1; }
inline int grid_for(int64_t N, int D, int64_t most) {
  const int64_t per = rows_per_wg(D);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((N + per - 1) / per, most)));
}
constexpr int kFwdGrid = 65536, kBwdGrid = 1024;
inline int bwd_grid(int64_t N, int D) { return grid_for(N, D, D <= 4096 ? kBwdGrid : kBwdGrid / 4); }

#define MG_BN_STEPS(T)                             \
  switch ((D + 4 * T - 1) / (4 * T)) {             \
    case 1: GO(T, 1) break;                        \
    case 2: GO(T, 2) break;                        \
    case 3: GO(T, 3) break;                        \
    default: GO(T, 4)                              \
  }
#define MG_BN_SIZES \
  if (D <= 1024) { MG_BN_STEPS(64) } else if (D <= 4096) { MG_BN_STEPS(256) } else { MG_BN_STEPS(1024) }

template <typename Tf, typename Ty>
int launch_fwd(const Fwd& a, hipStream_t st) {
  const int D = a.D, grid = grid_for(a.N, D, kFwdGrid);
#define GO(T, S) hipLaunchKernelGGL((fwd_kernel<Tf, Ty, T, S>), dim3(grid), dim3(threads_of(T)), 0, st, a);
  MG_BN_SIZES
#undef GO
  return check_launch("mg_block_norm_fwd");
}

template <typename Tf, typename Ty>
int launch_bwd(const Bwd& a, float* dw, float* dwf, float* dscale, hipStream_t st) {
  const int D = a.D, grid = bwd_grid(a.N, D);
#define GO(T, S) hipLaunchKernelGGL((bwd_kernel<Tf, Ty, T, S>), dim3(grid), dim3(threads_of(T)), 0, st, a);
  MG_BN_SIZES
#undef GO
  if (a.part)
    hipLaunchKernelGGL(sum_parts_kernel, dim3((2 * D + 15) / 16), dim3(256), 0, st, a.part, grid, D, a.wf, a.scale, dw, dwf, dscale);
  return check_launch("mg_block_norm_bwd");
}

inline int check_dt(const char* fn, const char* name, int dt) {
  return dt == MG_F32 || dt == MG_BF16 ? MG_OK : fail(MG_ERR_DTYPE, "%s: %s dtype %d unsupported", fn, name, dt);
}
inline int check_p(const char* fn, const char* name, const void* p, int dt, bool required) {
  if (!p) return required ? fail(MG_ERR_ARG, "%s: %s is NULL", fn, name) : MG_OK;
  if (!aligned(p, dt == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: %s misaligned", fn, name);
  return MG_OK;
}
inline int check_shape(const char* fn, int64_t N, int D, int act) {
  if (N < 1 || D < 1 || D > kMaxD) return fail(MG_ERR_ARG, "%s: N=%lld must be >= 1 and D=%d in [1, %d]", fn, (long long)N, D, kMaxD);
  if (act < kNone || act > kSilu) return fail(MG_ERR_ARG, "%s: activation %d unknown", fn, act);
  return MG_OK;
}

}  // namespace blocknorm
}  // namespace mg

using namespace mg;

extern "C" int mg_block_norm_fwd(const float* x, int f_dtype, const void* f, const void* g, int act, const float* w_branch,
                                 const float* scale, const float* w, float* x_out, int y_dtype, void* y, float* rstd_branch, float* rstd,
                                 int64_t N, int D, float eps, void* stream) {
  using namespace blocknorm;
  const char* fn = "mg_block_norm_fwd";
  int rc;
  if ((rc = check_shape(fn, N, D, act)) || (rc = check_dt(fn, "f", f_dtype)) || (rc = check_dt(fn, "y", y_dtype)) ||
      (rc = check_p(fn, "x", x, MG_F32, true)) || (rc = check_p(fn, "f", f, f_dtype, true)) ||
      (rc = check_p(fn, "g", g, f_dtype, act != kNone)) || (rc = check_p(fn, "w_branch", w_branch, MG_F32, true)) ||
      (rc = check_p(fn, "scale", scale, MG_F32, false)) || (rc = check_p(fn, "w", w, MG_F32, true)) ||
      (rc = check_p(fn, "x_out", x_out, MG_F32, true)) || (rc = check_p(fn, "y", y, y_dtype, true)) ||
      (rc = check_p(fn, "rstd_branch", rstd_branch, MG_F32, false)) || (rc = check_p(fn, "rstd", rstd, MG_F32, rstd_branch != nullptr)))
    return rc;
  const Fwd a = {x, f, g, w_branch, w, scale, x_out, y, rstd_branch, rstd, N, D, act, eps};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (f_dtype == MG_BF16) return y_dtype == MG_BF16 ? launch_fwd<bf16_t, bf16_t>(a, st) : launch_fwd<bf16_t, float>(a, st);
  return y_dtype == MG_BF16 ? launch_fwd<float, bf16_t>(a, st) : launch_fwd<float, float>(a, st);
}

extern "C" size_t mg_block_norm_bwd_workspace_bytes(int64_t N, int D) {
  if (N < 1 || D < 1 || D > blocknorm::kMaxD) return 0;
  return static_cast<size_t>(blocknorm::bwd_grid(N, D)) * 2 * D * sizeof(float);
}

extern "C" int mg_block_norm_bwd(const float* xn, int f_dtype, const void* f, const void* g, int act, const float* w_branch,
                                 const float* scale, const float* w, const float* rstd_branch, const float* rstd, int dy_dtype,
                                 const void* dy, const float* dres, float* dx, void* df, void* dg, float* dw_branch, float* dscale,
                                 float* dw, int64_t N, int D, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace blocknorm;
  const char* fn = "mg_block_norm_bwd";
  int rc;
  if ((rc = check_shape(fn, N, D, act)) || (rc = check_dt(fn, "f", f_dtype)) || (rc = check_dt(fn, "dy", dy_dtype)) ||
      (rc = check_p(fn, "xn", xn, MG_F32, true)) || (rc = check_p(fn, "f", f, f_dtype, true)) ||
      (rc = check_p(fn, "g", g, f_dtype, act != kNone)) || (rc = check_p(fn, "w_branch", w_branch, MG_F32, true)) ||
      (rc = check_p(fn, "scale", scale, MG_F32, false)) || (rc = check_p(fn, "w", w, MG_F32, true)) ||
      (rc = check_p(fn, "rstd_branch", rstd_branch, MG_F32, true)) || (rc = check_p(fn, "rstd", rstd, MG_F32, true)) ||
      (rc = check_p(fn, "dy", dy, dy_dtype, true)) || (rc = check_p(fn, "dres", dres, MG_F32, false)) ||
      (rc = check_p(fn, "dx", dx, MG_F32, false)) || (rc = check_p(fn, "df", df, f_dtype, false)) ||
      (rc = check_p(fn, "dg", dg, f_dtype, false)) || (rc = check_p(fn, "dw_branch", dw_branch, MG_F32, false)) ||
      (rc = check_p(fn, "dscale", dscale, MG_F32, false)) || (rc = check_p(fn, "dw", dw, MG_F32, false)))
    return rc;
  if (dg && act == kNone) return fail(MG_ERR_ARG, "%s: dg without a gate", fn);
  const bool sums = dw_branch || dscale || dw;
  const size_t need = mg_block_norm_bwd_workspace_bytes(N, D);
  if (sums && (!workspace || workspace_bytes < need || !aligned(workspace, 16)))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or misaligned)", fn, workspace_bytes, need);
  const Bwd a = {xn, f, g, w_branch, w, scale, rstd_branch, rstd, dy, dres, dx, df, dg, sums ? static_cast<float*>(workspace) : nullptr,
                 N, D, act};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (f_dtype == MG_BF16)
    return dy_dtype == MG_BF16 ? launch_bwd<bf16_t, bf16_t>(a, dw, dw_branch, dscale, st) : launch_bwd<bf16_t, float>(a, dw, dw_branch, dscale, st);
  return dy_dtype == MG_BF16 ? launch_bwd<float, bf16_t>(a, dw, dw_branch, dscale, st) : launch_bwd<float, float>(a, dw, dw_branch, dscale, st);
}
