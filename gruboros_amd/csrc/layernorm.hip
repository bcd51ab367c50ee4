// Layer norm, forward and backward, with a residual add and dropout of the
// added branch in the same pass, for gfx950. Per row of D elements:
//   xn = x + keep(delta) delta / (1 - p)   (delta optional; keep: mg_random.h)
//   mu = mean(xn), r = 1 / sqrt(mean((xn - mu)^2) + eps)
//   y  = (xn - mu) r w + b
// Backward, with dy the gradient of y and dres that of xn from its other use,
// h = (xn - mu) r and g = dy w:
//   dxn = r (g - mean(g) - h mean(g h)) + dres,  ddelta = keep(delta) dxn / (1 - p)
//   dw  = sum over rows of dy h,  db = sum over rows of dy
//
// A row belongs to one wave up to 1024 columns (16 bytes of fp32 per lane and step), else to a workgroup of 256
// threads, and stays in registers between its passes: the variance is that of the centred values, not a difference of
// two sums. How many steps a row of D has is known at compile time, and all but the last ones are whole, so that they
// carry no masks (with a mask per element a row's masks alone overflowed the scalar registers: 134 us for the forward
// below, against 76). Any D: the loads are 16 bytes wide at whatever alignment the rows have (the memory pipe takes
// them), and the last vector of a row is done element by element.
// The weight's gradients: lanes sum over their rows, a workgroup's lanes in LDS, its sum goes to a partial row, and a
// second kernel adds the partial rows in order. The backward's grid is what the device holds at once, 1024 workgroups
// (768: 3% slower at D 1024, as fast at D 2048).
//
// Bound by memory. fp32 stream, bf16 branch, N 16376 D 1024: forward 42 us (4.7 TB/s), backward 45 us (5.9), partial
// rows 5 us; N 16380 D 2048 with dropout: 76 us (5.3), 104 us (5.2).

#include <algorithm>

#include "mg_random.h"
#include "mg_vec.h"

namespace mg {
namespace layernorm {

constexpr int kThreads = 256;

// The sums of (a, b) over the threads of a row; every thread gets them
template <int TPR>
__device__ __forceinline__ void row_sum(float& a, float& b, float2* red) {
  a = wave_sum(a), b = wave_sum(b);
  if constexpr (TPR > 64) {
    __syncthreads();
    if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = make_float2(a, b);
    __syncthreads();
    a = (red[0].x + red[1].x) + (red[2].x + red[3].x);
    b = (red[0].y + red[1].y) + (red[2].y + red[3].y);
  }
}

// The first row of this wave (of this workgroup, where a row has more waves than one)
template <int TPR>
__device__ __forceinline__ int64_t first_row() {
  return static_cast<int64_t>(blockIdx.x) * (kThreads / TPR) + (TPR == 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x / 64) : 0);
}

__device__ __forceinline__ void drop4(f4& v, uint64_t e, bool even, const Drop& d, uint64_t key) {
  uint32_t w[4];
  if (even)
    drop_words<true>(e, d.offset, key, w);
  else
    drop_words<false>(e, d.offset, key, w);
#pragma unroll
  for (int j = 0; j < 4; ++j) v.v[j] = w[j] >= d.threshold ? v.v[j] * d.scale : 0.0f;
}

struct Fwd {
  const void *x, *delta;
  const float *w, *b;
  float* x_out;
  void* y;
  float *mean, *rstd;
  int64_t N;
  int D;
  float eps;
  Drop drop;
};

template <typename Tx, typename Td, typename Ty, int TPR, int STEPS, int WHOLE>
__global__ __launch_bounds__(kThreads) void fwd_kernel(Fwd a) {
  __shared__ float2 red[4];
  constexpr int kRows = kThreads / TPR;
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.D);
  const auto left = [&](int i, int c) { return i < WHOLE ? 4 : a.D - c; };
  const bool even = a.D % 4 == 0, drop = a.delta && a.drop.threshold;
  const uint64_t key = drop ? a.drop.key() : 0;
  for (int64_t row = first_row<TPR>(); row < a.N; row += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t base = row * a.D;
    f4 v[STEPS];
    float s = 0.0f, ss = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      v[i] = load4(static_cast<const Tx*>(a.x) + base + c, left(i, c));
    }
    if (a.delta) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        const int c = 4 * (t + TPR * i);
        f4 d = load4(static_cast<const Td*>(a.delta) + base + c, left(i, c));
        if (drop && left(i, c) > 0) drop4(d, static_cast<uint64_t>(base + c), even, a.drop, key);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[i].v[j] += d.v[j];
      }
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[i].v[j];  // (0 past the row)
      if (a.delta) store4(a.x_out + base + c, v[i], left(i, c));
    }
    row_sum<TPR>(s, none, red);
    const float mu = s * inv;
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float d = v[i].v[j] - mu;
        v[i].v[j] = d;
        ss += j < left(i, 4 * (t + TPR * i)) ? d * d : 0.0f;
      }
    row_sum<TPR>(ss, none, red);
    const float r = 1.0f / sqrtf(ss * inv + a.eps);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      const f4 w = load4(a.w + c, left(i, c));
      f4 b = io4<float>::fill(0.0f), o;
      if (a.b) b = load4(a.b + c, left(i, c));
#pragma unroll
      for (int j = 0; j < 4; ++j) o.v[j] = v[i].v[j] * r * w.v[j] + b.v[j];
      store4(static_cast<Ty*>(a.y) + base + c, o, left(i, c));
    }
    if (t == 0 && a.mean) a.mean[row] = mu, a.rstd[row] = r;
  }
}

struct Bwd {
  const void* xn;
  const float *w, *mean, *rstd;
  const void* dy;
  const float* dres;
  void *dx, *ddelta;
  float* part;  // [workgroups][2][D]
  int64_t N;
  int D;
  Drop drop;
};

template <typename Tx, typename Tg, typename Td, int TPR, int STEPS, int WHOLE>
__global__ __launch_bounds__(kThreads, TPR == 64 || STEPS <= 2 ? 4 : STEPS <= 4 ? 2 : 1) void bwd_kernel(Bwd a) {
  __shared__ float2 red[4];
  __shared__ f4 s_sum[2][4][64];
  constexpr int kRows = kThreads / TPR;
  const int t = threadIdx.x % TPR;
  const float inv = 1.0f / static_cast<float>(a.D);
  const auto left = [&](int i, int c) { return i < WHOLE ? 4 : a.D - c; };
  const bool even = a.D % 4 == 0, drop = a.ddelta && a.drop.threshold;
  const uint64_t key = drop ? a.drop.key() : 0;
  f4 dw[STEPS], db[STEPS];
#pragma unroll
  for (int i = 0; i < STEPS; ++i) dw[i] = db[i] = io4<float>::fill(0.0f);
  for (int64_t row = first_row<TPR>(); row < a.N; row += static_cast<int64_t>(gridDim.x) * kRows) {
    const int64_t base = row * a.D;
    const float mu = a.mean[row], r = a.rstd[row];
    f4 h[STEPS], g[STEPS], d[STEPS];
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      h[i] = load4(static_cast<const Tx*>(a.xn) + base + c, left(i, c));
      g[i] = load4(static_cast<const Tg*>(a.dy) + base + c, left(i, c));  // (0 past the row: adds nothing below)
      d[i] = io4<float>::fill(0.0f);
      if (a.dres) d[i] = load4(a.dres + base + c, left(i, c));
    }
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      const f4 w = load4(a.w + c, left(i, c));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        h[i].v[j] = (h[i].v[j] - mu) * r;
        dw[i].v[j] += g[i].v[j] * h[i].v[j];
        db[i].v[j] += g[i].v[j];
        g[i].v[j] *= w.v[j];
        s1 += g[i].v[j];
        s2 += g[i].v[j] * h[i].v[j];
      }
    }
    row_sum<TPR>(s1, s2, red);
    s1 *= inv, s2 *= inv;
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      const int c = 4 * (t + TPR * i);
      if (left(i, c) > 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) d[i].v[j] += r * (g[i].v[j] - s1 - h[i].v[j] * s2);
        if (a.dx) store4(static_cast<Tx*>(a.dx) + base + c, d[i], left(i, c));
        if (a.ddelta) {
          if (drop) drop4(d[i], static_cast<uint64_t>(base + c), even, a.drop, key);
          store4(static_cast<Td*>(a.ddelta) + base + c, d[i], left(i, c));
        }
      }
    }
  }
  float* part = a.part + static_cast<int64_t>(blockIdx.x) * 2 * a.D;
#pragma unroll
  for (int i = 0; i < STEPS; ++i) {
    const int c = 4 * (t + TPR * i);
    if constexpr (TPR > 64) {
      store4(part + c, dw[i], left(i, c));
      store4(part + a.D + c, db[i], left(i, c));
    } else {
      const int wave = threadIdx.x / 64;
      __syncthreads();
      s_sum[0][wave][t] = dw[i];
      s_sum[1][wave][t] = db[i];
      __syncthreads();
      if (wave < 2) {
        f4 x = s_sum[wave][0][t];
#pragma unroll
        for (int q = 1; q < 4; ++q)
#pragma unroll
          for (int j = 0; j < 4; ++j) x.v[j] += s_sum[wave][q][t].v[j];
        store4(part + wave * a.D + c, x, left(i, c));
      }
    }
  }
}

// [P][n] partial rows to n sums: 16 columns per workgroup, four to a thread, 64 threads' rows of each
__global__ __launch_bounds__(256) void sum_parts_kernel(const float* __restrict__ part, int P, int n, int D,
                                                        float* __restrict__ dw, float* __restrict__ db) {
  __shared__ float s[64][17];
  const int c = 16 * blockIdx.x + 4 * (threadIdx.x % 4), g = threadIdx.x / 4;
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
  if (q == 0 && e < n) {
    if (e < D) {
      if (dw) dw[e] = sum;
    } else if (db) {
      db[e - D] = sum;
    }
  }
}

constexpr int kMaxD = 16384;

constexpr int kWaveD = 1024;  // rows up to here belong to one wave

// Workgroups. A backward's are as many as the device holds at once, so that the partial rows stay few
inline int grid_for(int64_t N, int D, int64_t most) {
  const int64_t per = D <= kWaveD ? 4 : 1;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((N + per - 1) / per, most)));
}
constexpr int kFwdGrid = 65536, kBwdGrid = 1024;

// Threads per row, steps of four values per thread, and how many of the steps lie within the row for
// every D that takes them
#define MG_LN_SIZES(GO)                                                                                          \
  if (D <= 256) { GO(64, 1, 0) } else if (D <= 512) { GO(64, 2, 1) } else if (D <= 768) { GO(64, 3, 2) }          \
  else if (D <= 1024) { GO(64, 4, 3) } else if (D <= 2048) { GO(256, 2, 1) } else if (D <= 4096) { GO(256, 4, 2) } \
  else if (D <= 8192) { GO(256, 8, 4) } else { GO(256, 16, 8) }

template <typename Tx, typename Td, typename Ty>
int launch_fwd(const Fwd& a, hipStream_t st) {
  const int D = a.D, grid = grid_for(a.N, D, kFwdGrid);
#define GO(T, S, F) hipLaunchKernelGGL((fwd_kernel<Tx, Td, Ty, T, S, F>), dim3(grid), dim3(kThreads), 0, st, a);
  MG_LN_SIZES(GO)
#undef GO
  return check_launch("mg_layernorm_fwd");
}

template <typename Tx, typename Tg, typename Td>
int launch_bwd(const Bwd& a, float* dw, float* db, hipStream_t st) {
  const int D = a.D, grid = grid_for(a.N, D, kBwdGrid);
#define GO(T, S, F) hipLaunchKernelGGL((bwd_kernel<Tx, Tg, Td, T, S, F>), dim3(grid), dim3(kThreads), 0, st, a);
  MG_LN_SIZES(GO)
#undef GO
  if (dw || db)
    hipLaunchKernelGGL(sum_parts_kernel, dim3((2 * D + 15) / 16), dim3(256), 0, st, a.part, grid, 2 * D, D, dw, db);
  return check_launch("mg_layernorm_bwd");
}

inline int check_dt(const char* fn, const char* name, int dt) {
  return dt == MG_F32 || dt == MG_BF16 ? MG_OK : fail(MG_ERR_DTYPE, "%s: %s dtype %d unsupported", fn, name, dt);
}
inline int check_p(const char* fn, const char* name, const void* p, int dt, bool required) {
  if (!p) return required ? fail(MG_ERR_ARG, "%s: %s is NULL", fn, name) : MG_OK;
  if (!aligned(p, dt == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: %s misaligned", fn, name);
  return MG_OK;
}
inline int check_shape(const char* fn, int64_t N, int D, double p, const int64_t* seed_p) {
  if (N < 1 || D < 1 || D > kMaxD) return fail(MG_ERR_ARG, "%s: N=%lld must be >= 1 and D=%d in [1, %d]", fn, (long long)N, D, kMaxD);
  if (!(p >= 0.0 && p < 1.0)) return fail(MG_ERR_ARG, "%s: p=%g must be in [0, 1)", fn, p);
  if (!aligned(seed_p, 8)) return fail(MG_ERR_ARG, "%s: seed_p misaligned", fn);
  return MG_OK;
}
inline Drop drop_of(double p, uint64_t seed, const int64_t* seed_p, uint64_t offset) {
  return {seed, offset, seed_p, static_cast<uint32_t>(p * 4294967296.0), static_cast<float>(1.0 / (1.0 - p))};
}

}  // namespace layernorm
}  // namespace mg

using namespace mg;

extern "C" int mg_layernorm_fwd(int x_dtype, const void* x, int delta_dtype, const void* delta, const float* w, const float* b,
                                float* x_out, int y_dtype, void* y, float* mean, float* rstd, int64_t N, int D, float eps,
                                double p, uint64_t seed, const int64_t* seed_p, uint64_t offset, void* stream) {
  using namespace layernorm;
  const char* fn = "mg_layernorm_fwd";
  int rc;
  if ((rc = check_shape(fn, N, D, p, seed_p)) || (rc = check_dt(fn, "x", x_dtype)) || (rc = check_dt(fn, "y", y_dtype)) ||
      (rc = check_p(fn, "x", x, x_dtype, true)) || (rc = check_p(fn, "w", w, MG_F32, true)) ||
      (rc = check_p(fn, "b", b, MG_F32, false)) || (rc = check_p(fn, "y", y, y_dtype, true)) ||
      (rc = check_p(fn, "mean", mean, MG_F32, false)) || (rc = check_p(fn, "rstd", rstd, MG_F32, mean != nullptr)))
    return rc;
  if (delta) {
    if ((rc = check_dt(fn, "delta", delta_dtype)) || (rc = check_p(fn, "delta", delta, delta_dtype, true)) ||
        (rc = check_p(fn, "x_out", x_out, MG_F32, true)))
      return rc;
    if (x_dtype != MG_F32) return fail(MG_ERR_DTYPE, "%s: a stream that a branch joins is fp32", fn);
  }
  const Fwd a = {x, delta, w, b, x_out, y, mean, rstd, N, D, eps, drop_of(p, seed, seed_p, offset)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == MG_BF16)
    return y_dtype == MG_BF16 ? launch_fwd<bf16_t, bf16_t, bf16_t>(a, st) : launch_fwd<bf16_t, bf16_t, float>(a, st);
  if (delta && delta_dtype == MG_BF16)
    return y_dtype == MG_BF16 ? launch_fwd<float, bf16_t, bf16_t>(a, st) : launch_fwd<float, bf16_t, float>(a, st);
  return y_dtype == MG_BF16 ? launch_fwd<float, float, bf16_t>(a, st) : launch_fwd<float, float, float>(a, st);
}

extern "C" size_t mg_layernorm_bwd_workspace_bytes(int64_t N, int D) {
  if (N < 1 || D < 1 || D > layernorm::kMaxD) return 0;
  return static_cast<size_t>(layernorm::grid_for(N, D, layernorm::kBwdGrid)) * 2 * D * sizeof(float);
}

extern "C" int mg_layernorm_bwd(int x_dtype, const void* xn, const float* w, const float* mean, const float* rstd, int dy_dtype,
                                const void* dy, const float* dres, void* dx, int ddelta_dtype, void* ddelta, float* dw, float* db,
                                int64_t N, int D, double p, uint64_t seed, const int64_t* seed_p, uint64_t offset,
                                void* workspace, size_t workspace_bytes, void* stream) {
  using namespace layernorm;
  const char* fn = "mg_layernorm_bwd";
  int rc;
  if ((rc = check_shape(fn, N, D, p, seed_p)) || (rc = check_dt(fn, "xn", x_dtype)) || (rc = check_dt(fn, "dy", dy_dtype)) ||
      (rc = check_p(fn, "xn", xn, x_dtype, true)) || (rc = check_p(fn, "w", w, MG_F32, true)) ||
      (rc = check_p(fn, "mean", mean, MG_F32, true)) || (rc = check_p(fn, "rstd", rstd, MG_F32, true)) ||
      (rc = check_p(fn, "dy", dy, dy_dtype, true)) || (rc = check_p(fn, "dres", dres, MG_F32, false)) ||
      (rc = check_p(fn, "dx", dx, x_dtype, false)) || (rc = check_p(fn, "dw", dw, MG_F32, false)) ||
      (rc = check_p(fn, "db", db, MG_F32, false)))
    return rc;
  if (ddelta) {
    if ((rc = check_dt(fn, "ddelta", ddelta_dtype)) || (rc = check_p(fn, "ddelta", ddelta, ddelta_dtype, true))) return rc;
    if (x_dtype != MG_F32) return fail(MG_ERR_DTYPE, "%s: a stream that a branch joins is fp32", fn);
  }
  const size_t need = mg_layernorm_bwd_workspace_bytes(N, D);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or misaligned)", fn, workspace_bytes, need);
  const Bwd a = {xn, w, mean, rstd, dy, dres, dx, ddelta, static_cast<float*>(workspace), N, D, drop_of(p, seed, seed_p, offset)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == MG_BF16)
    return dy_dtype == MG_BF16 ? launch_bwd<bf16_t, bf16_t, bf16_t>(a, dw, db, st) : launch_bwd<bf16_t, float, bf16_t>(a, dw, db, st);
  if (ddelta && ddelta_dtype == MG_BF16)
    return dy_dtype == MG_BF16 ? launch_bwd<float, bf16_t, bf16_t>(a, dw, db, st) : launch_bwd<float, float, bf16_t>(a, dw, db, st);
  return dy_dtype == MG_BF16 ? launch_bwd<float, bf16_t, float>(a, dw, db, st) : launch_bwd<float, float, float>(a, dw, db, st);
}
