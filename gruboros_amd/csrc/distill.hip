// Distillation from a teacher's top logits, with the cross-entropy against labels beside it: the loss and its gradient
// in one pass over the logits, for gfx950 (ce.hip has the cross-entropy alone, for small vocabularies).
// Per row of V logits z, with K entries (id_k, t_k) of the teacher and a temperature T:
//   p = softmax(t / T) over the entries that count, q = softmax(z / T),  KL = sum_k p_k (log p_k - log q_id_k)
//   CE = -log softmax(z)_label
//   loss = alpha T^2 mean(KL) + (1 - alpha) mean(CE)
//   dz = alpha T / n1 (q - sum_k p_k [id_k]) + (1 - alpha) / n2 (softmax(z) - [label])
// The means are over the n1 rows with an entry that counts (id in [0, V), t not -inf) and the n2 rows with a label in
// [0, V); a row that is in neither is not read and has a gradient of 0. An id that is listed twice counts twice.
//
// A workgroup takes a row and keeps it in registers, as loaded, from its maximum to its sums to its gradient: logits
// are read once and gradients written once. Rows of more than 64 registers to each of 1024 threads are read twice.
// Everything is in powers of two: with k = log2(e) / T a term is 2^((z - max z) k), in the sums and in the logarithms
// alike. (The difference first: with a product z k + b the rounding of b = -k max z overflows the power for logits of
// the type's lowest value.) The few places that an entry or the label changes are
// written again after the row, by the threads that hold the entries. Losses are summed in double, in a fixed order.
//
// A small kernel counts n1 and n2 first (a thread per row, which seldom reads past a row's first entry); the last adds
// the workgroups' losses.

#include <algorithm>

#include "mg_vec.h"

namespace mg {
namespace distill {

constexpr int kMaxTop = 512;
constexpr int kCountRows = 64, kCountWgs = 256, kRowWgs = 4096;

typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));

// 16 bytes of a row as loaded
template <typename T> struct Vec;
template <> struct Vec<bf16_t> {
  static constexpr int kN = 8;
  uint32_t w[4];
  __device__ __forceinline__ void load(const bf16_t* p) {
    const uint4 y = __builtin_bit_cast(uint4, *reinterpret_cast<const u16x8u*>(p));
    w[0] = y.x, w[1] = y.y, w[2] = y.z, w[3] = y.w;
  }
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = 0xff80ff80u; }  // -inf
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16); }
  __device__ __forceinline__ static void store(bf16_t* p, const float (&v)[kN]) {
    u16x8u x;
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = f32_to_bf16(v[j]);
    *reinterpret_cast<u16x8u*>(p) = x;
  }
};
template <> struct Vec<float> {
  static constexpr int kN = 4;
  float w[4];
  __device__ __forceinline__ void load(const float* p) {
    const f32x4u x = *reinterpret_cast<const f32x4u*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = x[j];
  }
  __device__ __forceinline__ void none() { w[0] = w[1] = w[2] = w[3] = -INFINITY; }
  __device__ __forceinline__ float get(int j) const { return w[j]; }
  __device__ __forceinline__ static void store(float* p, const float (&v)[kN]) {
    const f32x4u x = {v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4u*>(p) = x;
  }
};
// What was computed from v so far is not kept for later: v is all that stays in registers
template <typename T>
__device__ __forceinline__ void forget(Vec<T>& v) {
#pragma unroll
  for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(v.w[q]));
}
__device__ __forceinline__ float value(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ void put(bf16_t* p, float v) { *p = f32_to_bf16(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }

struct Args {
  const void* z;
  int64_t sb, st;
  int64_t T, N;
  int V, K;
  const void* ids;
  const void* top;
  const int64_t* labels;
  int wide, top_bf16;  // ids int64 (not int32); top bf16 (not fp32)
  int soft, hard;      // the parts of the loss that there are
  float alpha, temperature;
  void* dz;
  int* counts;      // [kCountWgs][2]
  double* losses;   // [workgroups][2]
  __device__ __forceinline__ int64_t id(int64_t i) const {
    return wide ? static_cast<const int64_t*>(ids)[i] : static_cast<const int32_t*>(ids)[i];
  }
  __device__ __forceinline__ float teacher(int64_t i) const {
    return top_bf16 ? bf16_to_f32(static_cast<const bf16_t*>(top)[i]) : static_cast<const float*>(top)[i];
  }
  __device__ __forceinline__ bool inside(int64_t v) const { return v >= 0 && v < V; }
  __device__ __forceinline__ bool counts_as(int64_t id, float t) const { return inside(id) && t != -INFINITY; }
};

// Rows that count, kCountRows at a time to a workgroup, a thread per row: its entries by eights, as few as it takes
__global__ __launch_bounds__(kCountRows) void count_kernel(Args a) {
  int n1 = 0, n2 = 0;
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * kCountRows + threadIdx.x; n < a.N; n += static_cast<int64_t>(gridDim.x) * kCountRows) {
    bool any = !a.soft;
    for (int k0 = 0; k0 < a.K && !any; k0 += 8) {
      int64_t id[8];
      float t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t i = n * a.K + std::min(k0 + j, a.K - 1);
        id[j] = a.id(i), t[j] = a.teacher(i);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) any |= a.counts_as(id[j], t[j]);
    }
    n1 += any;
    n2 += a.hard && a.inside(a.labels[n]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n1 += __shfl_xor(n1, o, 64), n2 += __shfl_xor(n2, o, 64);
  if (threadIdx.x == 0) a.counts[2 * blockIdx.x] = a.soft ? n1 : 0, a.counts[2 * blockIdx.x + 1] = n2;
}

// (n1, n2) by the first 256 threads of a workgroup; s is cleared, and everyone waits before and after
__device__ __forceinline__ void all_counts(const Args& a, int (&s)[2]) {
  const int64_t wgs = (a.N + kCountRows - 1) / kCountRows;
  const int g = static_cast<int>(std::min<int64_t>(wgs, kCountWgs));
  if (threadIdx.x < 2) s[threadIdx.x] = 0;
  __syncthreads();
  if (threadIdx.x < g) {
    const int2 c = reinterpret_cast<const int2*>(a.counts)[threadIdx.x];
    atomicAdd(&s[0], c.x);
    atomicAdd(&s[1], c.y);
  }
  __syncthreads();
}

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

// Over the NT threads of a workgroup; every thread gets them
template <int NT, int M>
__device__ __forceinline__ void all_max(float (&v)[M], float (&red)[M][NT / 64]) {
#pragma unroll
  for (int i = 0; i < M; ++i) v[i] = wave_max(v[i]);
  __syncthreads();
  if (threadIdx.x % 64 == 0)
#pragma unroll
    for (int i = 0; i < M; ++i) red[i][threadIdx.x / 64] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < M; ++i) {
    v[i] = red[i][0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) v[i] = fmaxf(v[i], red[i][w]);
  }
}
template <int NT, int M>
__device__ __forceinline__ void all_sum(float (&v)[M], float (&red)[M][NT / 64]) {
#pragma unroll
  for (int i = 0; i < M; ++i) v[i] = wave_sum(v[i]);
  __syncthreads();
  if (threadIdx.x % 64 == 0)
#pragma unroll
    for (int i = 0; i < M; ++i) red[i][threadIdx.x / 64] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < M; ++i) {
    v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v[i] += red[i][w];
  }
}

// S vectors of a row to each of NT threads, and one of the values behind the last whole vector to the first few;
// S = 0: rows of any length, read twice. A row that counts for one part alone has a share of 0 of the other's
// gradient.
template <typename T, int NT, int S, bool kHard>
__global__ __launch_bounds__(NT) void rows_kernel(Args a) {
  using V16 = Vec<T>;
  constexpr int kN = V16::kN, kEntries = (kMaxTop + NT - 1) / NT;
  constexpr float kLn2 = 0.6931471805599453f;
  __shared__ float s_red[4][NT / 64], s_redm[3][NT / 64];
  __shared__ int s_count[2], s_id[kMaxTop];
  __shared__ float s_p[kMaxTop];
  const int tid = threadIdx.x;
  const int whole = a.V / kN * kN, last = whole + tid;  // (last: this thread's value behind them, if it has one)
  const uint32_t whole_bytes = static_cast<uint32_t>(whole) * sizeof(T);
  // a thread's first byte of a row, computed anew wherever it is needed (kept from row to row, the places of all S
  // vectors take two registers each)
  const auto here = [](uint32_t t) {
    asm volatile("" : "+v"(t));
    return t * 16;
  };
  all_counts(a, s_count);
  const float w1 = s_count[0] ? a.alpha * a.temperature / static_cast<float>(s_count[0]) : 0.0f;
  const float w2 = s_count[1] ? (1.0f - a.alpha) / static_cast<float>(s_count[1]) : 0.0f;
  const float k1 = kLog2e / a.temperature, k2 = kLog2e;
  double l1 = 0.0, l2 = 0.0;
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    const T* z = static_cast<const T*>(a.z) + n / a.T * a.sb + n % a.T * a.st;
    T* dz = a.dz ? static_cast<T*>(a.dz) + n * a.V : nullptr;
    const int64_t label = kHard ? a.labels[n] : -1;
    const bool told = kHard && a.inside(label);
    V16 x[S ? S : 1];
    if constexpr (S > 0) {
      const uint32_t c0 = here(tid);
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const uint32_t c = c0 + s * (NT * 16);
        if (c < whole_bytes)
          x[s].load(reinterpret_cast<const T*>(reinterpret_cast<const char*>(z) + c));
        else
          x[s].none();
      }
    }
    const float xl = last < a.V ? value(z + last) : -INFINITY;
    // the teacher's entries of this thread: at `id` the logit `at`, u = log2 of the unnormalised probability
    int id[kEntries];
    float u[kEntries], at[kEntries];
    float most[3] = {xl, -INFINITY, 0.0f};  // of the row, of the teacher, whether an entry counts
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int k = tid + i * NT;
      id[i] = -1, u[i] = 0.0f, at[i] = 0.0f;
      if (a.soft && k < a.K) {
        const int64_t v = a.id(n * a.K + k);
        const float t = a.teacher(n * a.K + k);
        if (a.counts_as(v, t)) {
          id[i] = static_cast<int>(v), u[i] = t * k1, most[2] = 1.0f;
          most[1] = fmaxf(most[1], u[i]);
          at[i] = value(z + v);
        }
      }
    }
    const float zl = told ? value(z + label) : 0.0f;
    // f(vector, where it goes) over the row's whole vectors
    const auto each = [&](auto&& f) {
      if constexpr (S > 0) {
        const uint32_t c0 = here(tid);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const uint32_t c = c0 + s * (NT * 16);
          forget(x[s]);
          f(x[s], c < whole_bytes ? reinterpret_cast<T*>(reinterpret_cast<char*>(dz) + c) : nullptr);
          __builtin_amdgcn_sched_barrier(0);  // (or the vectors' values are in registers all at once)
        }
      } else {
        for (int c = tid * kN; c < whole; c += NT * kN) {
          x[0].load(z + c);
          f(x[0], dz + c);
        }
      }
    };
    each([&](const V16& v, T*) {
#pragma unroll
      for (int j = 0; j < kN; ++j) most[0] = fmaxf(most[0], v.get(j));
    });
    all_max<NT>(most, s_redm);
    const bool taught = most[2] != 0.0f;
    if (!taught && !told) {
      if (dz) {
        const float none[kN] = {};
        for (int c = tid * kN; c < whole; c += NT * kN) V16::store(dz + c, none);
        if (last < a.V) put(dz + last, 0.0f);
      }
      continue;
    }
    const float zm = most[0];
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // of 2^((z - zm) k1), of 2^((z - zm) k2), of the teacher's 2^u, of 2^u (u - log2 of the student's)
    const auto add = [&](float zj) {
      const float d = zj - zm;
      sum[0] += exp2_raw(d * k1);
      if constexpr (kHard) sum[1] += exp2_raw(d * k2);
    };
    each([&](const V16& v, T*) {
#pragma unroll
      for (int j = 0; j < kN; ++j) add(v.get(j));
    });
    add(xl);
    float p[kEntries];
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      p[i] = 0.0f;
      if (id[i] >= 0) {
        u[i] -= most[1];
        p[i] = exp2_raw(u[i]);
        sum[2] += p[i];
        if (p[i] != 0.0f) sum[3] += p[i] * (u[i] - (at[i] - zm) * k1);
      }
    }
    all_sum<NT>(sum, s_red);
    if (tid == 0) {
      if (taught) l1 += kLn2 * (sum[3] / sum[2] - log2f(sum[2]) + log2f(sum[0]));
      if (told) l2 += kLn2 * (log2f(sum[1]) - (zl - zm) * k2);
    }
    if (!dz) continue;
    const float c1 = taught ? w1 / sum[0] : 0.0f, c2 = told ? w2 / sum[1] : 0.0f;
    const float wp = taught ? w1 / sum[2] : 0.0f;
    const int entries = a.soft ? a.K : 0;
    const auto slope = [&](float zj) {
      const float e = zj - zm;
      float d = c1 * exp2_raw(e * k1);
      if constexpr (kHard) d = __builtin_fmaf(c2, exp2_raw(e * k2), d);
      return d;
    };
    each([&](const V16& v, T* to) {
      if (to) {
        float d[kN];
#pragma unroll
        for (int j = 0; j < kN; ++j) d[j] = slope(v.get(j));
        V16::store(to, d);
      }
    });
    if (last < a.V) put(dz + last, slope(xl));
    // the places of the entries and of the label, after the row
#pragma unroll
    for (int i = 0; i < kEntries; ++i)
      if (tid + i * NT < kMaxTop) s_id[tid + i * NT] = id[i], s_p[tid + i * NT] = p[i] * wp;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      if (id[i] < 0) continue;
      float all = told && id[i] == label ? w2 : 0.0f;
      bool first = true;
      for (int k = 0; k < entries; ++k) {
        const bool same = s_id[k] == id[i];
        all += same ? s_p[k] : 0.0f;
        first &= !(same && k < tid + i * NT);
      }
      if (first) put(dz + id[i], slope(at[i]) - all);
    }
    if (told && tid == NT - 1) {
      bool listed = false;
      for (int k = 0; k < entries; ++k) listed |= s_id[k] == label;
      if (!listed) put(dz + label, slope(zl) - w2);
    }
  }
  if (tid == 0) a.losses[2 * blockIdx.x] = l1, a.losses[2 * blockIdx.x + 1] = l2;
}

__global__ __launch_bounds__(1024) void loss_kernel(Args a, int wgs, float* loss) {
  __shared__ double s[1024][2];
  __shared__ int s_n[2];
  double l1 = 0.0, l2 = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < wgs; i += 1024) l1 += a.losses[2 * i], l2 += a.losses[2 * i + 1];
  s[threadIdx.x][0] = l1, s[threadIdx.x][1] = l2;
  all_counts(a, s_n);
  for (int o = 512; o > 0; o >>= 1) {
    if (threadIdx.x < o) s[threadIdx.x][0] += s[threadIdx.x + o][0], s[threadIdx.x][1] += s[threadIdx.x + o][1];
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    const double t = a.temperature, al = a.alpha;
    double l = 0.0;
    if (s_n[0]) l += al * t * t * s[0][0] / s_n[0];
    if (s_n[1]) l += (1.0 - al) * s[0][1] / s_n[1];
    *loss = static_cast<float>(l);
  }
}

// x *= *g in place; nothing where *g is 1
template <typename T>
__global__ __launch_bounds__(256) void scale_kernel(T* x, int64_t n, const float* __restrict__ g) {
  using V16 = Vec<T>;
  const float f = *g;
  if (f == 1.0f) return;
  const int64_t whole = n / V16::kN * V16::kN, t = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  for (int64_t i = t * V16::kN; i < whole; i += static_cast<int64_t>(gridDim.x) * 256 * V16::kN) {
    V16 v;
    v.load(x + i);
    float d[V16::kN];
#pragma unroll
    for (int j = 0; j < V16::kN; ++j) d[j] = v.get(j) * f;
    V16::store(x + i, d);
  }
  if (whole + t < n) put(x + whole + t, value(x + whole + t) * f);
}

inline int row_wgs(int64_t N) { return static_cast<int>(std::min<int64_t>(N, kRowWgs)); }

template <typename T, bool kHard>
void launch_rows(const Args& a, hipStream_t st) {
  const int64_t vecs = (a.V + int64_t(Vec<T>::kN) - 1) / Vec<T>::kN;
  const dim3 grid(row_wgs(a.N));
#define GO(NT, S) hipLaunchKernelGGL((rows_kernel<T, NT, S, kHard>), grid, dim3(NT), 0, st, a)
  if (vecs <= 256) GO(256, 1);
  else if (vecs <= 512) GO(256, 2);
  else if (vecs <= 1024) GO(256, 4);
  else if (vecs <= 2048) GO(256, 8);
  else if (vecs <= 4096) GO(512, 8);
  else if (vecs <= 8192) GO(1024, 8);
  else if (vecs <= 16384) GO(1024, 16);
  else GO(1024, 0);
#undef GO
}

}  // namespace distill
}  // namespace mg

using namespace mg;

extern "C" size_t mg_distill_workspace_bytes(int64_t N) {
  return N < 1 ? 0 : distill::kCountWgs * 2 * sizeof(int) + static_cast<size_t>(distill::row_wgs(N)) * 2 * sizeof(double);
}

extern "C" int mg_distill(int logits_dtype, const mg_seq* logits, int64_t B, int64_t T, int V, int id_bytes, const void* ids, int top_dtype,
                          const void* top, int K, const int64_t* labels, float temperature, float alpha, float* loss, void* dlogits,
                          void* workspace, size_t workspace_bytes, void* stream) {
  using namespace distill;
  const char* fn = "mg_distill";
  for (int dt : {logits_dtype, top_dtype})
    if (dt != MG_F32 && dt != MG_BF16) return fail(MG_ERR_DTYPE, "%s: dtype %d unsupported", fn, dt);
  if (id_bytes != 4 && id_bytes != 8) return fail(MG_ERR_DTYPE, "%s: ids of %d bytes", fn, id_bytes);
  if (B < 1 || T < 1 || B > INT32_MAX || T > INT32_MAX || V < 1 || V > (1 << 30) || K < 1 || K > kMaxTop || B * T > INT32_MAX)
    return fail(MG_ERR_ARG, "%s: B=%lld, T=%lld, V=%d, K=%d: at least 1, B T < 2^31, V <= 2^30, K <= %d", fn, (long long)B, (long long)T, V, K, kMaxTop);
  if (!(temperature >= 1e-4f && temperature <= 1e4f) || !(alpha >= 0.0f && alpha <= 1.0f))
    return fail(MG_ERR_ARG, "%s: temperature=%g must be in [1e-4, 1e4], alpha=%g in [0, 1]", fn, temperature, alpha);
  const int e = logits_dtype == MG_F32 ? 4 : 2;
  if (!logits || !logits->p || !aligned(logits->p, e) || logits->sb < 0 || logits->st < 0)
    return fail(MG_ERR_ARG, "%s: logits NULL, misaligned or with a negative stride", fn);
  if (!ids || !aligned(ids, id_bytes) || !top || !aligned(top, top_dtype == MG_F32 ? 4 : 2) || !aligned(labels, 8))
    return fail(MG_ERR_ARG, "%s: ids, top or labels NULL or misaligned", fn);
  if (!loss || !aligned(loss, 4) || !aligned(dlogits, e)) return fail(MG_ERR_ARG, "%s: loss NULL, or loss or dlogits misaligned", fn);
  const int64_t N = B * T;
  if (!workspace || workspace_bytes < mg_distill_workspace_bytes(N) || !aligned(workspace, 16))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or misaligned)", fn, workspace_bytes, mg_distill_workspace_bytes(N));
  Args a = {logits->p, logits->sb, logits->st, T, N, V, K, ids, top, labels, id_bytes == 8, top_dtype == MG_BF16, alpha > 0.0f,
            labels && alpha < 1.0f, alpha, temperature, dlogits, static_cast<int*>(workspace),
            reinterpret_cast<double*>(static_cast<char*>(workspace) + kCountWgs * 2 * sizeof(int))};
  hipStream_t st = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(count_kernel, dim3(std::min<int64_t>((N + kCountRows - 1) / kCountRows, kCountWgs)), dim3(kCountRows), 0, st, a);
  if (logits_dtype == MG_BF16)
    a.hard ? launch_rows<bf16_t, true>(a, st) : launch_rows<bf16_t, false>(a, st);
  else
    a.hard ? launch_rows<float, true>(a, st) : launch_rows<float, false>(a, st);
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(1024), 0, st, a, row_wgs(N), loss);
  return check_launch(fn);
}

extern "C" int mg_scale_inplace(int dtype, void* x, int64_t n, const float* factor, void* stream) {
  using namespace distill;
  const char* fn = "mg_scale_inplace";
  if (dtype != MG_F32 && dtype != MG_BF16) return fail(MG_ERR_DTYPE, "%s: dtype %d unsupported", fn, dtype);
  if (n < 1 || !x || !aligned(x, dtype == MG_F32 ? 4 : 2) || !factor || !aligned(factor, 4))
    return fail(MG_ERR_ARG, "%s: n=%lld must be at least 1, x and factor not NULL and aligned", fn, (long long)n);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const int per = 256 * (dtype == MG_F32 ? 4 : 8);
  const dim3 grid(std::min<int64_t>((n + per - 1) / per, 2048));
  if (dtype == MG_BF16)
    hipLaunchKernelGGL(scale_kernel<bf16_t>, grid, dim3(256), 0, st, static_cast<bf16_t*>(x), n, factor);
  else
    hipLaunchKernelGGL(scale_kernel<float>, grid, dim3(256), 0, st, static_cast<float*>(x), n, factor);
  return check_launch(fn);
}
