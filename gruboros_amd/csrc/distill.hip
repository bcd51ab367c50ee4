// Distillation from a teacher's top logits, with the cross-entropy against labels beside it: the loss and its gradient
// in one pass over the logits, for gfx950 (ce.hip has the cross-entropy alone, for small vocabularies).
// Per row of V logits z, with K entries (id_k, t_k) of the teacher and a temperature T:
//   p = softmax(t / T) over the entries that count, q = softmax(z / T),  KL = sum_k p_k (log p_k - log q_id_k)
//   CE = -log softmax(z)_label
//   loss = alpha T^2 mean(KL) + (1 - alpha) mean(CE)
//   dz = alpha T / n1 (q - sum_k p_k [id_k]) + (1 - alpha) / n2 (softmax(z) - [label])
// The means are over the n1 rows with an entry that counts (id in [0, V), t not -inf) and the n2 rows with a label in
// [0, V); what a row in neither holds does not matter, its gradient is 0. An id that is listed twice counts twice.
//
// A workgroup takes a row and keeps it in registers, as loaded, from its maximum to its sums to its gradient: logits
// are read once and gradients written once. Rows of more than 64 registers to each of 1024 threads (131072 values in
// bfloat16, 65536 in fp32) do not stay: they are read for their maximum, for their sums and for their gradient.
// Everything is in powers of two: with k = log2(e) / T a term is 2^((z - max z) k), in the sums and in the logarithms
// alike, of the student and of the teacher. (The difference first: with a product z k + b the rounding of b = -k max z
// overflows the power for logits of the type's lowest value.) The few places that an entry or the label changes are
// written again after the row, by the threads that hold the entries. Losses are summed in double, in a fixed order.
//
// A small kernel counts n1 and n2 first; the last adds the workgroups' losses.
//
// Bound by memory as long as a row's sums and another's loads overlap: with bfloat16, 16376 rows of 32000 (K 64, labels)
// take 455 us (2.1 GB, 4.6 TB/s; at a temperature without a power 30 us more), 2044 rows of 131071 (K 32), of which a CU
// holds one, 251 us (1.07 GB, 4.3 TB/s). Rows beyond the registers, 2044 of 151936 and of 262144 (K 64), whole calls: 395
// and 690 us, in fp32 128256 648 us, where a read and a write are 233, 402 and 393: the reads from memory again. At
// 131071 a CU's registers are full with one row, and memory waits while its sums are made; holding the beginning of the
// next row as well (4 to 8 of 16 vectors) costs registers that are missing elsewhere (278 to 310 us where 283 was the
// time without).

#include <algorithm>

#include "mg_vec.h"

namespace mg {
namespace distill {

constexpr int kMaxTop = 512;
constexpr int kCountRows = 32, kCountWgs = 256, kRowWgs = 6144;

// The teacher's part alone; with the labels': an exponential for each, or, at the temperatures 1, 2 and 4, that of the
// labels' as a power of the teacher's (e^z = (e^{z/T})^T).
constexpr int kSoft = 0, kBoth = 1, kT1 = 2, kT2 = 3, kT4 = 4;

// Entries that a workgroup has room for
constexpr int top_of(int nt) { return nt == 64 ? 64 : kMaxTop; }

constexpr bool ahead(int s) { return s >= 16; }

// Waves per SIMD that a kernel leaves room for
constexpr int waves_of(int nt, int s) { return s > 0 && s < 16 ? 6 : 4; }

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));

// 16 bytes of a row as loaded
template <typename T> struct Vec;
template <> struct Vec<bf16_t> {
  static constexpr int kN = 8;
  u32x4 w;
  __device__ __forceinline__ void load(const bf16_t* p) { w = __builtin_bit_cast(u32x4, *reinterpret_cast<const u16x8u*>(p)); }
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16); }
  __device__ __forceinline__ static void store(bf16_t* p, const float (&v)[kN]) {
    u16x8u x;
#pragma unroll
    for (int j = 0; j < kN; ++j) x[j] = f32_to_bf16(v[j]);
    __builtin_nontemporal_store(x, reinterpret_cast<u16x8u*>(p));
  }
};
template <> struct Vec<float> {
  static constexpr int kN = 4;
  u32x4 w;
  __device__ __forceinline__ void load(const float* p) { w = __builtin_bit_cast(u32x4, *reinterpret_cast<const f32x4u*>(p)); }
  __device__ __forceinline__ float get(int j) const { return __uint_as_float(w[j]); }
  __device__ __forceinline__ static void store(float* p, const float (&v)[kN]) {
    const f32x4u x = {v[0], v[1], v[2], v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4u*>(p));
  }
};
// What was computed from v so far is not kept for later: v is all that stays in registers
template <typename T>
__device__ __forceinline__ void forget(Vec<T>& v) {
  asm volatile("" : "+v"(v.w));
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

// Rows that count, kCountRows at a time to a workgroup: eight threads to a row, each reads every eighth entry
__global__ __launch_bounds__(8 * kCountRows) void count_kernel(Args a) {
  __shared__ int s[2];
  if (threadIdx.x < 2) s[threadIdx.x] = 0;
  __syncthreads();
  int n1 = 0, n2 = 0;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.x) * kCountRows; n0 < a.N; n0 += static_cast<int64_t>(gridDim.x) * kCountRows) {
    const int64_t n = std::min<int64_t>(n0 + threadIdx.x / 8, a.N - 1);
    const bool own = n == n0 + threadIdx.x / 8 && threadIdx.x % 8 == 0;
    bool any = false;
    if (a.soft)
      for (int k0 = threadIdx.x % 8; k0 < a.K; k0 += 64) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t i = n * a.K + std::min(k0 + 8 * j, a.K - 1);
          any |= a.counts_as(a.id(i), a.teacher(i));
        }
      }
    const bool row = (__ballot(any) >> (threadIdx.x % 64 / 8 * 8) & 0xff) != 0;
    n1 += own && row;
    n2 += own && a.hard && a.inside(a.labels[n]);
  }
  if (n1) atomicAdd(&s[0], n1);
  if (n2) atomicAdd(&s[1], n2);
  __syncthreads();
  if (threadIdx.x < 2) a.counts[2 * blockIdx.x + threadIdx.x] = s[threadIdx.x];
}

__host__ __device__ __forceinline__ int count_wgs(int64_t N) {
  return static_cast<int>(std::min<int64_t>((N + kCountRows - 1) / kCountRows, kCountWgs));
}
static_assert(kCountWgs == 256, "a thread of loss_kernel for each");

// (n1, n2), by the first wave (with counters in LDS that every thread adds to, 31000 rows of V 1001 take 61 us, not 52,
// 2044 of V 131071 264, not 259; 16376 of V 32000 with labels, whose workgroups then start apart, 473, not 480)
__device__ __forceinline__ void all_counts(const Args& a, int (&s)[2]) {
  const int g = count_wgs(a.N);
  if (threadIdx.x < 64) {
    int n1 = 0, n2 = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < g; i += 64) n1 += a.counts[2 * i], n2 += a.counts[2 * i + 1];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n1 += __shfl_xor(n1, o, 64), n2 += __shfl_xor(n2, o, 64);
    if (threadIdx.x == 0) s[0] = n1, s[1] = n2;
  }
  __syncthreads();
}

// The largest of a wave's lanes, in every lane (as wave_sum; a lane without a partner keeps its own)
__device__ __forceinline__ float wave_max(float x) {
  const auto most = [](float x, auto ctrl, auto rows) {
    const int y = __builtin_amdgcn_update_dpp(__float_as_int(x), __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 0xf, false);
    return fmaxf(x, __int_as_float(y));
  };
  x = most(x, int_c<0xb1>{}, int_c<0xf>{});
  x = most(x, int_c<0x4e>{}, int_c<0xf>{});
  x = most(x, int_c<0x141>{}, int_c<0xf>{});
  x = most(x, int_c<0x140>{}, int_c<0xf>{});
  x = most(x, int_c<0x142>{}, int_c<0xa>{});
  x = most(x, int_c<0x143>{}, int_c<0xc>{});
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Over the NT threads of a workgroup; every thread gets them. One wait each: a second use of the same `red` has to come
// after another wait of the workgroup.
// A value that is the same in all lanes, in a scalar register
__device__ __forceinline__ float uniform(float v) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))); }

template <int NT>
__device__ __forceinline__ float all_max(float v, float (&red)[NT / 64]) {
  v = wave_max(v);
  if (threadIdx.x % 64 == 0) red[threadIdx.x / 64] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < NT / 64; ++w) v = fmaxf(v, red[w]);
  return uniform(v);
}
template <int NT, int M>
__device__ __forceinline__ void all_sum(float (&v)[M], float (&red)[M][NT / 64]) {
#pragma unroll
  for (int i = 0; i < M; ++i) v[i] = wave_sum(v[i]);
  if (threadIdx.x % 64 == 0)
#pragma unroll
    for (int i = 0; i < M; ++i) red[i][threadIdx.x / 64] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < M; ++i) {
    v[i] = 0.0f;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) v[i] += red[i][w];
    v[i] = uniform(v[i]);
  }
}

// S vectors of a row to each of NT threads, and one of the values before and behind them to the first few; S = 0: rows
// of any length, read three times (twice without a gradient). The vectors begin where the row's gradient, which is
// dense, has a multiple of 16 bytes (with all rows' vectors from their first values, V 50001 took 844 us where V 50000
// took 723, 16376 rows). A row that counts for one part alone has a share of 0 of the other's gradient.
// After a row's gradient (where a row has 16 vectors to a thread and few workgroups share a CU: while it is written,
// each vector's registers in turn) the next row is loaded, and its entries before that, so that a row begins with all
// of its loads under way; what is loaded early stays as it comes until it is needed, or the wait for it would come
// early too. The last row's successor is itself (its first vectors, for all S). What the entries are made into waits
// in LDS. Up to 64 entries are the first wave's business alone.
template <typename T, int NT, int S, int kMode>
__global__ __launch_bounds__(NT, waves_of(NT, S)) void rows_kernel(Args a) {
  constexpr bool kHard = kMode != kSoft, kAhead = ahead(S);
  using V16 = Vec<T>;
  constexpr int kN = V16::kN, kTop = top_of(NT), kEntries = (kTop + NT - 1) / NT;
  constexpr float kLn2 = 0.6931471805599453f, kSmall = 0x1p-24f;
  __shared__ float s_max[NT / 64], s_teacher[NT / 64], s_sum[kHard ? 2 : 1][NT / 64], s_teach[2][NT / 64];
  __shared__ int s_count[2], s_any[NT / 64], s_mine[NT / 64];
  __shared__ double s_loss[2];
  // of the entries: id (-1: none), unnormalised probability; of those that are the first of their id the place (else
  // -1), the logit there and what the gradient there has beyond the student's
  __shared__ int s_id[kTop], s_place[kTop];
  __shared__ float s_p[kTop], s_at[kTop], s_put[kTop];
  const int tid = threadIdx.x;
  // of row n: the values before the vectors, the values in vectors and this thread's value outside of them, if it has one
  const auto head_of = [&](int64_t n) {
    const uint32_t off = static_cast<uint32_t>(n) * static_cast<uint32_t>(a.V) % kN;
    return std::min<int>(off ? kN - off : 0, a.V);
  };
  const auto whole_of = [&](int head) { return (a.V - head) / kN * kN; };
  const auto own_of = [&](int head) { return tid < head ? tid : whole_of(head) + tid; };
  // a thread's first byte of a row, computed anew wherever it is needed (kept from row to row, the places of all S
  // vectors take two registers each)
  const auto here = [](uint32_t t) {
    asm volatile("" : "+v"(t));
    return t * 16;
  };
  const auto at_byte = [](auto* p, uint32_t c) {
    using C = std::conditional_t<std::is_const_v<std::remove_pointer_t<decltype(p)>>, const char, char>;
    return reinterpret_cast<decltype(p)>(reinterpret_cast<C*>(p) + c);
  };
  const auto row_of = [&](int64_t b, int64_t t) { return static_cast<const T*>(a.z) + b * a.sb + t * a.st; };
  const int entries = a.soft ? a.K : 0;
  const bool narrow = kTop == 64 || a.K <= 64;
  all_counts(a, s_count);
  const float w1 = uniform(s_count[0] ? a.alpha * a.temperature / static_cast<float>(s_count[0]) : 0.0f);
  const float w2 = uniform(s_count[1] ? (1.0f - a.alpha) / static_cast<float>(s_count[1]) : 0.0f);
  const float k1 = uniform(kLog2e / a.temperature), k2 = kLog2e;
  if (tid < 2) s_loss[tid] = 0.0;  // (the first thread's)

  V16 x[S ? S : 1];
  // this thread's entries, as loaded, then their ids; the logits there, at the label (-1: none) and beside the vectors
  uint32_t raw_lo[kEntries], raw_hi[kEntries], raw_t[kEntries];
  int id[kEntries], label = -1;
  T at[kEntries], zl, xl;
  int64_t raw_label = -1;
  bool twice;  // an id of this wave's entries may be listed twice
  const auto fetch_entries = [&](int64_t n) {
    if (entries) {
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        const int64_t k = n * a.K + std::min(tid + i * NT, entries - 1);
        if (a.wide) {
          const uint2 v = static_cast<const uint2*>(a.ids)[k];
          raw_lo[i] = v.x, raw_hi[i] = v.y;
        } else {
          raw_lo[i] = static_cast<const uint32_t*>(a.ids)[k];
        }
        raw_t[i] = a.top_bf16 ? static_cast<const uint16_t*>(a.top)[k] : static_cast<const uint32_t*>(a.top)[k];
      }
    }
    if (kHard) raw_label = a.labels[n];
  };
  const auto teacher = [&](int i) { return __uint_as_float(a.top_bf16 ? raw_t[i] << 16 : raw_t[i]); };
  const auto fetch_places = [&](const T* z, int head) {
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      id[i] = -1;
      if (tid + i * NT < entries) {
        const int64_t v = a.wide ? static_cast<int64_t>(static_cast<uint64_t>(raw_hi[i]) << 32 | raw_lo[i]) : static_cast<int32_t>(raw_lo[i]);
        if (a.counts_as(v, teacher(i))) id[i] = static_cast<int>(v);
      }
      at[i] = z[std::max(id[i], 0)];
    }
    if (kHard) {
      label = a.inside(raw_label) ? static_cast<int>(raw_label) : -1;
      zl = z[std::max(label, 0)];
    }
    xl = z[std::min(own_of(head), a.V - 1)];
    twice = !narrow;
    if (narrow && tid < 64) {  // (while the loads are under way; every entry that is none differs from all)
      const int own = id[0] >= 0 ? id[0] : -1 - tid;
      uint64_t same = 0;
      for (int k = 0; k < entries; ++k) {
        const uint64_t m = __ballot(own == __builtin_amdgcn_readlane(own, k));
        same |= m & (m - 1);
      }
      twice = same != 0;
    }
  };
  // a vector that the row does not have is its last one
  const auto fetch = [&](V16& v, const T* z, uint32_t c, uint32_t whole_bytes) { v.load(at_byte(z, std::min(c, whole_bytes - 16))); };
  int64_t row_b = blockIdx.x / a.T, row_t = blockIdx.x % a.T;
  const int64_t next_b = gridDim.x / a.T, next_t = gridDim.x % a.T;
  const T* z = row_of(row_b, row_t);
  const auto fetch_row = [&](const T* z, int head, uint32_t step) {
    if constexpr (S > 0) {
      const uint32_t c0 = here(tid), bytes = whole_of(head) * static_cast<uint32_t>(sizeof(T));
#pragma unroll
      for (int s = 0; s < S; ++s) fetch(x[s], z + head, c0 + s * step, bytes);
    }
  };
  fetch_entries(blockIdx.x);
  int head = head_of(blockIdx.x);
  fetch_row(z, head, NT * 16);
  fetch_places(z, head);
  for (int64_t n = blockIdx.x; n < a.N; n += gridDim.x) {
    T* dz = a.dz ? static_cast<T*>(a.dz) + n * a.V : nullptr;
    const bool more_rows = n + gridDim.x < a.N, told = kHard && label >= 0;
    const int64_t n_next = more_rows ? n + gridDim.x : n;
    if (more_rows) {
      row_b += next_b, row_t += next_t;
      if (row_t >= a.T) row_t -= a.T, ++row_b;
    }
    const T* z_next = row_of(row_b, row_t);
    const int head_next = head_of(n_next), whole = whole_of(head), own = own_of(head);
    const uint32_t whole_bytes = static_cast<uint32_t>(whole) * sizeof(T);
    const uint32_t next_bytes = static_cast<uint32_t>(whole_of(head_next)) * sizeof(T);
    const uint32_t step = more_rows ? NT * 16 : 0;
    // f(vector, its first byte) over the row's whole vectors; `then`: after each of the S, with its number
    const auto each = [&](auto&& f, auto&& then) {
      if constexpr (S > 0) {
        const uint32_t c0 = here(tid);
#pragma unroll
        for (int s = 0; s < S; ++s) {
          const uint32_t c = c0 + s * (NT * 16);
          forget(x[s]);
          if (c < whole_bytes) f(x[s], c);
          then(x[s], c0, s);
          __builtin_amdgcn_sched_barrier(0);  // (or the vectors' values are in registers all at once)
        }
      } else {
        for (int c = tid * kN; c < whole; c += NT * kN) {
          x[0].load(z + head + c);
          f(x[0], static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T)));
        }
      }
    };
    const auto nothing = [](V16&, uint32_t, int) {};

    float zm = -INFINITY, tm = -INFINITY;
    bool any = false;
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      if (id[i] >= 0) tm = fmaxf(tm, teacher(i)), any = true;
      if (tid + i * NT < entries) s_id[tid + i * NT] = id[i];
    }
    each([&](const V16& v, uint32_t) {
#pragma unroll
      for (int j = 0; j < kN; ++j) zm = fmaxf(zm, v.get(j));
    }, nothing);
    const float beside = own < a.V ? value(&xl) : -INFINITY;
    zm = fmaxf(zm, beside);
    if (const int one = __any(any); tid % 64 == 0) s_any[tid / 64] = one;
    zm = all_max<NT>(zm, s_max);
    bool taught = false;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) taught |= s_any[w] != 0;
    tm = narrow ? wave_max(tm) : all_max<NT>(tm, s_teacher);

    // the teacher's distribution: the sums of 2^u and of 2^u (u - log2 of the student's), the latter times kSmall: logits
    // of the type's lowest value, times k1 and 512 of them, stay finite
    float teach[2] = {};
    bool mine = false;  // the label is one of this thread's entries
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int k = tid + i * NT;
      if (k >= entries) continue;
      float p = 0.0f;
      if (id[i] >= 0) {
        const float u = (teacher(i) - tm) * k1, zk = value(&at[i]);
        p = exp2_raw(u);
        teach[0] += p;
        if (p != 0.0f) teach[1] += p * __builtin_fmaf(zm - zk, k1 * kSmall, u * kSmall);
        s_at[k] = zk;
        mine |= told && id[i] == label;
      }
      s_p[k] = p;
    }
    if constexpr (kHard)
      if (const int one = __any(mine); tid % 64 == 0) s_mine[tid / 64] = one;
    if (narrow)
      teach[0] = uniform(wave_sum(teach[0])), teach[1] = uniform(wave_sum(teach[1]));
    else
      all_sum<NT>(teach, s_teach);
    const float wp = taught ? w1 / teach[0] : 0.0f;
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int k = tid + i * NT;
      if (k >= entries) continue;
      bool first = id[i] >= 0;
      float all = s_p[k];
      if (twice && first) {
        all = 0.0f;
#pragma unroll 8
        for (int j = 0; j < entries; ++j) {
          const bool same = s_id[j] == id[i];
          first &= !(same && j < k);
          all += same ? s_p[j] : 0.0f;
        }
      }
      s_place[k] = first ? id[i] : -1;
      s_put[k] = -wp * all - (told && id[i] == label ? w2 : 0.0f);
    }

    // 2^((z - zm) k1) and 2^((z - zm) k2) of a logit
    const auto powers = [&](float zj, float& e1, float& e2) {
      const float d = zj - zm;
      e1 = exp2_raw(d * k1);
      if constexpr (kMode == kBoth) e2 = exp2_raw(d * k2);
      if constexpr (kMode == kT1) e2 = e1;
      if constexpr (kMode == kT2) e2 = e1 * e1;
      if constexpr (kMode == kT4) e2 = (e1 * e1) * (e1 * e1);
    };
    float sum[kHard ? 2 : 1] = {};
    const auto add = [&](float zj) {
      float e1, e2;
      powers(zj, e1, e2);
      sum[0] += e1;
      if constexpr (kHard) sum[1] += e2;
    };
    each([&](const V16& v, uint32_t) {
#pragma unroll
      for (int j = 0; j < kN; ++j) add(v.get(j));
    }, nothing);
    if (own < a.V) add(beside);
    all_sum<NT>(sum, s_sum);
    const float c1 = uniform(taught ? w1 / sum[0] : 0.0f), c2 = uniform(told ? w2 / sum[kHard ? 1 : 0] : 0.0f);
    const bool counted = taught || told;
    const auto slope = [&](float zj) {
      float e1, e2;
      powers(zj, e1, e2);
      e1 *= c1;
      if constexpr (kHard) e1 = __builtin_fmaf(c2, e2, e1);
      return e1;
    };
    float label_put = 0.0f;
    bool label_own = false;  // the label's place is this thread's to write: it is listed nowhere
    if constexpr (kHard) {
      const float zk = value(&zl);
      bool listed = false;
#pragma unroll
      for (int w = 0; w < NT / 64; ++w) listed |= s_mine[w] != 0;
      label_own = told && !listed && tid == NT - 1;
      label_put = slope(zk) - w2;
      if (tid == 0 && told) s_loss[1] += static_cast<double>(kLn2 * __builtin_amdgcn_logf(sum[kHard ? 1 : 0])) + (zm - zk);
    }
    if (tid == 0 && taught)
      s_loss[0] += __builtin_fma(teach[1] / teach[0], static_cast<double>(kLn2 / kSmall),
                                 kLn2 * (__builtin_amdgcn_logf(sum[0]) - __builtin_amdgcn_logf(teach[0])));
    if (dz && own < a.V) put(dz + own, counted ? slope(beside) : 0.0f);
    const int label_place = label;
    fetch_entries(n_next);
    each([&](const V16& v, uint32_t c) {
      if (!dz) return;
      float d[kN] = {};  // (a row that does not count may hold anything: nothing is made of it)
      if (counted) {
#pragma unroll
        for (int j = 0; j < kN; ++j) d[j] = slope(v.get(j));
      }
      V16::store(at_byte(dz + head, c), d);
    }, [&](V16& v, uint32_t c0, int s) {
      if constexpr (kAhead) fetch(v, z_next + head_next, c0 + s * step, next_bytes);
    });
    if constexpr (!kAhead) fetch_row(z_next, head_next, step);
    fetch_places(z_next, head_next);
    __syncthreads();  // the row, and what lies beside its vectors, then its places
    if (dz) {
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        const int k = tid + i * NT;
        if (k < entries && s_place[k] >= 0) put(dz + s_place[k], slope(s_at[k]) + s_put[k]);
      }
      if (label_own) put(dz + label_place, label_put);
    }
    z = z_next, head = head_next;
  }
  if (tid == 0) a.losses[2 * blockIdx.x] = s_loss[0], a.losses[2 * blockIdx.x + 1] = s_loss[1];
}

// (all loads first, and no counters in LDS: 6.8 -> 4.6 us)
__global__ __launch_bounds__(256) void loss_kernel(Args a, int wgs, float* loss) {
  __shared__ double s[4][2];
  __shared__ int s_n[4][2];
  const int groups = count_wgs(a.N), i0 = threadIdx.x;
  int n1 = 0, n2 = 0;
  if (i0 < groups) n1 = a.counts[2 * i0], n2 = a.counts[2 * i0 + 1];
  double l1 = 0.0, l2 = 0.0;
#pragma unroll 8
  for (int i = i0; i < wgs; i += 256) {
    const double2 l = reinterpret_cast<const double2*>(a.losses)[i];
    l1 += l.x, l2 += l.y;
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    l1 += __shfl_xor(l1, o, 64), l2 += __shfl_xor(l2, o, 64);
    n1 += __shfl_xor(n1, o, 64), n2 += __shfl_xor(n2, o, 64);
  }
  if (threadIdx.x % 64 == 0) {
    const int w = threadIdx.x / 64;
    s[w][0] = l1, s[w][1] = l2, s_n[w][0] = n1, s_n[w][1] = n2;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double t = a.temperature, al = a.alpha;
    l1 = (s[0][0] + s[1][0]) + (s[2][0] + s[3][0]), l2 = (s[0][1] + s[1][1]) + (s[2][1] + s[3][1]);
    n1 = s_n[0][0] + s_n[1][0] + s_n[2][0] + s_n[3][0], n2 = s_n[0][1] + s_n[1][1] + s_n[2][1] + s_n[3][1];
    double l = 0.0;
    if (n1) l += al * t * t * l1 / n1;
    if (n2) l += (1.0 - al) * l2 / n2;
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

// As many workgroups as the device holds at once: 256 CUs of four SIMDs
constexpr int wgs_of(int nt, int s) { return 256 * 4 * 64 * waves_of(nt, s) / nt; }
inline int row_wgs(int64_t N, int most) { return static_cast<int>(std::min<int64_t>(N, most)); }

// Few threads and many vectors to each: a row costs each of its waves about the same beyond its vectors (sums over the
// workgroup, entries). With half the threads and twice the vectors 16376 rows of V 16001 and 32000 take 266 and 469 us,
// with twice the threads and half the vectors 254 and 731, with these 257 and 470. Of up to 64 entries a row of few
// vectors is one wave's business, which waits for no other: at V 1001 (31000 rows), 2040, 4001, 6001 and 8001, 55, 51,
// 67, 91 and 128 us, with two waves 91, 74, 87, 121 and 146. Returns the workgroups
template <typename T, int kMode>
int launch_rows(const Args& a, hipStream_t st) {
  const int64_t vecs = a.V / Vec<T>::kN;
  int wgs;
#define GO(NT, S)                                                                            \
  {                                                                                          \
    static_assert(wgs_of(NT, S) <= kRowWgs, "a place for each workgroup's losses");          \
    wgs = row_wgs(a.N, wgs_of(NT, S));                                                       \
    hipLaunchKernelGGL((rows_kernel<T, NT, S, kMode>), dim3(wgs), dim3(NT), 0, st, a);       \
  }
  if (a.V < 2 * Vec<T>::kN - 1) GO(128, 0)  // (some row may have no vector)
  else if (a.K <= 64 && vecs <= 128) GO(64, 2)
  else if (a.K <= 64 && vecs <= 256) GO(64, 4)
  else if (a.K <= 64 && vecs <= 512) GO(64, 8)
  else if (a.K <= 64 && vecs <= 768) GO(64, 12)
  else if (a.K <= 64 && vecs <= 1024) GO(64, 16)
  else if (vecs <= 512) GO(128, 4)
  else if (vecs <= 1024) GO(128, 8)
  else if (vecs <= 2048) GO(256, 8)
  else if (vecs <= 4096) GO(512, 8)
  else if (vecs <= 8192) GO(512, 16)
  else if (vecs <= 16384) GO(1024, 16)
  else GO(1024, 0)
#undef GO
  return wgs;
}

template <typename T>
int launch_modes(const Args& a, hipStream_t st) {
  if (!a.hard) return launch_rows<T, kSoft>(a, st);
  if (a.temperature == 1.0f) return launch_rows<T, kT1>(a, st);
  if (a.temperature == 2.0f) return launch_rows<T, kT2>(a, st);
  if (a.temperature == 4.0f) return launch_rows<T, kT4>(a, st);
  return launch_rows<T, kBoth>(a, st);
}

}  // namespace distill
}  // namespace mg

using namespace mg;

extern "C" size_t mg_distill_workspace_bytes(int64_t N) {
  return N < 1 ? 0 : distill::kCountWgs * 2 * sizeof(int) + static_cast<size_t>(distill::row_wgs(N, distill::kRowWgs)) * 2 * sizeof(double);
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
  hipLaunchKernelGGL(count_kernel, dim3(count_wgs(N)), dim3(8 * kCountRows), 0, st, a);
  const int wgs = logits_dtype == MG_BF16 ? launch_modes<bf16_t>(a, st) : launch_modes<float>(a, st);
  hipLaunchKernelGGL(loss_kernel, dim3(1), dim3(256), 0, st, a, wgs, loss);
  return check_launch(fn);
}

extern "C" unsigned long long mg_capture_id(void* stream) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &id) != hipSuccess) {
    (void)hipGetLastError();  // (the launches that follow report what is wrong with the stream)
    return 0;
  }
  return status == hipStreamCaptureStatusActive ? id : 0;
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
