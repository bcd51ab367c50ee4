// Gated linear recurrence over sequences, forward and backward, and for single tokens, for gfx950.
// Per channel, with sigma the logistic function and rate = softplus(decay):
//   r_t = sigma(decay_gate_t), i_t = sigma(input_gate_t), l_t = -c rate r_t, a_t = e^{l_t} (at a reset none: -0)
//   m_t = sqrt(1 - a_t^2),  h_t = a_t h_{t-1} + m_t i_t x_t
// Backward, with dh the gradient of h:
//   lam_t = dh_t + a_{t+1} lam_{t+1}
//   dx = lam m i,  dinput_gate = lam m i x (1 - i),  w = lam (a h_{t-1} l - i x a^2 l / m)
//   ddecay_gate = w (1 - r),  ddecay = sigma(decay) / rate sum(w),  dh0 = a_0 lam_0
// (dm/da = -a/m; l/m has a limit where the gate is shut and m is 0, which a/m has not: it is 0.)
//
// 1 - a^2 = 1 - e^{2l} is a difference of nearly equal numbers wherever the state decays slowly, so up to |2l| = 1/4
// it is the series of 1 - e^{-w} (six terms, 5e-8), past it 1 - a a. States and sums are fp32.
//
// Work: as the minGRU scan (scan.hip) a workgroup takes a tile of 64 channels by 128 steps (backward 64), a thread 4
// channels by a run of 8 (4) steps; a run is an affine map of the state entering it, runs are combined in LDS, and a
// tile's carry comes from the tiles before it by look-back over self-validating words. One pass over the operands
// each way. Unlike the minGRU's, the words live in a workspace of the call, which a small kernel clears first:
// nothing is kept between calls, so any two calls may overlap, captured ones too. Sequences of one tile need neither.
// Tiles are taken in ticket order, so a tile waits only for tiles that run already; a wait of 2^22 polls ends with NaN.
// The order of every sum is fixed, whatever the timing.
//
// The state is kept every 8 steps in fp32 for the backward (half a byte per value); the steps between are made again.
//
// Bound by memory and, by a fifth, arithmetic. bfloat16, B8 T2047 D1024: forward 40 us (142 MB, 3.5 TB/s; 33 with no
// arithmetic and no carries, 36 with the carries alone), backward 60 (243 MB, 4.0 TB/s). B2 T16381 D2048, forward: 132
// us (537 MB, 4.1 TB/s), with resets 141: forgetting also what is not finite takes selects with every value.

#include <algorithm>

#include "mg_vec.h"

namespace mg {
namespace recurrence {

constexpr int kVec = 4;
constexpr int kLanes = 16;           // threads across channels
constexpr int kCh = kLanes * kVec;   // channels of a tile
constexpr int kRuns = 16;
constexpr int kThreads = kLanes * kRuns;
constexpr int kKeep = 8;             // steps between the states kept
constexpr int kFwdRows = 8, kBwdRows = 4;
constexpr uint32_t kMaxPolls = 1u << 22;
// the last cache: operands beyond it are loaded past the caches (B2 T16381 D2048 forward 138 -> 130 us, backward 288 ->
// 266; B8 T2047 D1024, which it holds, 43 -> 47, 68 -> 76)
constexpr size_t kCacheBytes = size_t(256) << 20;
static_assert(kKeep % kFwdRows == 0 && 2 * kBwdRows == kKeep, "runs and kept states");

// Results are read by other kernels, and by then from the next cache: past this one
template <typename T>
__device__ __forceinline__ void store4_nt(T* p, const f4& v, int left) {
  if (left < kVec) return store4(p, v, left);
  if constexpr (sizeof(T) == 2) {
    u16x4u x;
#pragma unroll
    for (int j = 0; j < kVec; ++j) x[j] = f32_to_bf16(v.v[j]);
    __builtin_nontemporal_store(x, reinterpret_cast<u16x4u*>(p));
  } else {
    const f32x4u x = {v.v[0], v.v[1], v.v[2], v.v[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<f32x4u*>(p));
  }
}

struct Seq {
  const void* p;
  int64_t sb;
  int st;
};

// Chains of tiles (channel blocks of every batch row), tiles of a chain
struct Grid {
  int B, T, D, blocks, chains, tiles;
};

// ------------------------------------------------------------------ values as loaded

template <typename T> struct Raw;
template <> struct Raw<bf16_t> {
  uint2 r;
  template <bool kOnce>
  __device__ __forceinline__ void load(const bf16_t* p) {
    const u16x4u* v = reinterpret_cast<const u16x4u*>(p);
    if constexpr (kOnce)
      r = __builtin_bit_cast(uint2, __builtin_nontemporal_load(v));
    else
      r = __builtin_bit_cast(uint2, *v);
  }
  __device__ __forceinline__ void load(const bf16_t* p, int left) {
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < left) v[j] = p[j];
    r = make_uint2(v[0] | v[1] << 16, v[2] | v[3] << 16);
  }
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = j < 2 ? r.x : r.y;
    return __uint_as_float(j & 1 ? w & 0xffff0000u : w << 16);
  }
};
template <> struct Raw<float> {
  float4 r;
  template <bool kOnce>
  __device__ __forceinline__ void load(const float* p) {
    const f32x4u* v = reinterpret_cast<const f32x4u*>(p);
    if constexpr (kOnce)
      r = __builtin_bit_cast(float4, __builtin_nontemporal_load(v));
    else
      r = __builtin_bit_cast(float4, *v);
  }
  __device__ __forceinline__ void load(const float* p, int left) {
    const f4 x = load4(p, left);
    r = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
  }
  __device__ __forceinline__ float get(int j) const { return j == 0 ? r.x : j == 1 ? r.y : j == 2 ? r.z : r.w; }
};

// kRows rows of four channels; those past the sequence or the last channel are zero. kOnce: without a place in the
// caches, for operands that are larger than those.
template <bool kOnce, typename T, int kRows>
__device__ __forceinline__ void load_rows(const T* p, int st, int rows, int left, Raw<T> (&v)[kRows]) {
  if (rows >= kRows && left >= kVec) {
#pragma unroll
    for (int i = 0; i < kRows; ++i) v[i].template load<kOnce>(p + i * st);
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i) v[i].load(p + i * st, i < rows ? left : 0);
  }
}

// Bit i: a sequence starts at the i-th of kRows steps from p on, `rows` of which exist
template <int kRows>
__device__ __forceinline__ uint32_t starts(const uint8_t* p, int rows) {
  typedef uint8_t u8s __attribute__((ext_vector_type(kRows), aligned(1)));
  uint32_t bits = 0;
  if (rows >= kRows) {
    const u8s v = *reinterpret_cast<const u8s*>(p);
#pragma unroll
    for (int i = 0; i < kRows; ++i) bits |= v[i] ? 1u << i : 0u;
  } else {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (i < rows && p[i]) bits |= 1u << i;
  }
  return bits;
}

// ------------------------------------------------------------------ a step's terms

__device__ __forceinline__ float sigma(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2_raw(x * -kLog2e)); }

// sigma(x) and 1 - sigma(x), each with all its digits (1 minus the rounded sigma has lost them all at x = 17), in one
// register: sigma where x is negative, else 1 - sigma with its sign turned. A value k of either kind is sigma or one
// less, so that the fraction of k is sigma, and that of -k is 1 - sigma; 2^-126 keeps the latter off 0, whose fraction
// is 0 on both sides. Hidden from the compiler, which would keep both. (A difference instead: B8 T2047 D1024 63 us, not
// 64, B2 T16381 D2048 packed 259, not 262; both sides by selects 65 and 268.)
struct Sides {
  float k;
  __device__ __forceinline__ float of(float x) {
    const float e = exp2_raw(x * -kLog2e), s = __builtin_amdgcn_rcpf(1.0f + e);
    k = x >= 0.0f ? -__builtin_fmaf(e, s, 0x1p-126f) : s;
    asm volatile("" : "+v"(k));
    return s;
  }
  __device__ __forceinline__ float open() const { return __builtin_amdgcn_fractf(k); }
  __device__ __forceinline__ float shut() const { return __builtin_amdgcn_fractf(-k); }
};

__device__ __forceinline__ float softplus(float x) { return log1pf(expf(-fabsf(x))) + fmaxf(x, 0.0f); }

// 1 - e^{-w}, w >= 0, of which a = e^{-w/2} is known
__device__ __forceinline__ float one_minus(float w, float a) {
  const float s = w * (1.0f + w * (-1.0f / 2 + w * (1.0f / 6 + w * (-1.0f / 24 + w * (1.0f / 120 + w * (-1.0f / 720))))));
  return w <= 0.25f ? s : 1.0f - a * a;
}

// a, m from l = c softplus(decay) sigma(decay_gate) (-l_t)
__device__ __forceinline__ void decay_terms(float l, float& a, float& m) {
  a = exp2_raw(l * -kLog2e);
  m = __builtin_amdgcn_sqrtf(one_minus(2.0f * l, a));
}

// The map h -> a h + v of a run or a tile. With kReset an a of -0 forgets what came before, be it finite or not: that is
// what a reset gives, and any product with it. A product of decays that underflows is +0: it forgets finite values, and
// what is not finite stays so.
constexpr float kCut = -0.0f;
__device__ __forceinline__ bool is_cut(float a) { return __float_as_uint(a) == __float_as_uint(kCut); }
template <bool kReset>
__device__ __forceinline__ float apply(float a, float h, float v) {
  return kReset && is_cut(a) ? v : __builtin_fmaf(a, h, v);
}

// ------------------------------------------------------------------ tiles and carries

struct Maps {
  f4 A[2][kRuns][kLanes], V[2][kRuns][kLanes];
};

// Maps of all runs up to (kReverse: from) each run of the tile, by doubling; returns the buffer that holds them
template <bool kReverse, bool kReset>
__device__ __forceinline__ int scan_runs(Maps& m, int s, int cl, f4 A, f4 V) {
  int buf = 0;
  m.A[0][s][cl] = A, m.V[0][s][cl] = V;
  __syncthreads();
#pragma unroll
  for (int o = 1; o < kRuns; o <<= 1) {
    const int src = kReverse ? s + o : s - o;
    if (kReverse ? src < kRuns : src >= 0) {
      const f4 pa = m.A[buf][src][cl], pv = m.V[buf][src][cl];
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        V.v[j] = apply<kReset>(A.v[j], pv.v[j], V.v[j]);
        A.v[j] = kReset && is_cut(A.v[j]) ? kCut : A.v[j] * pa.v[j];
      }
    }
    buf ^= 1;
    m.A[buf][s][cl] = A, m.V[buf][s][cl] = V;
    __syncthreads();
  }
  return buf;
}

// The chain and the tile of this workgroup, the tile in the order of arrival
__device__ __forceinline__ int take_tile(const Grid& g, uint32_t* tickets, uint32_t* s_ticket, int& chain) {
  chain = static_cast<int>(blockIdx.x % static_cast<uint32_t>(g.chains));
  if (g.tiles == 1) return 0;
  if (threadIdx.x == 0) *s_ticket = atomicAdd(tickets + chain, 1u);
  __syncthreads();
  return static_cast<int>(__builtin_amdgcn_readfirstlane(*s_ticket));
}

// A tile's map for the tiles after it: of an A without a sign, and the bit that calls that keep their words alternate
// instead (a NaN has that bit too: then the V beside it is NaN, and forgets or not)
template <bool kReset>
__device__ __forceinline__ void publish_map(uint64_t* word, float A, float V) {
  publish_agg(word, A, V, kReset && is_cut(A));
}
template <bool kReset>
__device__ __forceinline__ float map_of(uint32_t tag) {
  if (kReset && (tag & kTagParity)) return kCut;
  return __uint_as_float(tag & ~kTagAggBit);
}

// What enters tile k of channel c: back (step -1) or on (+1) to the nearest tile whose result is known, then through
// the maps of those between, in their order. A map becomes a result as this would compute it, so the carry does not
// depend on which of the two was seen. `end` always gives a result.
// Words are read four at a time: one at a time the walk over the tiles that run at once takes longer than their work.
template <bool kReset>
__device__ __forceinline__ float look_back(const uint64_t* words, int64_t BD, int k, int step, int end) {
  constexpr int kAt = 4;
  const auto read = [&](int first, int last, uint64_t (&x)[kAt]) {  // first, first + step, ..., none past `last`
#pragma unroll
    for (int q = 0; q < kAt; ++q) {
      const int i = first + q * step;
      x[q] = poll_word(words + (step < 0 ? std::max(i, last) : std::min(i, last)) * BD);
    }
  };
  const auto value = [](uint64_t x) { return __uint_as_float(static_cast<uint32_t>(x >> 32)); };
  int j = k + step;
  uint32_t polls = 0;
  float carry = 0.0f;
  for (bool found = false; !found;) {
    uint64_t x[kAt];
    read(j, end, x);
    bool ready = true;
#pragma unroll
    for (int q = 0; q < kAt; ++q) {
      if (!ready || found) continue;
      const uint32_t tag = static_cast<uint32_t>(x[q]);
      if (tag == kTagIncl) {
        carry = value(x[q]);
        found = true;
      } else if (j != end && (tag & kTagAggBit)) {
        j += step;
        polls = 0;
      } else {
        ready = false;
      }
    }
    if (!ready) {
      if (++polls > kMaxPolls) return __builtin_nanf("");
      __builtin_amdgcn_s_sleep(1);
    }
  }
  for (int i = j - step; i != k;) {
    uint64_t x[kAt];
    // (back towards k: the words of tiles that were seen ready)
#pragma unroll
    for (int q = 0; q < kAt; ++q) {
      const int n = i - q * step;
      x[q] = poll_word(words + (step < 0 ? std::min(n, k - 1) : std::max(n, k + 1)) * BD);
    }
#pragma unroll
    for (int q = 0; q < kAt; ++q) {
      if (i == k) continue;
      const uint32_t tag = static_cast<uint32_t>(x[q]);
      carry = tag == kTagIncl ? value(x[q]) : apply<kReset>(map_of<kReset>(tag), carry, value(x[q]));
      i -= step;
    }
  }
  return carry;
}

// ------------------------------------------------------------------ forward

struct Fwd {
  Seq x, gi, gr;
  const float *decay, *h0;
  const uint8_t* reset;
  void* h;
  float *last, *keep;
  float c;
  Grid g;
  uint32_t* tickets;
  uint64_t* words;
};

template <typename T, bool kReset, bool kOnce>
__global__ __launch_bounds__(kThreads) void fwd_kernel(Fwd p) {
  __shared__ uint32_t s_ticket;
  __shared__ Maps s_maps;
  __shared__ f4 s_carry[kLanes];
  __shared__ float s_rate[kCh];
  const Grid& g = p.g;
  const int tid = threadIdx.x, cl = tid % kLanes, s = tid / kLanes;
  int chain;
  const int k = take_tile(g, p.tickets, &s_ticket, chain);
  if (k >= g.tiles) return;
  const int b = chain / g.blocks, d0 = (chain % g.blocks) * kCh, d = d0 + cl * kVec, left = g.D - d;
  const int t0 = k * (kRuns * kFwdRows) + s * kFwdRows, rows = g.T - t0;
  const auto at = [&](const Seq& q) { return static_cast<const T*>(q.p) + b * q.sb + static_cast<int64_t>(t0) * q.st + d; };

  Raw<T> x[kFwdRows], gi[kFwdRows], gr[kFwdRows];
  load_rows<kOnce>(at(p.gr), p.gr.st, rows, left, gr);
  load_rows<kOnce>(at(p.gi), p.gi.st, rows, left, gi);
  load_rows<kOnce>(at(p.x), p.x.st, rows, left, x);
  uint32_t fresh = 0;  // bit i: a sequence starts at step t0 + i
  if constexpr (kReset) fresh = starts<kFwdRows>(p.reset + static_cast<int64_t>(b) * g.T + t0, rows);
  if (tid < kCh) s_rate[tid] = d0 + tid < g.D ? p.c * softplus(p.decay[d0 + tid]) : 0.0f;
  __syncthreads();
  const f4 rate = *reinterpret_cast<const f4*>(&s_rate[cl * kVec]);

  float a[kFwdRows][kVec], v[kFwdRows][kVec];
  f4 A = io4<float>::fill(1.0f), V = io4<float>::fill(0.0f);
#pragma unroll
  for (int i = 0; i < kFwdRows; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      float m;
      decay_terms(rate.v[j] * sigma(gr[i].get(j)), a[i][j], m);
      const bool cut = kReset && (fresh >> i & 1);
      if (cut) m = 1.0f;
      v[i][j] = m * (sigma(gi[i].get(j)) * x[i].get(j));
      if (i >= rows) a[i][j] = 1.0f, v[i][j] = 0.0f;  // past the end nothing changes
      // (the bits themselves, not a made 0 and compared again: B2 T16381 D2048 149 -> 141 us)
      V.v[j] = cut ? v[i][j] : __builtin_fmaf(a[i][j], V.v[j], v[i][j]);
      A.v[j] = cut ? kCut : A.v[j] * a[i][j];
    }
  }
  const int buf = scan_runs<false, kReset>(s_maps, s, cl, A, V);

  // the tile's carry, one channel to a lane of the first wave: lane (s, cl) has channel 4 cl + s
  const int64_t BD = static_cast<int64_t>(g.B) * g.D, row = static_cast<int64_t>(b) * g.D + d;
  if (tid < kCh && s < left) {
    const float TA = s_maps.A[buf][kRuns - 1][cl].v[s], TV = s_maps.V[buf][kRuns - 1][cl].v[s];
    uint64_t* words = p.words + row + s;
    float carry;
    if (k == 0) {
      carry = p.h0 ? p.h0[row + s] : 0.0f;
    } else {
      publish_map<kReset>(words + k * BD, TA, TV);
      carry = look_back<kReset>(words, BD, k, -1, 0);
    }
    if (k + 1 < g.tiles) publish_incl(words + k * BD, apply<kReset>(TA, carry, TV), 0);
    s_carry[cl].v[s] = carry;
  }
  __syncthreads();
  if (left <= 0 || rows <= 0) return;

  f4 h = s_carry[cl];
  if (s > 0) {
    const f4 pa = s_maps.A[buf][s - 1][cl], pv = s_maps.V[buf][s - 1][cl];
#pragma unroll
    for (int j = 0; j < kVec; ++j) h.v[j] = apply<kReset>(pa.v[j], h.v[j], pv.v[j]);
  }
  T* out = static_cast<T*>(p.h) + (static_cast<int64_t>(b) * g.T + t0) * g.D + d;
#pragma unroll
  for (int i = 0; i < kFwdRows; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) h.v[j] = kReset && (fresh >> i & 1) ? v[i][j] : __builtin_fmaf(a[i][j], h.v[j], v[i][j]);
    if (i < rows) store4_nt(out + static_cast<int64_t>(i) * g.D, h, left);
    if (i + 1 == rows && p.last) store4(p.last + row, h, left);
  }
  const int t1 = t0 + kFwdRows;
  if (p.keep && rows >= kFwdRows && t1 % kKeep == 0) store4(p.keep + (t1 / kKeep - 1) * BD + row, h, left);
}

// ------------------------------------------------------------------ backward

struct Bwd {
  Seq x, gi, gr, dh;
  const float *decay, *h0, *keep, *dlast;
  const uint8_t* reset;
  void *dx, *dgi, *dgr;
  float *dh0, *part;  // part: [B tiles][D] sums of w
  float c;
  Grid g;
  uint32_t* tickets;
  uint64_t* words;
};

// (four waves per SIMD fit bf16 operands without spills: B2 T16381 D2048 268 -> 248 us)
template <typename T, bool kReset, bool kOnce>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3) void bwd_kernel(Bwd p) {
  constexpr int kRows = kBwdRows;
  __shared__ uint32_t s_ticket;
  __shared__ Maps s_maps;
  __shared__ f4 s_carry[kLanes], s_mid[kRuns / 2][kLanes];
  __shared__ float s_rate[kCh];
  const Grid& g = p.g;
  // even runs, which start at a kept state, in the first half of the workgroup, odd ones in the second
  const int tid = threadIdx.x, cl = tid % kLanes;
  const int s = (tid / kLanes % (kRuns / 2)) * 2 + tid / (kThreads / 2);
  int chain;
  const int n = take_tile(g, p.tickets, &s_ticket, chain);
  if (n >= g.tiles) return;
  const int k = g.tiles - 1 - n;
  const int b = chain / g.blocks, d0 = (chain % g.blocks) * kCh, d = d0 + cl * kVec, left = g.D - d;
  const int t0 = k * (kRuns * kRows) + s * kRows, rows = g.T - t0;
  const int64_t BD = static_cast<int64_t>(g.B) * g.D, row = static_cast<int64_t>(b) * g.D + d;
  const auto at = [&](const Seq& q) { return static_cast<const T*>(q.p) + b * q.sb + static_cast<int64_t>(t0) * q.st + d; };

  Raw<T> x[kRows], gi[kRows], gr[kRows], dh[kRows];
  load_rows<kOnce>(at(p.gr), p.gr.st, rows, left, gr);
  load_rows<kOnce>(at(p.gi), p.gi.st, rows, left, gi);
  load_rows<kOnce>(at(p.x), p.x.st, rows, left, x);
  load_rows<kOnce>(at(p.dh), p.dh.st, rows, left, dh);
  uint32_t fresh = 0;
  if constexpr (kReset) fresh = starts<kRows>(p.reset + static_cast<int64_t>(b) * g.T + t0, rows);
  f4 h = io4<float>::fill(0.0f);  // the state that enters the run
  if (!(s & 1) && rows > 0 && left > 0) {
    if (t0 > 0)
      h = load4(p.keep + (t0 / kKeep - 1) * BD + row, left);
    else if (p.h0)
      h = load4(p.h0 + row, left);
  }
  if (tid < kCh) s_rate[tid] = d0 + tid < g.D ? p.c * softplus(p.decay[d0 + tid]) : 0.0f;
  __syncthreads();
  const f4 rate = *reinterpret_cast<const f4*>(&s_rate[cl * kVec]);

  float a[kRows][kVec], m[kRows][kVec];
  Sides r[kRows][kVec], gate[kRows][kVec];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      decay_terms(rate.v[j] * r[i][j].of(gr[i].get(j)), a[i][j], m[i][j]);
      if (kReset && (fresh >> i & 1)) a[i][j] = kCut, m[i][j] = 1.0f;
      if (i >= rows) a[i][j] = 1.0f, m[i][j] = 0.0f;
      gate[i][j].of(gi[i].get(j));
    }
    __builtin_amdgcn_sched_barrier(0);  // (B2 T16381 D2048 packed 267 us, 270 without)
  }
  if (!(s & 1)) {  // the next run's entering state
    f4 e = h;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
#pragma unroll
      for (int j = 0; j < kVec; ++j) e.v[j] = apply<kReset>(a[i][j], e.v[j], m[i][j] * (gate[i][j].open() * x[i].get(j)));
    s_mid[s / 2][cl] = e;
  }
  // the run as a map of what comes back through it: mu -> A mu + M, mu_t = a_t lam_t
  f4 A = io4<float>::fill(1.0f), M = io4<float>::fill(0.0f);
#pragma unroll
  for (int i = kRows - 1; i >= 0; --i)
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      const bool cut = kReset && is_cut(a[i][j]);
      M.v[j] = cut ? 0.0f : a[i][j] * (dh[i].get(j) + M.v[j]);
      A.v[j] = cut ? kCut : A.v[j] * a[i][j];
    }
  const int buf = scan_runs<true, kReset>(s_maps, s, cl, A, M);

  if (tid < kCh) {
    const int q = tid / kLanes;
    if (q < left) {
      const float TA = s_maps.A[buf][0][cl].v[q], TM = s_maps.V[buf][0][cl].v[q];
      uint64_t* words = p.words + row + q;
      float carry = 0.0f;
      if (k == g.tiles - 1) {
        // (the steps past the end pass it on unchanged)
        if (p.dlast) carry = p.dlast[row + q];
      } else {
        publish_map<kReset>(words + k * BD, TA, TM);
        carry = look_back<kReset>(words, BD, k, 1, g.tiles - 1);
      }
      if (k > 0) publish_incl(words + k * BD, apply<kReset>(TA, carry, TM), 0);
      s_carry[cl].v[q] = carry;
    }
  }
  __syncthreads();

  f4 mu = s_carry[cl], sum = io4<float>::fill(0.0f);
  if (s + 1 < kRuns) {
    const f4 pa = s_maps.A[buf][s + 1][cl], pm = s_maps.V[buf][s + 1][cl];
#pragma unroll
    for (int j = 0; j < kVec; ++j) mu.v[j] = apply<kReset>(pa.v[j], mu.v[j], pm.v[j]);
  }
  if (s & 1) h = s_mid[s / 2][cl];
  if (left > 0 && rows > 0) {
    float lam[kRows][kVec];
#pragma unroll
    for (int i = kRows - 1; i >= 0; --i)
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        lam[i][j] = dh[i].get(j) + mu.v[j];
        mu.v[j] = kReset && is_cut(a[i][j]) ? 0.0f : a[i][j] * lam[i][j];
      }
    if (p.dh0 && t0 == 0) store4(p.dh0 + row, mu, left);
    const int64_t out = (static_cast<int64_t>(b) * g.T + t0) * g.D + d;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      f4 ox, oi, og;
#pragma unroll
      for (int j = 0; j < kVec; ++j) {
        const float u = gate[i][j].open() * x[i].get(j), lm = lam[i][j] * m[i][j];
        ox.v[j] = lm * gate[i][j].open();
        oi.v[j] = lm * (u * gate[i][j].shut());
        // l / m is 0 with m, and its square with a
        const float l = -rate.v[j] * r[i][j].open(), q = l * __builtin_amdgcn_rcpf(fmaxf(m[i][j], 1e-30f));
        float w = lam[i][j] * (a[i][j] * (h.v[j] * l - u * (a[i][j] * q)));
        if (kReset && (fresh >> i & 1)) w = 0.0f;
        og.v[j] = w * r[i][j].shut();
        if (i < rows) sum.v[j] += w;
        h.v[j] = apply<kReset>(a[i][j], h.v[j], m[i][j] * u);
      }
      if (i < rows) {
        const int64_t o = out + static_cast<int64_t>(i) * g.D;
        store4_nt(static_cast<T*>(p.dx) + o, ox, left);
        store4_nt(static_cast<T*>(p.dgi) + o, oi, left);
        store4_nt(static_cast<T*>(p.dgr) + o, og, left);
      }
    }
  }
  // the tile's sum of w, runs in order (the maps' first buffer is free: the last one read is the other)
  f4(&s_sum)[kRuns][kLanes] = s_maps.A[buf ^ 1];
  s_sum[s][cl] = sum;
  __syncthreads();
  if (tid < kCh && d0 + tid < g.D) {
    float t = 0.0f;
#pragma unroll
    for (int q = 0; q < kRuns; ++q) t += s_sum[q][tid / kVec].v[tid % kVec];
    p.part[(static_cast<int64_t>(b) * g.tiles + k) * g.D + d0 + tid] = t;
  }
}

// ddecay = sigma(decay) / softplus(decay) times the sum of the tiles' rows: 16 columns to a workgroup, 16 threads to a
// column (the ratio is 1 where e^decay underflows)
__global__ __launch_bounds__(256) void ddecay_kernel(const float* __restrict__ part, int P, int D, const float* __restrict__ decay,
                                                     float* __restrict__ ddecay) {
  __shared__ float s[16][17];
  const int c = threadIdx.x % 16, q = threadIdx.x / 16, d = 16 * blockIdx.x + c;
  float t = 0.0f;
  if (d < D) {
#pragma unroll 4
    for (int p = q; p < P; p += 16) t += part[static_cast<int64_t>(p) * D + d];
  }
  s[q][c] = t;
  __syncthreads();
  if (q == 0 && d < D) {
    t = 0.0f;
    for (int i = 0; i < 16; ++i) t += s[i][c];
    const float x = decay[d], e = expf(-fabsf(x));
    const float up = x >= 0.0f ? 1.0f : e;  // sigma(x) (1 + e^-|x|)
    const float sp = softplus(x);
    ddecay[d] = t * (sp > 0.0f ? up / ((1.0f + e) * sp) : 1.0f);
  }
}

// ------------------------------------------------------------------ single tokens

struct Step {
  Seq x, gi, gr;
  const float* decay;
  float* state;
  void* h;
  float c;
  int B, D;
};

template <typename T>
__global__ __launch_bounds__(64) void step_kernel(Step p) {
  const int d = 4 * (blockIdx.x * 64 + threadIdx.x), left = p.D - d;
  if (left <= 0) return;
  const f4 decay = load4(p.decay + d, left);
  for (int b = blockIdx.y; b < p.B; b += gridDim.y) {
    const auto at = [&](const Seq& q) { return load4(static_cast<const T*>(q.p) + b * q.sb + d, left); };
    const f4 x = at(p.x), gi = at(p.gi), gr = at(p.gr);
    float* sp = p.state + static_cast<int64_t>(b) * p.D + d;
    f4 h = load4(sp, left);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float a, m;
      decay_terms(p.c * softplus(decay.v[j]) * sigma(gr.v[j]), a, m);
      h.v[j] = __builtin_fmaf(a, h.v[j], m * (sigma(gi.v[j]) * x.v[j]));
    }
    store4(sp, h, left);
    store4(static_cast<T*>(p.h) + static_cast<int64_t>(b) * p.D + d, h, left);
  }
}

// ------------------------------------------------------------------ host

__global__ __launch_bounds__(256) void clear_kernel(uint4* p, int64_t n) {
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += static_cast<int64_t>(gridDim.x) * 256)
    p[i] = make_uint4(0, 0, 0, 0);
}

inline Grid grid_of(int B, int T, int D, int rows) {
  const int blocks = (D + kCh - 1) / kCh, span = kRuns * rows;
  return {B, T, D, blocks, B * blocks, static_cast<int>((static_cast<int64_t>(T) + span - 1) / span)};
}
inline size_t up16(size_t n) { return (n + 15) / 16 * 16; }
// tickets, then a word per tile and channel; nothing where a chain is one tile
inline size_t words_at(const Grid& g) { return up16(static_cast<size_t>(g.chains) * 4); }
inline size_t clear_bytes(const Grid& g) {
  return g.tiles == 1 ? 0 : words_at(g) + up16(static_cast<size_t>(g.tiles) * g.B * g.D * 8);
}

inline int check_sizes(const char* fn, int B, int T, int D) {
  if (B < 1 || T < 1 || D < 1) return fail(MG_ERR_ARG, "%s: B=%d, T=%d, D=%d must be at least 1", fn, B, T, D);
  const int64_t chains = static_cast<int64_t>(B) * ((D + int64_t(kCh) - 1) / kCh);
  if (static_cast<int64_t>(B) * D > INT32_MAX || chains * ((T + int64_t(63)) / 64) > (int64_t(1) << 24) - 1)
    return fail(MG_ERR_ARG, "%s: B=%d, T=%d, D=%d: too many tiles", fn, B, T, D);
  return MG_OK;
}
// a run's rows are reached by 32-bit offsets
inline int check_seq(const char* fn, const char* name, const mg_seq* q, int dtype, Seq& out) {
  if (!q || !q->p) return fail(MG_ERR_ARG, "%s: %s is NULL", fn, name);
  if (!aligned(q->p, dtype == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: %s misaligned", fn, name);
  if (q->st < 0 || q->sb < 0 || q->st >= (int64_t(1) << 28)) return fail(MG_ERR_ARG, "%s: %s strides (%lld, %lld) out of range", fn, name, (long long)q->sb, (long long)q->st);
  out = {q->p, q->sb, static_cast<int>(q->st)};
  return MG_OK;
}
inline int check_vec(const char* fn, const char* name, const void* p, int align, bool required) {
  if (!p) return required ? fail(MG_ERR_ARG, "%s: %s is NULL", fn, name) : MG_OK;
  return aligned(p, align) ? MG_OK : fail(MG_ERR_ARG, "%s: %s misaligned", fn, name);
}
inline int check_dtype(const char* fn, int dtype, float c) {
  if (dtype != MG_F32 && dtype != MG_BF16) return fail(MG_ERR_DTYPE, "%s: dtype %d unsupported", fn, dtype);
  if (!(c >= 0.0f && c < 1e30f)) return fail(MG_ERR_ARG, "%s: c=%g must be in [0, 1e30)", fn, c);
  return MG_OK;
}
inline int check_ws(const char* fn, const void* ws, size_t bytes, size_t need) {
  if (need && (!ws || bytes < need || !aligned(ws, 16)))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or misaligned)", fn, bytes, need);
  return MG_OK;
}
inline void clear(void* ws, size_t bytes, hipStream_t st) {
  const int64_t n = bytes / 16;
  if (n) hipLaunchKernelGGL(clear_kernel, dim3(std::min<int64_t>((n + 255) / 256, 1024)), dim3(256), 0, st, static_cast<uint4*>(ws), n);
}

}  // namespace recurrence
}  // namespace mg

using namespace mg;

extern "C" int64_t mg_recurrence_keep_elems(int B, int T, int D) {
  return B < 1 || T < 1 || D < 1 ? 0 : static_cast<int64_t>(T / recurrence::kKeep) * B * D;
}

extern "C" size_t mg_recurrence_fwd_workspace_bytes(int B, int T, int D) {
  using namespace recurrence;
  return check_sizes("mg_recurrence_fwd_workspace_bytes", B, T, D) ? 0 : clear_bytes(grid_of(B, T, D, kFwdRows));
}

extern "C" int mg_recurrence_fwd(int dtype, const mg_seq* x, const mg_seq* input_gate, const mg_seq* decay_gate, const float* decay,
                                 float c, const float* h0, const uint8_t* reset, void* h, float* h_last, float* keep, int B, int T,
                                 int D, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace recurrence;
  const char* fn = "mg_recurrence_fwd";
  const int e = dtype == MG_F32 ? 4 : 2;
  Fwd p = {};
  int rc;
  if ((rc = check_dtype(fn, dtype, c)) || (rc = check_sizes(fn, B, T, D)) || (rc = check_seq(fn, "x", x, dtype, p.x)) ||
      (rc = check_seq(fn, "input_gate", input_gate, dtype, p.gi)) || (rc = check_seq(fn, "decay_gate", decay_gate, dtype, p.gr)) ||
      (rc = check_vec(fn, "decay", decay, 4, true)) || (rc = check_vec(fn, "h0", h0, 4, false)) ||
      (rc = check_vec(fn, "h", h, e, true)) || (rc = check_vec(fn, "h_last", h_last, 4, false)) ||
      (rc = check_vec(fn, "keep", keep, 4, false)))
    return rc;
  p.g = grid_of(B, T, D, kFwdRows);
  if ((rc = check_ws(fn, workspace, workspace_bytes, clear_bytes(p.g)))) return rc;
  p.decay = decay, p.h0 = h0, p.reset = reset, p.h = h, p.last = h_last, p.keep = keep, p.c = c;
  p.tickets = static_cast<uint32_t*>(workspace);
  p.words = p.g.tiles == 1 ? nullptr : reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + words_at(p.g));
  hipStream_t st = static_cast<hipStream_t>(stream);
  clear(workspace, clear_bytes(p.g), st);
  const dim3 grid(static_cast<unsigned>(p.g.chains) * p.g.tiles), block(kThreads);
  const bool once = static_cast<size_t>(B) * T * D * e * 3 > kCacheBytes;
  const auto go = [&](auto t, auto cut, auto single) {
    hipLaunchKernelGGL((fwd_kernel<decltype(t), decltype(cut)::value, decltype(single)::value>), grid, block, 0, st, p);
  };
  const auto by_size = [&](auto t, auto cut) { once ? go(t, cut, std::true_type{}) : go(t, cut, std::false_type{}); };
  const auto by_reset = [&](auto t) { reset ? by_size(t, std::true_type{}) : by_size(t, std::false_type{}); };
  dtype == MG_BF16 ? by_reset(bf16_t{}) : by_reset(0.0f);
  return check_launch(fn);
}

extern "C" size_t mg_recurrence_bwd_workspace_bytes(int B, int T, int D) {
  using namespace recurrence;
  if (check_sizes("mg_recurrence_bwd_workspace_bytes", B, T, D)) return 0;
  const Grid g = grid_of(B, T, D, kBwdRows);
  return clear_bytes(g) + static_cast<size_t>(B) * g.tiles * D * 4;
}

extern "C" int mg_recurrence_bwd(int dtype, const mg_seq* x, const mg_seq* input_gate, const mg_seq* decay_gate, const float* decay,
                                 float c, const float* h0, const uint8_t* reset, const float* keep, const mg_seq* dh,
                                 const float* dh_last, void* dx, void* dinput_gate, void* ddecay_gate, float* ddecay, float* dh0,
                                 int B, int T, int D, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace recurrence;
  const char* fn = "mg_recurrence_bwd";
  const int e = dtype == MG_F32 ? 4 : 2;
  Bwd p = {};
  int rc;
  if ((rc = check_dtype(fn, dtype, c)) || (rc = check_sizes(fn, B, T, D)) || (rc = check_seq(fn, "x", x, dtype, p.x)) ||
      (rc = check_seq(fn, "input_gate", input_gate, dtype, p.gi)) || (rc = check_seq(fn, "decay_gate", decay_gate, dtype, p.gr)) ||
      (rc = check_seq(fn, "dh", dh, dtype, p.dh)) || (rc = check_vec(fn, "decay", decay, 4, true)) ||
      (rc = check_vec(fn, "h0", h0, 4, false)) || (rc = check_vec(fn, "keep", keep, 4, T >= kKeep)) ||
      (rc = check_vec(fn, "dh_last", dh_last, 4, false)) || (rc = check_vec(fn, "dx", dx, e, true)) ||
      (rc = check_vec(fn, "dinput_gate", dinput_gate, e, true)) || (rc = check_vec(fn, "ddecay_gate", ddecay_gate, e, true)) ||
      (rc = check_vec(fn, "ddecay", ddecay, 4, false)) || (rc = check_vec(fn, "dh0", dh0, 4, false)))
    return rc;
  p.g = grid_of(B, T, D, kBwdRows);
  if ((rc = check_ws(fn, workspace, workspace_bytes, mg_recurrence_bwd_workspace_bytes(B, T, D)))) return rc;
  const size_t cleared = clear_bytes(p.g);
  p.decay = decay, p.h0 = h0, p.keep = keep, p.dlast = dh_last, p.reset = reset, p.c = c;
  p.dx = dx, p.dgi = dinput_gate, p.dgr = ddecay_gate, p.dh0 = dh0;
  p.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + cleared);
  p.tickets = static_cast<uint32_t*>(workspace);
  p.words = p.g.tiles == 1 ? nullptr : reinterpret_cast<uint64_t*>(static_cast<char*>(workspace) + words_at(p.g));
  hipStream_t st = static_cast<hipStream_t>(stream);
  clear(workspace, cleared, st);
  const dim3 grid(static_cast<unsigned>(p.g.chains) * p.g.tiles), block(kThreads);
  const bool once = static_cast<size_t>(B) * T * D * e * 4 > kCacheBytes;
  const auto go = [&](auto t, auto cut, auto single) {
    hipLaunchKernelGGL((bwd_kernel<decltype(t), decltype(cut)::value, decltype(single)::value>), grid, block, 0, st, p);
  };
  const auto by_size = [&](auto t, auto cut) { once ? go(t, cut, std::true_type{}) : go(t, cut, std::false_type{}); };
  const auto by_reset = [&](auto t) { reset ? by_size(t, std::true_type{}) : by_size(t, std::false_type{}); };
  dtype == MG_BF16 ? by_reset(bf16_t{}) : by_reset(0.0f);
  if (ddecay) hipLaunchKernelGGL(ddecay_kernel, dim3((D + 15) / 16), dim3(256), 0, st, p.part, B * p.g.tiles, D, decay, ddecay);
  return check_launch(fn);
}

extern "C" int mg_recurrence_step(int dtype, const void* x, int64_t x_ld, const void* input_gate, int64_t input_gate_ld,
                                  const void* decay_gate, int64_t decay_gate_ld, const float* decay, float c, float* state, void* h,
                                  int B, int D, void* stream) {
  using namespace recurrence;
  const char* fn = "mg_recurrence_step";
  const int e = dtype == MG_F32 ? 4 : 2;
  const mg_seq rows[3] = {{x, x_ld, 0}, {input_gate, input_gate_ld, 0}, {decay_gate, decay_gate_ld, 0}};
  Step p = {};
  int rc;
  if ((rc = check_dtype(fn, dtype, c)) || (rc = check_sizes(fn, B, 1, D)) || (rc = check_seq(fn, "x", &rows[0], dtype, p.x)) ||
      (rc = check_seq(fn, "input_gate", &rows[1], dtype, p.gi)) || (rc = check_seq(fn, "decay_gate", &rows[2], dtype, p.gr)) ||
      (rc = check_vec(fn, "decay", decay, 4, true)) || (rc = check_vec(fn, "state", state, 4, true)) ||
      (rc = check_vec(fn, "h", h, e, true)))
    return rc;
  p.decay = decay, p.state = state, p.h = h, p.c = c, p.B = B, p.D = D;
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid((D + 255) / 256, std::min(B, 65535));
  if (dtype == MG_BF16)
    hipLaunchKernelGGL(step_kernel<bf16_t>, grid, dim3(64), 0, st, p);
  else
    hipLaunchKernelGGL(step_kernel<float>, grid, dim3(64), 0, st, p);
  return check_launch(fn);
}
