// Scaled token embedding for any vocabulary and its gradient by sorted tokens, for gfx950 (embed.hip has the gradient
// of byte-sized vocabularies).
//   y[n, :] = scale table[ids[n], :]
//   dw[v, :] = scale sum over n with ids[n] = v of dy[n, :]
// An id outside the table has a row of NaN and no gradient; the padding id has no gradient.
//
// The gradient: the tokens are sorted by id, stably, so that the rows of one id are one run of the sorted order and
// are summed in token order whatever the timing; every row of dw is then written once, those of no token with zeros.
//   1. Radix sort of (id, token) in passes of up to 10 bits, least digit first. hist_kernel counts a chunk's digits,
//      scatter_kernel turns the counts of all chunks into first places and moves its chunk's pairs there; a token's
//      rank among the wave's lanes of its digit comes from one ballot per bit. Up to 4096 tokens one workgroup does
//      all passes in one launch. Ids without a gradient sort behind the table as id V.
//   2. pieces_kernel: every 16 places that are all one id become one row of partial sums, so that an id of many
//      tokens is not one wave's work; beside them, every id's first place is searched within its last digit's places.
//   3. rows_kernel: a wave has four rows of dw, and where they have few tokens loads those all at once. Else it adds a
//      row's places before its first piece, its pieces, and those after the last. An id of more than 16 pieces is a
//      workgroup's.
// Sums are fp32, rounded once to the table's type.
//
// Bound by memory (dy is read once, dw written once), and for fewer tokens by the chain of launches. Measured, bfloat16
// gradients, D 1024, tokens drawn by rank: 16376 tokens, V 32000, fp32 table: lookup 13.5 us, sort 18, pieces 5, rows
// 30 (131 MB written, 4.4 TB/s); 65528 tokens, V 131071, bfloat16 table: lookup 48, sort 25, pieces 17, rows 89 us (268
// MB written, 4.5 TB/s with the gradients read).

#include <algorithm>

#include "mg_vec.h"

namespace mg {
namespace embed_sorted {

constexpr int kDigit = 10, kBins = 1 << kDigit;  // at most
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / 64;
// Tokens that one workgroup sorts (3000 tokens: 50 us either way, in three launches fewer; 5000 and 8000: 69 and 74 us
// in one workgroup, 46 and 47 in several)
constexpr int kSmall = 4096;
constexpr int kMaxChunks = 256;
constexpr int kPiece = 16;
constexpr int kManyPieces = 16;    // an id of more is a workgroup's
constexpr int kThreads = 256, kWaves = 4;
constexpr int kVec = 8, kCols = 64 * kVec;  // columns of a lane and of a wave
constexpr int kRows = 4;                    // rows of dw per wave
constexpr int kFew = 4;                     // tokens of a wave's rows that are loaded at once
constexpr int64_t kMaxN = 1 << 27, kMaxV = 1 << 28;
constexpr int kMaxD = 1 << 30;  // (columns of a row are counted in 32 bits, a workgroup's share past the last one too)

struct Pairs {
  uint32_t *key, *pos;
};

// Passes and their digits: `bits` in all, `digit` each
struct Plan {
  int bits, passes, digit, bins, chunks;
  int64_t chunk;  // tokens of a chunk
};

struct Ids {
  const void* p;
  int wide;  // int64, not int32
  int64_t N, padding;
  uint32_t V;
  __device__ __forceinline__ uint32_t key(int64_t n) const {
    const int64_t v = wide ? static_cast<const int64_t*>(p)[n] : static_cast<const int32_t*>(p)[n];
    return v < 0 || v >= V || v == padding ? V : static_cast<uint32_t>(v);
  }
};

// ------------------------------------------------------------------ lookup

// N values (4 or 8) as loaded, of which the first `left` exist
template <typename T, int N> struct Pack {
  typedef T Raw __attribute__((ext_vector_type(N), aligned(sizeof(T))));
  Raw v;
  __device__ __forceinline__ void load(const T* p, int left) {
    if (left >= N) {
      v = *reinterpret_cast<const Raw*>(p);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = j < left ? p[j] : T(0);
    }
  }
  __device__ __forceinline__ float get(int j) const {
    if constexpr (sizeof(T) == 2)
      return bf16_to_f32(v[j]);
    else
      return v[j];
  }
  __device__ __forceinline__ void add_to(float (&acc)[N]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) acc[j] += get(j);
  }
  // kPast: past the nearest caches, as nothing here reads it again
  template <bool kPast>
  __device__ __forceinline__ static void store(T* p, int left, const float (&x)[N]) {
    Raw r;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if constexpr (sizeof(T) == 2)
        r[j] = f32_to_bf16(x[j]);
      else
        r[j] = x[j];
    }
    if (left >= N) {
      if constexpr (kPast)
        __builtin_nontemporal_store(r, reinterpret_cast<Raw*>(p));
      else
        *reinterpret_cast<Raw*>(p) = r;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < left) p[j] = r[j];
    }
  }
};
template <typename T>
constexpr int wide_of() { return 16 / sizeof(T); }  // values of an output that a lane stores at once: a wave's stores have no gaps
// Results larger than most of the last cache (256 MB) go past the caches where their rows fill cache lines: the
// gradient of a V131071 D1024 bf16 table 157 -> 115 us, of its fp32 one 256 -> 195; one that stays there is read from
// there next, and V32000 D1024 in fp32 takes 64 us, not 70. Lines that two rows share are better put together in the
// caches (V50001 D777: 78, not 91).
template <typename T>
inline bool past_caches(const T* p, int64_t rows, int D) {
  return aligned(p, 64) && D * sizeof(T) % 64 == 0 && static_cast<size_t>(rows) * D * sizeof(T) > size_t(192) << 20;
}

// `per` threads (a power of two) to a row
template <typename Tw, typename Ty, bool kPast>
__global__ __launch_bounds__(kThreads) void lookup_kernel(Ids ids, const Tw* __restrict__ table, Ty* __restrict__ y, int D, float scale,
                                                          int per) {
  constexpr int N = wide_of<Ty>();
  const int rows = kThreads / per, t = threadIdx.x & (per - 1);
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * rows + threadIdx.x / per; n < ids.N; n += static_cast<int64_t>(gridDim.x) * rows) {
    const uint32_t v = ids.key(n);
    const Tw* row = table + static_cast<int64_t>(v) * D;
    for (int c = t * N; c < D; c += per * N) {
      float x[N];
      if (v < ids.V) {
        Pack<Tw, N> w;
        w.load(row + c, D - c);
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = w.get(j) * scale;
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = __builtin_nanf("");
      }
      Pack<Ty, N>::template store<kPast>(y + n * D + c, D - c, x);
    }
  }
}

// ------------------------------------------------------------------ sort

// Lanes of the wave with this lane's digit d (live lanes only)
__device__ __forceinline__ uint64_t peers_of(bool live, uint32_t d, int bits) {
  uint64_t m = __ballot(live);
  for (int b = 0; b < bits; ++b) {
    const bool one = d >> b & 1;
    const uint64_t with = __ballot(live && one);
    m &= one ? with : ~with;
  }
  return m;
}

// A pass's source: the ids themselves first, then the pairs of the pass before
struct Source {
  Ids ids;
  const uint32_t *key, *pos;
  __device__ __forceinline__ uint32_t key_of(int64_t n) const { return key ? key[n] : ids.key(n); }
  __device__ __forceinline__ uint32_t pos_of(int64_t n) const { return key ? pos[n] : static_cast<uint32_t>(n); }
};

// counts[chunk][bin] of the digit at `shift` (added up by scatter_kernel where it moves the pairs, with atomics, the
// counts take 10 us of 65528 tokens, of which a few ids are many; this launch takes 3 to 5)
__global__ __launch_bounds__(kSortThreads) void hist_kernel(Source src, int64_t chunk, int shift, int bins, int* __restrict__ counts) {
  __shared__ int s_cnt[kBins];
  for (int i = threadIdx.x; i < bins; i += kSortThreads) s_cnt[i] = 0;
  __syncthreads();
  const int64_t n0 = blockIdx.x * chunk, n1 = std::min<int64_t>(src.ids.N, n0 + chunk);
  for (int64_t n = n0 + threadIdx.x; n < n1; n += kSortThreads) atomicAdd(&s_cnt[src.key_of(n) >> shift & (bins - 1)], 1);
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += kSortThreads) counts[static_cast<int64_t>(blockIdx.x) * bins + i] = s_cnt[i];
}

struct SortShared {
  int cnt[kSortWaves][kBins];  // of each wave's share of the chunk, then where its tokens of a digit go
  int wave[kSortWaves];
  int all[kSortThreads], before[kSortThreads];  // a bin's tokens by shares of the chunks
};

// One pass over a chunk by the whole workgroup. counts: those of all chunks, or null where this is the only one;
// starts (nullable): receives the first place of every bin, and N behind them.
__device__ void scatter(SortShared& s, const Source& src, int64_t n0, int64_t n1, int chunk_i, int chunks, const int* counts, int shift,
                        int digit, const Pairs& out, int* starts) {
  const int bins = 1 << digit, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t per = (n1 - n0 + kSortWaves - 1) / kSortWaves;
  const int64_t w0 = std::min<int64_t>(n1, n0 + wave * per), w1 = std::min<int64_t>(n1, w0 + per);
  // all loads at once: the wave's first tokens (up to 262144 tokens in all they are its only ones), and the bin's counts
  // of all chunks by as many threads as there are for it (one for each bin: 9.1 us at 64 chunks, for 7.9)
  uint32_t key0 = 0, pos0 = 0;
  if (w0 + lane < w1) key0 = src.key_of(w0 + lane), pos0 = src.pos_of(w0 + lane);
  int all = 0, before = 0;
  if (counts) {
    const int bin = threadIdx.x & (bins - 1), step = kSortThreads >> digit;
#pragma unroll 16
    for (int g = threadIdx.x >> digit; g < chunks; g += step) {
      const int c = counts[static_cast<int64_t>(g) * bins + bin];
      all += c;
      before += g < chunk_i ? c : 0;
    }
    s.all[threadIdx.x] = all, s.before[threadIdx.x] = before;
  }
  for (int w = 0; w < kSortWaves; ++w)
    for (int i = threadIdx.x; i < bins; i += kSortThreads) s.cnt[w][i] = 0;
  __syncthreads();
  for (int64_t n = w0 + lane; n < w1; n += 64)
    atomicAdd(&s.cnt[wave][(n == w0 + lane ? key0 : src.key_of(n)) >> shift & (bins - 1)], 1);
  __syncthreads();
  // a thread per bin: the waves' first places within the chunk's tokens of the bin; all tokens of the bin, and those
  // of the chunks before
  const int bin = threadIdx.x;
  if (bin < bins) {
    int own = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = s.cnt[w][bin];
      s.cnt[w][bin] = own;
      own += c;
    }
    if (counts) {
      for (int i = bin + bins; i < kSortThreads; i += bins) all += s.all[i], before += s.before[i];
    } else {
      all = own;
    }
  } else {
    all = 0;
  }
  // exclusive sums over the bins: within the wave, then over the waves
  int sum = all;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(sum, o, 64);
    if (lane >= o) sum += x;
  }
  if (lane == 63) s.wave[wave] = sum;
  __syncthreads();
  int first = sum - all;
  for (int w = 0; w < wave; ++w) first += s.wave[w];
  if (bin < bins) {
    if (starts) {
      starts[bin] = first;
      if (bin == bins - 1) starts[bins] = first + all;
    }
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) s.cnt[w][bin] += first + before;
  }
  __syncthreads();
  // (a wave's accesses to its counters are in program order)
  for (int64_t base = w0; base < w1; base += 64) {
    const int64_t n = base + lane;
    const bool live = n < w1;
    const bool again = base > w0 && live;
    const uint32_t key = again ? src.key_of(n) : key0, pos = again ? src.pos_of(n) : pos0, d = key >> shift & (bins - 1);
    const uint64_t m = peers_of(live, d, digit);
    if (live) {
      const int at = s.cnt[wave][d];
      const int p = at + __popcll(m & ((1ull << lane) - 1ull));
      out.key[p] = key;
      out.pos[p] = pos;
      if (63 - __clzll(m) == lane) s.cnt[wave][d] = at + __popcll(m);
    }
  }
}

__global__ __launch_bounds__(kSortThreads) void scatter_kernel(Source src, int64_t chunk, const int* __restrict__ counts, int shift,
                                                               int digit, Pairs out, int* __restrict__ starts) {
  __shared__ SortShared s;
  const int64_t n0 = blockIdx.x * chunk, n1 = std::min<int64_t>(src.ids.N, n0 + chunk);
  scatter(s, src, n0, n1, blockIdx.x, gridDim.x, counts, shift, digit, out, blockIdx.x == 0 ? starts : nullptr);
}

// All passes for up to kSmall tokens; the last one ends in `to`
__global__ __launch_bounds__(kSortThreads) void sort_small_kernel(Ids ids, int passes, int digit, Pairs other, Pairs to, int* __restrict__ starts) {
  __shared__ SortShared s;
  Source src = {ids, nullptr, nullptr};
  for (int p = 0; p < passes; ++p) {
    const Pairs& out = (passes - 1 - p) % 2 ? other : to;
    scatter(s, src, 0, ids.N, 0, 1, nullptr, p * digit, digit, out, p == passes - 1 ? starts : nullptr);
    __threadfence_block();
    __syncthreads();
    src.key = out.key, src.pos = out.pos;
  }
}

// ------------------------------------------------------------------ sums

// acc += rows pos[i], i = i0 .. i1 - 1, in order, of N columns from c on
template <int N, typename T>
__device__ __forceinline__ void add_rows(const T* __restrict__ dy, const uint32_t* __restrict__ pos, int64_t i0, int64_t i1, int D, int c,
                                         int left, float (&acc)[N]) {
  constexpr int kAhead = 8;
  int64_t i = i0;
  for (; i + kAhead <= i1; i += kAhead) {
    Pack<T, N> x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u].load(dy + static_cast<int64_t>(pos[i + u]) * D + c, left);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u].add_to(acc);
  }
  for (; i < i1; ++i) {
    Pack<T, N> x;
    x.load(dy + static_cast<int64_t>(pos[i]) * D + c, left);
    x.add_to(acc);
  }
}
template <int N>
__device__ __forceinline__ void add_parts(const float* __restrict__ part, int64_t p0, int64_t p1, int D, int c, int left, float (&acc)[N]) {
#pragma unroll 8
  for (int64_t p = p0; p < p1; ++p) {
    Pack<float, N> x;
    x.load(part + p * D + c, left);
    x.add_to(acc);
  }
}

// first[v]: the first place of id v, and of V
__device__ __forceinline__ void place(const uint32_t* __restrict__ key, const int* __restrict__ starts, int shift, uint32_t V, int64_t n,
                                      int* __restrict__ first) {
  if (n > V) return;
  const uint32_t v = static_cast<uint32_t>(n);
  int lo = starts[v >> shift], hi = starts[(v >> shift) + 1];
  while (lo < hi) {
    const int mid = lo + (hi - lo) / 2;
    if (key[mid] < v)
      lo = mid + 1;
    else
      hi = mid;
  }
  first[v] = lo;
}

// The first `piece_wgs` workgroups: part[p, :] = the sum of places [16 p, 16 p + 16) where they are all one id of the
// table, a wave per piece and kCols columns. The others: the ids' first places.
template <typename T>
__global__ __launch_bounds__(kThreads) void pieces_kernel(const T* __restrict__ dy, Pairs sorted, int64_t pieces, int piece_wgs, int cols, int D,
                                                          uint32_t V, float* __restrict__ part, const int* __restrict__ starts, int shift,
                                                          int* __restrict__ first) {
  if (blockIdx.x >= static_cast<uint32_t>(piece_wgs))
    return place(sorted.key, starts, shift, V, static_cast<int64_t>(blockIdx.x - piece_wgs) * kThreads + threadIdx.x, first);
  const int64_t p = static_cast<int64_t>(blockIdx.x / cols) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (p >= pieces) return;
  const uint32_t key = sorted.key[p * kPiece];
  if (key >= V || key != sorted.key[p * kPiece + kPiece - 1]) return;
  for (int c = (threadIdx.x % 64) * kVec + blockIdx.x % cols * kCols; c < D; c += cols * kCols) {
    float acc[kVec] = {};
    add_rows(dy, sorted.pos, p * kPiece, (p + 1) * kPiece, D, c, D - c, acc);
    Pack<float, kVec>::template store<false>(part + p * D + c, D - c, acc);
  }
}

// The pieces of the run [i0, i1): [p0, p1)
struct Run {
  int64_t i0, i1, p0, p1;
  __device__ __forceinline__ Run(int64_t a, int64_t b) : i0(a), i1(b), p0((a + kPiece - 1) / kPiece), p1(b / kPiece) {}
  __device__ __forceinline__ bool many() const { return p1 - p0 > kManyPieces; }
};

// An id of many pieces is a workgroup's: each wave sums a share of the pieces, the first wave the places before them
// too, the last those behind, and the shares are added in order. Such an id has at least one piece whose number is a
// multiple of kManyPieces; the workgroup of its first such piece has it.
template <typename T, typename Tw>
__device__ __forceinline__ void sum_run(const T* __restrict__ dy, const Pairs& sorted, const int* __restrict__ first,
                                        const float* __restrict__ part, Tw* __restrict__ dw, int D, uint32_t V, float scale, int64_t p) {
  constexpr int N = wide_of<Tw>();
  __shared__ float s_sum[kWaves][64 * N];
  const uint32_t key = sorted.key[p * kPiece];
  if (key >= V) return;
  const Run r(first[key], first[key + 1]);
  if (r.p0 > p || r.p0 <= p - kManyPieces || !r.many()) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int64_t share = (r.p1 - r.p0 + kWaves - 1) / kWaves, q0 = std::min(r.p1, r.p0 + wave * share), q1 = std::min(r.p1, q0 + share);
  for (int c0 = blockIdx.y * 64 * N; c0 < D; c0 += gridDim.y * 64 * N) {
    const int c = c0 + lane * N, left = D - c;
    float acc[N] = {};
    if (left > 0) {
      if (wave == 0) add_rows(dy, sorted.pos, r.i0, r.p0 * kPiece, D, c, left, acc);
      add_parts(part, q0, q1, D, c, left, acc);
      if (wave == kWaves - 1) add_rows(dy, sorted.pos, r.p1 * kPiece, r.i1, D, c, left, acc);
    }
#pragma unroll
    for (int j = 0; j < N; ++j) s_sum[wave][j * 64 + lane] = acc[j];
    __syncthreads();
    if (wave == 0 && left > 0) {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float t = s_sum[0][j * 64 + lane];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) t += s_sum[w][j * 64 + lane];
        acc[j] = t * scale;
      }
      Pack<Tw, N>::template store<false>(dw + static_cast<int64_t>(key) * D + c, left, acc);
    }
    __syncthreads();
  }
}

// The first `run_wgs` workgroups: ids of many pieces. The others: kRows rows of dw to a wave.
template <typename T, typename Tw, bool kPast>
__global__ __launch_bounds__(kThreads) void rows_kernel(const T* __restrict__ dy, Pairs sorted, const int* __restrict__ first,
                                                        const float* __restrict__ part, Tw* __restrict__ dw, int D, uint32_t V, float scale,
                                                        uint32_t run_wgs) {
  const uint32_t wg = blockIdx.z * gridDim.x + blockIdx.x;
  if (wg < run_wgs) return sum_run(dy, sorted, first, part, dw, D, V, scale, static_cast<int64_t>(wg) * kManyPieces);
  const int64_t v0 = (static_cast<int64_t>(wg - run_wgs) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / 64)) * kRows;
  if (v0 >= V) return;
  int at[kRows + 1];
#pragma unroll
  for (int q = 0; q <= kRows; ++q) at[q] = first[std::min<int64_t>(v0 + q, V)];
  const int n = at[kRows] - at[0];
  constexpr int N = wide_of<Tw>(), kWide = 64 * N;
  for (int c = (threadIdx.x % 64) * N + blockIdx.y * kWide; c < D; c += gridDim.y * kWide) {
    const int left = D - c;
    Tw* out = dw + v0 * D + c;
    const auto write = [&](int q, float (&acc)[N]) {
#pragma unroll
      for (int j = 0; j < N; ++j) acc[j] *= scale;
      Pack<Tw, N>::template store<kPast>(out + static_cast<int64_t>(q) * D, left, acc);
    };
    if (n <= kFew) {
      Pack<T, N> x[kFew];
#pragma unroll
      for (int u = 0; u < kFew; ++u)
        if (u < n) x[u].load(dy + static_cast<int64_t>(sorted.pos[at[0] + u]) * D + c, left);
#pragma unroll
      for (int q = 0; q < kRows; ++q) {
        if (v0 + q >= V) break;
        float acc[N] = {};
#pragma unroll
        for (int u = 0; u < kFew; ++u)
          if (at[0] + u >= at[q] && at[0] + u < at[q + 1]) x[u].add_to(acc);
        write(q, acc);
      }
    } else {
#pragma unroll 1
      for (int q = 0; q < kRows; ++q) {
        if (v0 + q >= V) break;
        const Run r(first[v0 + q], first[v0 + q + 1]);
        if (r.many()) continue;
        float acc[N] = {};
        if (r.p0 < r.p1) {
          add_rows(dy, sorted.pos, r.i0, r.p0 * kPiece, D, c, left, acc);
          add_parts(part, r.p0, r.p1, D, c, left, acc);
          add_rows(dy, sorted.pos, r.p1 * kPiece, r.i1, D, c, left, acc);
        } else {
          add_rows(dy, sorted.pos, r.i0, r.i1, D, c, left, acc);
        }
        write(q, acc);
      }
    }
  }
}

// ------------------------------------------------------------------ host

inline Plan plan_of(int64_t N, int64_t V) {
  Plan p = {};
  p.bits = 1;
  while (V >> p.bits) ++p.bits;  // (ids to V, which is the one without a gradient)
  p.passes = (p.bits + kDigit - 1) / kDigit;
  p.digit = (p.bits + p.passes - 1) / p.passes;
  p.bins = 1 << p.digit;
  if (N <= kSmall) {
    p.chunks = 1, p.chunk = N;
  } else {
    p.chunk = std::max<int64_t>(kSortThreads, (N + kMaxChunks - 1) / kMaxChunks);
    p.chunks = static_cast<int>((N + p.chunk - 1) / p.chunk);
  }
  return p;
}

// Workspace: [pieces][D] partial sums, counts of each chunk, first places of the last digits and of the ids, two sets
// of pairs
struct Layout {
  size_t counts, starts, first, pairs, total;
  int64_t pieces;
};
inline Layout layout_of(int64_t N, int D, int64_t V, const Plan& p) {
  const auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  Layout l;
  l.pieces = N / kPiece;
  l.counts = up(static_cast<size_t>(l.pieces) * D * 4);
  l.starts = l.counts + up(static_cast<size_t>(p.chunks) * p.bins * 4);
  l.first = l.starts + up((static_cast<size_t>(p.bins) + 1) * 4);
  l.pairs = l.first + up((static_cast<size_t>(V) + 1) * 4);
  l.total = l.pairs + 4 * up(static_cast<size_t>(N) * 4);
  return l;
}

inline int check_ids(const char* fn, int id_bytes, const void* ids, int64_t N, int D, int64_t V) {
  if (N < 1 || N >= kMaxN || D < 1 || D >= kMaxD || V < 1 || V >= kMaxV)
    return fail(MG_ERR_ARG, "%s: N=%lld, D=%d, V=%lld must be at least 1, N below 2^27, D below 2^30, V below 2^28", fn, (long long)N, D, (long long)V);
  if (id_bytes != 4 && id_bytes != 8) return fail(MG_ERR_DTYPE, "%s: ids of %d bytes", fn, id_bytes);
  if (!ids || !aligned(ids, id_bytes)) return fail(MG_ERR_ARG, "%s: ids NULL or misaligned", fn);
  return MG_OK;
}
inline int check_p(const char* fn, const char* name, const void* p, int dt) {
  if (dt != MG_F32 && dt != MG_BF16) return fail(MG_ERR_DTYPE, "%s: %s dtype %d unsupported", fn, name, dt);
  if (!p || !aligned(p, dt == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: %s NULL or misaligned", fn, name);
  return MG_OK;
}

template <typename Tw, typename Ty>
void launch_lookup(const Ids& ids, const void* table, void* y, int D, float scale, hipStream_t st) {
  int per = 1;
  while (per < kThreads && per * wide_of<Ty>() < D) per *= 2;
  const int64_t wgs = (ids.N + kThreads / per - 1) / (kThreads / per);
  const auto go = [&](auto past) {
    hipLaunchKernelGGL((lookup_kernel<Tw, Ty, decltype(past)::value>), dim3(std::min<int64_t>(wgs, 1 << 20)), dim3(kThreads), 0, st, ids,
                       static_cast<const Tw*>(table), static_cast<Ty*>(y), D, scale, per);
  };
  past_caches(static_cast<Ty*>(y), ids.N, D) ? go(std::true_type{}) : go(std::false_type{});
}

template <typename T, typename Tw>
void launch_sums(const void* dy, const Pairs& sorted, const int* starts, int shift, int* first, float* part, int64_t pieces, void* dw, int D,
                 int64_t V, float scale, hipStream_t st) {
  const int cols = std::min((D + kCols - 1) / kCols, 16);
  const uint32_t v = static_cast<uint32_t>(V);
  const T* g = static_cast<const T*>(dy);
  Tw* w = static_cast<Tw*>(dw);
  const int64_t piece_wgs = (pieces + kWaves - 1) / kWaves * cols, place_wgs = (V + kThreads) / kThreads;
  hipLaunchKernelGGL((pieces_kernel<T>), dim3(piece_wgs + place_wgs), dim3(kThreads), 0, st, g, sorted, pieces, static_cast<int>(piece_wgs), cols, D,
                     v, part, starts, shift, first);
  const uint32_t run_wgs = pieces > kManyPieces ? (pieces + kManyPieces - 1) / kManyPieces : 0;
  constexpr int kWide = 64 * wide_of<Tw>();
  const uint32_t wgs = run_wgs + (v + kWaves * kRows - 1) / (kWaves * kRows), z = (wgs >> 20) + 1;  // (x below 2^32 threads)
  const auto rows = [&](auto past) {
    hipLaunchKernelGGL((rows_kernel<T, Tw, decltype(past)::value>), dim3((wgs + z - 1) / z, std::min((D + kWide - 1) / kWide, 64), z), dim3(kThreads),
                       0, st, g, sorted, first, part, w, D, v, scale, run_wgs);
  };
  past_caches(w, V, D) ? rows(std::true_type{}) : rows(std::false_type{});
}

}  // namespace embed_sorted
}  // namespace mg

using namespace mg;

extern "C" int mg_embedding_fwd(int id_bytes, const void* ids, int64_t N, int table_dtype, const void* table, int64_t V, int D, float scale,
                                int y_dtype, void* y, void* stream) {
  using namespace embed_sorted;
  const char* fn = "mg_embedding_fwd";
  int rc;
  if ((rc = check_ids(fn, id_bytes, ids, N, D, V)) || (rc = check_p(fn, "table", table, table_dtype)) || (rc = check_p(fn, "y", y, y_dtype)))
    return rc;
  const Ids in = {ids, id_bytes == 8, N, -1, static_cast<uint32_t>(V)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (table_dtype == MG_BF16)
    y_dtype == MG_BF16 ? launch_lookup<bf16_t, bf16_t>(in, table, y, D, scale, st) : launch_lookup<bf16_t, float>(in, table, y, D, scale, st);
  else
    y_dtype == MG_BF16 ? launch_lookup<float, bf16_t>(in, table, y, D, scale, st) : launch_lookup<float, float>(in, table, y, D, scale, st);
  return check_launch(fn);
}

extern "C" size_t mg_embedding_sorted_bwd_workspace_bytes(int64_t N, int D, int64_t V) {
  using namespace embed_sorted;
  if (N < 1 || N >= kMaxN || D < 1 || D >= kMaxD || V < 1 || V >= kMaxV) return 0;
  return layout_of(N, D, V, plan_of(N, V)).total;
}

extern "C" int mg_embedding_sorted_bwd(int id_bytes, const void* ids, int64_t N, int dy_dtype, const void* dy, int D, int64_t V, float scale,
                                       int64_t padding, int dw_dtype, void* dw, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace embed_sorted;
  const char* fn = "mg_embedding_sorted_bwd";
  int rc;
  if ((rc = check_ids(fn, id_bytes, ids, N, D, V)) || (rc = check_p(fn, "dy", dy, dy_dtype)) || (rc = check_p(fn, "dw", dw, dw_dtype))) return rc;
  const Plan p = plan_of(N, V);
  const Layout l = layout_of(N, D, V, p);
  if (!workspace || workspace_bytes < l.total || !aligned(workspace, 256))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or misaligned)", fn, workspace_bytes, l.total);
  char* ws = static_cast<char*>(workspace);
  float* part = reinterpret_cast<float*>(ws);
  int* counts = reinterpret_cast<int*>(ws + l.counts);
  int* starts = reinterpret_cast<int*>(ws + l.starts);
  const size_t each = (l.total - l.pairs) / 4;
  uint32_t* arr[4];
  for (int i = 0; i < 4; ++i) arr[i] = reinterpret_cast<uint32_t*>(ws + l.pairs + i * each);
  const Pairs set[2] = {{arr[0], arr[1]}, {arr[2], arr[3]}};
  const Ids in = {ids, id_bytes == 8, N, padding, static_cast<uint32_t>(V)};
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Pairs& sorted = set[0];
  if (p.chunks == 1 && N <= kSmall) {
    hipLaunchKernelGGL(sort_small_kernel, dim3(1), dim3(kSortThreads), 0, st, in, p.passes, p.digit, set[1], set[0], starts);
  } else {
    Source src = {in, nullptr, nullptr};
    for (int i = 0; i < p.passes; ++i) {
      const Pairs& out = set[(p.passes - 1 - i) % 2];
      hipLaunchKernelGGL(hist_kernel, dim3(p.chunks), dim3(kSortThreads), 0, st, src, p.chunk, i * p.digit, p.bins, counts);
      hipLaunchKernelGGL(scatter_kernel, dim3(p.chunks), dim3(kSortThreads), 0, st, src, p.chunk, counts, i * p.digit, p.digit, out,
                         i == p.passes - 1 ? starts : nullptr);
      src.key = out.key, src.pos = out.pos;
    }
  }
  int* first = reinterpret_cast<int*>(ws + l.first);
  const int shift = (p.passes - 1) * p.digit;
  if (dy_dtype == MG_BF16)
    dw_dtype == MG_BF16 ? launch_sums<bf16_t, bf16_t>(dy, sorted, starts, shift, first, part, l.pieces, dw, D, V, scale, st)
                        : launch_sums<bf16_t, float>(dy, sorted, starts, shift, first, part, l.pieces, dw, D, V, scale, st);
  else
    dw_dtype == MG_BF16 ? launch_sums<float, bf16_t>(dy, sorted, starts, shift, first, part, l.pieces, dw, D, V, scale, st)
                        : launch_sums<float, float>(dy, sorted, starts, shift, first, part, l.pieces, dw, D, V, scale, st);
  return check_launch(fn);
}
