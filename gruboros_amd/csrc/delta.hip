// The gated delta rule for gfx950: over sequences in chunks (forward and
// backward) and for single tokens.
//
// Per (batch, head), with a state S in R^{K x V}, decay e^{g_t} and write
// strength beta_t:
//   S_t = e^{g_t} S_{t-1} + beta_t k_t (v_t - e^{g_t} S_{t-1}^T k_t)^T,
//   o_t = scale S_t^T q_t.
// A chunk of C = 64 tokens with entry state S, G = cumsum(g) in the chunk and
// D_ij = e^{G_i - G_j} (j <= i):
//   A_ij = beta_i D_ij k_i.k_j (j < i),  T = (I + A)^-1,  P_ij = scale D_ij q_i.k_j (j <= i)
//   y = beta (v - e^G (K S)),  d = T y,
//   o = scale e^G (Q S) + P d,
//   S' = e^{G_C} S + K^T (e^{G_C - G} d).
// Backward, from do and dS' (the gradient of the chunk's exit state):
//   dd = P^T do + e^{G_C - G} (K dS'),  dy = T^T dd,  dv = beta dy,
//   dS = e^{G_C} dS' + Q^T (scale e^G do) - K^T (e^G beta dy);
//   N_ij = scale D_ij do_i.d_j (j <= i),  F_ij = D_ij dy_i.d_j (j < i),
//   Z = e^G (dy S^T) + F K,
//   dq = scale e^G (do S^T) + N K,
//   dk = e^{G_C - G} (d dS'^T) + N^T Q - F^T (beta K) - beta Z,
//   dbeta = dy.v - k.Z,
//   dg_t = <S', dS'> + sum_{i >= t in the chunk} (q_i.dq_i - v_i.dv_i).
// The last line: with c_i = e^{G_i}, the rule for S_i / c_i has no decay and
// sees v_i / c_i, c_i q_i and (at the end) c_C; the gradient of log c_i follows
// from theirs.
//
// Three kinds of kernel:
//   chunk_kernel  one workgroup per (chunk, head), all in parallel: T, P and the decays;
//   state_kernel, dstate_kernel  the pass over the chunks in order. A wave owns
//     16 value columns of S for good, in the accumulators of its matrix
//     instructions: every product of the chain (K S, T y, P d, K^T d) contracts
//     the rows and keeps the columns, and the accumulator layout (lane = column,
//     registers = rows) is the B operand's layout up to the order of the rows,
//     which the A operands read from LDS make up for. So the chain never leaves
//     the wave's registers, and waves only share the chunk's A operands in LDS;
//   grad_kernel   one workgroup per (chunk, head): what contracts the value columns.
//
// Matrix operands are bf16. An fp32 value enters as limbs, x = h + m + l with 8
// bits each (exact), and the limb products down to 2^-16 of the leading one are
// summed in fp32: states, T, y and d are never rounded to bf16. bf16 inputs are
// one limb, so a product with one costs three instructions at most; fp32 inputs
// are three, and a product six.

#include <algorithm>

#include "mg_common.h"

namespace mg {
namespace delta {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

constexpr int C = 64;           // tokens per chunk
constexpr int kPlane = C * C;   // elements of one limb of T or P
constexpr float kMinLog = -200.0f;  // decays below e^-104 are zero in fp32: kept finite for the differences

struct Args {
  int B, T, Hk, H, K, V, NC, VP;
  float scale;
  const char *q, *k, *v, *g, *beta;
  int64_t q_sb, q_st, q_sh, k_sb, k_st, k_sh, v_sb, v_st, v_sh, g_sb, g_st, g_sh, b_sb, b_st, b_sh;
  const float* h0;       // [B, H, K, V] or null
  char* o;               // [B, T, H, V]
  float* state;          // [B, H, K, V] or null
  // chunk data, index c = (b H + h) NC + n
  char* img;             // [c][Tile::kBytes]: the chunk's operands as they lie in LDS
  double* Gd;            // [c][64]
  bf16_t* Sw;            // kept for the backward: each chunk's entry state, [c][VP / 32][NW][32][KP]
  bf16_t* dw;            // d, [c][VP / 32][NW][32][64]
  // backward
  const char* dout;      // [B, T, H, V]
  int64_t do_sb, do_st, do_sh;
  const float* dstate;   // or null
  bf16_t* dSw;           // the gradients of the exit states, as Sw
  bf16_t* yw;            // dy, as dw
  char *dq, *dk, *dv, *dg, *db;
  float* dh0;
  float *dqp, *dkp;      // shared heads: [B, T, H, K] before their sum
};

// ---------------------------------------------------------------- limbs

__device__ __forceinline__ uint32_t hi16x2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t lo16x2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x05040100u); }

// 8 fp32 values as N limbs. N = 3: by cutting the mantissa (8 + 8 + 8 bits, exact). N = 2: the second
// limb rounded to nearest, off by 2^-17 at most.
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&out)[N]) {
  u32x4 w[N];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
    w[0][i] = hi16x2(__float_as_uint(a), __float_as_uint(b));
    if constexpr (N > 1) {
      a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
      b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
      if constexpr (N == 2) {
        w[1][i] = pack_bf16x2(a, b);
      } else {
        w[1][i] = hi16x2(__float_as_uint(a), __float_as_uint(b));
        a -= __uint_as_float(__float_as_uint(a) & 0xffff0000u);
        b -= __uint_as_float(__float_as_uint(b) & 0xffff0000u);
        w[2][i] = hi16x2(__float_as_uint(a), __float_as_uint(b));
      }
    }
  }
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = __builtin_bit_cast(bf16x8, w[l]);
}

// Limbs of what is kept for the backward's products: two of a state or update of bf16 inputs (2^-16,
// far below the rounding of the gradients they end in), all three of fp32 inputs.
template <int NI>
constexpr int kKept = NI == 3 ? 3 : 2;

// c += a b over the limb products (i, j) with i + j < ORD, the small ones first
template <int ORD, int NA, int NB>
__device__ __forceinline__ f32x4 mm(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 c) {
#pragma unroll
  for (int s = ORD - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c, 0, 0, 0);
  return c;
}

// ---------------------------------------------------------------- elements

template <int NI> struct elem { using type = bf16_t; };
template <> struct elem<3> { using type = float; };

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void st(float* p, float x) { *p = x; }
__device__ __forceinline__ void st(bf16_t* p, float x) { *p = f32_to_bf16(x); }

// Column accesses of the passes over the chunks: a buffer over the chunk's rows of one head, the lane's
// column and first row in its offset, a scalar offset per register. Rows and columns past the end are
// out of the buffer's range: they read as zero and are not written.
constexpr uint32_t kOutOfRange = 0x80000000u;
template <typename E>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const E* p, int64_t st_, int rows, int cols) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(p), static_cast<short>(0),
                                           static_cast<int>(((rows - 1) * st_ + cols) * sizeof(E)), 0x00020000);
}
template <typename E>
__device__ __forceinline__ uint32_t load_col(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t row_off) {  // raw
  if constexpr (sizeof(E) == 2)
    return __builtin_amdgcn_raw_buffer_load_b16(r, off, row_off, 0);
  else
    return __builtin_amdgcn_raw_buffer_load_b32(r, off, row_off, 0);
}
template <typename E>
__device__ __forceinline__ float value(uint32_t raw) {
  return __uint_as_float(sizeof(E) == 2 ? raw << 16 : raw);
}
template <typename E>
__device__ __forceinline__ void store_col(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t row_off, float x) {
  if constexpr (sizeof(E) == 2)
    __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(x), r, off, row_off, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), r, off, row_off, 0);
}

// 8 consecutive values as limbs; nothing (zero) unless ok
__device__ __forceinline__ void load8(const bf16_t* p, bool ok, bf16x8 (&out)[1]) {
  const u32x4 z = {0, 0, 0, 0};
  out[0] = __builtin_bit_cast(bf16x8, ok ? *reinterpret_cast<const u32x4*>(p) : z);
}
__device__ __forceinline__ void load8(const float* p, bool ok, bf16x8 (&out)[3]) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float4 v = ok ? reinterpret_cast<const float4*>(p)[i] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
  }
  split<3>(x, out);
}

// ---------------------------------------------------------------- LDS operands
//
// A matrix of U 16-byte units per row; unit u of row r lies at u ^ swz(r), so that the 16 rows of a
// fragment (in the row order below) spread over the banks.

__device__ __forceinline__ int swz(int r) { return (r & 3) | ((r >> 1) & 4); }
template <int U>
__device__ __forceinline__ int at(int r, int u) { return (r * U + (u ^ swz(r))) * 16; }

// Row order of 16-row tile t of a matrix whose rows are contracted next: accumulator rows 4 g + i of
// the tiles 2 p and 2 p + 1 are rows 32 p + 8 g + i and 32 p + 8 g + 4 + i, so that lane group g holds
// rows 32 p + 8 g ... + 7: the k order of the B operand.
__device__ __forceinline__ int row_of(int t, int m) { return 32 * (t >> 1) + 8 * (m >> 2) + 4 * (t & 1) + (m & 3); }

// A operand: tile t (in row_of order) of a row-major matrix, k = 32 kb ... + 31
template <int U>
__device__ __forceinline__ bf16x8 frag(const char* m, int t, int kb, int lane) {
  return *reinterpret_cast<const bf16x8*>(m + at<U>(row_of(t, lane & 15), 4 * kb + (lane >> 4)));
}
// the same with rows in their own order
template <int U>
__device__ __forceinline__ bf16x8 frag_plain(const char* m, int t, int kb, int lane) {
  return *reinterpret_cast<const bf16x8*>(m + at<U>(16 * t + (lane & 15), 4 * kb + (lane >> 4)));
}
// Operand whose rows are the matrix's columns and whose k are its rows 32 p ... + 31, through the
// transposing LDS read: in each 16 lanes, lane 4 j + q addresses row j, columns 4 q ... 4 q + 3, and
// lane i receives column i of the four rows. PERM: columns of tile t in row_of order.
template <int U, bool PERM>
__device__ __forceinline__ bf16x8 frag_t(const char* m, int t, int p, int lane) {
  const int g = lane >> 4, j = (lane >> 2) & 3, q = lane & 3;
  const int u = PERM ? 4 * (t >> 1) + q : 2 * t + (q >> 1), half = PERM ? t & 1 : q & 1;
  const int r = 32 * p + 8 * g + j;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(m + at<U>(r, u) + 8 * half));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(m + at<U>(r + 4, u) + 8 * half));
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// One chunk's operands as chunk_kernel leaves them in memory and the other kernels keep them in LDS:
// limb planes of k and q [64][KP], of T and P [64][64], all with their units at at<>(), and the vectors
// e^G, e^{G_C - G}, beta. An image is copied as it is, 1 KiB per wave instruction and straight into LDS:
// no strides, masks or swizzles where the time counts, at the price of writing k and q once more.
template <int KP, int NI>
struct Tile {
  static constexpr int NP = NI == 3 ? 3 : 2;
  static constexpr int U = KP / 8;
  static constexpr int kK = 0, kQ = NI * C * KP * 2, kT = 2 * kQ, kP = kT + 3 * kPlane * 2, kGate = kP + NP * kPlane * 2;
  static constexpr int kBytes = kGate + 1024;
  static constexpr int kStages = 2 * kBytes <= 160 * 1024 ? 2 : 1;
};

template <int BYTES, int WAVES>
__device__ __forceinline__ void stage(char* lds, const void* src, int lane, int wave) {
  const __amdgpu_buffer_rsrc_t rsrc =
      __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(src), static_cast<short>(0), BYTES, 0x00020000);
  int off = wave * 1024;
#pragma unroll
  for (int i = 0; i < (BYTES / 1024 + WAVES - 1) / WAVES; ++i) {
    asm volatile("" : "+s"(off));  // (one running offset: else every copy's is kept in registers of its own)
    if ((i + 1) * WAVES <= BYTES / 1024 || i * WAVES + wave < BYTES / 1024)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(lds + off), 16, lane * 16, off, 0, 0);
    off += WAVES * 1024;
  }
}

__device__ __forceinline__ void staged() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

// ---------------------------------------------------------------- T, P and the decays of a chunk

constexpr int LD = 68;  // floats per row of the 64 x 64 matrices in LDS

__device__ __forceinline__ f32x4 mm16(const float* a, int lda, const float* b, f32x4 c, int lane) {
  const int m = lane & 15, g = lane >> 4;  // 16 x 16 x 16 in fp32, k = 4 g + s
#pragma unroll
  for (int s = 0; s < 4; ++s)
    c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m * lda + 4 * g + s], b[(4 * g + s) * LD + m], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 mm16(const float* a, f32x4 b, f32x4 c, int lane) {  // b: an accumulator
  const int m = lane & 15, g = lane >> 4;
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[m * LD + 4 * g + s], b[s], c, 0, 0, 0);
  return c;
}

// A 64 x 64 lower triangle from LDS to N limb planes, 16 values per thread
template <int N>
__device__ __forceinline__ void put_planes(const float* m, char* out, int tid) {
  const int r = tid >> 2, c0 = 16 * (tid & 3);
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int c = c0 + 8 * u + i;
      x[i] = c <= r ? m[r * LD + c] : 0.0f;
    }
    bf16x8 l[N];
    split<N>(x, l);
#pragma unroll
    for (int i = 0; i < N; ++i) *reinterpret_cast<bf16x8*>(out + i * kPlane * 2 + at<8>(r, c0 / 8 + u)) = l[i];
  }
}

template <int KP, int NI>
__global__ __launch_bounds__(256) void chunk_kernel(Args a) {
  using E = typename elem<NI>::type;
  using L = Tile<KP, NI>;
  __shared__ float sA[C * LD], sP[C * LD], sT[C * LD];
  __shared__ double sG[C];
  __shared__ float sB[C];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x;
  const int n = static_cast<int>(c % a.NC), bh = static_cast<int>(c / a.NC), h = bh % a.H, b = bh / a.H, grp = a.H / a.Hk;
  const int hk = h / grp, t0 = n * C, rows = min(C, a.T - t0);
  const E* k = reinterpret_cast<const E*>(a.k) + b * a.k_sb + t0 * a.k_st + hk * a.k_sh;
  const E* q = reinterpret_cast<const E*>(a.q) + b * a.q_sb + t0 * a.q_st + hk * a.q_sh;
  char* img = a.img + c * L::kBytes;
  if (wave == 0) {
    float gv = 0.0f, bv = 0.0f;
    if (lane < rows) {
      gv = ld(reinterpret_cast<const E*>(a.g) + b * a.g_sb + (t0 + lane) * a.g_st + h * a.g_sh);
      bv = ld(reinterpret_cast<const E*>(a.beta) + b * a.b_sb + (t0 + lane) * a.b_st + h * a.b_sh);
      gv = gv < kMinLog ? kMinLog : gv;
    }
    // the sums in 64 bits: what counts is their differences, also behind a token that forgets all
    double s = gv;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_up(s, o, 64);
      if (lane >= o) s += x;
    }
    const double last = __shfl(s, 63, 64);
    sG[lane] = s;
    sB[lane] = bv;
    float* gt = reinterpret_cast<float*>(img + L::kGate);
    gt[lane] = expf(static_cast<float>(s));
    gt[64 + lane] = expf(static_cast<float>(last - s));
    gt[128 + lane] = bv;
    gt[192 + lane] = 0.0f;
    a.Gd[c * 64 + lane] = s;
  }
  // k k^T, rows 16 wave ...; q k^T, rows 16 (3 - wave) ...: five blocks of the lower triangles each
  const int wq = 3 - wave;
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kk[i] = f32x4{0, 0, 0, 0}, qk[i] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int kb = 0; kb < KP / 32; ++kb) {
    const int d = 32 * kb + 8 * g;
    bf16x8 ak[NI], aq[NI];
    load8(k + (16 * wave + m) * a.k_st + d, 16 * wave + m < rows && d < a.K, ak);
    load8(q + (16 * wq + m) * a.q_st + d, 16 * wq + m < rows && d < a.K, aq);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i <= wave || i <= wq) {
        bf16x8 bk[NI];
        load8(k + (16 * i + m) * a.k_st + d, 16 * i + m < rows && d < a.K, bk);
        if (i <= wave) kk[i] = mm<NI>(ak, bk, kk[i]);
        if (i <= wq) qk[i] = mm<NI>(aq, bk, qk[i]);
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int col = 16 * i + m;
      if (i <= wave) {
        const int row = 16 * wave + 4 * g + r;
        sA[row * LD + col] = col < row ? sB[row] * expf(static_cast<float>(sG[row] - sG[col])) * kk[i][r] : 0.0f;
      }
      if (i <= wq) {
        const int row = 16 * wq + 4 * g + r;
        sP[row * LD + col] = col <= row ? a.scale * expf(static_cast<float>(sG[row] - sG[col])) * qk[i][r] : 0.0f;
      }
    }
  }
  __syncthreads();
  // (I + A)^-1: diagonal blocks of 16 by forward substitution (a lane per column), then the blocks
  // below them, X_ij = -T_ii (A X)_ij, on the fp32 matrix instructions
  if (lane < 16) {
    const float* A = sA + 16 * wave * LD + 16 * wave;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == lane ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) s -= A[i * LD + j] * x[j];
      x[i] = s;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) sT[(16 * wave + i) * LD + 16 * wave + lane] = x[i];
  }
  __syncthreads();
  const auto blk = [](float* p, int i, int j) { return p + 16 * i * LD + 16 * j; };
  const auto put = [&](int i, int j, f32x4 x) {
#pragma unroll
    for (int r = 0; r < 4; ++r) sT[(16 * i + 4 * g + r) * LD + 16 * j + m] = -x[r];
  };
  const f32x4 zero = {0, 0, 0, 0};
  if (wave < 2) {
    const int j = 2 * wave, i = j + 1;
    const f32x4 y = mm16(blk(sA, i, j), LD, blk(sT, j, j), zero, lane);
    put(i, j, mm16(blk(sT, i, i), y, zero, lane));
  }
  __syncthreads();
  {
    const int i = 2 + (wave >> 1), j = wave & 1;
    f32x4 y2 = mm16(blk(sA, 2, j), LD, blk(sT, j, j), zero, lane), x;
    if (j == 0) y2 = mm16(blk(sA, 2, 1), LD, blk(sT, 1, 0), y2, lane);
    x = mm16(blk(sT, i, 2), y2, zero, lane);
    if (i == 3) {
      f32x4 y3 = mm16(blk(sA, 3, j), LD, blk(sT, j, j), zero, lane);
      if (j == 0) y3 = mm16(blk(sA, 3, 1), LD, blk(sT, 1, 0), y3, lane);
      x = mm16(blk(sT, 3, 3), y3, x, lane);
    }
    put(i, j, x);
  }
  __syncthreads();
  put_planes<3>(sT, img + L::kT, tid);
  put_planes<L::NP>(sP, img + L::kP, tid);
  for (int i = tid; i < C * L::U; i += 256) {
    const int r = i / L::U, u = i % L::U;
    const bool ok = r < rows && 8 * u < a.K;
    bf16x8 lk[NI], lq[NI];
    load8(k + r * a.k_st + 8 * u, ok, lk);
    load8(q + r * a.q_st + 8 * u, ok, lq);
#pragma unroll
    for (int l = 0; l < NI; ++l) {
      *reinterpret_cast<bf16x8*>(img + L::kK + l * C * KP * 2 + at<L::U>(r, u)) = lk[l];
      *reinterpret_cast<bf16x8*>(img + L::kQ + l * C * KP * 2 + at<L::U>(r, u)) = lq[l];
    }
  }
}

// ---------------------------------------------------------------- the pass over the chunks

// Workgroups of one (batch, head) differ by the value columns and read the same chunk operands: ids
// that are equal modulo the 8 XCDs, so that they share an L2.
__device__ __forceinline__ void place(int id, int BH, int tiles, int& bh, int& tile) {
  const int full = BH / 8 * 8 * tiles;
  if (id < full) {
    const int r = id % (8 * tiles);
    bh = id / (8 * tiles) * 8 + r % 8;
    tile = r / 8;
  } else {
    const int r = id - full, rest = BH % 8;
    bh = BH / 8 * 8 + r % rest;
    tile = r / rest;
  }
}

// Rows (accumulator order) of two adjacent tiles as 8 values of a B operand
__device__ __forceinline__ void pair8(const f32x4& a, const f32x4& b, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
template <int N>
__device__ __forceinline__ void split_pair(const f32x4& a, const f32x4& b, bf16x8 (&out)[N]) {
  float x[8];
  pair8(a, b, x);
  split<N>(x, out);
}

template <int U, int N>
__device__ __forceinline__ void frags(const char* m, int plane, int t, int kb, int lane, bf16x8 (&out)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = frag<U>(m + l * plane, t, kb, lane);
}
template <int U, bool PERM, int N>
__device__ __forceinline__ void frags_t(const char* m, int plane, int t, int p, int lane, bf16x8 (&out)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = frag_t<U, PERM>(m + l * plane, t, p, lane);
}

// Limbs of an operand (lane = column, 8 rows per register group) to an image of [columns][rows]
template <int U, int NW, int N>
__device__ __forceinline__ void keep(bf16_t* img, int plane, int row, int u, const bf16x8 (&x)[N]) {
#pragma unroll
  for (int l = 0; l < NW; ++l) *reinterpret_cast<bf16x8*>(reinterpret_cast<char*>(img) + l * plane + at<U>(row, u)) = x[l];
}

// What a wave of the passes works on
template <int KP, int NI, int W>
struct Place {
  int lane, wave, m, g, bh, h, b, col;
  bool in;
  __device__ __forceinline__ Place(const Args& a, int tiles) {
    lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), m = lane & 15, g = lane >> 4;
    int tile;
    place(blockIdx.x, a.B * a.H, tiles, bh, tile);
    h = bh % a.H, b = bh / a.H, col = (tile * W + wave) * 16 + m;
    in = col < a.V;
  }
};

// The state (or its gradient) of a head's columns from dense [K][V] fp32, or zero
template <int KT, typename P>
__device__ __forceinline__ void load_state(f32x4 (&S)[KT], const float* s, const Args& a, const P& w) {
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      S[t][r] = s && w.in && row_of(t, 4 * w.g) < a.K  // (K % 8 == 0)
                    ? s[(static_cast<int64_t>(w.bh) * a.K + row_of(t, 4 * w.g + r)) * a.V + w.col] : 0.0f;
}
template <int KT, typename P>
__device__ __forceinline__ void store_state(const f32x4 (&S)[KT], float* s, const Args& a, const P& w) {
#pragma unroll
  for (int t = 0; t < KT; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (w.in && row_of(t, 4 * w.g) < a.K) s[(static_cast<int64_t>(w.bh) * a.K + row_of(t, 4 * w.g + r)) * a.V + w.col] = S[t][r];
}

template <int KP, int NI, bool KEEP, int W>
__global__ __launch_bounds__(512) void state_kernel(Args a, int tiles) {  // (bounds of 8 waves: no accumulator registers apart)
  using E = typename elem<NI>::type;
  using L = Tile<KP, NI>;
  constexpr int KT = KP / 16, KB = KP / 32, NP = L::NP, U = L::U, NW = kKept<NI>;
  __shared__ __attribute__((aligned(16))) char lds[L::kStages * L::kBytes];
  const Place<KP, NI, W> w(a, tiles);
  const int lane = w.lane, g = w.g;
  const int64_t o_st = static_cast<int64_t>(a.H) * a.V;
  const E* v = reinterpret_cast<const E*>(a.v) + w.b * a.v_sb + w.h * a.v_sh;
  E* o = reinterpret_cast<E*>(a.o) + (static_cast<int64_t>(w.b) * a.T * a.H + w.h) * a.V;
  const uint32_t vs = static_cast<uint32_t>(a.v_st * sizeof(E)), os = static_cast<uint32_t>(o_st * sizeof(E));
  const uint32_t v_off = w.in ? 8 * g * vs + w.col * sizeof(E) : kOutOfRange, o_off = w.in ? 8 * g * os + w.col * sizeof(E) : kOutOfRange;
  const char* img = a.img + static_cast<int64_t>(w.bh) * a.NC * L::kBytes;

  // v of a chunk, loaded one chunk ahead, and before the copy of its operands: loads come back in order
  uint32_t next[4][4];
  const auto load_v = [&](int n) {
    const __amdgpu_buffer_rsrc_t vr = rows_buffer(v + static_cast<int64_t>(n) * C * a.v_st, a.v_st, min(C, a.T - n * C), a.V);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) next[t][r] = load_col<E>(vr, v_off, row_of(t, r) * vs);
  };
  f32x4 S[KT];
  load_state(S, a.h0, a, w);
  stage<L::kBytes, W>(lds, img, lane, w.wave);
  load_v(0);
  for (int n = 0; n < a.NC; ++n) {
    char* cur = lds + (L::kStages == 2 ? (n & 1) * L::kBytes : 0);
    const int t0 = n * C, rows = min(C, a.T - t0);
    const int64_t c = static_cast<int64_t>(w.bh) * a.NC + n;
    f32x4 vv[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) vv[t][r] = value<E>(next[t][r]);
    bf16x8 sb[KB][3];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      split_pair<3>(S[2 * kb], S[2 * kb + 1], sb[kb]);
      if constexpr (KEEP)
        keep<U, NW>(a.Sw + (c * (a.VP / 32) + w.col / 32) * NW * 32 * KP, 32 * KP * 2, w.col % 32, 4 * kb + g, sb[kb]);
    }
    staged();
    if (n + 1 < a.NC) load_v(n + 1);
    if constexpr (L::kStages == 2)
      if (n + 1 < a.NC) stage<L::kBytes, W>(lds + ((n + 1) & 1) * L::kBytes, img + static_cast<int64_t>(n + 1) * L::kBytes, lane, w.wave);
    const float* gt = reinterpret_cast<const float*>(cur + L::kGate);
    f32x4 y[4], oa[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 ks = {0, 0, 0, 0}, qs = {0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        bf16x8 x[NI];
        frags<U>(cur + L::kK, C * KP * 2, t, kb, lane, x);
        ks = mm<3>(x, sb[kb], ks);
        frags<U>(cur + L::kQ, C * KP * 2, t, kb, lane, x);
        qs = mm<NP>(x, sb[kb], qs);  // only o, which is rounded to the inputs' type, sees this product
      }
      const f32x4 eg = *reinterpret_cast<const f32x4*>(gt + row_of(t, 4 * g));
      const f32x4 be = *reinterpret_cast<const f32x4*>(gt + 128 + row_of(t, 4 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        y[t][r] = be[r] * (vv[t][r] - eg[r] * ks[r]);
        oa[t][r] = a.scale * eg[r] * qs[r];
      }
    }
    bf16x8 yb[2][3];
#pragma unroll
    for (int p = 0; p < 2; ++p) split_pair<3>(y[2 * p], y[2 * p + 1], yb[p]);
    f32x4 d[4], e[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      d[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = 0; p <= t / 2; ++p) {
        bf16x8 x[3];
        frags<8>(cur + L::kT, kPlane * 2, t, p, lane, x);
        d[t] = mm<3>(x, yb[p], d[t]);
      }
      const f32x4 tail = *reinterpret_cast<const f32x4*>(gt + 64 + row_of(t, 4 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) e[t][r] = tail[r] * d[t][r];
    }
    bf16x8 db[2][NP], eb[2][3];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      split_pair<NP>(d[2 * p], d[2 * p + 1], db[p]);
      split_pair<3>(e[2 * p], e[2 * p + 1], eb[p]);
      if constexpr (KEEP)
        keep<8, NW>(a.dw + (c * (a.VP / 32) + w.col / 32) * NW * 32 * C, 32 * C * 2, w.col % 32, 4 * p + g, db[p]);
    }
    const float last = gt[63];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      S[t] *= last;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        bf16x8 x[NI];
        frags_t<U, true>(cur + L::kK, C * KP * 2, t, p, lane, x);
        S[t] = mm<3>(x, eb[p], S[t]);
      }
    }
    const __amdgpu_buffer_rsrc_t orr = rows_buffer(o + t0 * o_st, o_st, rows, a.V);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int p = 0; p <= t / 2; ++p) {
        bf16x8 x[NP];
        frags<8>(cur + L::kP, kPlane * 2, t, p, lane, x);
        oa[t] = mm<NP>(x, db[p], oa[t]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) store_col<E>(orr, o_off, row_of(t, r) * os, oa[t][r]);
    }
    if constexpr (L::kStages == 1) {
      __syncthreads();
      if (n + 1 < a.NC) stage<L::kBytes, W>(lds, img + static_cast<int64_t>(n + 1) * L::kBytes, lane, w.wave);
    }
  }
  if (a.state) store_state(S, a.state, a, w);
}

template <int KP, int NI, int W>
__global__ __launch_bounds__(512) void dstate_kernel(Args a, int tiles) {
  using E = typename elem<NI>::type;
  using L = Tile<KP, NI>;
  constexpr int KT = KP / 16, KB = KP / 32, NP = L::NP, U = L::U, NW = kKept<NI>;
  __shared__ __attribute__((aligned(16))) char lds[L::kStages * L::kBytes];
  const Place<KP, NI, W> w(a, tiles);
  const int lane = w.lane, g = w.g;
  const int64_t v_st = static_cast<int64_t>(a.H) * a.V;
  const E* dout = reinterpret_cast<const E*>(a.dout) + w.b * a.do_sb + w.h * a.do_sh;
  E* dv = reinterpret_cast<E*>(a.dv) + (static_cast<int64_t>(w.b) * a.T * a.H + w.h) * a.V;
  const uint32_t is = static_cast<uint32_t>(a.do_st * sizeof(E)), os = static_cast<uint32_t>(v_st * sizeof(E));
  const uint32_t i_off = w.in ? 8 * g * is + w.col * sizeof(E) : kOutOfRange, o_off = w.in ? 8 * g * os + w.col * sizeof(E) : kOutOfRange;
  const char* img = a.img + static_cast<int64_t>(w.bh) * a.NC * L::kBytes;

  uint32_t next[4][4];
  const auto load_go = [&](int n) {
    const __amdgpu_buffer_rsrc_t ir = rows_buffer(dout + static_cast<int64_t>(n) * C * a.do_st, a.do_st, min(C, a.T - n * C), a.V);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) next[t][r] = load_col<E>(ir, i_off, row_of(t, r) * is);
  };
  f32x4 S[KT];  // the gradient of the state
  load_state(S, a.dstate, a, w);
  load_go(a.NC - 1);
  stage<L::kBytes, W>(lds + (L::kStages == 2 ? ((a.NC - 1) & 1) * L::kBytes : 0), img + static_cast<int64_t>(a.NC - 1) * L::kBytes, lane, w.wave);
  for (int n = a.NC - 1; n >= 0; --n) {
    char* cur = lds + (L::kStages == 2 ? (n & 1) * L::kBytes : 0);
    const int t0 = n * C, rows = min(C, a.T - t0);
    const int64_t c = static_cast<int64_t>(w.bh) * a.NC + n;
    f32x4 go[4];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) go[t][r] = value<E>(next[t][r]);
    bf16x8 sb[KB][3], gb[2][NI];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      split_pair<3>(S[2 * kb], S[2 * kb + 1], sb[kb]);
      keep<U, NW>(a.dSw + (c * (a.VP / 32) + w.col / 32) * NW * 32 * KP, 32 * KP * 2, w.col % 32, 4 * kb + g, sb[kb]);
    }
    staged();
    if (n > 0) load_go(n - 1);
    if constexpr (L::kStages == 2)
      if (n > 0) stage<L::kBytes, W>(lds + ((n - 1) & 1) * L::kBytes, img + static_cast<int64_t>(n - 1) * L::kBytes, lane, w.wave);
#pragma unroll
    for (int p = 0; p < 2; ++p) split_pair<NI>(go[2 * p], go[2 * p + 1], gb[p]);
    const float* gt = reinterpret_cast<const float*>(cur + L::kGate);
    f32x4 dd[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 x = {0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        bf16x8 f[NI];
        frags<U>(cur + L::kK, C * KP * 2, t, kb, lane, f);
        x = mm<3>(f, sb[kb], x);
      }
      x *= *reinterpret_cast<const f32x4*>(gt + 64 + row_of(t, 4 * g));
#pragma unroll
      for (int p = t / 2; p < 2; ++p) {
        bf16x8 f[NP];
        frags_t<8, true>(cur + L::kP, kPlane * 2, t, p, lane, f);
        x = mm<3>(f, gb[p], x);
      }
      dd[t] = x;
    }
    bf16x8 ddb[2][3], xb[2][3], wb[2][3], yb[2][NW];
#pragma unroll
    for (int p = 0; p < 2; ++p) split_pair<3>(dd[2 * p], dd[2 * p + 1], ddb[p]);
    f32x4 dy[4], x[4], u[4];
    const __amdgpu_buffer_rsrc_t orr = rows_buffer(dv + t0 * v_st, v_st, rows, a.V);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      dy[t] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int p = t / 2; p < 2; ++p) {
        bf16x8 f[3];
        frags_t<8, true>(cur + L::kT, kPlane * 2, t, p, lane, f);
        dy[t] = mm<3>(f, ddb[p], dy[t]);
      }
      const f32x4 eg = *reinterpret_cast<const f32x4*>(gt + row_of(t, 4 * g));
      const f32x4 be = *reinterpret_cast<const f32x4*>(gt + 128 + row_of(t, 4 * g));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float dvv = be[r] * dy[t][r];
        store_col<E>(orr, o_off, row_of(t, r) * os, dvv);
        x[t][r] = -eg[r] * dvv;
        u[t][r] = a.scale * eg[r] * go[t][r];
      }
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      split_pair<3>(x[2 * p], x[2 * p + 1], xb[p]);
      split_pair<3>(u[2 * p], u[2 * p + 1], wb[p]);
      split_pair<NW>(dy[2 * p], dy[2 * p + 1], yb[p]);
      keep<8, NW>(a.yw + (c * (a.VP / 32) + w.col / 32) * NW * 32 * C, 32 * C * 2, w.col % 32, 4 * p + g, yb[p]);
    }
    const float last = gt[63];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
      S[t] *= last;
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        bf16x8 f[NI];
        frags_t<U, true>(cur + L::kK, C * KP * 2, t, p, lane, f);
        S[t] = mm<3>(f, xb[p], S[t]);
        frags_t<U, true>(cur + L::kQ, C * KP * 2, t, p, lane, f);
        S[t] = mm<3>(f, wb[p], S[t]);
      }
    }
    if constexpr (L::kStages == 1) {
      __syncthreads();
      if (n > 0) stage<L::kBytes, W>(lds, img + static_cast<int64_t>(n - 1) * L::kBytes, lane, w.wave);
    }
  }
  if (a.dh0) store_state(S, a.dh0, a, w);
}

// ---------------------------------------------------------------- dq, dk, dg, dbeta of a chunk

template <int KP, int NI>
struct GradTile {
  static constexpr int W = KP / 16;                                           // a wave for 16 columns of dq, dk
  static constexpr int NW = kKept<NI>;
  static constexpr int kState = NW * 32 * KP * 2, kVec = NW * 32 * C * 2;     // bytes of 32 columns of a state, of d or dy
  static constexpr int kS = 0, kE = kState, kD = 2 * kState, kY = kD + kVec;  // S, dS', d, dy, 32 columns at a time;
  static constexpr int kK = 0, kQ = NI * C * KP * 2;                          // then in their place k, q
  static constexpr int kF = 2 * kQ, kN = kF + NW * kPlane * 2;                // and F, N
  static constexpr int kSums = kY + kVec > kN + NW * kPlane * 2 ? kY + kVec : kN + NW * kPlane * 2;
  static constexpr int kBytes = kSums + (2 * W * 64 + 64 + W) * 4;            // floats: q.dq, k.Z [W][64], dy.v [64], [W]
};

template <int KP, int NI>
__global__ __launch_bounds__(64 * (KP / 16)) void grad_kernel(Args a) {
  using E = typename elem<NI>::type;
  using L = GradTile<KP, NI>;
  constexpr int NW = L::NW, U = KP / 8, W = L::W;
  __shared__ __attribute__((aligned(16))) char lds[L::kBytes];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x;
  const int n = static_cast<int>(c % a.NC), bh = static_cast<int>(c / a.NC), h = bh % a.H, b = bh / a.H, grp = a.H / a.Hk;
  const int hk = h / grp, t0 = n * C, rows = min(C, a.T - t0);
  float* vec = reinterpret_cast<float*>(lds + L::kSums);
  const char* img = a.img + c * Tile<KP, NI>::kBytes;
  const float* gt = reinterpret_cast<const float*>(img + Tile<KP, NI>::kGate);
  const double* Gd = a.Gd + c * 64;

  // Products over the value columns, 32 at a time, in this wave's 16 columns of K: W1 = dy S^T, W2 = do S^T,
  // W3 = d dS'^T, and a diagonal block of S dS'^T. Of the 64 x 64 products dy d^T and do d^T a wave takes 16 rows of
  // both (W = 4) or of one (W = 8: waves 0 to 3 the first, 4 to 7 the second); waves 0 to 3 also a diagonal block of dy v^T.
  f32x4 w1[4], w2[4], w3[4], m1[4], m2[W == 4 ? 4 : 1], ss = {0, 0, 0, 0}, yv = ss;
#pragma unroll
  for (int t = 0; t < 4; ++t) w1[t] = w2[t] = w3[t] = m1[t] = m2[W == 4 ? t : 0] = f32x4{0, 0, 0, 0};
  const int mr = wave & 3;
  const E* orow = reinterpret_cast<const E*>(a.dout) + b * a.do_sb + t0 * a.do_st + h * a.do_sh + 8 * g;
  const E* vrow = reinterpret_cast<const E*>(a.v) + b * a.v_sb + (t0 + 16 * mr + m) * a.v_st + h * a.v_sh + 8 * g;
  for (int vb = 0; vb < a.VP / 32; ++vb) {
    const int64_t blk = c * (a.VP / 32) + vb;
    if (vb) __syncthreads();
    stage<L::kState, W>(lds + L::kS, a.Sw + blk * NW * 32 * KP, lane, wave);
    stage<L::kState, W>(lds + L::kE, a.dSw + blk * NW * 32 * KP, lane, wave);
    stage<L::kVec, W>(lds + L::kD, a.dw + blk * NW * 32 * C, lane, wave);
    stage<L::kVec, W>(lds + L::kY, a.yw + blk * NW * 32 * C, lane, wave);
    bf16x8 fo[4][NI], fv[NI];
    const bool cols = 32 * vb + 8 * g < a.V;
#pragma unroll
    for (int t = 0; t < 4; ++t) load8(orow + (16 * t + m) * a.do_st + 32 * vb, 16 * t + m < rows && cols, fo[t]);
    if (wave < 4) {
      float x[8];  // (v may lie at any alignment)
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = 16 * mr + m < rows && cols ? ld(vrow + 32 * vb + j) : 0.0f;
      split<NI>(x, fv);
    }
    staged();
    bf16x8 s[NW], ds[NW];
    frags_t<U, false>(lds + L::kS, 32 * KP * 2, wave, 0, lane, s);
    frags_t<U, false>(lds + L::kE, 32 * KP * 2, wave, 0, lane, ds);
    ss = mm<NW>(s, ds, ss);
    bf16x8 yr[NW], orr[NI];
    frags_t<8, false>(lds + L::kY, 32 * C * 2, mr, 0, lane, yr);
    if (wave < 4) yv = mm<NW>(yr, fv, yv);
    load8(orow + (16 * mr + m) * a.do_st + 32 * vb, 16 * mr + m < rows && cols, orr);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bf16x8 fy[NW], fd[NW];
      frags_t<8, false>(lds + L::kY, 32 * C * 2, t, 0, lane, fy);
      frags_t<8, false>(lds + L::kD, 32 * C * 2, t, 0, lane, fd);
      w1[t] = mm<NW>(fy, s, w1[t]);
      w2[t] = mm<NW>(fo[t], s, w2[t]);
      w3[t] = mm<NW>(fd, ds, w3[t]);
      if (t <= mr) {
        if constexpr (W == 4) {
          m1[t] = mm<NW>(yr, fd, m1[t]);
          m2[t] = mm<NW>(orr, fd, m2[t]);
        } else if (wave < 4) {
          m1[t] = mm<NW>(yr, fd, m1[t]);
        } else {
          m1[t] = mm<NW>(orr, fd, m1[t]);
        }
      }
    }
  }
  __syncthreads();
  stage<2 * L::kQ, W>(lds, img, lane, wave);  // k and q
  // F and N, in this wave's rows, to LDS
  const auto put = [&](int plane, int row, int col, float x) {
    const int pos = at<8>(row, col >> 3) + (col & 7) * 2;
#pragma unroll
    for (int l = 0; l < NW; ++l) {
      const uint32_t u = __float_as_uint(x);
      *reinterpret_cast<bf16_t*>(lds + plane + l * kPlane * 2 + pos) = NW == 2 && l == 1 ? f32_to_bf16(x) : static_cast<bf16_t>(u >> 16);
      x -= __uint_as_float(u & 0xffff0000u);
    }
  };
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * mr + 4 * g + r, col = 16 * t + m;
      const float dec = col <= row ? expf(static_cast<float>(Gd[row] - Gd[col])) : 0.0f;
      if (W == 4 || wave < 4) put(L::kF, row, col, col < row ? dec * m1[t][r] : 0.0f);
      if (W == 4 || wave >= 4) put(L::kN, row, col, col <= row ? a.scale * dec * (W == 4 ? m2[W == 4 ? t : 0][r] : m1[t][r]) : 0.0f);
    }
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * t + 4 * g + r;
      w1[t][r] *= gt[i], w2[t][r] *= a.scale * gt[i], w3[t][r] *= gt[64 + i];
    }
  if (wave < 4) {  // the diagonals' lanes
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * g + r == m) vec[2 * W * 64 + 16 * mr + m] = yv[r];
  }
  staged();
  // <S', dS'> = e^{G_C} <S, dS'> + sum_j k_j.(e^{G_C - G_j} (d dS'^T)_j): its first part from the diagonals
  float dot = 0.0f;
#pragma unroll
  for (int r = 0; r < 4; ++r) dot += 4 * g + r == m ? ss[r] : 0.0f;
  dot *= gt[63];
  const int d = 16 * wave + m;
  // k and q where this wave's accumulators are
  const auto at_acc = [&](int base, int row) {
    float x = 0.0f;
#pragma unroll
    for (int l = 0; l < NI; ++l)
      x += bf16_to_f32(*reinterpret_cast<const bf16_t*>(lds + base + l * C * KP * 2 + at<U>(row, d >> 3) + (d & 7) * 2));
    return x;
  };
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) dot += at_acc(L::kK, 16 * t + 4 * g + r) * w3[t][r];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    bf16x8 kf[NI], qf[NI], bk[NW];
    frags_t<U, false>(lds + L::kK, C * KP * 2, wave, p, lane, kf);
    frags_t<U, false>(lds + L::kQ, C * KP * 2, wave, p, lane, qf);
    {
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float kv = static_cast<float>(kf[0][j]);
#pragma unroll
        for (int l = 1; l < NI; ++l) kv += static_cast<float>(kf[l][j]);
        x[j] = -kv * gt[128 + 32 * p + 8 * g + j];
      }
      split<NW>(x, bk);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bf16x8 f[NW];
      if (p <= t / 2) {
#pragma unroll
        for (int l = 0; l < NW; ++l) f[l] = frag_plain<8>(lds + L::kF + l * kPlane * 2, t, p, lane);
        w1[t] = mm<NW>(f, kf, w1[t]);
#pragma unroll
        for (int l = 0; l < NW; ++l) f[l] = frag_plain<8>(lds + L::kN + l * kPlane * 2, t, p, lane);
        w2[t] = mm<NW>(f, kf, w2[t]);
      }
      if (p >= t / 2) {
        frags_t<8, false>(lds + L::kN, kPlane * 2, t, p, lane, f);
        w3[t] = mm<NW>(f, qf, w3[t]);
        frags_t<8, false>(lds + L::kF, kPlane * 2, t, p, lane, f);
        w3[t] = mm<NW>(f, bk, w3[t]);
      }
    }
  }
  // outputs, and the row sums q.dq and k.Z
  const int64_t tok0 = static_cast<int64_t>(b) * a.T + t0;
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * t + 4 * g + r;
      const float dq = w2[t][r], z = w1[t][r], dk = w3[t][r] - gt[128 + row] * z;
      float qd = at_acc(L::kQ, row) * dq, kz = at_acc(L::kK, row) * z;
      if (row < rows && d < a.K) {
        if (grp == 1) {
          st(reinterpret_cast<E*>(a.dq) + ((tok0 + row) * a.Hk + hk) * a.K + d, dq);
          st(reinterpret_cast<E*>(a.dk) + ((tok0 + row) * a.Hk + hk) * a.K + d, dk);
        } else {
          a.dqp[((tok0 + row) * a.H + h) * a.K + d] = dq;
          a.dkp[((tok0 + row) * a.H + h) * a.K + d] = dk;
        }
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) qd += __shfl_xor(qd, o, 64), kz += __shfl_xor(kz, o, 64);
      if (m == 0) vec[wave * 64 + row] = qd, vec[(W + wave) * 64 + row] = kz;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
  if (lane == 0) vec[(2 * W + 1) * 64 + wave] = dot;
  __syncthreads();
  if (wave == 0) {
    float qd = 0.0f, kz = 0.0f, all = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) qd += vec[w * 64 + lane], kz += vec[(W + w) * 64 + lane], all += vec[(2 * W + 1) * 64 + w];
    const float y = vec[2 * W * 64 + lane], be = gt[128 + lane];
    double s = static_cast<double>(qd) - static_cast<double>(be) * y;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double x = __shfl_down(s, o, 64);
      if (lane + o < 64) s += x;
    }
    if (lane < rows) {
      const int64_t tok = (tok0 + lane) * a.H + h;
      const float gv = ld(reinterpret_cast<const E*>(a.g) + b * a.g_sb + (t0 + lane) * a.g_st + h * a.g_sh);
      // a decay that is zero in fp32 passes nothing on
      st(reinterpret_cast<E*>(a.dg) + tok, gv < -104.0f ? 0.0f : static_cast<float>(s + all));
      st(reinterpret_cast<E*>(a.db) + tok, y - kz);
    }
  }
}

// dq, dk of shared heads: the sum over the H / Hk value heads of a key head
template <typename E>
__global__ __launch_bounds__(256) void sum_heads_kernel(const float* dqp, const float* dkp, E* dq, E* dk, int64_t n, int K, int grp) {
  const int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const int64_t src = i / K * grp * K + i % K;
  f4 x = io4<float>::load(dqp + src), y = io4<float>::load(dkp + src);
  for (int j = 1; j < grp; ++j) {
    const f4 u = io4<float>::load(dqp + src + j * K), w = io4<float>::load(dkp + src + j * K);
#pragma unroll
    for (int e = 0; e < 4; ++e) x.v[e] += u.v[e], y.v[e] += w.v[e];
  }
  io4<E>::store(dq + i, x);
  io4<E>::store(dk + i, y);
}

// ---------------------------------------------------------------- single tokens
//
// One workgroup per (batch, head, 32 value columns): thread (r, c) holds rows r, r + 32, ... and columns
// 4 c ... 4 c + 3 of the state, read and written once. k S and q S are taken together from the old
// state: o = scale (e^g q S + (q.k) d), d = beta (v - e^g k S).
template <typename E, int KR>
__global__ __launch_bounds__(256) void step_kernel(const E* __restrict__ q, const E* __restrict__ k, const E* __restrict__ v,
                                                   const E* __restrict__ gg, const E* __restrict__ beta, float* __restrict__ state,
                                                   E* __restrict__ o, int H, int Hk, int K, int V, float scale) {
  __shared__ float red[4][8][8];
  __shared__ float dots[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = tid >> 3, cc = tid & 7;
  const int64_t bh = blockIdx.x;
  const int h = static_cast<int>(bh % H), hk = h / (H / Hk);
  const int64_t bk = bh / H * Hk + hk;
  const int col = blockIdx.y * 32 + 4 * cc;
  const bool in = col < V;
  float* s = state + bh * K * V + col;
  f4 x[KR];
  float kr[KR], qr[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int d = r + 32 * i;
    x[i] = in && d < K ? io4<float>::load(s + static_cast<int64_t>(d) * V) : io4<float>::fill(0.0f);
    kr[i] = d < K ? ld(k + bk * K + d) : 0.0f;
    qr[i] = d < K ? ld(q + bk * K + d) : 0.0f;
  }
  const float decay = expf(ld(gg + bh)), be = ld(beta + bh);
  f4 vv = in ? io4<E>::load(v + bh * V + col) : io4<float>::fill(0.0f);
  float ks[4] = {0, 0, 0, 0}, qs[4] = {0, 0, 0, 0}, qk = 0.0f;
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    qk += qr[i] * kr[i];
#pragma unroll
    for (int j = 0; j < 4; ++j) ks[j] += kr[i] * x[i].v[j], qs[j] += qr[i] * x[i].v[j];
  }
#pragma unroll
  for (int off = 8; off < 64; off <<= 1) {
    qk += __shfl_xor(qk, off, 64);
#pragma unroll
    for (int j = 0; j < 4; ++j) ks[j] += __shfl_xor(ks[j], off, 64), qs[j] += __shfl_xor(qs[j], off, 64);
  }
  if (lane < 8) {
#pragma unroll
    for (int j = 0; j < 4; ++j) red[wave][lane][j] = ks[j], red[wave][lane][4 + j] = qs[j];
    if (lane == 0) dots[wave] = qk;
  }
  __syncthreads();
  qk = dots[0] + dots[1] + dots[2] + dots[3];
  float d[4];
  f4 out;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float kk = red[0][cc][j] + red[1][cc][j] + red[2][cc][j] + red[3][cc][j];
    const float qq = red[0][cc][4 + j] + red[1][cc][4 + j] + red[2][cc][4 + j] + red[3][cc][4 + j];
    d[j] = be * (vv.v[j] - decay * kk);
    out.v[j] = scale * (decay * qq + qk * d[j]);
  }
  if (in) {
    if (r == 0) io4<E>::store(o + bh * V + col, out);
#pragma unroll
    for (int i = 0; i < KR; ++i) {
      const int row = r + 32 * i;
      if (row < K) {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i].v[j] = decay * x[i].v[j] + kr[i] * d[j];
        io4<float>::store(s + static_cast<int64_t>(row) * V, x[i]);
      }
    }
  }
}

// ---------------------------------------------------------------- host side

constexpr int kCUs = 256;

inline size_t up(size_t x) { return (x + 255) / 256 * 256; }

struct Layout {  // byte offsets of the forward's buffer
  size_t img, G, S, d, end;
};
inline int vpad(int V) { return (V + 31) / 32 * 32; }
inline int64_t chunks(const mg_delta_dims& s) { return (static_cast<int64_t>(s.T) + C - 1) / C; }

inline Layout layout(int dtype, const mg_delta_dims& s, bool keep_) {
  const size_t n = static_cast<size_t>(chunks(s)), bh = static_cast<size_t>(s.B) * s.H, c = bh * n;
  const size_t vp = vpad(s.V), image = dtype == MG_F32 ? (s.K <= 64 ? Tile<64, 3>::kBytes : Tile<128, 3>::kBytes)
                                                       : (s.K <= 64 ? Tile<64, 1>::kBytes : Tile<128, 1>::kBytes);
  Layout l;
  l.img = 0;
  l.G = c * image;
  l.S = l.G + c * 512;
  const size_t nw = dtype == MG_F32 ? 3 : 2;
  l.d = l.S + (keep_ ? c * vp * nw * (s.K <= 64 ? 64 : 128) * 2 : 0);
  l.end = l.d + (keep_ ? c * vp * nw * C * 2 : 0);
  return l;
}

struct BwdLayout {
  size_t dS, y, dqp, dkp, end;
};
inline BwdLayout bwd_layout(int dtype, const mg_delta_dims& s) {
  const size_t c = static_cast<size_t>(s.B) * s.H * chunks(s), vp = vpad(s.V);
  BwdLayout l;
  l.dS = 0;
  const size_t nw = dtype == MG_F32 ? 3 : 2;
  l.y = c * vp * nw * (s.K <= 64 ? 64 : 128) * 2;
  l.dqp = l.y + c * vp * nw * C * 2;
  l.dkp = l.dqp + (s.H > s.Hk ? up(static_cast<size_t>(s.B) * s.T * s.H * s.K * 4) : 0);
  l.end = l.dkp + (l.dkp - l.dqp);
  return l;
}

inline int check_dims(const char* fn, int dtype, const mg_delta_dims* s) {
  if (dtype != MG_F32 && dtype != MG_BF16) return fail(MG_ERR_DTYPE, "%s: dtype %d unsupported", fn, dtype);
  if (!s || s->B < 1 || s->T < 1 || s->H < 1 || s->Hk < 1 || s->H % s->Hk)
    return fail(MG_ERR_ARG, "%s: needs B, T, H, Hk >= 1 and H a multiple of Hk", fn);
  if (s->K < 8 || s->K % 8 || s->K > 128 || s->V < 8 || s->V % 8 || s->V > 256)
    return fail(MG_ERR_ARG, "%s: K=%d and V=%d must be multiples of 8, K <= 128, V <= 256", fn, s->K, s->V);
  if (static_cast<int64_t>(s->B) * s->H * chunks(*s) >= (int64_t(1) << 31))
    return fail(MG_ERR_ARG, "%s: B * H * ceil(T / 64) must be below 2^31", fn);
  return MG_OK;
}

// strides in elements; `vector`: rows of d elements read 16 bytes at a time
inline int check_rows(const char* fn, const char* name, int dtype, const mg_rows* r, bool vector) {
  const int64_t e = dtype == MG_F32 ? 4 : 2;
  if (!r || !r->p) return fail(MG_ERR_ARG, "%s: %s is NULL", fn, name);
  if (!aligned(r->p, vector ? 16 : e)) return fail(MG_ERR_ARG, "%s: %s not %d-byte aligned", fn, name, vector ? 16 : (int)e);
  if (r->sb < 0 || r->st < 0 || r->sh < 0) return fail(MG_ERR_ARG, "%s: %s has a negative stride", fn, name);
  if (vector && (r->sb * e % 16 || r->st * e % 16 || r->sh * e % 16))
    return fail(MG_ERR_ARG, "%s: strides of %s must be multiples of 16 bytes", fn, name);
  if (r->st * e * C >= (int64_t(1) << 31)) return fail(MG_ERR_ARG, "%s: token stride of %s too large", fn, name);
  return MG_OK;
}

// Waves per workgroup of the passes over the chunks: a workgroup takes a CU's LDS, so as few waves
// as spread the value columns over all CUs.
inline int waves_for(int64_t bh, int vp) {
  const int tiles = vp / 16;
  int w = 2;
  while (w < 8 && tiles % (2 * w) == 0 && bh * (tiles / w) > kCUs) w *= 2;
  return w;
}

inline void fill(Args& a, const mg_delta_dims& s, float scale, const mg_rows* q, const mg_rows* k, const mg_rows* v,
                 const mg_rows* g, const mg_rows* beta, char* ws, const Layout& l) {
  a.B = s.B, a.T = s.T, a.Hk = s.Hk, a.H = s.H, a.K = s.K, a.V = s.V, a.NC = static_cast<int>(chunks(s)), a.VP = vpad(s.V);
  a.scale = scale;
  a.q = static_cast<const char*>(q->p), a.q_sb = q->sb, a.q_st = q->st, a.q_sh = q->sh;
  a.k = static_cast<const char*>(k->p), a.k_sb = k->sb, a.k_st = k->st, a.k_sh = k->sh;
  a.v = static_cast<const char*>(v->p), a.v_sb = v->sb, a.v_st = v->st, a.v_sh = v->sh;
  a.g = static_cast<const char*>(g->p), a.g_sb = g->sb, a.g_st = g->st, a.g_sh = g->sh;
  a.beta = static_cast<const char*>(beta->p), a.b_sb = beta->sb, a.b_st = beta->st, a.b_sh = beta->sh;
  a.img = ws + l.img, a.Gd = reinterpret_cast<double*>(ws + l.G);
  a.Sw = reinterpret_cast<bf16_t*>(ws + l.S), a.dw = reinterpret_cast<bf16_t*>(ws + l.d);
}

template <int KP, int NI>
int launch_fwd(const Args& a, bool keep_, hipStream_t st_) {
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  hipLaunchKernelGGL((chunk_kernel<KP, NI>), dim3(bh * a.NC), dim3(256), 0, st_, a);
  const int w = waves_for(bh, a.VP), tiles = a.VP / 16 / w;
  const dim3 grid(bh * tiles), block(64 * w);
#define GO(W)                                                                                         \
  if (keep_)                                                                                          \
    hipLaunchKernelGGL((state_kernel<KP, NI, true, W>), grid, block, 0, st_, a, tiles);               \
  else                                                                                                \
    hipLaunchKernelGGL((state_kernel<KP, NI, false, W>), grid, block, 0, st_, a, tiles);
  if (w == 8) { GO(8) } else if (w == 4) { GO(4) } else { GO(2) }
#undef GO
  return check_launch("mg_delta_fwd");
}

template <int KP, int NI>
int launch_bwd(const Args& a, hipStream_t st_) {
  using E = typename elem<NI>::type;
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  const int w = waves_for(bh, a.VP), tiles = a.VP / 16 / w;
  const dim3 grid(bh * tiles), block(64 * w);
  if (w == 8)
    hipLaunchKernelGGL((dstate_kernel<KP, NI, 8>), grid, block, 0, st_, a, tiles);
  else if (w == 4)
    hipLaunchKernelGGL((dstate_kernel<KP, NI, 4>), grid, block, 0, st_, a, tiles);
  else
    hipLaunchKernelGGL((dstate_kernel<KP, NI, 2>), grid, block, 0, st_, a, tiles);
  hipLaunchKernelGGL((grad_kernel<KP, NI>), dim3(bh * a.NC), dim3(64 * GradTile<KP, NI>::W), 0, st_, a);
  if (a.H > a.Hk) {
    const int64_t n = static_cast<int64_t>(a.B) * a.T * a.Hk * a.K;
    hipLaunchKernelGGL((sum_heads_kernel<E>), dim3((n / 4 + 255) / 256), dim3(256), 0, st_, a.dqp, a.dkp,
                       reinterpret_cast<E*>(a.dq), reinterpret_cast<E*>(a.dk), n, a.K, a.H / a.Hk);
  }
  return check_launch("mg_delta_bwd");
}

template <typename E>
int launch_step(const mg_delta_dims& s, const void* q, const void* k, const void* v, const void* g, const void* beta, float scale,
                float* state, void* o, hipStream_t st_) {
  const dim3 grid(s.B * s.H, (s.V + 31) / 32);
  const E *qq = static_cast<const E*>(q), *kk = static_cast<const E*>(k), *vv = static_cast<const E*>(v),
          *gg = static_cast<const E*>(g), *bb = static_cast<const E*>(beta);
  E* oo = static_cast<E*>(o);
  if (s.K <= 32)
    hipLaunchKernelGGL((step_kernel<E, 1>), grid, dim3(256), 0, st_, qq, kk, vv, gg, bb, state, oo, s.H, s.Hk, s.K, s.V, scale);
  else if (s.K <= 64)
    hipLaunchKernelGGL((step_kernel<E, 2>), grid, dim3(256), 0, st_, qq, kk, vv, gg, bb, state, oo, s.H, s.Hk, s.K, s.V, scale);
  else
    hipLaunchKernelGGL((step_kernel<E, 4>), grid, dim3(256), 0, st_, qq, kk, vv, gg, bb, state, oo, s.H, s.Hk, s.K, s.V, scale);
  return check_launch("mg_delta_step");
}

}  // namespace delta
}  // namespace mg

using namespace mg;

extern "C" size_t mg_delta_fwd_workspace_bytes(int dtype, const mg_delta_dims* dims, int keep) {
  if (delta::check_dims("mg_delta_fwd_workspace_bytes", dtype, dims)) return 0;
  return delta::layout(dtype, *dims, keep != 0).end;
}

extern "C" size_t mg_delta_bwd_workspace_bytes(int dtype, const mg_delta_dims* dims) {
  if (delta::check_dims("mg_delta_bwd_workspace_bytes", dtype, dims)) return 0;
  return delta::bwd_layout(dtype, *dims).end;
}

extern "C" int mg_delta_fwd(int dtype, const mg_delta_dims* dims, const mg_rows* q, const mg_rows* k, const mg_rows* v,
                            const mg_rows* g, const mg_rows* beta, float scale, const float* h0, void* o, float* state,
                            int keep, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "mg_delta_fwd";
  int rc;
  if ((rc = delta::check_dims(fn, dtype, dims))) return rc;
  if ((rc = delta::check_rows(fn, "q", dtype, q, true)) || (rc = delta::check_rows(fn, "k", dtype, k, true)) ||
      (rc = delta::check_rows(fn, "v", dtype, v, false)) || (rc = delta::check_rows(fn, "g", dtype, g, false)) ||
      (rc = delta::check_rows(fn, "beta", dtype, beta, false)))
    return rc;
  if (!o || !aligned(o, dtype == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: o is NULL or misaligned", fn);
  if (!aligned(h0, 4) || !aligned(state, 4)) return fail(MG_ERR_ARG, "%s: state misaligned", fn);
  const delta::Layout l = delta::layout(dtype, *dims, keep != 0);
  if (!workspace || workspace_bytes < l.end || !aligned(workspace, 256))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or not 256-byte aligned)", fn, workspace_bytes, l.end);
  delta::Args a = {};
  delta::fill(a, *dims, scale, q, k, v, g, beta, static_cast<char*>(workspace), l);
  a.h0 = h0, a.o = static_cast<char*>(o), a.state = state;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MG_F32)
    return dims->K <= 64 ? delta::launch_fwd<64, 3>(a, keep, st) : delta::launch_fwd<128, 3>(a, keep, st);
  return dims->K <= 64 ? delta::launch_fwd<64, 1>(a, keep, st) : delta::launch_fwd<128, 1>(a, keep, st);
}

extern "C" int mg_delta_bwd(int dtype, const mg_delta_dims* dims, const mg_rows* q, const mg_rows* k, const mg_rows* v,
                            const mg_rows* g, const mg_rows* beta, float scale, const void* kept, size_t kept_bytes,
                            const mg_rows* dout, const float* dstate, void* dq, void* dk, void* dv, void* dg, void* dbeta,
                            float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "mg_delta_bwd";
  int rc;
  if ((rc = delta::check_dims(fn, dtype, dims))) return rc;
  if ((rc = delta::check_rows(fn, "q", dtype, q, true)) || (rc = delta::check_rows(fn, "k", dtype, k, true)) ||
      (rc = delta::check_rows(fn, "v", dtype, v, false)) || (rc = delta::check_rows(fn, "g", dtype, g, false)) ||
      (rc = delta::check_rows(fn, "beta", dtype, beta, false)) || (rc = delta::check_rows(fn, "dout", dtype, dout, true)))
    return rc;
  for (const void* p : {dq, dk, dv, dg, dbeta})
    if (!p || !aligned(p, dtype == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: a gradient is NULL or misaligned", fn);
  if (dims->H > dims->Hk && (!aligned(dq, 16) || !aligned(dk, 16)))
    return fail(MG_ERR_ARG, "%s: dq and dk must be 16-byte aligned", fn);
  if (!aligned(dstate, 4) || !aligned(dh0, 4)) return fail(MG_ERR_ARG, "%s: state gradient misaligned", fn);
  const delta::Layout l = delta::layout(dtype, *dims, true);
  if (!kept || kept_bytes < l.end || !aligned(kept, 256))
    return fail(MG_ERR_WORKSPACE, "%s: the forward's buffer has %zu bytes < %zu (or is not 256-byte aligned)", fn, kept_bytes, l.end);
  const delta::BwdLayout w = delta::bwd_layout(dtype, *dims);
  if (!workspace || workspace_bytes < w.end || !aligned(workspace, 256))
    return fail(MG_ERR_WORKSPACE, "%s: workspace %zu bytes < required %zu (or not 256-byte aligned)", fn, workspace_bytes, w.end);
  delta::Args a = {};
  delta::fill(a, *dims, scale, q, k, v, g, beta, const_cast<char*>(static_cast<const char*>(kept)), l);
  char* ws = static_cast<char*>(workspace);
  a.dout = static_cast<const char*>(dout->p), a.do_sb = dout->sb, a.do_st = dout->st, a.do_sh = dout->sh;
  a.dstate = dstate, a.dh0 = dh0;
  a.dSw = reinterpret_cast<bf16_t*>(ws + w.dS), a.yw = reinterpret_cast<bf16_t*>(ws + w.y);
  a.dqp = reinterpret_cast<float*>(ws + w.dqp), a.dkp = reinterpret_cast<float*>(ws + w.dkp);
  a.dq = static_cast<char*>(dq), a.dk = static_cast<char*>(dk), a.dv = static_cast<char*>(dv);
  a.dg = static_cast<char*>(dg), a.db = static_cast<char*>(dbeta);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (dtype == MG_F32) return dims->K <= 64 ? delta::launch_bwd<64, 3>(a, st) : delta::launch_bwd<128, 3>(a, st);
  return dims->K <= 64 ? delta::launch_bwd<64, 1>(a, st) : delta::launch_bwd<128, 1>(a, st);
}

extern "C" int mg_delta_step(int dtype, const mg_delta_dims* dims, const void* q, const void* k, const void* v, const void* g,
                             const void* beta, float scale, float* state, void* o, void* stream) {
  const char* fn = "mg_delta_step";
  int rc;
  if ((rc = delta::check_dims(fn, dtype, dims))) return rc;
  if (dims->T != 1) return fail(MG_ERR_ARG, "%s: T must be 1", fn);
  const size_t e = dtype == MG_F32 ? 4 : 2;
  if (!q || !k || !g || !beta || !aligned(q, e) || !aligned(k, e) || !aligned(g, e) || !aligned(beta, e))
    return fail(MG_ERR_ARG, "%s: an input is NULL or misaligned", fn);
  if (!v || !o || !aligned(v, 4 * e) || !aligned(o, 4 * e)) return fail(MG_ERR_ARG, "%s: v and o must be %zu-byte aligned", fn, 4 * e);
  if (!state || !aligned(state, 16)) return fail(MG_ERR_ARG, "%s: state is NULL or not 16-byte aligned", fn);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return dtype == MG_F32 ? delta::launch_step<float>(*dims, q, k, v, g, beta, scale, state, o, st)
                         : delta::launch_step<bf16_t>(*dims, q, k, v, g, beta, scale, state, o, st);
}
