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
//   dg_t = e^{G_C} <S, dS'> + sum_{i >= t > j} M_ij
//        + sum_{i >= t} (q_i.(scale e^G do S^T)_i - beta_i k_i.(e^G dy S^T)_i) + sum_{j < t} k_j.(e^{G_C - G} d dS'^T)_j,
//   M_ij = N_ij q_i.k_j - beta_i F_ij k_i.k_j (j < i).
// The last lines: every factor e^{G_i - G_j} that a result contains is multiplied with its gradient, and g_t is in those
// with i >= t > j. Only these are summed, all of them as small as e^{g_t}: what a token that forgets passes on is no
// difference of larger sums.
//
// The kernels:
//   chunk_kernel  one workgroup per (chunk, head), all in parallel: T, P, the decays, and the
//     chunk's operands in the order in which the passes load them;
//   state_kernel, dstate_kernel  the pass over the chunks in order, forward and backward, which alone
//     holds the state (or its gradient); the products that contract the tokens or K;
//   grad_kernel   one workgroup per (chunk, head): what contracts the value columns;
//   step_kernel   single tokens.
// Times below are for K = V = 128 in bf16: B8 T2047 H8, forward and backward, and B2 T16381 H16, forward.
//
// Matrix operands are bf16. An fp32 value enters as limbs, x = h + m + l (exact,
// |m| <= 2^-9 |x|, |l| <= 2^-18 |x|), and the limb products down to 2^-18 of the
// leading one are summed in fp32 (what is left out: 2^-26). States, T, y and d are
// never rounded to bf16 in the passes; o and the gradients that bf16 inputs take
// in their own type are made from two limbs (2^-18). bf16 inputs are one limb, so
// a product with one costs three instructions at most; fp32 inputs are three, and
// a product six.

#include <algorithm>

#include "mg_common.h"

namespace mg {
namespace delta {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

template <int N>
struct int_c { static constexpr int value = N; };

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
  char* Sw;            // kept for the backward: each chunk's entry state, [c][VP / 32][Kept::kState]
  char* dw;            // d, [c][VP / 32][Kept::kVec]
  // backward
  const char* dout;      // [B, T, H, V]
  int64_t do_sb, do_st, do_sh;
  const float* dstate;   // or null
  char* dSw;           // the gradients of the exit states, as Sw
  char* yw;            // dy, as dw
  char *dq, *dk, *dv, *dg, *db;
  float* dh0;
  float *dqp, *dkp;      // shared heads: [B, T, H, K] before their sum
};

// ---------------------------------------------------------------- limbs

__device__ __forceinline__ uint32_t hi16x2(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// Two fp32 values as limbs, each the rest rounded to nearest: off by 2^-9 after one, 2^-18 after two, and nothing is
// left after three. (Where three are made and two are used, as of a state, these are rounded too: cut limbs would be
// off by up to 2^-15, always towards zero.)
__device__ __forceinline__ void pair_limbs(float a, float b, uint32_t (&w)[2]) {
  w[0] = pack_bf16x2(a, b);
  w[1] = pack_bf16x2(a - __uint_as_float(w[0] << 16), b - __uint_as_float(w[0] & 0xffff0000u));
}
__device__ __forceinline__ void pair_limbs(float a, float b, uint32_t (&w)[3]) {
  w[0] = pack_bf16x2(a, b);
  a -= __uint_as_float(w[0] << 16), b -= __uint_as_float(w[0] & 0xffff0000u);
  w[1] = pack_bf16x2(a, b);
  w[2] = hi16x2(__float_as_uint(a - __uint_as_float(w[1] << 16)), __float_as_uint(b - __uint_as_float(w[1] & 0xffff0000u)));
}
__device__ __forceinline__ void pair_limbs(float a, float b, uint32_t (&w)[1]) { w[0] = hi16x2(__float_as_uint(a), __float_as_uint(b)); }
template <int N>
__device__ __forceinline__ void split(const float (&x)[8], bf16x8 (&out)[N]) {
  u32x4 w[N];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t l[N];
    pair_limbs(x[2 * i], x[2 * i + 1], l);
#pragma unroll
    for (int j = 0; j < N; ++j) w[j][i] = l[j];
  }
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = __builtin_bit_cast(bf16x8, w[l]);
}

// Limbs of what is kept for the backward's products: two of a state or update of bf16 inputs (2^-18,
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

// the same into two sums in turn: half as long a chain of products that wait for one another
template <int ORD, int NA, int NB>
__device__ __forceinline__ void mm2(const bf16x8 (&a)[NA], const bf16x8 (&b)[NB], f32x4 (&c)[2]) {
  int n = 0;
#pragma unroll
  for (int s = ORD - 1; s >= 0; --s)
#pragma unroll
    for (int i = 0; i < NA; ++i)
      if (s - i >= 0 && s - i < NB) c[n & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], b[s - i], c[n & 1], 0, 0, 0), ++n;
}

template <int NI> struct elem { using type = bf16_t; };
template <> struct elem<3> { using type = float; };

__device__ __forceinline__ float ld(const float* p) { return *p; }
__device__ __forceinline__ float ld(const bf16_t* p) { return bf16_to_f32(*p); }
__device__ __forceinline__ void st(float* p, float x) { *p = x; }
__device__ __forceinline__ void st(bf16_t* p, float x) { *p = f32_to_bf16(x); }
// four values, 16 (fp32) or 8 bytes aligned
__device__ __forceinline__ void st4(float* p, const f32x4& x) { *reinterpret_cast<f32x4*>(p) = x; }
__device__ __forceinline__ void st4(bf16_t* p, const f32x4& x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(static_cast<uint32_t>(f32_to_bf16(x[0])) | static_cast<uint32_t>(f32_to_bf16(x[1])) << 16,
                                            static_cast<uint32_t>(f32_to_bf16(x[2])) | static_cast<uint32_t>(f32_to_bf16(x[3])) << 16);
}

// Column accesses of the passes over the chunks. A lane has a column and, one register each, the rows `row` to
// row + 3: a buffer over the chunk's rows of one head from row r on for register r, and the lane's column and first
// row in its offset. Rows and columns past the end are out of that buffer's range (which is empty if the chunk ends
// before r): they read as zero and are not written. (A scalar offset for r would be left out of the range check; a
// check of every row by its lane took 40 registers more.) Rows that are closer than their length, a broadcast's, may
// read a row that is there in place of one that is not: beta, P and q are zero there, and what they multiply is an
// operand's own value.
constexpr uint32_t kOutOfRange = 0x80000000u;
template <typename E>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_buffer(const E* p, int64_t st_, int rows, int cols, int r = 0) {
  const int64_t records = rows > r ? (rows - 1 - r) * st_ + cols : 0;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<E*>(p) + (rows > r ? r * st_ : 0), static_cast<short>(0),
                                           static_cast<int>(records * sizeof(E)), 0x00020000);
}
template <typename E>
__device__ __forceinline__ uint32_t load_col(__amdgpu_buffer_rsrc_t r, uint32_t off) {  // raw
  if constexpr (sizeof(E) == 2)
    return __builtin_amdgcn_raw_buffer_load_b16(r, off, 0, 0);
  else
    return __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0);
}
template <typename E>
__device__ __forceinline__ float value(uint32_t raw) {
  return __uint_as_float(sizeof(E) == 2 ? raw << 16 : raw);
}
template <typename E>
__device__ __forceinline__ void store_col(__amdgpu_buffer_rsrc_t r, uint32_t off, float x) {
  if constexpr (sizeof(E) == 2)
    __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(x), r, off, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x), r, off, 0, 0);
}

// four columns of a row
template <typename E>
__device__ __forceinline__ void store_cols(__amdgpu_buffer_rsrc_t r, uint32_t off, const f32x4& x) {
  if constexpr (sizeof(E) == 2) {
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 v = {static_cast<uint32_t>(f32_to_bf16(x[0])) | static_cast<uint32_t>(f32_to_bf16(x[1])) << 16,
                     static_cast<uint32_t>(f32_to_bf16(x[2])) | static_cast<uint32_t>(f32_to_bf16(x[3])) << 16};
    __builtin_amdgcn_raw_buffer_store_b64(v, r, off, 0, 0);
  } else {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, x), r, off, 0, 0);
  }
}

// 8 values at any alignment: where one row's start and its length are multiples of 8 elements the memory
// pipe takes them in one piece (two of fp32)
typedef unsigned short u16x8u __attribute__((ext_vector_type(8), aligned(2)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
template <typename E> struct raw8;
template <> struct raw8<bf16_t> {
  u16x8u v = {0, 0, 0, 0, 0, 0, 0, 0};
  __device__ __forceinline__ void load(const bf16_t* p) { v = *reinterpret_cast<const u16x8u*>(p); }
  __device__ __forceinline__ void limbs(bf16x8 (&out)[1]) const { out[0] = __builtin_bit_cast(bf16x8, v); }
};
template <> struct raw8<float> {
  f32x4u v[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
  __device__ __forceinline__ void load(const float* p) {
    v[0] = reinterpret_cast<const f32x4u*>(p)[0], v[1] = reinterpret_cast<const f32x4u*>(p)[1];
  }
  __device__ __forceinline__ void limbs(bf16x8 (&out)[3]) const {
    const float x[8] = {v[0][0], v[0][1], v[0][2], v[0][3], v[1][0], v[1][1], v[1][2], v[1][3]};
    split<3>(x, out);
  }
};

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

// One chunk's operands as chunk_kernel leaves them in memory: fragments of the matrix instructions, 1 KiB for a
// limb of one (16 bytes per lane), each read by one wave of a pass straight into the registers that the instruction
// takes them from. Rows of k and q [tile of 16 tokens, in row_of order][32 of K]; k^T and q^T [16 of K, in row_of
// order][32 tokens]; of T and P the blocks of 16 rows and 32 columns that reach the diagonal, and of T^T and P^T;
// each with its limbs (of P two for bf16, whose o is rounded to it; of P^T
// three, as the state's gradient is fp32). And the vectors e^G, e^{G_C - G}, beta. What only the backward reads comes last.
template <int KP, int NI>
struct Tile {
  static constexpr int NP = NI == 3 ? 3 : 2, KB = KP / 32, U = KP / 8;
  static constexpr int F = 1024, kRows = 4 * KB * NI * F, nT = 6 * 3 * F, nP = 6 * NP * F;
  static constexpr int kK = 0, kKT = kRows, kQ = 2 * kRows, kT = 3 * kRows, kP = kT + nT, kGate = kP + nP, kOnce = kGate + F;
  static constexpr int kQT = kOnce, kTT = kQT + kRows, kPT = kTT + nT, kKept = kPT + nT;
  // limb 0 of block (tile t, 32 of K or 32 tokens b)
  static constexpr int rows(int t, int kb) { return (t * KB + kb) * NI * F; }
  static constexpr int cols(int t, int p) { return (t * 2 + p) * NI * F; }
  // the blocks (w, p) of T or P with p <= w / 2, and those of their transposes with p >= w / 2
  static constexpr int low(int w, int p, int n) { return ((w < 2 ? w : 2 * w - 2) + p) * n * F; }
  static constexpr int high(int w, int p, int n) { return (w < 2 ? 2 * w + p : w + 2) * n * F; }
  // unit u of row r of k or q (limb 0) in `rows`' order
  __device__ static int unit(int r, int u) {
    return rows(2 * (r >> 5) + ((r >> 2) & 1), u >> 2) + (16 * (u & 3) + 4 * ((r >> 3) & 3) + (r & 3)) * 16;
  }
};

template <int N>
__device__ __forceinline__ void load_frag(const char* p, int lane, bf16x8 (&out)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = *reinterpret_cast<const bf16x8*>(p + l * 1024 + lane * 16);
}
template <int N>
__device__ __forceinline__ void store_frag(char* p, int lane, const bf16x8 (&x)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) *reinterpret_cast<bf16x8*>(p + l * 1024 + lane * 16) = x[l];
}

template <int BYTES, int WAVES>
__device__ __forceinline__ void stage(char* lds, const void* src, int lane, int wave) {  // BYTES / 1024 / WAVES loads a wave, rounded up
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
// the same, columns in their own order, from k or q as they lie in a chunk's image
template <typename L, int NI>
__device__ __forceinline__ void frags_t_image(const char* x, int t, int p, int lane, bf16x8 (&out)[NI]) {
  const int g = lane >> 4, j = (lane >> 2) & 3, q = lane & 3, r = 32 * p + 8 * g + j;
#pragma unroll
  for (int l = 0; l < NI; ++l) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + L::unit(r, 2 * t + (q >> 1)) + l * 1024 + 8 * (q & 1)));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + L::unit(r + 4, 2 * t + (q >> 1)) + l * 1024 + 8 * (q & 1)));
    out[l] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// 4 values (one accumulator) as N limbs of half a fragment
template <int N>
__device__ __forceinline__ void split4(const f32x4& x, uint2 (&out)[N]) {
  uint32_t a[N], b[N];
  pair_limbs(x[0], x[1], a);
  pair_limbs(x[2], x[3], b);
#pragma unroll
  for (int l = 0; l < N; ++l) out[l] = make_uint2(a[l], b[l]);
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

// The blocks of a 64 x 64 lower triangle in LDS as N limbs, and with `both` those of its transpose as three, to the
// image: wave w's tiles w
template <int N>
__device__ __forceinline__ void put_blocks(const float* m, char* low, char* high, bool both, int lane, int w) {
  using L = Tile<64, 1>;
  const int r = row_of(w, lane & 15), g = lane >> 4;
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int c0 = 32 * p + 8 * g;
    float x[8];
    bf16x8 l[N], h[3];
    if (p <= w / 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = c0 + i <= r ? m[r * LD + c0 + i] : 0.0f;
      split<N>(x, l);
      store_frag(low + L::low(w, p, N), lane, l);
    }
    if (both && p >= w / 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = r <= c0 + i ? m[(c0 + i) * LD + r] : 0.0f;
      split<3>(x, h);
      store_frag(high + L::high(w, p, 3), lane, h);
    }
  }
}

// k and q are read once, all loads of a thread under way at a time, and go to LDS and from there, as fragments, to the
// image; A and T take over the LDS once k k^T and q k^T are in registers, P A's once T is done: 36 KB, four workgroups
// to a CU. Bound by memory, by what the image takes: 69 us for 340 MB (131 KB a chunk with what the backward
// reads), 184 us for 930 MB (79 KB a chunk): 5.0 and 5.1 TB/s. (Reading k and q where they were needed, one
// load after the other: 84 us for a smaller image, at 2.6 TB/s.)
template <int KP, int NI>
__global__ __launch_bounds__(256, NI == 1 ? 4 : 1) void chunk_kernel(Args a, bool keep) {
  using E = typename elem<NI>::type;
  using L = Tile<KP, NI>;
  constexpr int U = KP / 8, KB = KP / 32, kRows = NI * C * KP * 2, kLds = 2 * kRows > 2 * C * LD * 4 ? 2 * kRows : 2 * C * LD * 4;
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ double sG[C];
  __shared__ float sB[C];
  float *sA = reinterpret_cast<float*>(lds), *sT = sA + C * LD;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x;
  const int bh = blockIdx.x / a.NC, n = blockIdx.x - bh * a.NC, h = bh % a.H, b = bh / a.H, grp = a.H / a.Hk;
  const int hk = h / grp, t0 = n * C, rows = min(C, a.T - t0);
  const E* k = reinterpret_cast<const E*>(a.k) + b * a.k_sb + t0 * a.k_st + hk * a.k_sh;
  const E* q = reinterpret_cast<const E*>(a.q) + b * a.q_sb + t0 * a.q_st + hk * a.q_sh;
  char* img = a.img + c * (keep ? L::kKept : L::kOnce);
  float gv = 0.0f, bv = 0.0f;
  if (wave == 0 && lane < rows) {
    gv = ld(reinterpret_cast<const E*>(a.g) + b * a.g_sb + (t0 + lane) * a.g_st + h * a.g_sh);
    bv = ld(reinterpret_cast<const E*>(a.beta) + b * a.b_sb + (t0 + lane) * a.b_st + h * a.b_sh);
    gv = gv < kMinLog ? kMinLog : gv;
  }
  {
    raw8<E> rk[C * U / 256], rq[C * U / 256];
#pragma unroll
    for (int i = 0; i < C * U / 256; ++i) {  // (what is outside reads the chunk's first values: no branches between the loads)
      const int r = (tid + 256 * i) / U, u = tid % U;
      const bool ok = r < rows && 8 * u < a.K;
      rk[i].load(k + (ok ? r * a.k_st + 8 * u : 0));
      rq[i].load(q + (ok ? r * a.q_st + 8 * u : 0));
    }
#pragma unroll
    for (int i = 0; i < C * U / 256; ++i) {
      const int r = (tid + 256 * i) / U, u = tid % U;
      if (!(r < rows && 8 * u < a.K)) rk[i] = rq[i] = raw8<E>();
      bf16x8 lk[NI], lq[NI];
      rk[i].limbs(lk);
      rq[i].limbs(lq);
#pragma unroll
      for (int l = 0; l < NI; ++l) {
        const int pos = l * C * KP * 2 + at<U>(r, u);
        *reinterpret_cast<bf16x8*>(lds + pos) = lk[l];
        *reinterpret_cast<bf16x8*>(lds + kRows + pos) = lq[l];
      }
    }
  }
  if (wave == 0) {
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
  __syncthreads();
  {
    const auto put = [&](int base, int from, int t) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        bf16x8 f[NI];
        frags<U>(lds + from, C * KP * 2, t, kb, lane, f);
        store_frag(img + base + L::rows(t, kb), lane, f);
      }
    };
    const auto put_t = [&](int base, int from, int t) {
#pragma unroll
      for (int i = 0; i < KP / 64; ++i)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          bf16x8 f[NI];
          frags_t<U, true>(lds + from, C * KP * 2, t + 4 * i, p, lane, f);
          store_frag(img + base + L::cols(t + 4 * i, p), lane, f);
        }
    };
    put(L::kK, 0, wave);
    put(L::kQ, kRows, wave);
    put_t(L::kKT, 0, wave);
    if (keep) put_t(L::kQT, kRows, wave);
  }
  // k k^T, rows 16 wave ...; q k^T, rows 16 (3 - wave) ...: five blocks of the lower triangles each, transposed: a
  // lane has one row and four consecutive columns
  const int wq = 3 - wave;
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) kk[i] = qk[i] = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int kb = 0; kb < KP / 32; ++kb) {
    const auto rows_of = [&](int base, int t, bf16x8 (&out)[NI]) {
#pragma unroll
      for (int l = 0; l < NI; ++l) out[l] = frag_plain<U>(lds + base + l * C * KP * 2, t, kb, lane);
    };
    bf16x8 ak[NI], aq[NI];
    rows_of(0, wave, ak);
    rows_of(kRows, wq, aq);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i <= wave || i <= wq) {
        bf16x8 bk[NI];
        rows_of(0, i, bk);
        if (i <= wave) kk[i] = mm<NI>(bk, ak, kk[i]);
        if (i <= wq) qk[i] = mm<NI>(bk, aq, qk[i]);
      }
    }
  }
  __syncthreads();
  {
    const int ra = 16 * wave + m;
    const double ga = sG[ra];
    const float be = sB[ra];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 16 * i + 4 * g;
      f32x4 x;
      if (i <= wave) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float e = be * expf(col + r < ra ? static_cast<float>(ga - sG[col + r]) : 0.0f) * kk[i][r];
          x[r] = col + r < ra ? e : 0.0f;
        }
        *reinterpret_cast<f32x4*>(sA + ra * LD + col) = x;
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
  {  // P in A's place
    const int rp = 16 * wq + m;
    const double gp = sG[rp];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 16 * i + 4 * g;
      f32x4 x;
      if (i <= wq) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[r] = a.scale * expf(col + r <= rp ? static_cast<float>(gp - sG[col + r]) : 0.0f) * qk[i][r];
        *reinterpret_cast<f32x4*>(sA + rp * LD + col) = x;
      }
    }
  }
  put_blocks<3>(sT, img + L::kT, img + L::kTT, keep, lane, wave);
  __syncthreads();
  put_blocks<L::NP>(sA, img + L::kP, img + L::kPT, keep, lane, wave);
}

// ---------------------------------------------------------------- the pass over the chunks
//
// A workgroup of eight waves owns 16 CT value columns of one head's state and takes the chunks in order. Four of
// them are the chain: the state never leaves their accumulators. Wave w holds rows 32 w ... 32 w + 31 of S and, in
// each chunk, makes 16 of the 64 tokens' y and d (dd and dy in the backward). What other waves need as a B
// operand, S for K S, y for T y, d for K^T d, goes through LDS as limbs, already in the operand's register order (an
// accumulator's lane is the operand's lane: a fragment is 16 bytes per lane, written and read without conflicts).
// The A operands are different for every wave, so they pass no LDS: each wave loads its own fragments from the
// chunk's image into registers, a chunk ahead. Three barriers a chunk. The other four waves do what the chain does
// not wait for, between the same barriers: o = scale e^G Q S + P d and what is kept; in the backward P^T do and
// Q^T (scale e^G do), a chunk ahead.
//
// Bound by the chain: 521 us for 256 chunks are 2.0 us a chunk, of which 1.3 pass with no loads at all (dependent
// products, limbs, three exchanges) and the rest are loads that come late when all CUs draw on the L2s (each of a head's
// workgroups loads all of its image). B8 T2047 H8: state 135, its gradient 144 us, 3.1 TB/s for the 430 MB each that
// cross memory. Tried before, B2 T16381 H16: a wave of its own for each 16 columns with no exchange, 1053 us; the
// operands through LDS by asynchronous copies, 553; no separate waves for o, 504. Asking for the image two chunks
// ahead so that the loads find it in L2 changed nothing.

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

// B operands in LDS, kFrag bytes per fragment and limb: fragment f of F, limb l at (l F + f) kFrag
constexpr int kFrag = 1024;
template <int F, int N>
__device__ __forceinline__ void put_half(char* x, int f, int lane, int half, const uint2 (&v)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) *reinterpret_cast<uint2*>(x + (l * F + f) * kFrag + lane * 16 + half * 8) = v[l];
}
template <int F, int N>
__device__ __forceinline__ void put_full(char* x, int f, int lane, const bf16x8 (&v)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) *reinterpret_cast<bf16x8*>(x + (l * F + f) * kFrag + lane * 16) = v[l];
}
template <int F, int N>
__device__ __forceinline__ void get(const char* x, int f, int lane, bf16x8 (&v)[N]) {
#pragma unroll
  for (int l = 0; l < N; ++l) v[l] = *reinterpret_cast<const bf16x8*>(x + (l * F + f) * kFrag + lane * 16);
}

// All waves' LDS accesses so far are done; loads to registers stay under way
__device__ __forceinline__ void sync() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// All loads so far are there, as far as the compiler's own waits go too: what it counts in a loop are then the
// loop's operations alone (0x0f70: vmcnt 0, the other counters as they are)
__device__ __forceinline__ void settled() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// What a wave of a pass works on
template <int CT>
struct Place {
  int lane, w, m, g, bh, h, b, tile;
  bool chain;  // one of the waves 0 to 3
  __device__ __forceinline__ explicit Place(const Args& a) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    lane = threadIdx.x & 63, w = wave & 3, m = lane & 15, g = lane >> 4, chain = wave < 4;
    place(blockIdx.x, a.B * a.H, a.VP / 16 / CT, bh, tile);
    h = bh % a.H, b = bh / a.H;
  }
  __device__ __forceinline__ int col(int i) const { return (tile * CT + i) * 16 + m; }
};

// This wave's rows of the state (or its gradient), from dense [K][V] fp32, or zero
template <int CT, typename P>
__device__ __forceinline__ void load_state(f32x4 (&S)[CT][2], const float* s, const Args& a, const P& p) {
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = row_of(2 * p.w + t, 4 * p.g + r);
        S[i][t][r] = s && p.col(i) < a.V && d < a.K ? s[(static_cast<int64_t>(p.bh) * a.K + d) * a.V + p.col(i)] : 0.0f;
      }
}
template <int CT, typename P>
__device__ __forceinline__ void store_state(const f32x4 (&S)[CT][2], float* s, const Args& a, const P& p) {
#pragma unroll
  for (int i = 0; i < CT; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = row_of(2 * p.w + t, 4 * p.g + r);
        if (p.col(i) < a.V && d < a.K) s[(static_cast<int64_t>(p.bh) * a.K + d) * a.V + p.col(i)] = S[i][t][r];
      }
}

// What is kept of 32 value columns for the gradients, in the order of the accumulators, so that a wave writes whole
// lines: S and dS' [16 columns][32 of K][limb], unit g (8 of K) of column m at 16 g + m; d and dy [16 columns]
// [32 tokens][limb][wave's half], four tokens of column m at 16 g + m. Odd units and halves have m ^ 4: grad_kernel
// reads across the columns, and these land on other banks then.
template <int KP, int NI>
struct Kept {
  static constexpr int NW = kKept<NI>, kState = 2 * (KP / 32) * NW * 1024, kVec = 2 * 2 * NW * 1024;  // bytes of 32 columns
  __device__ static int state(int col, int u) {  // limb 0 of unit u
    return ((col >> 4) * (KP / 32) + (u >> 2)) * NW * 1024 + (16 * (u & 3) + ((col & 15) ^ (4 * (u & 1)))) * 16;
  }
  __device__ static int vec(int col, int t) {  // limb 0 of tokens t ... t + 3 (t a multiple of 4)
    const int h = (t >> 2) & 1;
    return ((col >> 4) * 2 + (t >> 5)) * NW * 1024 + h * 512 + (16 * ((t >> 3) & 3) + ((col & 15) ^ (4 * h))) * 8;
  }
};
// Operand through the transposing read as frag_t: columns 16 t ... (of K, tokens) of the matrix, its 32 rows (value columns)
template <typename P, int N>
__device__ __forceinline__ void kept_frags(const char* x, P pos, int lane, bf16x8 (&out)[N]) {
  const int g = lane >> 4, j = (lane >> 2) & 3, q = lane & 3, a0 = pos(8 * g + j, q), a1 = pos(8 * g + j + 4, q);
#pragma unroll
  for (int l = 0; l < N; ++l) {
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + a0 + l * 1024));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(x + a1 + l * 1024));
    out[l] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
  }
}

// This wave's rows of the state to the other waves
template <int KP, int CT, typename P>
__device__ __forceinline__ void publish(const f32x4 (&S)[CT][2], char* xs, const P& p) {
  if (KP == 128 || p.w < KP / 32) {  // (four waves)
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const float x[8] = {S[i][0][0], S[i][0][1], S[i][0][2], S[i][0][3], S[i][1][0], S[i][1][1], S[i][1][2], S[i][1][3]};
      bf16x8 l[3];
      split<3>(x, l);
      put_full<CT * (KP / 32)>(xs, i * (KP / 32) + p.w, p.lane, l);
    }
  }
}
// What lies in LDS of the state, and of d, to memory: a fragment's limbs, or halves of one, by one wave each
template <int KP, int NI, int CT, typename P>
__device__ __forceinline__ void keep_state(char* kept, int64_t c, const char* xs, const Args& a, const P& p) {
  using L = Kept<KP, NI>;
  constexpr int KB = KP / 32, N = CT * KB;
#pragma unroll
  for (int j = 0; j < (N + 3) / 4; ++j) {
    const int f = 4 * j + p.w;
    if (N % 4 == 0 || f < N) {
      const int col = (p.tile * CT + f / KB) * 16 + p.m;
      char* out = kept + (c * (a.VP / 32) + col / 32) * L::kState + L::state(col % 32, 4 * (f % KB) + p.g);
#pragma unroll
      for (int q = 0; q < L::NW; ++q)
        *reinterpret_cast<bf16x8*>(out + q * 1024) = *reinterpret_cast<const bf16x8*>(xs + (q * N + f) * kFrag + p.lane * 16);
    }
  }
}
template <int KP, int NI, int CT, typename P>
__device__ __forceinline__ void keep_vec(char* kept, int64_t c, const char* xd, const Args& a, const P& p) {
  using L = Kept<KP, NI>;
  constexpr int N = 2 * CT * L::NW;
#pragma unroll
  for (int j = 0; j < (N + 3) / 4; ++j) {
    const int x = 4 * j + p.w, f = x % (2 * CT), q = x / (2 * CT);
    if (N % 4 == 0 || x < N) {
      const int col = (p.tile * CT + f / 2) * 16 + p.m;
      char* out = kept + (c * (a.VP / 32) + col / 32) * L::kVec + q * 1024;
      const uint4 v = *reinterpret_cast<const uint4*>(xd + x * kFrag + p.lane * 16);
      *reinterpret_cast<uint2*>(out + L::vec(col % 32, 32 * (f % 2) + 8 * p.g)) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(out + L::vec(col % 32, 32 * (f % 2) + 8 * p.g + 4)) = make_uint2(v.z, v.w);
    }
  }
}
// Half a fragment of dy
template <int KP, int NI, typename P>
__device__ __forceinline__ void keep_half(char* kept, int64_t c, int col, const uint2 (&l)[kKept<NI>], const Args& a, const P& p) {
  using L = Kept<KP, NI>;
  char* out = kept + (c * (a.VP / 32) + col / 32) * L::kVec + L::vec(col % 32, row_of(p.w, 4 * p.g));
#pragma unroll
  for (int q = 0; q < L::NW; ++q) *reinterpret_cast<uint2*>(out + q * 1024) = l[q];
}

template <int KP, int NI, bool KEEP, int CT>
__global__ __launch_bounds__(512) void state_kernel(Args a) {
  using E = typename elem<NI>::type;
  using I = Tile<KP, NI>;
  constexpr int KB = I::KB, NP = I::NP;
  __shared__ __attribute__((aligned(16))) char xs[CT * KB * 3 * kFrag], xy[CT * 6 * kFrag], xe[CT * 6 * kFrag], xd[CT * 2 * NP * kFrag];
  const Place<CT> p(a);
  const int lane = p.lane, g = p.g, w = p.w, pw = w / 2;
  constexpr int64_t kImage = KEEP ? I::kKept : I::kOnce;
  const char* img = a.img + static_cast<int64_t>(p.bh) * a.NC * kImage;

  // What a chunk takes from memory is loaded anew for the next one once its last reader is through. (A loop for each
  // half of the waves: how many blocks of T and P a wave has is then known, and so is how many operations later than
  // its loads a wait may leave under way.)
  const auto chain = [&](auto half) __attribute__((always_inline)) {
    const E* v = reinterpret_cast<const E*>(a.v) + p.b * a.v_sb + p.h * a.v_sh;
    const uint32_t vs = static_cast<uint32_t>(a.v_st * sizeof(E));
    const int row = row_of(w, 4 * g);  // the lane's first of four tokens
    uint32_t next[CT][4];
    bf16x8 fk[KB][NI], ft[2][3], kt[2][2][NI];
    f32x4 eg, tail, be;
    float last;
    const auto load_v = [&](int n) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const __amdgpu_buffer_rsrc_t vr = rows_buffer(v + static_cast<int64_t>(n) * C * a.v_st, a.v_st, min(C, a.T - n * C), a.V, r);
#pragma unroll
        for (int i = 0; i < CT; ++i) next[i][r] = load_col<E>(vr, p.col(i) < a.V ? row * vs + p.col(i) * sizeof(E) : kOutOfRange);
      }
    };
    const auto load_rows = [&](int n) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) load_frag(img + n * kImage + I::kK + I::rows(w, kb), lane, fk[kb]);
    };
    const auto load_gates = [&](int n) {
      const float* gt = reinterpret_cast<const float*>(img + n * kImage + I::kGate);
      eg = *reinterpret_cast<const f32x4*>(gt + row), tail = *reinterpret_cast<const f32x4*>(gt + 64 + row);
      be = *reinterpret_cast<const f32x4*>(gt + 128 + row), last = gt[63];
    };
    const auto load_t = [&](int n) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (q <= half.value) load_frag(img + n * kImage + I::kT + I::low(w, q, 3), lane, ft[q]);
    };
    const auto load_cols = [&](int n) {
      if (KB == 4 || w < KB) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) load_frag(img + n * kImage + I::kKT + I::cols(2 * w + t, q), lane, kt[t][q]);
      }
    };
    f32x4 S[CT][2];
    load_state(S, a.h0, a, p);
    load_rows(0), load_gates(0), load_v(0), load_t(0), load_cols(0);
    publish<KP>(S, xs, p);
    settled();
    sync();
#pragma unroll 1
    for (int n = 0; n < a.NC; ++n) {
      const int n1 = min(n + 1, a.NC - 1);  // (the last chunk loads itself once more)
      f32x4 ks[CT];  // y: this wave's 16 tokens
#pragma unroll
      for (int i = 0; i < CT; ++i) ks[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          bf16x8 sb[3];
          get<CT * KB>(xs, i * KB + kb, lane, sb);
          ks[i] = mm<3>(fk[kb], sb, ks[i]);
        }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        f32x4 vv;
#pragma unroll
        for (int r = 0; r < 4; ++r) vv[r] = value<E>(next[i][r]);
        uint2 l[3];
        split4(be * (vv - eg * ks[i]), l);
        put_half<2 * CT>(xy, 2 * i + pw, lane, w & 1, l);
      }
      const f32x4 tl = tail;
      const float decay = last;
      load_rows(n1), load_gates(n1), load_v(n1);
      sync();  // y is there
      f32x4 d2[CT][2], d[CT];
#pragma unroll
      for (int i = 0; i < CT; ++i) d2[i][0] = d2[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q <= half.value) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            bf16x8 yb[3];
            get<2 * CT>(xy, 2 * i + q, lane, yb);
            mm2<3>(ft[q], yb, d2[i]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        uint2 l[3], dl[NP];
        d[i] = d2[i][0] + d2[i][1];
        split4(tl * d[i], l);
        put_half<2 * CT>(xe, 2 * i + pw, lane, w & 1, l);
        split4(d[i], dl);
        put_half<2 * CT>(xd, 2 * i + pw, lane, w & 1, dl);
      }
      load_t(n1);
      sync();  // d is there
      if (KB == 4 || w < KB) {
#pragma unroll
        for (int i = 0; i < CT; ++i) S[i][0] *= decay, S[i][1] *= decay;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            bf16x8 eb[3];
            get<2 * CT>(xe, 2 * i + q, lane, eb);
            S[i][0] = mm<3>(kt[0][q], eb, S[i][0]);
            S[i][1] = mm<3>(kt[1][q], eb, S[i][1]);
          }
        }
      }
      load_cols(n1);
      publish<KP>(S, xs, p);
      sync();  // the state is there
    }
    if (a.state && w < KB) store_state(S, a.state, a, p);
  };

  // o, transposed (a lane has a token and four columns), and what is kept
  const auto beside = [&](auto half) __attribute__((always_inline)) {
    const int64_t o_st = static_cast<int64_t>(a.H) * a.V;
    E* o = reinterpret_cast<E*>(a.o) + (static_cast<int64_t>(p.b) * a.T * a.H + p.h) * a.V;
    const uint32_t os = static_cast<uint32_t>(o_st * sizeof(E));
    const int row = row_of(w, p.m);
    bf16x8 fq[KB][NI], fp[2][NP];
    float eg;
    const auto load_rows = [&](int n) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) load_frag(img + n * kImage + I::kQ + I::rows(w, kb), lane, fq[kb]);
      eg = reinterpret_cast<const float*>(img + n * kImage + I::kGate)[row];
    };
    const auto load_p = [&](int n) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (q <= half.value) load_frag(img + n * kImage + I::kP + I::low(w, q, NP), lane, fp[q]);
    };
    load_rows(0), load_p(0);
    settled();
    sync();
#pragma unroll 1
    for (int n = 0; n < a.NC; ++n) {
      const int t0 = n * C, rows = min(C, a.T - t0), n1 = min(n + 1, a.NC - 1);
      const int64_t c = static_cast<int64_t>(p.bh) * a.NC + n;
      f32x4 oa[CT];
#pragma unroll
      for (int i = 0; i < CT; ++i) oa[i] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          bf16x8 sb[3];
          get<CT * KB>(xs, i * KB + kb, lane, sb);
          oa[i] = mm<NP>(sb, fq[kb], oa[i]);  // (only o, which is rounded to the inputs' type, sees this product)
        }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) oa[i] *= a.scale * eg;
      if constexpr (KEEP) keep_state<KP, NI, CT>(a.Sw, c, xs, a, p);
      load_rows(n1);
      sync();
      sync();  // d is there
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q <= half.value) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            bf16x8 db[NP];
            get<2 * CT>(xd, 2 * i + q, lane, db);
            oa[i] = mm<NP>(db, fp[q], oa[i]);
          }
        }
      }
      load_p(n1);
      const __amdgpu_buffer_rsrc_t orr = rows_buffer(o + t0 * o_st, o_st, rows, a.V);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        const int col = (p.tile * CT + i) * 16 + 4 * g;
        store_cols<E>(orr, col < a.V ? row * os + col * sizeof(E) : kOutOfRange, oa[i]);
      }
      if constexpr (KEEP) keep_vec<KP, NI, CT>(a.dw, c, xd, a, p);
      sync();  // the state is there
    }
  };
  if (p.chain) {
    if (pw == 0)
      chain(int_c<0>{});
    else
      chain(int_c<1>{});
  } else {
    if (pw == 0)
      beside(int_c<0>{});
    else
      beside(int_c<1>{});
  }
}

template <int KP, int NI, int CT>
__global__ __launch_bounds__(512) void dstate_kernel(Args a) {
  using E = typename elem<NI>::type;
  using I = Tile<KP, NI>;
  constexpr int KB = I::KB, NW = kKept<NI>;
  __shared__ __attribute__((aligned(16))) char xs[CT * KB * 3 * kFrag], xy[CT * 6 * kFrag], xe[CT * 6 * kFrag];
  __shared__ __attribute__((aligned(16))) char xu[CT * 6 * kFrag], xo[CT * 2 * NI * kFrag];
  __shared__ f32x4 xp[4][CT][64], xq[4][CT][2][64];  // P^T do and Q^T (scale e^G do) in the accumulators' order
  const Place<CT> p(a);
  const int lane = p.lane, g = p.g, w = p.w, pw = w / 2;
  constexpr int64_t kImage = I::kKept;
  const char* img = a.img + static_cast<int64_t>(p.bh) * a.NC * kImage;
  const int row = row_of(w, 4 * g), last_n = a.NC - 1;

  const auto chain = [&](auto half) __attribute__((always_inline)) {
    const int64_t v_st = static_cast<int64_t>(a.H) * a.V;
    E* dv = reinterpret_cast<E*>(a.dv) + (static_cast<int64_t>(p.b) * a.T * a.H + p.h) * a.V;
    const uint32_t os = static_cast<uint32_t>(v_st * sizeof(E));
    bf16x8 fk[KB][NI], ft[2][3], kt[2][2][NI];
    f32x4 eg, tail, be;
    float last;
    const auto load_rows = [&](int n) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) load_frag(img + n * kImage + I::kK + I::rows(w, kb), lane, fk[kb]);
    };
    const auto load_gates = [&](int n) {
      const float* gt = reinterpret_cast<const float*>(img + n * kImage + I::kGate);
      eg = *reinterpret_cast<const f32x4*>(gt + row), tail = *reinterpret_cast<const f32x4*>(gt + 64 + row);
      be = *reinterpret_cast<const f32x4*>(gt + 128 + row), last = gt[63];
    };
    const auto load_t = [&](int n) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (q >= half.value) load_frag(img + n * kImage + I::kTT + I::high(w, q, 3), lane, ft[q]);
    };
    const auto load_cols = [&](int n) {
      if (KB == 4 || w < KB) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) load_frag(img + n * kImage + I::kKT + I::cols(2 * w + t, q), lane, kt[t][q]);
      }
    };
    f32x4 S[CT][2];  // the gradient of the state
    load_state(S, a.dstate, a, p);
    load_rows(last_n), load_gates(last_n), load_t(last_n), load_cols(last_n);
    publish<KP>(S, xs, p);
    settled();
    sync();
    sync();
#pragma unroll 1
    for (int n = last_n; n >= 0; --n) {
      const int t0 = n * C, rows = min(C, a.T - t0), n1 = max(n - 1, 0);  // (the last chunk loads itself once more)
      const int64_t c = static_cast<int64_t>(p.bh) * a.NC + n;
      f32x4 dd[CT], add[CT][2];
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        dd[i] = f32x4{0, 0, 0, 0};
        add[i][0] = xq[w][i][0][lane], add[i][1] = xq[w][i][1][lane];
      }
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          bf16x8 sb[3];
          get<CT * KB>(xs, i * KB + kb, lane, sb);
          dd[i] = mm<3>(fk[kb], sb, dd[i]);
        }
      }
      load_rows(n1);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        uint2 l[3];
        split4(tail * dd[i] + xp[w][i][lane], l);
        put_half<2 * CT>(xy, 2 * i + pw, lane, w & 1, l);
      }
      sync();  // dd is there
      f32x4 d2[CT][2], dy[CT];
#pragma unroll
      for (int i = 0; i < CT; ++i) d2[i][0] = d2[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q >= half.value) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            bf16x8 b[3];
            get<2 * CT>(xy, 2 * i + q, lane, b);
            mm2<3>(ft[q], b, d2[i]);
          }
        }
      }
      load_t(n1);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        dy[i] = d2[i][0] + d2[i][1];
        const f32x4 x = be * dy[i];
        uint2 l[3];
        split4(-eg * x, l);
        put_half<2 * CT>(xe, 2 * i + pw, lane, w & 1, l);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          store_col<E>(rows_buffer(dv + t0 * v_st, v_st, rows, a.V, r), p.col(i) < a.V ? row * os + p.col(i) * sizeof(E) : kOutOfRange, x[r]);
      }
      const float decay = last;
      load_gates(n1);
      sync();  // e^G beta dy is there
      if (KB == 4 || w < KB) {
#pragma unroll
        for (int i = 0; i < CT; ++i) S[i][0] = decay * S[i][0] + add[i][0], S[i][1] = decay * S[i][1] + add[i][1];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
          for (int i = 0; i < CT; ++i) {
            bf16x8 b[3];
            get<2 * CT>(xe, 2 * i + q, lane, b);
            S[i][0] = mm<3>(kt[0][q], b, S[i][0]);
            S[i][1] = mm<3>(kt[1][q], b, S[i][1]);
          }
        }
      }
      load_cols(n1);
      publish<KP>(S, xs, p);
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        uint2 l[NW];
        split4(dy[i], l);
        keep_half<KP, NI>(a.yw, c, p.col(i), l, a, p);
      }
      sync();  // the state is there
    }
    if (a.dh0 && w < KB) store_state(S, a.dh0, a, p);
  };

  // What depends on do alone, a chunk ahead of the chain, and what is kept of the state's gradient
  const auto beside = [&](auto half) __attribute__((always_inline)) {
    const E* dout = reinterpret_cast<const E*>(a.dout) + p.b * a.do_sb + p.h * a.do_sh;
    const uint32_t is = static_cast<uint32_t>(a.do_st * sizeof(E));
    uint32_t next[CT][4];
    bf16x8 fp[2][3], qt[2][2][NI];
    f32x4 eg;
    const auto load_go = [&](int n) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const __amdgpu_buffer_rsrc_t ir = rows_buffer(dout + static_cast<int64_t>(n) * C * a.do_st, a.do_st, min(C, a.T - n * C), a.V, r);
#pragma unroll
        for (int i = 0; i < CT; ++i) next[i][r] = load_col<E>(ir, p.col(i) < a.V ? row * is + p.col(i) * sizeof(E) : kOutOfRange);
      }
      eg = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(img + n * kImage + I::kGate) + row);
    };
    const auto put_go = [&]() {
#pragma unroll
      for (int i = 0; i < CT; ++i) {
        f32x4 go;
#pragma unroll
        for (int r = 0; r < 4; ++r) go[r] = value<E>(next[i][r]);
        uint2 l[NI], u[3];
        split4(go, l);
        put_half<2 * CT>(xo, 2 * i + pw, lane, w & 1, l);
        split4(a.scale * eg * go, u);
        put_half<2 * CT>(xu, 2 * i + pw, lane, w & 1, u);
      }
    };
    const auto load_pq = [&](int n) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        if (q >= half.value) load_frag(img + n * kImage + I::kPT + I::high(w, q, 3), lane, fp[q]);
      if (KB == 4 || w < KB) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int q = 0; q < 2; ++q) load_frag(img + n * kImage + I::kQT + I::cols(2 * w + t, q), lane, qt[t][q]);
      }
    };
    const auto products = [&]() {
      f32x4 x[CT], y[CT][2];
#pragma unroll
      for (int i = 0; i < CT; ++i) x[i] = y[i][0] = y[i][1] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int q = 0; q < 2; ++q) {
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          if (q >= half.value) {
            bf16x8 b[NI];
            get<2 * CT>(xo, 2 * i + q, lane, b);
            x[i] = mm<3>(fp[q], b, x[i]);
          }
          if (KB == 4 || w < KB) {
            bf16x8 b[3];
            get<2 * CT>(xu, 2 * i + q, lane, b);
            y[i][0] = mm<3>(qt[0][q], b, y[i][0]);
            y[i][1] = mm<3>(qt[1][q], b, y[i][1]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < CT; ++i) xp[w][i][lane] = x[i], xq[w][i][0][lane] = y[i][0], xq[w][i][1][lane] = y[i][1];
    };
    load_go(last_n), load_pq(last_n);
    put_go();
    load_go(max(last_n - 1, 0));
    sync();
    products();
    load_pq(max(last_n - 1, 0));
    settled();
    sync();
#pragma unroll 1
    for (int n = last_n; n >= 0; --n) {
      const int64_t c = static_cast<int64_t>(p.bh) * a.NC + n;
      put_go();
      load_go(max(n - 2, 0));
      keep_state<KP, NI, CT>(a.dSw, c, xs, a, p);
      sync();  // do is there, and the last products have been read
      products();
      load_pq(max(n - 2, 0));
      sync();
      sync();  // the state is there
    }
  };
  if (p.chain) {
    if (pw == 0)
      chain(int_c<0>{});
    else
      chain(int_c<1>{});
  } else {
    if (pw == 0)
      beside(int_c<0>{});
    else
      beside(int_c<1>{});
  }
}

// ---------------------------------------------------------------- sums over lanes

template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ float dpp(float x) {  // another lane's value, 0 where there is none or the row of 16 is not in ROWS
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xf, false));
}
// x: a in even rows of 16 lanes and the even rows' b in odd ones; y: the odd rows' a in even rows and b in odd ones
__device__ __forceinline__ void swap16(float a, float b, float& x, float& y) {
  const auto v = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  x = __uint_as_float(v[0]), y = __uint_as_float(v[1]);
}
__device__ __forceinline__ void swap32(float a, float b, float& x, float& y) {  // the same with halves of 32
  const auto v = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  x = __uint_as_float(v[0]), y = __uint_as_float(v[1]);
}
// The sums of four values over the four lanes m, m + 16, ...: of value g in row g
__device__ __forceinline__ float sum_groups(const float (&v)[4]) {
  float a, b, c, d;
  swap32(v[0], v[2], a, b);
  swap32(v[1], v[3], c, d);
  swap16(a + b, c + d, a, b);
  return a + b;
}
// The sums over the lanes up to each, and from each on (g: its row)
__device__ __forceinline__ float sum_up_to(float x) {
  x += dpp<0x111>(x);
  x += dpp<0x112>(x);
  x += dpp<0x114>(x);
  x += dpp<0x118>(x);
  x += dpp<0x142, 0xa>(x);  // row 0 into 1, 2 into 3
  return x + dpp<0x143, 0xc>(x);
}
__device__ __forceinline__ float sum_from(float x, int g) {
  x += dpp<0x101>(x);
  x += dpp<0x102>(x);
  x += dpp<0x104>(x);
  x += dpp<0x108>(x);
  const auto row = [&](int r) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 16 * r)); };
  const float r1 = row(1), r2 = row(2), r3 = row(3);
  return x + ((g < 1 ? r1 : 0.0f) + (g < 2 ? r2 : 0.0f) + (g < 3 ? r3 : 0.0f));
}

// ---------------------------------------------------------------- dq, dk, dg, dbeta of a chunk

template <int KP, int NI>
struct GradTile {
  static constexpr int W = KP / 16;                                           // a wave for 16 columns of dq, dk
  static constexpr int NW = kKept<NI>;
  static constexpr int kState = Kept<KP, NI>::kState, kVec = Kept<KP, NI>::kVec;  // bytes of 32 columns of a state, of d or dy,
  static constexpr int kRows = NI * C * 32 * 2;                               // of do or v
  static constexpr int kK = 0, kS = NI * C * KP * 2;                          // k; S, dS', d, dy, do, v, 32 columns at a time;
  static constexpr int kE = kS + kState, kD = kE + kState, kY = kD + kVec, kO = kY + kVec, kV = kO + kRows;
  static constexpr int kQ = kS, kF = kQ + NI * C * KP * 2, kN = kF + NW * kPlane * 2;  // then in their place q, F, N
  static constexpr int kEnd = kV + kRows > kN + NW * kPlane * 2 ? kV + kRows : kN + NW * kPlane * 2;
  static constexpr int kG = kEnd, kGate = kG + 512;                           // the chunk's G (doubles) and gates
  static constexpr int kSums = kGate + 1024;                                  // floats: dg, k.Z [W][64], dy.v [64]
  static constexpr int kBytes = kSums + (2 * W * 64 + 64) * 4;
};

// 16-byte unit u of row r of a matrix with four: a fragment's 16 rows spread over all banks
__device__ __forceinline__ int at4(int r, int u) { return (r * 4 + (u ^ ((r >> 2) & 3))) * 16; }

// A wave has 16 columns of K. The kept operands come through LDS, 32 value columns at a time; two workgroups to a CU (bf16:
// 128 registers, 78 KB), one of which works while the other waits for its operands. Bound by memory: 161 us for 600 MB,
// 3.7 TB/s, 7 of them for the terms of dg (with the sums over lanes through LDS, 17). (One workgroup to a CU, do read
// by every wave that needed it, and a lane per column, whose sums over K crossed lanes and whose stores were of two
// bytes: 278 us.)
template <int KP, int NI>
__global__ __launch_bounds__(64 * (KP / 16), NI == 3 ? 1 : KP == 128 ? 4 : 3) void grad_kernel(Args a) {
  using E = typename elem<NI>::type;
  using L = GradTile<KP, NI>;
  using I = Tile<KP, NI>;
  constexpr int NW = L::NW, W = L::W;
  __shared__ __attribute__((aligned(16))) char lds[L::kBytes];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int lane = tid & 63, m = lane & 15, g = lane >> 4;
  const int64_t c = blockIdx.x;
  const int bh = blockIdx.x / a.NC, n = blockIdx.x - bh * a.NC, h = bh % a.H, b = bh / a.H, grp = a.H / a.Hk;
  const int hk = h / grp, t0 = n * C, rows = min(C, a.T - t0);
  float* vec = reinterpret_cast<float*>(lds + L::kSums);
  const char* img = a.img + c * I::kKept;
  const float* gt = reinterpret_cast<const float*>(lds + L::kGate);
  const double* Gd = reinterpret_cast<const double*>(lds + L::kG);

  // do and v go through registers, one 32-column block ahead: 4 threads to a row, of both (W = 4) or of one each
  const int lr = (tid >> 2) & 63, lu = tid & 3;
  const bool second = W == 8 && wave >= 4;
  const E* orow = reinterpret_cast<const E*>(a.dout) + b * a.do_sb + (t0 + lr) * a.do_st + h * a.do_sh + 8 * lu;
  const E* vrow = reinterpret_cast<const E*>(a.v) + b * a.v_sb + (t0 + lr) * a.v_st + h * a.v_sh + 8 * lu;
  raw8<E> ro[W == 4 ? 2 : 1];
  const auto load_rows = [&](int vb) {
    if (lr < rows && 32 * vb + 8 * lu < a.V) {
      ro[0].load((second ? vrow : orow) + 32 * vb);
      if constexpr (W == 4) ro[1].load(vrow + 32 * vb);
    } else {
      ro[0] = raw8<E>();
      if constexpr (W == 4) ro[1] = raw8<E>();
    }
  };
  const auto put_rows = [&](const raw8<E>& x, int base) {
    bf16x8 l[NI];
    x.limbs(l);
#pragma unroll
    for (int q = 0; q < NI; ++q) *reinterpret_cast<bf16x8*>(lds + base + q * C * 64 + at4(lr, lu)) = l[q];
  };
  const auto row_frags = [&](int base, int t, int ln, bf16x8 (&out)[NI]) {
#pragma unroll
    for (int q = 0; q < NI; ++q) out[q] = *reinterpret_cast<const bf16x8*>(lds + base + q * C * 64 + at4(16 * t + (ln & 15), ln >> 4));
  };
  load_rows(0);
  stage<I::kRows, W>(lds + L::kK, img + I::kK, lane, wave);
  if (wave == 0) {
    reinterpret_cast<float4*>(lds + L::kGate)[lane] = reinterpret_cast<const float4*>(img + I::kGate)[lane];
    reinterpret_cast<double*>(lds + L::kG)[lane] = a.Gd[c * 64 + lane];
  }

  // Products over the value columns, 32 at a time, in this wave's 16 columns of K: W1 = dy S^T, W2 = do S^T,
  // W3 = d dS'^T, and a diagonal block of S dS'^T. Of the 64 x 64 products dy d^T and do d^T a wave takes 16 rows of
  // both (W = 4) or of one (W = 8: waves 0 to 3 the first, 4 to 7 the second); waves 0 to 3 also a diagonal block of dy v^T.
  // All but the diagonals are held transposed: a lane has one token (of F and N one row) and four consecutive
  // columns, so that gates are a value per lane, sums over K stay in registers and the outputs are stored four at a time.
  f32x4 w1[4], w2[4], w3[4], m1[4], m2[W == 4 ? 4 : 1], ss = {0, 0, 0, 0}, yv = ss;
#pragma unroll
  for (int t = 0; t < 4; ++t) w1[t] = w2[t] = w3[t] = m1[t] = m2[W == 4 ? t : 0] = f32x4{0, 0, 0, 0};
  const int mr = wave & 3, blocks = a.VP / 32;
#pragma unroll 1
  for (int vb = 0; vb < blocks; ++vb) {
    const int64_t blk = c * blocks + vb;
    __syncthreads();
    stage<L::kState, W>(lds + L::kS, a.Sw + blk * L::kState, lane, wave);
    stage<L::kState, W>(lds + L::kE, a.dSw + blk * L::kState, lane, wave);
    stage<L::kVec, W>(lds + L::kD, a.dw + blk * L::kVec, lane, wave);
    stage<L::kVec, W>(lds + L::kY, a.yw + blk * L::kVec, lane, wave);
    put_rows(ro[0], second ? L::kV : L::kO);
    if constexpr (W == 4) put_rows(ro[1], L::kV);
    staged();
    if (vb + 1 < blocks) load_rows(vb + 1);
    int ln = lane;
    asm volatile("" : "+v"(ln));  // (addresses made anew in each block: kept, they cost the registers of the products)
    const auto state_at = [&](int r, int q) { return Kept<KP, NI>::state(r, 2 * wave + (q >> 1)) + 8 * (q & 1); };
    bf16x8 s[NW], ds[NW], yr[NW], vr[NI], orr[W == 4 ? NI : 1];
    kept_frags(lds + L::kS, state_at, ln, s);
    kept_frags(lds + L::kE, state_at, ln, ds);
    ss = mm<NW>(s, ds, ss);
    if (second) {  // (do as the first limbs)
      bf16x8 x[NI];
      row_frags(L::kO, mr, ln, x);
#pragma unroll
      for (int q = 0; q < NW; ++q) yr[q] = q < NI ? x[q < NI ? q : 0] : bf16x8{};
    } else {
      kept_frags(lds + L::kY, [&](int r, int q) { return Kept<KP, NI>::vec(r, 16 * mr + 4 * q); }, ln, yr);
    }
    row_frags(L::kV, mr, ln, vr);
    yv = mm<NW>(yr, vr, yv);  // (read where W = 4 or not `second`)
    if constexpr (W == 4) row_frags(L::kO, mr, ln, orr);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const auto tokens_at = [&](int r, int q) { return Kept<KP, NI>::vec(r, 16 * t + 4 * q); };
      bf16x8 f[NW], fo[NI];
      kept_frags(lds + L::kY, tokens_at, ln, f);
      w1[t] = mm<NW>(s, f, w1[t]);
      row_frags(L::kO, t, ln, fo);
      w2[t] = mm<NW>(s, fo, w2[t]);
      kept_frags(lds + L::kD, tokens_at, ln, f);
      w3[t] = mm<NW>(ds, f, w3[t]);
      m1[t] = mm<NW>(f, yr, m1[t]);  // (above the diagonal too: fewer branches are worth more than the products)
      if constexpr (W == 4) m2[t] = mm<NW>(f, orr, m2[t]);
    }
  }
  asm volatile("" : "+v"(lane));  // (as in the blocks: the places below are not held through them)
  m = lane & 15, g = lane >> 4;
  __syncthreads();
  stage<I::kRows, W>(lds + L::kQ, img + I::kQ, lane, wave);
  // F and N, in this wave's rows, to LDS, and what of them M takes
  const auto put = [&](int plane, int row, int col, const f32x4& x) {
    uint2 l[NW];
    split4<NW>(x, l);
#pragma unroll
    for (int q = 0; q < NW; ++q) *reinterpret_cast<uint2*>(lds + plane + q * kPlane * 2 + at<8>(row, col >> 3) + (col & 7) * 2) = l[q];
  };
  {
    const int row = 16 * mr + m;
    const double Gr = Gd[row];
    const float be = gt[128 + row];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int col = 16 * t + 4 * g;
      f32x4 f, x;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float dec = expf(col + r <= row ? static_cast<float>(Gr - Gd[col + r]) : 0.0f);
        f[r] = col + r < row ? dec * m1[t][r] : 0.0f;
        x[r] = col + r <= row ? a.scale * dec * (W == 4 ? m2[W == 4 ? t : 0][r] : m1[t][r]) : 0.0f;
      }
      if (W == 4 || !second) put(L::kF, row, col, f);
      if (W == 4 || second) put(L::kN, row, col, x);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = col + r < row ? x[r] : 0.0f;
      m1[t] = W == 8 && second ? x : -be * f;
      if constexpr (W == 4) m2[t] = x;
    }
  }
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const float e = gt[16 * t + m], tail = gt[64 + 16 * t + m];
#pragma unroll
    for (int r = 0; r < 4; ++r) w1[t][r] *= e, w2[t][r] *= a.scale * e, w3[t][r] *= tail;
  }
  if (wave < 4) {  // the diagonals' lanes
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (4 * g + r == m) vec[2 * W * 64 + 16 * mr + m] = yv[r];
  }
  staged();
  const int d = 16 * wave + 4 * g;
  // k and q where this wave's accumulators are
  const auto at_acc = [&](int base, int row) {
    f32x4 x = {0, 0, 0, 0};
#pragma unroll
    for (int l = 0; l < NI; ++l) {
      const uint2 u = *reinterpret_cast<const uint2*>(lds + base + l * 1024 + I::unit(row, d >> 3) + (d & 7) * 2);
      x[0] += __uint_as_float(u.x << 16), x[1] += __uint_as_float(u.x & 0xffff0000u);
      x[2] += __uint_as_float(u.y << 16), x[3] += __uint_as_float(u.y & 0xffff0000u);
    }
    return x;
  };
  {
    // This wave's part of dg. M in its 16 rows: tiles left of the diagonal one are summed over the rows first, then
    // over the columns up to each; in the diagonal tile a row adds its columns up to each that lies before it.
    const auto rows_of = [&](int base, int t, int kb, bf16x8 (&out)[NI]) {
#pragma unroll
      for (int l = 0; l < NI; ++l) out[l] = *reinterpret_cast<const bf16x8*>(lds + base + l * 1024 + I::unit(16 * t + m, 4 * kb + g));
    };
    float c[16], before = 0.0f;  // columns 16 t + 4 g + r at 4 t + r
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 x = {0, 0, 0, 0}, y = x;
      if (t <= mr) {
#pragma unroll
        for (int kb = 0; kb < KP / 32; ++kb) {
          bf16x8 col[NI], row[NI];
          rows_of(L::kK, t, kb, col);
          rows_of(second ? L::kQ : L::kK, mr, kb, row);
          x = mm<NI>(col, row, x);
          if constexpr (W == 4) {
            rows_of(L::kQ, mr, kb, row);
            y = mm<NI>(col, row, y);
          }
        }
        x *= m1[t];
        if constexpr (W == 4) x += m2[t] * y;
        if (t == mr) {
          x[1] += x[0], x[2] += x[1], x[3] += x[2];
          float r0, r1, r2, r3, all, other;
          swap16(x[3], x[3], r0, r1);
          swap32(r0, r0, r0, r2);
          swap32(r1, r1, r1, r3);
          swap16(before, before, all, other);
          all += other;
          swap32(all, all, all, other);
          all += other + ((g > 0 ? r0 : 0.0f) + (g > 1 ? r1 : 0.0f) + (g > 2 ? r2 : 0.0f));
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = 4 * g + r < m ? all + x[r] : 0.0f;
        } else {
          before += (x[0] + x[1]) + (x[2] + x[3]);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) c[4 * t + r] = x[r];
      __builtin_amdgcn_sched_barrier(0);
    }
    // the sum over the rows m, half of the values to each half of the lanes at a time: value m is left
    const auto halve = [&](auto o, auto ctrl) {
#pragma unroll
      for (int i = 0; i < decltype(o)::value; ++i) {
        const bool hi = m & decltype(o)::value;
        const float mine = hi ? c[i + decltype(o)::value] : c[i], other = hi ? c[i] : c[i + decltype(o)::value];
        c[i] = mine + dpp<decltype(ctrl)::value>(other);
      }
    };
    halve(int_c<8>{}, int_c<0x140>{});  // lanes mirrored in 16
    halve(int_c<4>{}, int_c<0x141>{});  // mirrored in 8
    halve(int_c<2>{}, int_c<0x4e>{});   // lane ^ 2
    halve(int_c<1>{}, int_c<0xb1>{});   // lane ^ 1
    vec[wave * 64 + 16 * (m >> 2) + 4 * g + (m & 3)] = c[0];
    __builtin_amdgcn_wave_barrier();
    // what goes through the chunk's first and last state, in this wave's 16 columns of K: a lane's token is `lane`
    float in[4], out[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      asm volatile("" ::: "memory");  // (one tile's operands in registers at a time, and none kept for what follows)
      const f32x4 k = at_acc(L::kK, 16 * t + m), q = at_acc(L::kQ, 16 * t + m);
      const float be = gt[128 + 16 * t + m];
      in[t] = out[t] = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) in[t] += q[r] * w2[t][r] - be * (k[r] * w1[t][r]), out[t] += k[r] * w3[t][r];
    }
    float from = sum_groups(in), before_it = sum_groups(out);
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // (<S, dS'> is in every sum once: each lane's part is before a token or not)
      const float dot = 4 * g + r == m ? gt[63] * ss[r] : 0.0f;
      from += dot, before_it += dot;
    }
    const float col = vec[wave * 64 + lane], cols = sum_up_to(lane < 16 * mr ? col : 0.0f);
    before_it = __shfl_up(sum_up_to(before_it) + (lane < 16 * mr ? cols : col), 1, 64);
    vec[wave * 64 + lane] = sum_from(from, g) + (lane > 0 ? before_it : 0.0f);
    asm volatile("" ::: "memory");
  }
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    bf16x8 kf[NI], qf[NI], bk[NW];
    frags_t_image<I>(lds + L::kK, wave, p, lane, kf);
    frags_t_image<I>(lds + L::kQ, wave, p, lane, qf);
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
        w1[t] = mm<NW>(kf, f, w1[t]);
#pragma unroll
        for (int l = 0; l < NW; ++l) f[l] = frag_plain<8>(lds + L::kN + l * kPlane * 2, t, p, lane);
        w2[t] = mm<NW>(kf, f, w2[t]);
      }
      if (p >= t / 2) {
        frags_t<8, false>(lds + L::kN, kPlane * 2, t, p, lane, f);
        w3[t] = mm<NW>(qf, f, w3[t]);
        frags_t<8, false>(lds + L::kF, kPlane * 2, t, p, lane, f);
        w3[t] = mm<NW>(bk, f, w3[t]);
      }
    }
  }
  // outputs, and the row sums k.Z
  const int64_t tok0 = static_cast<int64_t>(b) * a.T + t0;
  float kz[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int row = 16 * t + m;
    const float be = gt[128 + row];
    const f32x4 dq = w2[t], z = w1[t], k = at_acc(L::kK, row);
    f32x4 dk;
    kz[t] = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) dk[r] = w3[t][r] - be * z[r], kz[t] += k[r] * z[r];
    if (row < rows && d < a.K) {
      if (grp == 1) {
        st4(reinterpret_cast<E*>(a.dq) + ((tok0 + row) * a.Hk + hk) * a.K + d, dq);
        st4(reinterpret_cast<E*>(a.dk) + ((tok0 + row) * a.Hk + hk) * a.K + d, dk);
      } else {
        st4(a.dqp + ((tok0 + row) * a.H + h) * a.K + d, dq);
        st4(a.dkp + ((tok0 + row) * a.H + h) * a.K + d, dk);
      }
    }
  }
  vec[(W + wave) * 64 + lane] = sum_groups(kz);
  __syncthreads();
  if (wave == 0 && lane < rows) {
    float kz = 0.0f, dg = 0.0f;
#pragma unroll
    for (int w = 0; w < W; ++w) dg += vec[w * 64 + lane], kz += vec[(W + w) * 64 + lane];
    const int64_t tok = (tok0 + lane) * a.H + h;
    st(reinterpret_cast<E*>(a.dg) + tok, dg);
    st(reinterpret_cast<E*>(a.db) + tok, vec[2 * W * 64 + lane] - kz);
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
// 4 c ... 4 c + 3 of the state, read and written once: bound by memory, B128 H16 49 us for 270 MB, 5.5 TB/s. k S and
// q S are taken together from the old state: o = scale (e^g q S + (q.k) d), d = beta (v - e^g k S). ONCE: past the caches, see launch_step.
template <bool ONCE>
__device__ __forceinline__ f4 load_state4(const float* p) {
  f4 r;
  const f32x4 v = ONCE ? __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(p)) : *reinterpret_cast<const f32x4*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) r.v[j] = v[j];
  return r;
}
template <bool ONCE>
__device__ __forceinline__ void store_state4(float* p, const f4& x) {
  const f32x4 v = {x.v[0], x.v[1], x.v[2], x.v[3]};
  if constexpr (ONCE)
    __builtin_nontemporal_store(v, reinterpret_cast<f32x4*>(p));
  else
    *reinterpret_cast<f32x4*>(p) = v;
}
template <typename E, int KR, bool ONCE>
__global__ __launch_bounds__(256) void step_kernel(const E* __restrict__ q, const E* __restrict__ k, const E* __restrict__ v,
                                                   const E* __restrict__ gg, const E* __restrict__ beta, float* __restrict__ state,
                                                   E* __restrict__ o, int H, int Hk, int K, int V, float scale) {
  __shared__ float red[4][8][8];
  __shared__ float dots[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = tid >> 3, cc = tid & 7;
  const int tiles = (V + 31) / 32;  // (neighbours in memory at the same time)
  const int64_t bh = blockIdx.x / tiles;
  const int h = static_cast<int>(bh % H), hk = h / (H / Hk);
  const int64_t bk = bh / H * Hk + hk;
  const int col = static_cast<int>(blockIdx.x % tiles) * 32 + 4 * cc;
  const bool in = col < V;
  float* s = state + bh * K * V + col;
  f4 x[KR];
  float kr[KR], qr[KR];
#pragma unroll
  for (int i = 0; i < KR; ++i) {
    const int d = r + 32 * i;
    x[i] = in && d < K ? load_state4<ONCE>(s + static_cast<int64_t>(d) * V) : io4<float>::fill(0.0f);
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
        store_state4<ONCE>(s + static_cast<int64_t>(row) * V, x[i]);
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

template <int KP, int NI>
inline size_t image_bytes(bool keep) { return keep ? Tile<KP, NI>::kKept : Tile<KP, NI>::kOnce; }
inline Layout layout(int dtype, const mg_delta_dims& s, bool keep_) {
  const size_t n = static_cast<size_t>(chunks(s)), bh = static_cast<size_t>(s.B) * s.H, c = bh * n;
  const size_t vp = vpad(s.V), nw = dtype == MG_F32 ? 3 : 2;
  const size_t image = dtype == MG_F32 ? (s.K <= 64 ? image_bytes<64, 3>(keep_) : image_bytes<128, 3>(keep_))
                                       : (s.K <= 64 ? image_bytes<64, 1>(keep_) : image_bytes<128, 1>(keep_));
  Layout l;
  l.img = 0;
  l.G = c * image;
  l.S = l.G + c * 512;
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
  return MG_OK;
}

// A launch has less than 2^32 threads: a workgroup of up to 512 for every chunk, of 512 for every 16 value columns
// of a head (a pass over the chunks), or of 256 for every 32 (a step).
inline int check_launches(const char* fn, const mg_delta_dims* s, bool step) {
  const int64_t bh = static_cast<int64_t>(s->B) * s->H, tiles = (s->V + 31) / 32;
  const auto below = [&](int bits, int64_t each) { return bh <= ((int64_t(1) << bits) - 1) / each; };
  if (step) return below(24, tiles) ? MG_OK : fail(MG_ERR_ARG, "%s: B * H * ceil(V / 32) must be below 2^24", fn);
  if (!below(23, chunks(*s)) || !below(22, tiles))
    return fail(MG_ERR_ARG, "%s: B * H * ceil(T / 64) must be below 2^23, B * H * ceil(V / 32) below 2^22", fn);
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

// o and dv are dense: their rows' offsets in a chunk are held in 31 bits, as the operands' are
inline int check_out(const char* fn, int dtype, const mg_delta_dims* s) {
  if (static_cast<int64_t>(s->H) * s->V * (dtype == MG_F32 ? 4 : 2) * C >= (int64_t(1) << 31))
    return fail(MG_ERR_ARG, "%s: 64 tokens' o must be below 2 GiB", fn);
  return MG_OK;
}

// Value columns per workgroup of the passes over the chunks, in tiles of 16: one as long as every tile has a CU of its
// own, for more of them, else two, so that a chunk's operands are loaded for twice the columns. T 2048, K = V = 128,
// forward (the backward alike), one against two: 256 tiles 107 and 125 us, 264 133 and 125, 320 159 and 140, 512 245
// and 201, 2048 878 and 716; T 16384, 264 tiles, 1192 and 1098; K = V = 64, 256 tiles 109 and 122, 264 136 and 131.
// fp32 loads three limbs for one and is kept at one.
inline int columns_for(int64_t bh, int vp, int dtype_limbs) {
  return dtype_limbs == 1 && bh * (vp / 16) > kCUs ? 2 : 1;
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
  a.Sw = ws + l.S, a.dw = ws + l.d;
}

template <int KP, int NI>
int launch_fwd(const Args& a, bool keep_, hipStream_t st_) {
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  hipLaunchKernelGGL((chunk_kernel<KP, NI>), dim3(bh * a.NC), dim3(256), 0, st_, a, keep_);
  const int ct = columns_for(bh, a.VP, NI);
  const dim3 grid(bh * (a.VP / 16 / ct));
  if constexpr (NI == 1) {
    if (ct == 2) {
      if (keep_)
        hipLaunchKernelGGL((state_kernel<KP, NI, true, 2>), grid, dim3(512), 0, st_, a);
      else
        hipLaunchKernelGGL((state_kernel<KP, NI, false, 2>), grid, dim3(512), 0, st_, a);
      return check_launch("mg_delta_fwd");
    }
  }
  if (keep_)
    hipLaunchKernelGGL((state_kernel<KP, NI, true, 1>), grid, dim3(512), 0, st_, a);
  else
    hipLaunchKernelGGL((state_kernel<KP, NI, false, 1>), grid, dim3(512), 0, st_, a);
  return check_launch("mg_delta_fwd");
}

template <int KP, int NI>
int launch_bwd(const Args& a, hipStream_t st_) {
  using E = typename elem<NI>::type;
  const int64_t bh = static_cast<int64_t>(a.B) * a.H;
  const int ct = columns_for(bh, a.VP, NI);
  const dim3 grid(bh * (a.VP / 16 / ct));
  if constexpr (NI == 1) {
    if (ct == 2) hipLaunchKernelGGL((dstate_kernel<KP, NI, 2>), grid, dim3(512), 0, st_, a);
  }
  if (ct == 1) hipLaunchKernelGGL((dstate_kernel<KP, NI, 1>), grid, dim3(512), 0, st_, a);
  hipLaunchKernelGGL((grad_kernel<KP, NI>), dim3(bh * a.NC), dim3(64 * GradTile<KP, NI>::W), 0, st_, a);
  if (a.H > a.Hk) {
    const int64_t n = static_cast<int64_t>(a.B) * a.T * a.Hk * a.K;
    hipLaunchKernelGGL((sum_heads_kernel<E>), dim3((n / 4 + 255) / 256), dim3(256), 0, st_, a.dqp, a.dkp,
                       reinterpret_cast<E*>(a.dq), reinterpret_cast<E*>(a.dk), n, a.K, a.H / a.Hk);
  }
  return check_launch("mg_delta_bwd");
}

template <typename E, bool ONCE>
void launch_step(const mg_delta_dims& s, const E* q, const E* k, const E* v, const E* g, const E* beta, float scale, float* state, E* o,
                 hipStream_t st_) {
  const dim3 grid(static_cast<int64_t>(s.B) * s.H * ((s.V + 31) / 32));
#define GO(KR) hipLaunchKernelGGL((step_kernel<E, KR, ONCE>), grid, dim3(256), 0, st_, q, k, v, g, beta, state, o, s.H, s.Hk, s.K, s.V, scale)
  if (s.K <= 32)
    GO(1);
  else if (s.K <= 64)
    GO(2);
  else
    GO(4);
#undef GO
}

// A call's states from 64 MiB on are taken to be out of the 256 MiB cache by the next token: a model steps
// several layers' in between. Then it is no use to send them through it. Through the caches and past them, one layer
// over and over, and 16 in turn: 32 MiB 10.1 and 12.7 us, 15.3 and 12.5; 64 MiB 22.6 and 22.5, 30.6 and 25.1; 128 MiB
// 43 and 48, 54 and 50; 256 MiB 87 and 96, 107 and 97.
template <typename E>
int launch_step(const mg_delta_dims& s, const void* q, const void* k, const void* v, const void* g, const void* beta, float scale,
                float* state, void* o, hipStream_t st_) {
  const auto go = [&](auto once) {
    launch_step<E, decltype(once)::value != 0>(s, static_cast<const E*>(q), static_cast<const E*>(k), static_cast<const E*>(v),
                                               static_cast<const E*>(g), static_cast<const E*>(beta), scale, state, static_cast<E*>(o), st_);
  };
  if (static_cast<int64_t>(s.B) * s.H * s.K * s.V * 4 >= int64_t(64) << 20)
    go(int_c<1>{});
  else
    go(int_c<0>{});
  return check_launch("mg_delta_step");
}

}  // namespace delta
}  // namespace mg

using namespace mg;

extern "C" size_t mg_delta_fwd_workspace_bytes(int dtype, const mg_delta_dims* dims, int keep) {
  const char* fn = "mg_delta_fwd_workspace_bytes";
  if (delta::check_dims(fn, dtype, dims) || delta::check_launches(fn, dims, false)) return 0;
  return delta::layout(dtype, *dims, keep != 0).end;
}

extern "C" size_t mg_delta_bwd_workspace_bytes(int dtype, const mg_delta_dims* dims) {
  const char* fn = "mg_delta_bwd_workspace_bytes";
  if (delta::check_dims(fn, dtype, dims) || delta::check_launches(fn, dims, false)) return 0;
  return delta::bwd_layout(dtype, *dims).end;
}

extern "C" int mg_delta_fwd(int dtype, const mg_delta_dims* dims, const mg_rows* q, const mg_rows* k, const mg_rows* v,
                            const mg_rows* g, const mg_rows* beta, float scale, const float* h0, void* o, float* state,
                            int keep, void* workspace, size_t workspace_bytes, void* stream) {
  const char* fn = "mg_delta_fwd";
  int rc;
  if ((rc = delta::check_dims(fn, dtype, dims)) || (rc = delta::check_launches(fn, dims, false)) ||
      (rc = delta::check_out(fn, dtype, dims)))
    return rc;
  if ((rc = delta::check_rows(fn, "q", dtype, q, true)) || (rc = delta::check_rows(fn, "k", dtype, k, true)) ||
      (rc = delta::check_rows(fn, "v", dtype, v, false)) || (rc = delta::check_rows(fn, "g", dtype, g, false)) ||
      (rc = delta::check_rows(fn, "beta", dtype, beta, false)))
    return rc;
  if (!o || !aligned(o, 16)) return fail(MG_ERR_ARG, "%s: o must be 16-byte aligned", fn);
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
  if ((rc = delta::check_dims(fn, dtype, dims)) || (rc = delta::check_launches(fn, dims, false)) ||
      (rc = delta::check_out(fn, dtype, dims)))
    return rc;
  if ((rc = delta::check_rows(fn, "q", dtype, q, true)) || (rc = delta::check_rows(fn, "k", dtype, k, true)) ||
      (rc = delta::check_rows(fn, "v", dtype, v, false)) || (rc = delta::check_rows(fn, "g", dtype, g, false)) ||
      (rc = delta::check_rows(fn, "beta", dtype, beta, false)) || (rc = delta::check_rows(fn, "dout", dtype, dout, true)))
    return rc;
  for (const void* p : {dq, dk, dv, dg, dbeta})
    if (!p || !aligned(p, dtype == MG_F32 ? 4 : 2)) return fail(MG_ERR_ARG, "%s: a gradient is NULL or misaligned", fn);
  if (!aligned(dq, 16) || !aligned(dk, 16))
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
  a.dSw = ws + w.dS, a.yw = ws + w.y;
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
  if ((rc = delta::check_dims(fn, dtype, dims)) || (rc = delta::check_launches(fn, dims, true))) return rc;
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
