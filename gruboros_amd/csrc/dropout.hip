// Dropout with a counter-based generator, for gfx950: y = residual + keep(x) x / (1 - p), and its
// backward dx = keep(x) dy / (1 - p). Which elements are kept follows from (seed, offset, index)
// alone (mg_random.h), so no mask is stored and the backward is the forward's kernel without a residual.
//
// One pass, eight consecutive elements and two Philox calls per thread and step. Bound by memory: 16376 x 1024 bf16 added
// to an fp32 residual 26 us (6.5 TB/s), its backward 17 us (5.8 TB/s).

#include <algorithm>

#include "mg_random.h"

namespace mg {
namespace dropout {

constexpr int kThreads = 256;

template <typename Tin, typename Tout>
__global__ __launch_bounds__(kThreads) void dropout_kernel(const Tin* __restrict__ x, const Tout* __restrict__ residual,
                                                           Tout* __restrict__ y, int64_t n, Drop d) {
  const bool drop = d.threshold;  // (none are dropped else: nothing is drawn)
  const uint64_t key = drop ? d.key() : 0;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; 8 * i < n; i += step) {
    uint32_t w[2][4] = {};
    if (drop) {
      philox(2 * i, d.offset, key, w[0]);
      philox(2 * i + 1, d.offset, key, w[1]);
    }
    if (8 * i + 8 <= n) {
      fv<8> v = iov<Tin, 8>::load(x + 8 * i);
      fv<8> r = residual ? iov<Tout, 8>::load(residual + 8 * i) : iov<Tout, 8>::fill(0.0f);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float k = w[j / 4][j % 4] >= d.threshold ? v.v[j] * d.scale : 0.0f;
        r.v[j] = residual ? r.v[j] + k : k;
      }
      iov<Tout, 8>::store(y + 8 * i, r);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (8 * i + j < n) {
          float k, r = 0.0f;
          if constexpr (sizeof(Tin) == 2) k = bf16_to_f32(x[8 * i + j]); else k = x[8 * i + j];
          k = w[j / 4][j % 4] >= d.threshold ? k * d.scale : 0.0f;
          if (residual) {
            if constexpr (sizeof(Tout) == 2) r = bf16_to_f32(residual[8 * i + j]); else r = residual[8 * i + j];
            k = r + k;
          }
          if constexpr (sizeof(Tout) == 2) y[8 * i + j] = f32_to_bf16(k); else y[8 * i + j] = k;
        }
      }
    }
  }
}

template <typename Tin, typename Tout>
int launch(const void* x, const void* residual, void* y, int64_t n, const Drop& d, hipStream_t st) {
  const int64_t wgs = (n + 8 * kThreads - 1) / (8 * kThreads);
  hipLaunchKernelGGL((dropout_kernel<Tin, Tout>), dim3(std::min<int64_t>(wgs, 4096)), dim3(kThreads), 0, st,
                     static_cast<const Tin*>(x), static_cast<const Tout*>(residual), static_cast<Tout*>(y), n, d);
  return check_launch("mg_dropout");
}

}  // namespace dropout
}  // namespace mg

using namespace mg;

extern "C" int mg_dropout(int x_dtype, const void* x, int y_dtype, const void* residual, void* y, int64_t n, double p,
                          uint64_t seed, const int64_t* seed_p, uint64_t offset, void* stream) {
  const char* fn = "mg_dropout";
  for (int dt : {x_dtype, y_dtype})
    if (dt != MG_F32 && dt != MG_BF16) return fail(MG_ERR_DTYPE, "%s: dtype %d unsupported", fn, dt);
  if (n < 1) return fail(MG_ERR_ARG, "%s: n=%lld must be at least 1", fn, (long long)n);
  if (!(p >= 0.0 && p < 1.0)) return fail(MG_ERR_ARG, "%s: p=%g must be in [0, 1)", fn, p);
  if (!x || !y || !aligned(x, 16) || !aligned(y, 16) || !aligned(residual, 16))
    return fail(MG_ERR_ARG, "%s: x, y and residual must be 16-byte aligned (x, y not NULL)", fn);
  if (!aligned(seed_p, 8)) return fail(MG_ERR_ARG, "%s: seed_p misaligned", fn);
  const Drop d = {seed, offset, seed_p, static_cast<uint32_t>(p * 4294967296.0), static_cast<float>(1.0 / (1.0 - p))};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (x_dtype == MG_BF16)
    return y_dtype == MG_BF16 ? dropout::launch<bf16_t, bf16_t>(x, residual, y, n, d, st)
                              : dropout::launch<bf16_t, float>(x, residual, y, n, d, st);
  return y_dtype == MG_BF16 ? dropout::launch<float, bf16_t>(x, residual, y, n, d, st)
                            : dropout::launch<float, float>(x, residual, y, n, d, st);
}
