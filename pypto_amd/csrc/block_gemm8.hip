// projection_fp8_block: out = (a8 * a_scale) @ (w8 * w_scale)^T with a scale per 128 k of a row and per 128 x 128 weights.
#include <hip/hip_runtime.h>

#include "block_gemm8.h"
#include "common.h"

namespace pto_hip {
namespace block8 {

template <typename OutT>
int launch_projection(const Params& p, hipStream_t st) {
  constexpr int CT = 2;
  const int tiles_n = (p.n + 16 * CT - 1) / (16 * CT);
  auto go = [&](auto kern, int height, int waves) {
    const int64_t tiles = (int64_t)tiles_n * ((p.m + height - 1) / height);
    hipLaunchKernelGGL(kern, dim3((unsigned)tiles), dim3(waves * 64), 0, st, p, tiles_n);
  };
  if (p.m <= 16) go(narrow_kernel<kPlain, CT, 1, 4, 3, OutT>, 16, 4);
  else go(narrow_kernel<kPlain, CT, 2, 4, 3, OutT>, 32, 4);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

}  // namespace block8
}  // namespace pto_hip

extern "C" int pto_hip_projection_fp8_block(const void* a8, const float* a_scale, const void* w8, const float* w_scale, void* out,
                                            int64_t m, int64_t k, int64_t n, int out_dtype, void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  PTO_CHECK_ARG(m >= 0 && k > 0 && n > 0 && m < (1 << 24) && n < (1 << 24), "projection_fp8_block: bad shape M=%lld K=%lld N=%lld",
                (long long)m, (long long)k, (long long)n);
  PTO_CHECK_ARG(out_dtype == PTO_HIP_FP32 || out_dtype == PTO_HIP_BF16 || out_dtype == PTO_HIP_FP16,
                "projection_fp8_block: output dtype %s not in {FP32, BF16, FP16}", dtype_name(out_dtype));
  if (k % block8::kBlock != 0 || k > block8::kMaxK)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "projection_fp8_block: k %lld must be a multiple of %d and at most %d", (long long)k, block8::kBlock,
                block8::kMaxK);
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  if (m == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(a8 && a_scale && w8 && w_scale && out, "projection_fp8_block: null tensor pointer");
  PTO_CHECK_ARG(((uintptr_t)a8 | (uintptr_t)w8) % 16 == 0 && ((uintptr_t)a_scale | (uintptr_t)w_scale) % 4 == 0 &&
                    (uintptr_t)out % (size_t)dtype_bytes(out_dtype) == 0,
                "projection_fp8_block: codes must be 16-byte aligned, scales and out to their elements");
  block8::Params p{};
  p.a = reinterpret_cast<const uint8_t*>(a8);
  p.sa = a_scale;
  p.b0 = reinterpret_cast<const uint8_t*>(w8);
  p.sb0 = w_scale;
  p.c = out;
  p.m = (int)m;
  p.n = (int)n;
  p.k = (int)k;
  p.kb = (int)(k / block8::kBlock);
  hipStream_t st = (hipStream_t)stream;
  switch (out_dtype) {
    case PTO_HIP_FP32: return block8::launch_projection<float>(p, st);
    case PTO_HIP_BF16: return block8::launch_projection<__bf16>(p, st);
    default: return block8::launch_projection<_Float16>(p, st);
  }
}
