// projection_fp8_block: out = (a8 * a_scale) @ (w8 * w_scale)^T with a scale per 128 k of a row and per 128 x 128 weights.
#include <hip/hip_runtime.h>

#include "block_gemm8.h"
#include "block_tiled8.h"
#include "common.h"
#include "launch_choice.h"

namespace pto_hip {
namespace block8 {

// out = the sum of the k ranges' slabs, in their order
template <typename OutT>
__global__ __launch_bounds__(256) void sum_ranges_kernel(const float* __restrict__ slabs, int ranges, int64_t count, OutT* __restrict__ out) {
  const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= count) return;
  const int here = (int)(count - at < 4 ? count - at : 4);
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int r = 0; r < ranges; ++r) {
    const float* src = slabs + r * count + at;
    if (here == 4) {
      f32x4 v;
      __builtin_memcpy(&v, src, sizeof(v));
      sum += v;
    } else {
      for (int e = 0; e < here; ++e) sum[e] += src[e];
    }
  }
  store_upto4(out + at, sum, here);
}

// `launch` with p, or with ranges of k into slabs that are summed behind it.  launch(p, type of the results)
template <typename OutT, typename F>
int launch_ranges(Params p, int per_split, hipStream_t st, F launch) {
  if (per_split <= 0 || per_split >= p.kb) return launch(p, OutT{});
  const int ranges = (p.kb + per_split - 1) / per_split;
  const int64_t count = (int64_t)p.m * p.n;
  void* slabs = nullptr;
  int rc = gemm_slabs((size_t)ranges * count * sizeof(float), st, &slabs);
  if (rc) return rc;
  if (!slabs) return launch(p, OutT{});
  OutT* const out = reinterpret_cast<OutT*>(p.c);
  p.c = slabs;
  p.per_split = per_split;
  rc = launch(p, float{});
  if (rc) return rc;
  hipLaunchKernelGGL(sum_ranges_kernel<OutT>, dim3((unsigned)((count + 1023) / 1024)), dim3(256), 0, st, reinterpret_cast<const float*>(slabs),
                     ranges, count, out);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

template <typename OutT>
int launch_projection(const Params& p, hipStream_t st) {
  constexpr bool kExact = std::is_same<OutT, float>::value;
  const BlockTile t = choose_block_tile(p.m, p.n, p.kb, kExact, ctx().num_cu, (int)ctx().block_gemm_rows, (int)ctx().block_gemm_cols,
                                        (int)ctx().gemm_splits);
  if (t.rows == 16) {
    const int tiles_n = (p.n + t.cols - 1) / t.cols;
    const int64_t wgs = (int64_t)tiles_n * ((p.m + 15) / 16);
    if (wgs >= (1 << 23)) return fail(PTO_HIP_ERR_UNSUPPORTED, "a product of %lld tiles is more than one launch holds", (long long)wgs);
    const dim3 grid((unsigned)wgs);
    if (t.cols == 16) hipLaunchKernelGGL((narrow_kernel<1, 8, 4, OutT>), grid, dim3(512), 0, st, p, tiles_n);
    else if (t.tiles[0] == 8) hipLaunchKernelGGL((narrow_kernel<2, 8, 3, OutT>), grid, dim3(512), 0, st, p, tiles_n);
    else hipLaunchKernelGGL((narrow_kernel<2, 4, 3, OutT>), grid, dim3(256), 0, st, p, tiles_n);
    PTO_CHECK_HIP(hipGetLastError());
    return PTO_HIP_OK;
  }
  return launch_ranges<OutT>(p, t.per_split, st, [&](const Params& q, auto type) {
    typedef decltype(type) C;
    if (t.cols == 64) return launch_tiled<64, kExact, C>(q, st);
    if (t.cols == 128) return launch_tiled<128, kExact, C>(q, st);
    if (t.rows == 64) return launch_tiled_rows<64, kExact, C>(q, t.tiles, st);
    if constexpr (!kExact) {
      if (t.rows == 256) return launch_tiled_rows<256, kExact, C>(q, t.tiles, st);
    }
    return launch_tiled_rows<128, kExact, C>(q, t.tiles, st);
  });
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
  const int64_t kb = k / block8::kBlock, out_bytes = m * n * dtype_bytes(out_dtype);
  PTO_CHECK_ARG(!block8::overlap(out, out_bytes, a8, m * k) && !block8::overlap(out, out_bytes, a_scale, m * kb * 4) &&
                    !block8::overlap(out, out_bytes, w8, n * k) &&
                    !block8::overlap(out, out_bytes, w_scale, (n + block8::kBlock - 1) / block8::kBlock * kb * 4),
                "projection_fp8_block: out overlaps an operand");
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
