// The experts' FFN of a mixture layer on e4m3 operands with a scale for each block of 128:
//
//   out[t] = sum_j weights[t, j] * FFN_e(x[t]),  e = ids[t, j],   FFN_e(x) = (SiLU(x Wg_e) * (x Wu_e)) Wd_e
//
// The slots (t, j) are put in order of their experts, so that the rows of a tile of either product share one expert's
// matrices; the tiles of all experts are one launch.  h = SiLU(g) * u is quantised per 128 channels in the
// first product's epilogue, from 32 bits; the second product's rows stay in 32 bits until the sum over a token's experts.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_gemm8.h"
#include "common.h"

namespace pto_hip {
namespace block8 {

constexpr int kMaxExperts = 1024;
constexpr int kPlanThreads = 1024;

// The plan: slots by expert, and tiles of `height` rows of one expert each.  One workgroup; a slot with a negative expert is in no
// tile, one with an expert that there is not is reported.  Places inside an expert are taken in the order of atomics: which row of
// which tile a slot becomes changes no bit of its result.
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(const int32_t* __restrict__ ids, int slots, int experts, int height,
                                                            int32_t* __restrict__ order, int4* __restrict__ tiles, int* __restrict__ n_tiles,
                                                            int* __restrict__ flag) {
  __shared__ int count[kMaxExperts], first[kMaxExperts], waves[2][kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int e = tid; e < experts; e += kPlanThreads) count[e] = 0;
  __syncthreads();
  for (int s = tid; s < slots; s += kPlanThreads) {
    const int e = ids[s];
    if (e >= experts) *flag = 1;
    else if (e >= 0) atomicAdd(&count[e], 1);
  }
  __syncthreads();
  // thread e: exclusive sums over the experts in front, of rows and of tiles
  const int rows = tid < experts ? count[tid] : 0, mine = (rows + height - 1) / height;
  int sum[2] = {rows, mine};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(sum[q], off);
      if (lane >= off) sum[q] += o;
    }
    if (lane == 63) waves[q][wave] = sum[q];
  }
  __syncthreads();
  int before[2] = {sum[0] - rows, sum[1] - mine};
  for (int w = 0; w < wave; ++w) {
    before[0] += waves[0][w];
    before[1] += waves[1][w];
  }
  if (tid < experts) {
    first[tid] = before[0];
    for (int i = 0; i < mine; ++i) tiles[before[1] + i] = int4{tid, before[0] + i * height, min(height, rows - i * height), 0};
  }
  if (tid == kPlanThreads - 1) *n_tiles = before[1] + mine;
  __syncthreads();
  for (int s = tid; s < slots; s += kPlanThreads) {
    const int e = ids[s];
    if (e >= 0 && e < experts) order[atomicAdd(&first[e], 1)] = s;
  }
}

// out[t] = sum over j of weights[t, j] * y[t * top_k + j], the slots without an expert left out.
template <typename OutT>
__global__ __launch_bounds__(256) void combine_kernel(const float* __restrict__ y, const int32_t* __restrict__ ids,
                                                      const float* __restrict__ weights, OutT* __restrict__ out, int hidden, int experts,
                                                      int top_k) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * 4;
  if (col >= hidden) return;
  const int64_t token = blockIdx.y;
  f32x4 sum = {0.f, 0.f, 0.f, 0.f};
  for (int j = 0; j < top_k; ++j) {
    const int64_t slot = token * top_k + j;
    const int e = ids[slot];
    if (e < 0 || e >= experts) continue;
    const float w = weights[slot];
    const f32x4 v = *reinterpret_cast<const f32x4*>(y + slot * hidden + col);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = fmaf(w, v[i], sum[i]);
  }
  store_upto4(out + token * hidden + col, sum, 4);
}

struct Experts {
  const uint8_t* x;
  const float* x_scale;
  const int32_t* ids;
  const float* weights;
  const uint8_t *gate, *up, *down;
  const float *gate_scale, *up_scale, *down_scale;
  void* out;
  int hidden, inter, experts, top_k;
};

// Scratch of a pass over `tokens` tokens.
struct Scratch {
  size_t order, tiles, n_tiles, h, h_scale, y, bytes;
  int max_tiles;
  Scratch(int64_t tokens, const Experts& x, int height) {
    const int64_t slots = tokens * x.top_k;
    max_tiles = (int)(std::min<int64_t>(slots, x.experts) + slots / height);
    size_t at = 0;
    auto take = [&](size_t b) {
      const size_t here = at;
      at += (b + 255) / 256 * 256;
      return here;
    };
    order = take((size_t)slots * 4);
    tiles = take((size_t)max_tiles * sizeof(int4));
    n_tiles = take(sizeof(int));
    h = take((size_t)slots * x.inter);
    h_scale = take((size_t)slots * (x.inter / kBlock) * 4);
    y = take((size_t)slots * x.hidden * 4);
    bytes = at;
  }
};

template <typename OutT>
int run_pass(const Experts& x, int64_t tokens, const Scratch& s, int height, char* ws, hipStream_t st) {
  const int slots = (int)(tokens * x.top_k);
  int32_t* order = reinterpret_cast<int32_t*>(ws + s.order);
  int4* tiles = reinterpret_cast<int4*>(ws + s.tiles);
  int* n_tiles = reinterpret_cast<int*>(ws + s.n_tiles);
  float* y = reinterpret_cast<float*>(ws + s.y);
  hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, x.ids, slots, x.experts, height, order, tiles, n_tiles, ctx().flags + 3);
  Params p{};
  p.tiles = tiles;
  p.n_tiles = n_tiles;
  p.order = order;
  p.top_k = x.top_k;
  p.a = x.x;
  p.sa = x.x_scale;
  p.b0 = x.gate;
  p.sb0 = x.gate_scale;
  p.b1 = x.up;
  p.sb1 = x.up_scale;
  p.c = ws + s.h;
  p.c_scale = reinterpret_cast<float*>(ws + s.h_scale);
  p.n = x.inter;
  p.k = x.hidden;
  p.kb = x.hidden / kBlock;
  const int groups = x.inter / kBlock;
  if (height == 16) hipLaunchKernelGGL((narrow_gate_up_kernel<1, 1, 4>), dim3((unsigned)(s.max_tiles * groups)), dim3(512), 0, st, p, groups);
  else hipLaunchKernelGGL((narrow_gate_up_kernel<2, 1, 3>), dim3((unsigned)(s.max_tiles * groups)), dim3(512), 0, st, p, groups);
  Params d = p;
  d.a = reinterpret_cast<const uint8_t*>(ws + s.h);
  d.sa = reinterpret_cast<const float*>(ws + s.h_scale);
  d.b0 = x.down;
  d.sb0 = x.down_scale;
  d.c = y;
  d.n = x.hidden;
  d.k = x.inter;
  d.kb = x.inter / kBlock;
  const int tiles_n = x.hidden / 32;
  if (height == 16) hipLaunchKernelGGL((narrow_kernel<kDown, 2, 1, 4, 3, float>), dim3((unsigned)(s.max_tiles * tiles_n)), dim3(256), 0, st, d, tiles_n);
  else hipLaunchKernelGGL((narrow_kernel<kDown, 2, 2, 4, 3, float>), dim3((unsigned)(s.max_tiles * tiles_n)), dim3(256), 0, st, d, tiles_n);
  hipLaunchKernelGGL(combine_kernel<OutT>, dim3((unsigned)((x.hidden + 1023) / 1024), (unsigned)tokens), dim3(256), 0, st, y, x.ids, x.weights,
                     reinterpret_cast<OutT*>(x.out), x.hidden, x.experts, x.top_k);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

// Tokens are worked through in passes, so that the scratch stays below a gigabyte or two and every index inside 32 bits.
constexpr int64_t kPassSlots = 32768;

template <typename OutT>
int run_experts(Experts x, int64_t tokens, hipStream_t st) {
  const int64_t pass = std::min(tokens, std::max<int64_t>(1, kPassSlots / x.top_k));
  const int height = pass * x.top_k <= 24 * (int64_t)x.experts ? 16 : 32;
  const Scratch s(pass, x, height);
  void* ws = nullptr;
  const int rc = workspace(s.bytes, &ws);
  if (rc) return rc;
  for (int64_t t = 0; t < tokens; t += pass) {
    Experts part = x;
    part.x += t * x.hidden;
    part.x_scale += t * (x.hidden / kBlock);
    part.ids += t * x.top_k;
    part.weights += t * x.top_k;
    part.out = reinterpret_cast<OutT*>(x.out) + t * x.hidden;
    const int rc2 = run_pass<OutT>(part, std::min(pass, tokens - t), s, height, reinterpret_cast<char*>(ws), st);
    if (rc2) return rc2;
  }
  return PTO_HIP_OK;
}

}  // namespace block8
}  // namespace pto_hip

extern "C" int pto_hip_experts_ffn_fp8_block(const void* x8, const float* x_scale, const int32_t* expert_ids, const float* expert_weights,
                                             const void* w_gate8, const float* w_gate_scale, const void* w_up8, const float* w_up_scale,
                                             const void* w_down8, const float* w_down_scale, void* out, int64_t tokens, int64_t hidden,
                                             int64_t intermediate, int64_t experts, int64_t top_k, int out_dtype, void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  PTO_CHECK_ARG(tokens >= 0 && tokens < (1ll << 30) && hidden > 0 && intermediate > 0 && experts > 0 && top_k > 0,
                "experts_ffn_fp8_block: bad shape T=%lld H=%lld I=%lld E=%lld top_k=%lld", (long long)tokens, (long long)hidden,
                (long long)intermediate, (long long)experts, (long long)top_k);
  PTO_CHECK_ARG(out_dtype == PTO_HIP_FP32 || out_dtype == PTO_HIP_BF16 || out_dtype == PTO_HIP_FP16,
                "experts_ffn_fp8_block: output dtype %s not in {FP32, BF16, FP16}", dtype_name(out_dtype));
  if (hidden % block8::kBlock != 0 || intermediate % block8::kBlock != 0 || hidden > block8::kMaxK || intermediate > block8::kMaxK)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "experts_ffn_fp8_block: hidden %lld and intermediate %lld must be multiples of %d and at most %d",
                (long long)hidden, (long long)intermediate, block8::kBlock, block8::kMaxK);
  if (experts > block8::kMaxExperts || top_k > 64)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "experts_ffn_fp8_block: at most %d experts and top_k 64, got %lld and %lld", block8::kMaxExperts,
                (long long)experts, (long long)top_k);
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  if (tokens == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(x8 && x_scale && expert_ids && expert_weights && w_gate8 && w_gate_scale && w_up8 && w_up_scale && w_down8 &&
                    w_down_scale && out,
                "experts_ffn_fp8_block: null tensor pointer");
  PTO_CHECK_ARG(((uintptr_t)x8 | (uintptr_t)w_gate8 | (uintptr_t)w_up8 | (uintptr_t)w_down8 | (uintptr_t)out) % 16 == 0 &&
                    ((uintptr_t)x_scale | (uintptr_t)expert_ids | (uintptr_t)expert_weights | (uintptr_t)w_gate_scale |
                     (uintptr_t)w_up_scale | (uintptr_t)w_down_scale) % 4 == 0,
                "experts_ffn_fp8_block: codes and out must be 16-byte aligned, scales, ids and weights to their elements");
  const block8::Experts x{reinterpret_cast<const uint8_t*>(x8), x_scale, expert_ids, expert_weights, reinterpret_cast<const uint8_t*>(w_gate8),
                          reinterpret_cast<const uint8_t*>(w_up8), reinterpret_cast<const uint8_t*>(w_down8), w_gate_scale, w_up_scale,
                          w_down_scale, out, (int)hidden, (int)intermediate, (int)experts, (int)top_k};
  hipStream_t st = (hipStream_t)stream;
  switch (out_dtype) {
    case PTO_HIP_FP32: return block8::run_experts<float>(x, tokens, st);
    case PTO_HIP_BF16: return block8::run_experts<__bf16>(x, tokens, st);
    default: return block8::run_experts<_Float16>(x, tokens, st);
  }
}
