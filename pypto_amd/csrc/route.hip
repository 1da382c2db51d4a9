// Routing of tokens to experts: scores, a bias for balance, groups, the best top_k, renormalised weights.
//
//   score = softmax(logits) or sigmoid(logits)        key = score + bias, or the logits themselves without a bias
//   group key = the sum of its two best keys with a bias, its best key without; the topk_groups best groups stay
//   ids = the top_k experts of those groups by key    weight = score [/ the chosen ones' sum] * scale
//
// Ties go to the lowest index.  Keys with a bias are compared in 64 bits: two experts' scores differ by less than an ulp of 32 bits
// often enough to matter among thousands of tokens times hundreds of experts.  Without one the order of the scores is the order of
// the logits, which are compared as they are.  NaN counts as -inf; equal infinities share a softmax's mass evenly.
//
// One wavefront per token, expert e in lane e % 64.  Keys are mapped to unsigned integers of the same order, so that the
// best of a wavefront is a maximum of their upper halves by six lane exchanges, and of the lower halves only among equals.
#include <hip/hip_runtime.h>

#include "common.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopK = 64;
constexpr int kWaves = 4;  // tokens of a workgroup

struct Params {
  const void* logits;
  const float* bias;
  int32_t* ids;
  float* weights;
  int tokens, experts, top_k, groups, kept, group_size;
  bool sigmoid, renormalize;
  float scale;
};

// Unsigned integers in the order of the values.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);  // -0 and 0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v == 0.0 ? 0.0 : v);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// ... and what no value maps to, below all of them: taken, left out, or not there
constexpr uint64_t kNone = 0;

__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off));
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor(v, off));
  return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}

template <typename T, int J, bool BIAS>
__global__ __launch_bounds__(kWaves * 64) void route_kernel(Params p) {
  __shared__ double keys[kWaves][J * 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * kWaves + wave;
  const bool live = token < p.tokens;  // every wavefront reaches the barriers
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)(live ? token : 0) * p.experts;
  float logit[J];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    const float v = e < p.experts ? (float)row[e] : -INFINITY;
    logit[j] = v == v ? v : -INFINITY;
    top = fmaxf(top, logit[j]);
  }
  double score[J];
  if (p.sigmoid) {
#pragma unroll
    for (int j = 0; j < J; ++j) score[j] = 1.0 / (1.0 + exp(-(double)logit[j]));
  } else {
    top = wave_max(top);
    double sum = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      score[j] = lane + 64 * j >= p.experts ? 0.0 : logit[j] == top ? 1.0 : exp((double)logit[j] - (double)top);
      sum += score[j];
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int j = 0; j < J; ++j) score[j] /= sum;
  }
  uint64_t key[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = lane + 64 * j;
    double k = (double)logit[j];
    if (BIAS && e < p.experts) k = score[j] + (double)p.bias[e];
    if (!(k == k)) k = -INFINITY;
    if (p.groups > 1) keys[wave][e] = k;
    key[j] = e < p.experts ? ordered(k) : kNone;
  }
  if (p.groups > 1) {
    __syncthreads();
    // lane g: the key of group g
    double best = -INFINITY, second = -INFINITY;
    const int g = lane < p.groups ? lane : 0;
    for (int i = 0; i < p.group_size; ++i) {
      const double k = keys[wave][g * p.group_size + i];
      second = fmax(second, fmin(best, k));
      best = fmax(best, k);
    }
    const double worth = BIAS && p.group_size > 1 ? best + second : best;
    const uint64_t mine = lane < p.groups ? ordered(worth == worth ? worth : -INFINITY) : kNone;
    int ahead = 0;
    for (int o = 0; o < p.groups; ++o) {
      const uint64_t other = (uint64_t)__shfl((long long)mine, o);
      ahead += other > mine || (other == mine && o < lane);
    }
    const uint64_t stay = __ballot(lane < p.groups && ahead < p.kept);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e = lane + 64 * j;
      if (e < p.experts && !((stay >> (e / p.group_size)) & 1)) key[j] = kNone;
    }
  }
  int my_id = 0;
  double my_score = 0.0, total = 0.0;
  for (int i = 0; i < p.top_k; ++i) {
    uint64_t best = key[0];
    int at = 0;
#pragma unroll
    for (int j = 1; j < J; ++j)
      if (key[j] > best) {
        best = key[j];
        at = j;
      }
    const uint32_t hi = (uint32_t)(best >> 32), top_hi = wave_max(hi);
    const uint32_t lo = hi == top_hi ? (uint32_t)best : 0u, top_lo = wave_max(lo);
    const bool candidate = hi == top_hi && lo == top_lo;
    const int e = (int)~wave_max(candidate ? ~(uint32_t)(lane + 64 * at) : 0u);  // the lowest index among equals
    double s = 0.0;
#pragma unroll
    for (int j = 0; j < J; ++j)
      if (lane + 64 * j == e) {
        s = score[j];
        key[j] = kNone;
      }
    s = __shfl(s, e & 63);
    total += s;
    if (lane == i) {
      my_id = e;
      my_score = s;
    }
  }
  if (live && lane < p.top_k) {
    const int64_t at = (int64_t)token * p.top_k + lane;
    p.ids[at] = my_id;
    const double w = p.renormalize ? (total > 0.0 ? my_score / total : 0.0) : my_score;
    p.weights[at] = (float)(w * (double)p.scale);
  }
}

template <typename T, bool BIAS>
void launch(const Params& p, hipStream_t st) {
  auto go = [&](auto kern) { hipLaunchKernelGGL(kern, dim3((unsigned)((p.tokens + kWaves - 1) / kWaves)), dim3(kWaves * 64), 0, st, p); };
  if (p.experts <= 64) go(route_kernel<T, 1, BIAS>);
  else if (p.experts <= 128) go(route_kernel<T, 2, BIAS>);
  else if (p.experts <= 256) go(route_kernel<T, 4, BIAS>);
  else if (p.experts <= 512) go(route_kernel<T, 8, BIAS>);
  else go(route_kernel<T, 16, BIAS>);
}

}  // namespace

extern "C" int pto_hip_route_experts(const void* logits, const float* bias, int32_t* expert_ids, float* expert_weights, int64_t tokens,
                                     int64_t experts, int64_t top_k, int64_t n_groups, int64_t topk_groups, int score_fn, int renormalize,
                                     float scale, int logits_dtype, void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  PTO_CHECK_ARG(tokens >= 0 && tokens < (1ll << 30) && experts > 0 && top_k > 0, "route_experts: bad shape T=%lld E=%lld top_k=%lld",
                (long long)tokens, (long long)experts, (long long)top_k);
  PTO_CHECK_ARG(logits_dtype == PTO_HIP_FP32 || logits_dtype == PTO_HIP_BF16 || logits_dtype == PTO_HIP_FP16,
                "route_experts: logits dtype %s not in {FP32, BF16, FP16}", dtype_name(logits_dtype));
  PTO_CHECK_ARG(score_fn == PTO_HIP_SCORE_SOFTMAX || score_fn == PTO_HIP_SCORE_SIGMOID, "route_experts: score function %d is neither softmax (0) nor sigmoid (1)",
                score_fn);
  PTO_CHECK_ARG(renormalize == 0 || renormalize == 1, "route_experts: renormalize must be 0 or 1, got %d", renormalize);
  PTO_CHECK_ARG(n_groups >= 1 && experts % n_groups == 0, "route_experts: %lld experts do not divide into %lld groups", (long long)experts,
                (long long)n_groups);
  PTO_CHECK_ARG(topk_groups >= 1 && topk_groups <= n_groups, "route_experts: topk_groups %lld outside [1, n_groups %lld]",
                (long long)topk_groups, (long long)n_groups);
  PTO_CHECK_ARG(top_k <= topk_groups * (experts / n_groups), "route_experts: top_k %lld of the %lld experts in %lld groups", (long long)top_k,
                (long long)(topk_groups * (experts / n_groups)), (long long)topk_groups);
  if (experts > kMaxExperts || top_k > kMaxTopK || n_groups > kMaxGroups)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "route_experts: at most %d experts, %d groups and top_k %d, got %lld, %lld and %lld", kMaxExperts,
                kMaxGroups, kMaxTopK, (long long)experts, (long long)n_groups, (long long)top_k);
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  if (tokens == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(logits && expert_ids && expert_weights, "route_experts: null tensor pointer");
  PTO_CHECK_ARG(((uintptr_t)bias | (uintptr_t)expert_ids | (uintptr_t)expert_weights) % 4 == 0 &&
                    (uintptr_t)logits % (size_t)dtype_bytes(logits_dtype) == 0,
                "route_experts: misaligned operand");
  const Params p{logits, bias, expert_ids, expert_weights, (int)tokens, (int)experts, (int)top_k, (int)n_groups, (int)topk_groups,
                 (int)(experts / n_groups), score_fn == PTO_HIP_SCORE_SIGMOID, renormalize != 0, scale};
  hipStream_t st = (hipStream_t)stream;
  if (logits_dtype == PTO_HIP_FP32) bias ? launch<float, true>(p, st) : launch<float, false>(p, st);
  else if (logits_dtype == PTO_HIP_BF16) bias ? launch<__bf16, true>(p, st) : launch<__bf16, false>(p, st);
  else bias ? launch<_Float16, true>(p, st) : launch<_Float16, false>(p, st);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
