// Routing of tokens to experts: scores, a bias for balance, groups, the best top_k, renormalised weights.
//
//   score = softmax(logits) or sigmoid(logits)        key = score + bias, or the logits themselves without a bias
//   group key = the sum of its two best keys with a bias, its best key without; the topk_groups best groups stay
//   ids = the top_k experts of those groups by key    weight = score [/ the chosen ones' sum] * scale
//
// Ties go to the lowest index.  Without a bias the order of the scores is the order of the logits, which are compared as they are.
// With one, the order is that of the 64-bit keys: two experts' scores differ by less than an ulp of 32 bits often enough to matter
// among thousands of tokens times hundreds of experts.  The choice is made on 32-bit keys all the same, and made again on 64-bit
// ones where two keys next to each other in it, or the last group or expert chosen and the first that is not, are nearer than the
// 32-bit keys' error: about one token in a hundred.  NaN counts as -inf; equal infinities share a softmax's mass evenly.
//
// One wavefront per token, expert e in lane e % 64.  Keys are mapped to unsigned integers of the same order, so that the
// best of a wavefront is an integer maximum.  Bound by instructions, not by memory: 4096 tokens, eight of 256 experts in four of eight groups,
// sigmoid and bias, 8.7 us a call, where the 4.5 MB take 1 us; 11.6 us with loads waited for one by one, the lanes' best looked for again
// behind every choice and groups ranked on exact keys, 14.7 with the whole choice on 64-bit keys.  One token 7 us, the call's own time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_fp8.h"
#include "common.h"

namespace {

constexpr int kMaxExperts = 1024, kMaxGroups = 64, kMaxTopK = 64;
constexpr int kWaves = 4;  // tokens of a workgroup
constexpr int64_t kLaunchTokens = 1 << 25;  // a launch holds fewer than 2^32 threads

struct Params {
  const void* logits;
  const float* bias;
  int32_t* ids;
  float* weights;
  int tokens, experts, top_k, groups, kept, group_size;
  int group_lanes;  // lanes that look through a group together: the largest power of two that lets all groups be looked through at once
  bool sigmoid, renormalize;
  float scale;
};

// Unsigned integers in the order of the values, and back.  No value maps to 0: a key that is taken, left out, or not there.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v);  // -0 and 0 are equal
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t ordered(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v == 0.0 ? 0.0 : v);
  return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t max_with(uint32_t v) {
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, true));  // one instruction: 0 where no lane is read
}
// The largest of a wavefront's values (wave-uniform): along rows of 16 lanes, then from row to row; lane 63 has seen all.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  v = max_with<0x111, 0xf>(v);
  v = max_with<0x112, 0xf>(v);
  v = max_with<0x114, 0xf>(v);
  v = max_with<0x118, 0xf>(v);
  v = max_with<0x142, 0xa>(v);
  v = max_with<0x143, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
// The sum of a wavefront's values (wave-uniform), over the same lanes.
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_from(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double add_from(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, true);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float of_lane(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ double of_lane(double v, int lane) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
  v = add_from<0x111, 0xf>(v);
  v = add_from<0x112, 0xf>(v);
  v = add_from<0x114, 0xf>(v);
  v = add_from<0x118, 0xf>(v);
  v = add_from<0x142, 0xa>(v);
  v = add_from<0x143, 0xc>(v);
  return of_lane(v, 63);
}

// The lane with the best key of a wavefront, ties to the lowest expert (ANY: to any); `top` is that key.
template <bool ANY>
__device__ __forceinline__ int best_lane(uint32_t key, int expert, uint32_t* top) {
  *top = wave_max(key);
  uint64_t equal = __ballot(key == *top);
  if (!ANY && __builtin_expect((equal & (equal - 1)) != 0, 0)) {
    const uint32_t lowest = wave_max(key == *top ? ~(uint32_t)expert : 0u);  // all lanes take part
    equal = __ballot(~(uint32_t)expert == lowest);
  }
  return __builtin_ctzll(equal);
}
template <bool ANY>
__device__ __forceinline__ int best_lane(uint64_t key, int expert, uint64_t* top) {
  const uint32_t hi = wave_max((uint32_t)(key >> 32));
  const bool first = (uint32_t)(key >> 32) == hi;
  const uint32_t lo = wave_max(first ? (uint32_t)key : 0u);
  const bool equal = first && (uint32_t)key == lo;
  *top = (uint64_t)hi << 32 | lo;
  uint64_t lanes = __ballot(equal);
  if (__builtin_expect((lanes & (lanes - 1)) != 0, 0)) {
    const uint32_t lowest = wave_max(equal ? ~(uint32_t)expert : 0u);
    lanes = __ballot(~(uint32_t)expert == lowest);
  }
  return __builtin_ctzll(lanes);
}

// How far apart two 32-bit keys have to be for their order to be the 64-bit keys'.  A sigmoid's exponential is off by (|v| + 2) 2^-24 of itself,
// which moves the score by at most 2^-23, as do sum and quotient: 2^-21 together with room.  A softmax's sum of up to 16 + 6 steps is off by
// 2^-19 of itself.  The sum with the bias adds 2^-24 of its size.  Both keys are off.  A group's key is the sum of two, off by as much as both:
// size is that of the keys' roundings, |best| + |second|, whatever is left of them in the sum; this is then how far the one group's key may be off.
__device__ __forceinline__ float margin(float size, bool sigmoid) { return (sigmoid ? 0x1p-20f : 0x1p-17f) + 0x1p-21f * fabsf(size); }

template <typename V>
struct KeyOf {
  typedef uint32_t type;
};
template <>
struct KeyOf<double> {
  typedef uint64_t type;
};

__device__ __forceinline__ float exp_of(float v) { return expf(v); }
__device__ __forceinline__ double exp_of(double v) { return exp(v); }
__device__ __forceinline__ float over(float a, float b) { return a * __builtin_amdgcn_rcpf(b); }  // b in [1, 1024] or so
__device__ __forceinline__ double over(double a, double b) { return a / b; }

// The keys' exponential: off by (|v| + 2) 2^-24 of itself in 32 bits, where exp_of is off by an ulp.
__device__ __forceinline__ float key_exp(float v) { return __expf(v); }
__device__ __forceinline__ double key_exp(double v) { return exp(v); }

template <typename V>
__device__ __forceinline__ V sigmoid_key(V v) {
  const V e = key_exp(v >= V(0) ? -v : v);
  return over(v >= V(0) ? V(1) : e, V(1) + e);
}
template <typename V>
__device__ __forceinline__ V sigmoid_of(V v) {
  const V e = exp_of(v >= V(0) ? -v : v);
  return over(v >= V(0) ? V(1) : e, V(1) + e);
}

// The choice on keys of type V: lane i < top_k gets the i-th expert.  False: made on 32-bit keys that are too near to each other.
// top: the largest logit (softmax).  values: a row of LDS for the wavefront.
template <typename V, int J, bool BIAS>
__device__ __forceinline__ bool choose(const Params& p, const float (&logit)[J], const float (&bias)[J], float top, int lane, V* values, int* mine) {
  typedef typename KeyOf<V>::type Key;
  constexpr bool kNear = BIAS && sizeof(V) == 4;
  V value[J];
  if constexpr (BIAS) {
    if (p.sigmoid) {
#pragma unroll
      for (int j = 0; j < J; ++j) value[j] = sigmoid_key((V)logit[j]);
    } else {
      V sum = 0;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        value[j] = lane + 64 * j >= p.experts ? V(0) : logit[j] == top ? V(1) : key_exp((V)logit[j] - (V)top);
        sum += value[j];
      }
      sum = wave_sum(sum);
#pragma unroll
      for (int j = 0; j < J; ++j) value[j] = over(value[j], sum);
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
      value[j] += (V)bias[j];
      if (!(value[j] == value[j])) value[j] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < J; ++j) value[j] = (V)logit[j];
  }
  Key key[J];
#pragma unroll
  for (int j = 0; j < J; ++j) key[j] = lane + 64 * j < p.experts ? ordered(value[j]) : Key(0);
  bool near = false;
  if (p.groups > 1) {
#pragma unroll
    for (int j = 0; j < J; ++j) values[lane + 64 * j] = value[j];
    __builtin_amdgcn_wave_barrier();
    // group_lanes lanes look through group g together; its key ends up in all of them
    const int g = lane / p.group_lanes, part = lane % p.group_lanes;
    V best = -INFINITY, second = -INFINITY;
    if (g < p.groups)
      for (int i = part; i < p.group_size; i += p.group_lanes) {
        const V v = values[g * p.group_size + i];
        second = fmax(second, fmin(best, v));
        best = fmax(best, v);
      }
    for (int off = 1; off < p.group_lanes; off <<= 1) {
      const V ob = __shfl_xor(best, off), os = __shfl_xor(second, off);
      second = fmax(fmax(second, os), fmin(best, ob));
      best = fmax(best, ob);
    }
    V worth = BIAS && p.group_size > 1 ? best + second : best;
    if (!(worth == worth)) worth = -INFINITY;
    bool stays;
    if constexpr (kNear) {
      // how many of the others are surely better, and how many may be; one between the two can change sides
      const float size = fminf(p.group_size > 1 ? fabsf(best) + fabsf(second) : fabsf(best), 3e38f), off = margin(size, p.sigmoid);
      const float here = fminf(fmaxf(worth, -3e38f), 3e38f), least = here - off, most = here + off;
      int surely = 0, maybe = -1;  // (itself)
      for (int o = 0; o < p.groups; ++o) {
        surely += of_lane(least, o * p.group_lanes) > most;
        maybe += of_lane(most, o * p.group_lanes) >= least;
      }
      stays = g < p.groups && maybe < p.kept;
      if (__ballot(g < p.groups && !stays && surely < p.kept)) near = true;
    } else {
      const Key own = g < p.groups ? ordered(worth) : Key(0);
      int ahead = 0;
      for (int o = 0; o < p.groups; ++o) {
        const Key k = ordered(of_lane(worth, o * p.group_lanes));
        ahead += k > own || (k == own && o < g);
      }
      stays = g < p.groups && ahead < p.kept;
    }
    const uint64_t stay = __ballot(stays);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int e = lane + 64 * j;
      if (e < p.experts) {
        // e / group_size: (e + 1/2) / size lies at least 1 / (2 size) from a whole number, far more than this product's error
        const int group = (int)(((float)e + 0.5f) * (1.f / (float)p.group_size));
        if (!((stay >> (group * p.group_lanes)) & 1)) key[j] = Key(0);
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
  // Up to four keys a lane are put in descending order first, the lower expert first among equal ones; of more the best is looked for
  // again behind every choice (sorting sixteen takes longer than that).
  constexpr bool kSorted = J <= 4;
  int at[J];
#pragma unroll
  for (int j = 0; j < J; ++j) at[j] = lane + 64 * j;
  if constexpr (kSorted) {
#pragma unroll
    for (int end = J - 1; end > 0; --end)
#pragma unroll
      for (int j = 0; j < end; ++j) {
        const bool swap = key[j + 1] > key[j];
        const Key high = swap ? key[j + 1] : key[j], low = swap ? key[j] : key[j + 1];
        const int high_at = swap ? at[j + 1] : at[j], low_at = swap ? at[j] : at[j + 1];
        key[j] = high, key[j + 1] = low, at[j] = high_at, at[j + 1] = low_at;
      }
  }
  Key best = 0;  // this lane's
  int best_at = 0;
  auto look = [&] {
    best = key[0];
    best_at = at[0];
    if constexpr (!kSorted) {
#pragma unroll
      for (int j = 1; j < J; ++j)
        if (key[j] > best) {
          best = key[j];
          best_at = at[j];
        }
    }
  };
  look();
  Key taken = 0;  // lane i: key of the i-th expert
  for (int i = 0; i < p.top_k; ++i) {
    Key first;
    const int winner = best_lane<kNear>(best, best_at, &first);
    const int e = __builtin_amdgcn_readlane(best_at, winner);
    if (lane == i) {
      *mine = e;
      taken = first;
    }
    if (lane == winner) {
      if constexpr (kSorted) {
#pragma unroll
        for (int j = 0; j + 1 < J; ++j) {
          key[j] = key[j + 1];
          at[j] = at[j + 1];
        }
        key[J - 1] = 0;
      } else {
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (at[j] == best_at) key[j] = 0;
      }
      look();
    }
  }
  if constexpr (kNear) {
    const uint32_t left_out = wave_max(best);  // 0: nothing is
    const uint32_t next = (uint32_t)__shfl_down((int)taken, 1);
    const float a = value_of(taken), b = value_of(lane + 1 < p.top_k ? next : left_out);
    if (__ballot(lane < p.top_k && (lane + 1 < p.top_k || left_out) && !(a - b > margin(a, p.sigmoid)))) near = true;
  }
  return !near;
}

template <typename T, int J, bool BIAS>
__global__ __launch_bounds__(kWaves * 64) void route_kernel(Params p) {
  __shared__ double rows[kWaves][BIAS ? J * 64 : J * 32];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int token = blockIdx.x * kWaves + wave;
  if (token >= p.tokens) return;
  const T* row = reinterpret_cast<const T*>(p.logits) + (int64_t)token * p.experts;
  float logit[J], bias[J];
  float top = -INFINITY;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int e = min(lane + 64 * j, p.experts - 1);  // (all are asked for at once)
    logit[j] = (float)row[e];
    bias[j] = BIAS ? p.bias[e] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < J; ++j)
    if (lane + 64 * j >= p.experts || !(logit[j] == logit[j])) logit[j] = -INFINITY;
#pragma unroll
  for (int j = 0; j < J; ++j) top = fmaxf(top, logit[j]);
  top = value_of(wave_max(ordered(top)));
  int mine = 0;
  if (!choose<float, J, BIAS>(p, logit, bias, top, lane, reinterpret_cast<float*>(rows[wave]), &mine)) {
    if constexpr (BIAS) choose<double, J, BIAS>(p, logit, bias, top, lane, rows[wave], &mine);
  }
  // The chosen ones' scores, in 64 bits where a score is below what 32 bits hold well (a renormalised weight may be large all the same).
  const float chosen = (float)row[mine], l = chosen == chosen ? chosen : -INFINITY;
  const bool small = __ballot(lane < p.top_k && (p.sigmoid ? l < -60.f : l < top && !(l - top > -60.f))) != 0;
  float sum = 1.f;
  if (!p.sigmoid) {
    sum = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) sum += lane + 64 * j >= p.experts ? 0.f : logit[j] == top ? 1.f : expf(logit[j] - top);
    sum = wave_sum(sum);
  }
  float weight;
  auto weigh = [&](auto zero) {
    typedef decltype(zero) V;
    V s = p.sigmoid ? sigmoid_of((V)l) : over(l == top ? V(1) : exp_of((V)l - (V)top), (V)sum);
    if (p.renormalize) {
      const V total = wave_sum(lane < p.top_k ? s : V(0));
      s = total > V(0) ? s / total : V(0);  // (not over(): a total may be tiny)
    }
    weight = (float)(s * (V)p.scale);
  };
  if (small) weigh(0.0);
  else weigh(0.f);
  if (lane < p.top_k) {
    const int64_t at = (int64_t)token * p.top_k + lane;
    p.ids[at] = mine;
    p.weights[at] = weight;
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
  {
    using block8::overlap;
    const int64_t chosen = tokens * top_k * 4, all = tokens * experts * dtype_bytes(logits_dtype);
    PTO_CHECK_ARG(!overlap(expert_ids, chosen, expert_weights, chosen) && !overlap(expert_ids, chosen, logits, all) &&
                      !overlap(expert_weights, chosen, logits, all) && !overlap(expert_ids, chosen, bias, experts * 4) &&
                      !overlap(expert_weights, chosen, bias, experts * 4),
                  "route_experts: the results overlap an operand or each other");
  }
  int group_lanes = 64;
  while (group_lanes * n_groups > 64) group_lanes /= 2;
  Params p{logits, bias, expert_ids, expert_weights, (int)tokens, (int)experts, (int)top_k, (int)n_groups, (int)topk_groups,
           (int)(experts / n_groups), group_lanes, score_fn == PTO_HIP_SCORE_SIGMOID, renormalize != 0, scale};
  hipStream_t st = (hipStream_t)stream;
  for (int64_t t = 0; t < tokens; t += kLaunchTokens) {
    p.logits = reinterpret_cast<const char*>(logits) + t * experts * dtype_bytes(logits_dtype);
    p.ids = expert_ids + t * top_k;
    p.weights = expert_weights + t * top_k;
    p.tokens = (int)std::min(kLaunchTokens, tokens - t);
    if (logits_dtype == PTO_HIP_FP32) bias ? launch<float, true>(p, st) : launch<float, false>(p, st);
    else if (logits_dtype == PTO_HIP_BF16) bias ? launch<__bf16, true>(p, st) : launch<__bf16, false>(p, st);
    else bias ? launch<_Float16, true>(p, st) : launch<_Float16, false>(p, st);
  }
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
