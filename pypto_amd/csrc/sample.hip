// The next token of every row of logits, from a random number of the row's own.
//
//   w_i = exp((l_i - max l) / T)      the order: larger logits first, of equal ones the lower index
//   kept: the first top_k; of those the fewest from the front whose sum reaches top_p of all of theirs; of those the w_i >= min_p
//   token: the first index at which the running sum of the kept w, in the order of indices, passes u times their sum
//
// The kept tokens are what lies in front of a border (key, number of tokens of that key), and a filter only moves the border forward; min_p asks each
// weight by itself.  Weights are integers, w in units of 2^-44: their sums are exact in any order, so that a row's token does not depend on how
// the work is split, and next to a border or the random number the decision is that of the definition in 64 bits up to 2^-45 a token.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_fp8.h"
#include "common.h"
#include "token_seq.h"

namespace {

constexpr int kMaxVocab = 1 << 19;  // sums of 2^19 weights of 2^44 stay below 2^64
constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
constexpr int kTiles = kMaxVocab / kThreads;
constexpr int kUnit = 44;  // a weight of 1 is 2^44
constexpr uint64_t kOne = 1ull << kUnit;

struct Params {
  const void* logits;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* uniform;
  int32_t* tokens;
  float* probs;
  int rows, vocab;
};

// Unsigned integers in the order of the values; NaN is -inf.
__device__ __forceinline__ uint32_t ordered(float v) {
  const uint32_t b = __builtin_bit_cast(uint32_t, v == 0.f ? 0.f : v != v ? -INFINITY : v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kNone = 0x007fffffu;  // the key of -inf

// 2^-y for y >= 0, to 2^-50 or better of it: the fraction's power is its series in ln 2 times it.
__device__ __forceinline__ double power_of_two(double y) {
  const double n = rint(y);
  const double f = (n - y) * 0.69314718055994530942;  // [-0.35, 0.35]
  double s = 1.0 / 6227020800.0;
  s = fma(s, f, 1.0 / 479001600.0);
  s = fma(s, f, 1.0 / 39916800.0);
  s = fma(s, f, 1.0 / 3628800.0);
  s = fma(s, f, 1.0 / 362880.0);
  s = fma(s, f, 1.0 / 40320.0);
  s = fma(s, f, 1.0 / 5040.0);
  s = fma(s, f, 1.0 / 720.0);
  s = fma(s, f, 1.0 / 120.0);
  s = fma(s, f, 1.0 / 24.0);
  s = fma(s, f, 1.0 / 6.0);
  s = fma(s, f, 0.5);
  s = fma(s, f, 1.0);
  s = fma(s, f, 1.0);
  return ldexp(s, -(int)n);
}
struct Weights {
  float best;   // the largest logit
  double rate;  // log2(e) / T
  __device__ __forceinline__ double exponent(float v) const { return ((double)best - (double)v) * rate; }
  // in units of 2^-44, rounded to the nearest
  __device__ __forceinline__ uint64_t operator()(float v) const {
    if (v == best) return kOne;
    const double y = exponent(v);
    if (!(y < kUnit + 1.0)) return 0;
    const double big = 4503599627370496.0;  // 2^52: what is added to it is rounded to a whole number
    return __builtin_bit_cast(uint64_t, power_of_two(y) * (double)kOne + big) - __builtin_bit_cast(uint64_t, big);
  }
  __device__ __forceinline__ double exact(float v) const { return v == best ? 1.0 : power_of_two(fmin(exponent(v), 1000.0)); }
};

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off);
    v = o > v ? o : v;
  }
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_sum(V v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
  return v;
}
// Sums over a workgroup's threads in front of this one; all threads take part.
template <typename V>
__device__ __forceinline__ V sum_in_front(V v, V* waves, V* total) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  V s = v;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const V o = __shfl_up(s, off);
    if (lane >= off) s += o;
  }
  __syncthreads();  // `waves` may still be read
  if (lane == 63) waves[wave] = s;
  __syncthreads();
  V before = 0, all = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) before += waves[w];
    all += waves[w];
  }
  *total = all;
  return before + s - v;
}

// What a row keeps: keys above `key`, and of that key the first `ties` by index.
struct Border {
  uint32_t key;
  uint32_t ties;
};

struct Shared {
  unsigned int count[kBins];
  unsigned long long weight[kBins];
  unsigned long long tile_weight[kTiles];
  unsigned int tile_ties[kTiles];
  unsigned long long waves[kWaves];
  unsigned long long found[4];
};

template <typename T>
__device__ __forceinline__ float logit(const T* row, int i) { return (float)row[i]; }

// The border behind which the running sum, of tokens (by_weight: of weights) in the order, reaches `need`, from `in_front` on; it lies between the keys
// lo and hi, or nowhere (false).  Eleven bits of the key a pass over the row.
template <typename T>
__device__ bool find_border(Shared& sh, const T* row, int vocab, const Weights& w, bool by_weight, uint64_t need, uint32_t lo, uint32_t hi, Border* border,
                            uint64_t* weight_to_border) {
  uint64_t tokens_front = 0, weight_front = 0;
  while (true) {
    int shift = 0;
    while ((((uint64_t)hi - lo) >> shift) >= kBins) ++shift;
    for (int b = threadIdx.x; b < kBins; b += kThreads) {
      sh.count[b] = 0;
      sh.weight[b] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const float v = logit(row, i);
      const uint32_t key = ordered(v);
      if (key < lo || key > hi) continue;
      const int bin = (hi - key) >> shift;
      atomicAdd(&sh.count[bin], 1u);
      const uint64_t x = w(value_of(key));
      if (x) atomicAdd(&sh.weight[bin], (unsigned long long)x);
    }
    __syncthreads();
    // two bins a thread
    const int b0 = 2 * threadIdx.x;
    const uint64_t n0 = sh.count[b0], n1 = sh.count[b0 + 1], w0 = sh.weight[b0], w1 = sh.weight[b0 + 1];
    unsigned long long all;
    const uint64_t n_front = tokens_front + sum_in_front<unsigned long long>(n0 + n1, sh.waves, &all);
    const uint64_t w_front = weight_front + sum_in_front<unsigned long long>(w0 + w1, sh.waves, &all);
    if (threadIdx.x == 0) sh.found[0] = kBins;
    __syncthreads();
    const uint64_t front = by_weight ? w_front : n_front, own0 = by_weight ? w0 : n0, own1 = by_weight ? w1 : n1;
    if (front < need && front + own0 + own1 >= need) {
      const bool second = front + own0 < need;
      sh.found[0] = b0 + second;
      sh.found[1] = n_front + (second ? n0 : 0);
      sh.found[2] = w_front + (second ? w0 : 0);
    }
    __syncthreads();
    const int bin = (int)sh.found[0];
    if (bin == kBins) return false;
    tokens_front = sh.found[1];
    weight_front = sh.found[2];
    const uint32_t top = hi - ((uint32_t)bin << shift);
    __syncthreads();
    if (shift == 0) {
      const uint64_t each = w(value_of(top));
      const uint64_t ties = by_weight ? (need - weight_front + each - 1) / each : need - tokens_front;
      *border = Border{top, (uint32_t)ties};
      *weight_to_border = weight_front + ties * each;
      return true;
    }
    const uint32_t least = top - ((1u << shift) - 1);
    lo = least > top || least < lo ? lo : least;
    hi = top;
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(Params p) {
  __shared__ Shared sh;
  const int r = blockIdx.x, lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int vocab = p.vocab;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * vocab;
  // the best token: the largest key, of equal ones the lowest index
  uint64_t best = 0;
  for (int i = threadIdx.x; i < vocab; i += kThreads) {
    const uint64_t k = (uint64_t)ordered(logit(row, i)) << 32 | (uint32_t)~i;
    best = k > best ? k : best;
  }
  best = wave_max(best);
  if (lane == 0) sh.waves[wave] = best;
  __syncthreads();
  for (int i = 0; i < kWaves; ++i) best = sh.waves[i] > best ? sh.waves[i] : best;
  __syncthreads();
  const uint32_t top = (uint32_t)(best >> 32);
  const float t = p.temperature[r];
  if (top <= kNone || !(t > 0.f)) {  // nothing to choose from, or no choice
    if (threadIdx.x == 0) {
      p.tokens[r] = top <= kNone ? -1 : (int32_t)~(uint32_t)best;
      if (p.probs) p.probs[r] = top <= kNone ? 0.f : 1.f;
    }
    return;
  }
  const Weights w{value_of(top), 1.4426950408889634074 / (double)t};
  Border border{kNone, 0};
  uint64_t total = 0;
  bool bounded = false;
  const int k = p.top_k ? p.top_k[r] : 0;
  if (k > 0 && k < vocab) bounded = find_border(sh, row, vocab, w, false, (uint64_t)k, kNone + 1, top, &border, &total);
  const float top_p = p.top_p ? p.top_p[r] : 1.f;
  if (top_p < 1.f) {
    if (!bounded) {
      for (int i = threadIdx.x; i < vocab; i += kThreads) total += w(value_of(ordered(logit(row, i))));
      unsigned long long all;
      sum_in_front<unsigned long long>(total, sh.waves, &all);
      total = all;
    }
    const uint64_t need = max((uint64_t)ceil(fmax((double)top_p, 0.0) * (double)total), (uint64_t)1);
    Border nearer;
    uint64_t unused;
    if (find_border(sh, row, vocab, w, true, need, bounded ? border.key : kNone + 1, top, &nearer, &unused)) border = nearer;
  }
  const float min_p = p.min_p ? p.min_p[r] : 0.f;
  const uint64_t least = min_p > 0.f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * (double)kOne) : 1;  // weights of nothing are never chosen

  // kept weights and ties of each 1024 tokens, in the order of indices
  const int tiles = (vocab + kThreads - 1) / kThreads;
  for (int i = threadIdx.x; i < tiles; i += kThreads) {
    sh.tile_weight[i] = 0;
    sh.tile_ties[i] = 0;
  }
  __syncthreads();
  const uint64_t tie = w(value_of(border.key)), tie_weight = border.key > kNone && tie >= least ? tie : 0;
  for (int i = 0; i < tiles; ++i) {
    const int at = i * kThreads + threadIdx.x;
    const uint32_t key = at < vocab ? ordered(logit(row, at)) : 0;
    uint64_t x = key > border.key ? w(value_of(key)) : 0;
    x = wave_sum((unsigned long long)(x >= least ? x : 0));
    const int ties = __popcll(__ballot(key == border.key));
    if (lane == 0 && x) atomicAdd(&sh.tile_weight[i], (unsigned long long)x);
    if (lane == 0 && ties) atomicAdd(&sh.tile_ties[i], (unsigned)ties);
  }
  __syncthreads();
  // the sum, and the tile in which the running sum passes its share
  uint64_t ties_front = 0, front = 0;
  if (threadIdx.x == 0) {
    uint64_t ties = 0, sum = 0;
    for (int i = 0; i < tiles; ++i) {
      sum += sh.tile_weight[i] + (min((uint64_t)border.ties, ties + sh.tile_ties[i]) - min((uint64_t)border.ties, ties)) * tie_weight;
      ties += sh.tile_ties[i];
    }
    const double u = fmin(fmax((double)p.uniform[r], 0x1p-25), 1.0 - 0x1p-24);
    const uint64_t target = (uint64_t)(u * (double)sum);
    ties = 0;
    int at = 0;
    for (; at < tiles - 1; ++at) {
      const uint64_t more = sh.tile_weight[at] + (min((uint64_t)border.ties, ties + sh.tile_ties[at]) - min((uint64_t)border.ties, ties)) * tie_weight;
      if (front + more > target) break;
      front += more;
      ties += sh.tile_ties[at];
    }
    sh.found[0] = at;
    sh.found[1] = target;
    sh.found[2] = front;
    sh.found[3] = ties;
    sh.weight[0] = sum;
  }
  __syncthreads();
  const int tile = (int)sh.found[0];
  const uint64_t target = sh.found[1], sum = sh.weight[0];
  front = sh.found[2];
  ties_front = sh.found[3];
  const int at = tile * kThreads + threadIdx.x;
  const uint32_t key = at < vocab ? ordered(logit(row, at)) : 0;
  unsigned long long all;
  const uint64_t tie_number = ties_front + sum_in_front<unsigned long long>(key == border.key, sh.waves, &all);
  uint64_t x = key > border.key ? w(value_of(key)) : 0;
  x = x >= least ? x : 0;
  if (key == border.key && tie_number < border.ties) x = tie_weight;
  front += sum_in_front<unsigned long long>(x, sh.waves, &all);
  if (front <= target && front + x > target) {
    p.tokens[r] = at;
    if (p.probs) p.probs[r] = (float)(w.exact(value_of(key)) / ((double)sum * (1.0 / (double)kOne)));
  }
}

template <typename T>
void launch(const Params& p, hipStream_t st) {
  hipLaunchKernelGGL((sample_kernel<T>), dim3(p.rows), dim3(kThreads), 0, st, p);
}

}  // namespace

extern "C" int pto_hip_sample_tokens(const void* logits, const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                                     const float* uniform, int32_t* tokens, float* probs, int64_t rows, int64_t vocab, int logits_dtype,
                                     void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  PTO_CHECK_ARG(rows >= 0 && rows < (1ll << 22) && vocab > 0, "sample_tokens: bad shape R=%lld V=%lld", (long long)rows, (long long)vocab);
  PTO_CHECK_ARG(logits_dtype == PTO_HIP_FP32 || logits_dtype == PTO_HIP_BF16 || logits_dtype == PTO_HIP_FP16,
                "sample_tokens: logits dtype %s not in {FP32, BF16, FP16}", dtype_name(logits_dtype));
  if (vocab > kMaxVocab)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "sample_tokens: at most %d logits a row, got %lld", kMaxVocab, (long long)vocab);
  if (rows == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(logits && temperature && uniform && tokens, "sample_tokens: null tensor pointer");
  PTO_CHECK_ARG(((uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)uniform | (uintptr_t)tokens |
                 (uintptr_t)probs) % 4 == 0 && (uintptr_t)logits % (size_t)dtype_bytes(logits_dtype) == 0,
                "sample_tokens: misaligned operand");
  {
    using block8::overlap;
    const int64_t n = rows * 4, all = rows * vocab * dtype_bytes(logits_dtype);
    bool apart = !overlap(tokens, n, probs, n) && !overlap(tokens, n, logits, all) && !overlap(probs, n, logits, all);
    const void* ins[5] = {temperature, top_k, top_p, min_p, uniform};
    for (const void* in : ins) apart = apart && !overlap(tokens, n, in, n) && !overlap(probs, n, in, n);
    PTO_CHECK_ARG(apart, "sample_tokens: the results overlap an operand or each other");
  }
  const DeviceScope scope(ctx().device);
  hipStream_t st = (hipStream_t)stream;
  const Params p{logits, temperature, top_k, top_p, min_p, uniform, tokens, probs, (int)rows, (int)vocab};
  if (logits_dtype == PTO_HIP_FP32) launch<float>(p, st);
  else if (logits_dtype == PTO_HIP_BF16) launch<__bf16>(p, st);
  else launch<_Float16>(p, st);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
