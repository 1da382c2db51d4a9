// The next token of every row of logits, from a random number of the row's own.
//
//   w_i = exp((l_i - max l) / T)      the order: larger logits first, of equal ones the lower index
//   kept: the first top_k; of those the fewest from the front whose sum reaches top_p of all of theirs; of those the w_i >= min_p
//   token: the first index at which the running sum of the kept w, in the order of indices, passes u times their sum
//
// The kept tokens are what lies in front of a border in that order, and a filter only moves the border forward; min_p asks each weight by itself.
// Weights are integers, w in units of 2^-44: their sums are exact in any order, so that a row's token does not depend on how
// the work is split, and next to a border or the random number the decision is that of the definition up to half a unit a token.
//
// Four kernels, the first three over slices of the rows so that few rows fill the chip too: the largest logit; of rows with top_k or top_p, how many
// tokens or how much weight lie in each of 1472 intervals of 2^(1/32) below it (finer ones where its logits lie closer together, masked ones left out); for each 2048 tokens the sum of what they
// surely keep, and the tokens of the borders' intervals, top_k's and top_p's; and, a workgroup a row, the border among those (by 1024 cells of the intervals, then in order), the 2048 tokens in
// which the random number falls and the token among them.  Where more tokens share a border's interval than are collected (thousands of equal or nearly equal logits), the last kernel looks for
// the border in the row itself, eleven bits of the key a pass: 0.7 ms for a row of 151936 in one launch, 0.8 to 1.3 ms for 64 of them.
//
// A row is read two or three times and its weights are computed in 64 bits.  One row of 151936 bf16 logits with top_p: 24 to 31 us, of which the four kernels' chains of
// dependent loads and barriers 4 + 7 + 7 + 11; 64 rows of 151936 fp32 ones with mixed filters: 47 to 49 us (9 + 11 + 18 + 11), with top_k 20000 and top_p in every row 69; 320 rows of 32000 fp16 ones without: 31 us, collecting 16
// of them, bound by the exponentials; 500 rows of 128000 fp32 ones, mixed: 187 to 190 us, the first read at 5.1 TB/s, the histogram of half of the rows bound by LDS atomics
// (57 to 60 us; a second copy of it in LDS, for half of the conflicts, takes 66, as fewer workgroups fit), the collecting read 70 us, the vector units 85 % busy.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "block_fp8.h"
#include "common.h"
#include "token_seq.h"

namespace {

constexpr int kMaxVocab = 1 << 19;  // sums of 2^19 weights of 2^44 stay below 2^64
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2048;
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

// 2^(44 - i / 64), kept in LDS by every workgroup: 64 places in 64 banks, two at most in one.
struct Powers {
  double of[64];
};
__device__ __forceinline__ void fill(Powers& t) {  // and a barrier
  if (threadIdx.x < 64) {
    const int i = threadIdx.x;
    double v = i & 1 ? 0x1.fa7c1819e90d8p+43 : (double)kOne;  // 2^(-1 / 64)
    v *= i & 2 ? 0x1.f50765b6e4540p-1 : 1.0;
    v *= i & 4 ? 0x1.ea4afa2a490dap-1 : 1.0;
    v *= i & 8 ? 0x1.d5818dcfba487p-1 : 1.0;
    v *= i & 16 ? 0x1.ae89f995ad3adp-1 : 1.0;
    v *= i & 32 ? 0x1.6a09e667f3bcdp-1 : 1.0;
    t.of[i] = v;
  }
}
constexpr int kSteps = 46 * 64;          // weights end behind 45 of the 64ths of a power of two
constexpr int kIntervals = kSteps / 2;

constexpr double kBig = 4503599627370496.0;  // 2^52
// The whole number that was added to kBig.
__device__ __forceinline__ uint64_t whole(double sum) { return __builtin_bit_cast(uint64_t, sum) - __builtin_bit_cast(uint64_t, kBig); }

// What a logit of a row weighs.  With z = 64 log2(best's weight / its own): the whole number next to z is a place in the table and a power of two, the rest, half of
// a 64th at most, the exponential's series up to the fourth power, in its third and first coefficient what is next to the fifth (5/16 f^3 - 5/256 f: within 2^-9 of f^5; off by
// 2.5e-15 of the weight, a 23rd of a unit).
struct Weights {
  float best;     // the largest logit
  double rate;    // 64 log2(e) / T
  const Powers* powers;
  float half_best, fast_rate;  // intervals are by a difference in 32 bits, halved so that it stays finite
  float finer;                 // intervals of an interval of 2^(1/32): 1, or more where the row's logits lie closer together than all of those
  __device__ __forceinline__ double steps(float v) const { return v == best ? 0.0 : ((double)best - (double)v) * rate; }
  // of a finite best: nothing has to be asked.  (The minimum is for temperatures whose rate 32 bits do not hold.)
  __device__ __forceinline__ double finite_steps(float v) const { return fmin(((double)best - (double)v) * rate, kSteps + 63.0); }
  // The interval that a logit lies in, by a function that never falls with the distance from a finite best; kIntervals and more, or NaN: none, and no weight.  (Its 32-bit
  // roundings are a few 2^-23 of it: what lies behind the last interval is more than 45 powers of two down.)
  __device__ __forceinline__ float interval(float v) const { return fmaf(-0.5f, v, half_best) * fast_rate; }
  // A logit below it lies more than `limit` intervals down: one comparison leaves out what weighs nothing
  __device__ __forceinline__ float cut(double limit) const {
    const double v = (double)best - 2.0 * (limit + 1.0) / (double)fast_rate;
    const float f = (float)v;
    return f - fabsf(f) * 0x1p-23f;  // below it, whichever way it was rounded; of an infinite temperature -inf
  }
  // The weight in units of 2^-44, not yet rounded; z in [0, kSteps + 64).  Its lowest bit is set, so that it never lies halfway between two whole numbers: a sum that starts at
  // kBig, where doubles are whole, rounds each in the same way whatever it holds already.
  __device__ __forceinline__ double scaled(double z) const {
    constexpr double magic = 6755399441055744.0;  // 1.5 2^52: what is added to it is rounded to a whole number, its lowest bits
    const double t = z + magic;
    const int near = (int)(uint32_t)__builtin_bit_cast(uint64_t, t);
    constexpr double c = -0.69314718055994530942 / 64.0;
    const double f = z - (t - magic);
    constexpr double fifth = c * c * c * c * c / 120.0;
    double s = fma(c * c * c * c / 24.0, f, c * c * c / 6.0 + fifth * (5.0 / 16.0));
    s = fma(s, f, c * c / 2.0);
    s = fma(s, f, c - fifth * (5.0 / 256.0));
    s = fma(s, f, 1.0);
    const uint64_t power = __builtin_bit_cast(uint64_t, powers->of[near & 63]) - ((uint64_t)(uint32_t)(near >> 6) << 52);
    return __builtin_bit_cast(double, __builtin_bit_cast(uint64_t, s * __builtin_bit_cast(double, power)) | 1);
  }
  __device__ __forceinline__ uint64_t at(double z) const { return whole(scaled(z) + kBig); }
  __device__ __forceinline__ uint64_t operator()(float v) const {
    const double z = steps(v);
    return z < (double)kSteps ? at(z) : 0;  // NaN: nothing
  }
  __device__ __forceinline__ double exact(float v) const { return scaled(fmin(steps(v), 64000.0)) * (1.0 / (double)kOne); }
};

__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const uint64_t o = __shfl_xor((unsigned long long)v, off);
    v = o > v ? o : v;
  }
  return v;
}
__device__ __forceinline__ float wave_min(float v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = fminf(v, __shfl_xor(v, off));
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
  unsigned long long waves[kWaves];
  unsigned long long found[4];
};

constexpr int kSliceThreads = kThreads;
constexpr int kStep = 8 * kSliceThreads;  // elements of a workgroup's step

// Eight elements from i on, NaN behind the end: as a logit it is none.
template <typename T, bool WIDE>
__device__ __forceinline__ void load8(const T* row, int i, int end, float (&v)[8]) {
  if constexpr (WIDE) {
    if (i + 8 <= end) {
      if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(row + i)[0], b = reinterpret_cast<const float4*>(row + i)[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        typedef T T8 __attribute__((ext_vector_type(8)));
        const T8 a = *reinterpret_cast<const T8*>(row + i);
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = (float)a[u];
      }
      return;
    }
  }
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = i + u < end ? (float)row[i + u] : __builtin_nanf("");
}

// Two steps' worth of a thread's elements, on their way at once; NaN behind the end.
struct Two {
  float a[8], b[8];
};
template <typename T, bool WIDE>
__device__ __forceinline__ void load_two(const T* row, int i0, int end, Two& v) {
  load8<T, WIDE>(row, i0 + threadIdx.x * 8, end, v.a);
  load8<T, WIDE>(row, i0 + threadIdx.x * 8 + kStep, end, v.b);
}
// f(eight logits, index of the first) for a thread's elements of [first, end); v: the first of them, asked for before.
template <typename T, bool WIDE, typename F>
__device__ __forceinline__ void in_eights(const T* row, int first, int end, Two& v, F f) {
  for (int i0 = first; i0 < end; i0 += 2 * kStep) {
    const int i = i0 + threadIdx.x * 8;
    f(v.a, i);
    if (i0 + kStep < end) f(v.b, i + kStep);
    if (i0 + 2 * kStep < end) load_two<T, WIDE>(row, i0 + 2 * kStep, end, v);
  }
}
// f(logit, index) likewise.
template <typename T, bool WIDE, typename F>
__device__ __forceinline__ void in_steps(const T* row, int first, int end, F f) {
  Two v;
  if (first < end) load_two<T, WIDE>(row, first, end, v);
  in_eights<T, WIDE>(row, first, end, v, [&](const float (&v)[8], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 8; ++u) f(v[u], i + u);
  });
}

// A thread's eight elements as they lie in memory; NaN behind the end.
template <typename T>
using Raw8 = T __attribute__((ext_vector_type(8)));
template <typename T, bool WIDE>
__device__ __forceinline__ Raw8<T> load_raw(const T* row, int i, int end) {
  if constexpr (WIDE) {
    if (i + 8 <= end) return *reinterpret_cast<const Raw8<T>*>(row + i);
  }
  Raw8<T> v;
#pragma unroll
  for (int u = 0; u < 8; ++u) v[u] = i + u < end ? row[i + u] : (T)__builtin_nanf("");
  return v;
}
// f(logit, index) likewise and behind every step done(step), the next step's loads on their way meanwhile; `next`: the first step's, asked for long before.
template <typename T, bool WIDE, typename F, typename Done>
__device__ __forceinline__ void step_by_step(const T* row, int first, int end, Raw8<T> next, F f, Done done) {
  for (int i0 = first; i0 < end; i0 += kStep) {
    const int i = i0 + threadIdx.x * 8;
    const Raw8<T> v = next;
    if (i0 + kStep < end) next = load_raw<T, WIDE>(row, i + kStep, end);
#pragma unroll
    for (int u = 0; u < 8; ++u) f((float)v[u], i + u);
    done((i0 - first) / kStep);
  }
}

// The border behind which the running sum, of tokens (by_weight: of weights) in the order, reaches `need`, from `in_front` on; it lies between the keys
// lo and hi, or nowhere (false).  Eleven bits of the key a pass over the row.
template <typename T, bool WIDE>
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
    in_steps<T, WIDE>(row, 0, vocab, [&](float v, int) {
      const uint32_t key = ordered(v);
      if (key < lo || key > hi) return;
      const int bin = (hi - key) >> shift;
      atomicAdd(&sh.count[bin], 1u);
      const uint64_t x = w(v);
      if (x) atomicAdd(&sh.weight[bin], (unsigned long long)x);
    });
    __syncthreads();
    constexpr int kOwn = kBins / kThreads;
    uint64_t n_own = 0, x_own = 0;
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      n_own += sh.count[threadIdx.x * kOwn + u];
      x_own += sh.weight[threadIdx.x * kOwn + u];
    }
    unsigned long long all;
    uint64_t n_front = tokens_front + sum_in_front<unsigned long long>(n_own, sh.waves, &all);
    uint64_t x_front = weight_front + sum_in_front<unsigned long long>(x_own, sh.waves, &all);
    if (threadIdx.x == 0) sh.found[0] = kBins;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const uint64_t n = sh.count[threadIdx.x * kOwn + u], x = sh.weight[threadIdx.x * kOwn + u];
      const uint64_t front = by_weight ? x_front : n_front;
      if (front < need && front + (by_weight ? x : n) >= need) {
        sh.found[0] = threadIdx.x * kOwn + u;
        sh.found[1] = n_front;
        sh.found[2] = x_front;
      }
      n_front += n;
      x_front += x;
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

// A row's filters.
struct Filters {
  int k;        // 0: none
  bool by_sum;  // top_p
  double p;
  uint64_t least;  // a chosen token's weight
  __device__ __forceinline__ bool any() const { return k > 0 || by_sum; }
};
__device__ __forceinline__ Filters filters_of(const Params& p, int r) {
  Filters f;
  const int k = p.top_k ? p.top_k[r] : 0;
  const float top_p = p.top_p ? p.top_p[r] : 1.f, min_p = p.min_p ? p.min_p[r] : 0.f;
  f.k = k > 0 && k < p.vocab ? k : 0;
  f.by_sum = top_p < 1.f;
  f.p = fmax((double)top_p, 0.0);
  f.least = min_p > 0.f ? (uint64_t)ceil(fmin((double)min_p, 1.0) * (double)kOne) : 1;  // weights of nothing are never chosen
  return f;
}
__device__ __forceinline__ uint64_t needed(const Filters& f, uint64_t sum) { return max((uint64_t)ceil(f.p * (double)sum), (uint64_t)1); }

// A token's place in the order, larger ones in front: its key, then its index.
__device__ __forceinline__ uint64_t packed(float v, int i) { return (uint64_t)ordered(v) << 32 | (uint32_t)~i; }

// The place of the last token that a row's filters keep, from the row alone (all threads of a workgroup of kThreads).
template <typename T, bool WIDE>
__device__ __forceinline__ uint64_t border_of_row(Shared& sh, const T* row, int vocab, float low, const Weights& w, const Filters& f) {
  const uint32_t top = ordered(w.best), bottom = max(ordered(low), kNone + 1);
  Border border{kNone, 0};
  uint64_t total = 0;
  bool bounded = false;
  if (f.k) bounded = find_border<T, WIDE>(sh, row, vocab, w, false, (uint64_t)f.k, bottom, top, &border, &total);
  if (f.by_sum) {
    if (!bounded) {
      in_steps<T, WIDE>(row, 0, vocab, [&](float v, int) { total += w(v); });
      unsigned long long all;
      sum_in_front<unsigned long long>(total, sh.waves, &all);
      total = all;
    }
    Border nearer;
    uint64_t unused;
    if (find_border<T, WIDE>(sh, row, vocab, w, true, needed(f, total), bounded ? border.key : bottom, top, &nearer, &unused)) {
      border = nearer;
      bounded = true;
    }
  }
  if (!bounded) return (uint64_t)(kNone + 1) << 32;
  // the index of the last of its ties
  uint64_t before = 0;
  __syncthreads();
  if (threadIdx.x == 0) sh.found[0] = 0;
  __syncthreads();
  for (int i0 = 0; i0 < vocab && before < border.ties; i0 += kStep) {
    const int i = i0 + threadIdx.x * 8;
    float v[8];
    load8<T, WIDE>(row, i, vocab, v);
    uint64_t own = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) own += i + u < vocab && ordered(v[u]) == border.key;
    unsigned long long all;
    uint64_t number = before + sum_in_front<unsigned long long>(own, sh.waves, &all);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool tie = i + u < vocab && ordered(v[u]) == border.key;
      number += tie;
      if (tie && number == border.ties) sh.found[0] = (uint32_t)~(i + u);
    }
    before += all;
  }
  __syncthreads();
  return (uint64_t)border.key << 32 | sh.found[0];
}

// ---- slices ----
// Slices are for some four workgroups a CU, and at most this long: of 500 rows of 128000 the histogram takes 57 / 60 / 49 us and collecting 72 / 78 / 98 us by slices of
// 16384 / 32768 / 65536.
constexpr int kMaxSlice = 16384;
constexpr int kCollected = 4096;
constexpr int kGathered = 1024;  // by a workgroup for itself, with one place asked for in the row's list

constexpr int kFront = 9;

// What the kernels leave for each other, a row of each a row.
struct Scratch {
  unsigned long long* best;    // [slices] places of the slices' largest logits
  float* low;                  // [slices] and the smallest beside them (Beside)
  unsigned long long* weight;  // [kIntervals]
  unsigned int* count;         // [kIntervals]
  unsigned int* collected;     // [1] tokens of the border's intervals
  unsigned long long* tokens;  // [kCollected] their places
  unsigned long long* sums;    // [stretches] weights surely kept of each kStep elements
  unsigned long long* front;   // [kFront] of top_k's interval and of top_p's: the first, their number, tokens and weights in front; the weights of all
  int slices, slice;           // elements of a slice, a multiple of kStep
  int stretches;               // kStep elements each
};

// The smallest of a row's logits that weigh anything, or less: what lies 46 powers of two below the largest - masked logits, whatever they are masked by - has no part in how
// close together a row's logits lie.  Of a part of the row the largest is known before the row's: its smallest is not below the bound of its own largest, and moves up with that.
struct Beside {
  float span;  // 46 powers of two: 31.9 temperatures, somewhat more
  __device__ __forceinline__ explicit Beside(float temperature) : span(32.5f * temperature) {}
  // logits that are not above it weigh nothing beside `most`
  __device__ __forceinline__ float bound(float most) const { return most - span - fabsf(most) * 0x1p-22f; }
  // a part's smallest beside a larger logit than the part's; of a part that weighs nothing none
  __device__ __forceinline__ float moved(float low, float part_most, float bound) const { return part_most > bound ? fmaxf(low, bound) : INFINITY; }
};

template <typename T, bool WIDE>
__global__ __launch_bounds__(kSliceThreads) void best_kernel(Params p, Scratch s) {
  __shared__ unsigned long long waves[kSliceThreads / 64];
  __shared__ float lows[kSliceThreads / 64];
  const int slice = blockIdx.x, r = blockIdx.y;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.vocab;
  const int first = slice * s.slice, end = min(p.vocab, first + s.slice);
  Two ahead;
  load_two<T, WIDE>(row, first, end, ahead);
  const Beside beside(p.temperature[r]);
  // a thread meets its elements by rising index: of equal ones the first stays
  float most = -INFINITY, low = INFINITY;
  int where = first;
  auto more_of = [&](const float (&v)[8], int i) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const bool more = v[u] > most;
      most = more ? v[u] : most;
      where = more ? i + u : where;
    }
  };
  if (filters_of(p, r).any()) {
    in_eights<T, WIDE>(row, first, end, ahead, [&](const float (&v)[8], int i) __attribute__((always_inline)) {
      const float before = most;
      more_of(v, i);
      const float bound = beside.bound(most);
      low = beside.moved(low, before, bound);
#pragma unroll
      for (int u = 0; u < 8; ++u) low = fminf(low, v[u] > bound ? v[u] : INFINITY);
    });
  } else {
    in_eights<T, WIDE>(row, first, end, ahead, more_of);
  }
  uint64_t best = packed(most, where);
  // the histogram of the next kernel starts from nothing
  const int per = (kIntervals + s.slices - 1) / s.slices;
  for (int i = slice * per + threadIdx.x; i < min(kIntervals, (slice + 1) * per); i += kSliceThreads) {
    s.weight[(size_t)r * kIntervals + i] = 0;
    s.count[(size_t)r * kIntervals + i] = 0;
  }
  if (slice == 0 && threadIdx.x == 0) s.collected[r] = 0;
  best = wave_max(best);
  low = wave_min(beside.moved(low, most, beside.bound(value_of((uint32_t)(best >> 32)))));
  if (threadIdx.x % 64 == 0) {
    waves[threadIdx.x / 64] = best;
    lows[threadIdx.x / 64] = low;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kSliceThreads / 64; ++w) best = waves[w] > best ? waves[w] : best;
    const float bound = beside.bound(value_of((uint32_t)(best >> 32)));
    low = INFINITY;
    for (int w = 0; w < kSliceThreads / 64; ++w) low = fminf(low, beside.moved(lows[w], value_of((uint32_t)(waves[w] >> 32)), bound));
    s.best[(size_t)r * s.slices + slice] = best;
    s.low[(size_t)r * s.slices + slice] = low;
  }
}

// The place of a row's largest logit and, where it has filters, the smallest beside it, by every wavefront for itself.
struct Span {
  uint64_t best;
  float low;
};
__device__ __forceinline__ Span span_of_row(const Scratch& s, int r, bool filtered, float temperature) {
  const int lane = threadIdx.x % 64;
  const unsigned long long* bests = s.best + (size_t)r * s.slices;
  const float* lows = s.low + (size_t)r * s.slices;
  constexpr int kOwn = kMaxVocab / kStep / 64;
  uint64_t own[kOwn];
  float own_low[kOwn];
  auto ask = [&](int u) __attribute__((always_inline)) {  // behind the last slice the last again
    const int i = min(lane + 64 * u, s.slices - 1);
    own[u] = bests[i];
    own_low[u] = lows[i];
  };
  const bool many = s.slices > 64;
  ask(0);
  if (many) {
#pragma unroll
    for (int u = 1; u < kOwn; ++u) ask(u);
  }
  uint64_t best = own[0];
  if (many) {
#pragma unroll
    for (int u = 1; u < kOwn; ++u) best = max(best, own[u]);
  }
  best = wave_max(best);
  if (!filtered) return Span{best, -INFINITY};
  const Beside beside(temperature);
  const float bound = beside.bound(value_of((uint32_t)(best >> 32)));
  float low = beside.moved(own_low[0], value_of((uint32_t)(own[0] >> 32)), bound);
  if (many) {
#pragma unroll
    for (int u = 1; u < kOwn; ++u) low = fminf(low, beside.moved(own_low[u], value_of((uint32_t)(own[u] >> 32)), bound));
  }
  return Span{best, wave_min(low)};
}
__device__ __forceinline__ Weights weights_of(const Span& span, float temperature, const Powers* powers) {
  const float v = value_of((uint32_t)(span.best >> 32));
  const double rate = 64.0 * 1.4426950408889634074 / (double)temperature;
  // Half the distance and two steps an interval.  At a high temperature, or of an even distribution, that is few intervals for the whole row, and thousands of tokens in the
  // border's: then there are as many intervals between its logits as there is room for (64 rows of 151936 at a temperature of 30: 61 us, by the row's own passes 657; the same
  // with masked logits among them).
  const float whole = (float)(((double)v - (double)span.low) * rate * 0.5);
  const float finer = fminf(fmaxf((kIntervals - 2) * __builtin_amdgcn_rcpf(whole), 1.f), 1e6f);  // of no distance 1e6, of an infinite or undefined one 1
  return Weights{v, rate, powers, 0.5f * v, (float)fmin(rate * finer, 1e38), finer};
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kSliceThreads) void histogram_kernel(Params p, Scratch s) {
  __shared__ Powers powers;
  __shared__ unsigned long long weight[kIntervals];
  __shared__ unsigned int count[kIntervals];
  const int slice = blockIdx.x, r = blockIdx.y;
  const Filters f = filters_of(p, r);
  const float t = p.temperature[r];
  const Span span = span_of_row(s, r, f.any(), t);
  if (!(t > 0.f) || !f.any()) return;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.vocab;
  const int first = slice * s.slice, end = min(p.vocab, first + s.slice);
  const Raw8<T> ahead = load_raw<T, WIDE>(row, first + threadIdx.x * 8, end);
  const Weights w = weights_of(span, t, &powers);
  if (!(fabsf(w.best) <= 3.4028234664e38f)) return;  // nothing to choose from, or infinite: the last kernel looks at the row
  fill(powers);
  for (int i = threadIdx.x; i < kIntervals; i += kSliceThreads) {
    weight[i] = 0;
    count[i] = 0;
  }
  __syncthreads();
  const bool by_count = f.k > 0;
  auto each = [&](auto counts, auto weighs) {
    step_by_step<T, WIDE>(row, first, end, ahead, [&](float v, int) __attribute__((always_inline)) {
      const float i = w.interval(v);
      if (i < (float)kIntervals) {
        if constexpr (decltype(counts)::value != 0) atomicAdd(&count[(int)i], 1u);
        if constexpr (decltype(weighs)::value != 0) atomicAdd(&weight[(int)i], (unsigned long long)w.at(w.finite_steps(v)));
      }
    }, [](int) {});
  };
  using pto_hip::block8::IntConst;
  if (by_count && f.by_sum) each(IntConst<1>{}, IntConst<1>{});
  else if (by_count) each(IntConst<1>{}, IntConst<0>{});
  else each(IntConst<0>{}, IntConst<1>{});
  __syncthreads();
  for (int i = threadIdx.x; i < kIntervals; i += kSliceThreads) {
    if (by_count && count[i]) atomicAdd(&s.count[(size_t)r * kIntervals + i], count[i]);
    if (f.by_sum && weight[i]) atomicAdd(&s.weight[(size_t)r * kIntervals + i], weight[i]);
  }
}

// Neighbouring intervals and what lies in front of them; kIntervals: none.
struct Stretch {
  int first, last;
  uint64_t tokens_front, weight_front;
  __device__ __forceinline__ bool there() const { return first < kIntervals; }
};
// The intervals in which a row's borders may lie: top_k's, one, and top_p's, which are in front of it or end with it.  Thousands of tokens may lie between the two.
struct BorderIntervals {
  Stretch k, p;
  uint64_t weight_all;
};
// Each thread holds the sums of its kIntervals / kSliceThreads intervals.
__device__ __forceinline__ BorderIntervals find_intervals(const Scratch& s, int r, const Filters& f) {
  constexpr int kOwn = (kIntervals + kSliceThreads - 1) / kSliceThreads;
  __shared__ unsigned long long wave_n[kSliceThreads / 64], wave_w[kSliceThreads / 64];
  __shared__ unsigned long long found[8];
  uint64_t n[kOwn], x[kOwn], n_own = 0, x_own = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    const int at = threadIdx.x * kOwn + i;
    n[i] = at < kIntervals && f.k ? s.count[(size_t)r * kIntervals + at] : 0;
    x[i] = at < kIntervals && f.by_sum ? s.weight[(size_t)r * kIntervals + at] : 0;
    n_own += n[i];
    x_own += x[i];
  }
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  uint64_t n_to = n_own, x_to = x_own;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint64_t a = __shfl_up((unsigned long long)n_to, off), b = __shfl_up((unsigned long long)x_to, off);
    if (lane >= off) {
      n_to += a;
      x_to += b;
    }
  }
  if (lane == 63) {
    wave_n[wave] = n_to;
    wave_w[wave] = x_to;
  }
  if (threadIdx.x < 8) found[threadIdx.x] = kIntervals;
  __syncthreads();
  uint64_t all = 0, n_front = n_to - n_own, x_front = x_to - x_own;
  for (int i = 0; i < kSliceThreads / 64; ++i) {
    if (i < wave) {
      n_front += wave_n[i];
      x_front += wave_w[i];
    }
    all += wave_w[i];
  }
  // of top_k: found[0] its interval, the weights in front of it and up to its end in [1] and [2], the tokens in front in [3]
  if (f.k) {
    uint64_t a = n_front, b = x_front;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (a < (uint64_t)f.k && a + n[i] >= (uint64_t)f.k) {
        found[0] = threadIdx.x * kOwn + i;
        found[1] = b;
        found[2] = b + x[i];
        found[3] = a;
      }
      a += n[i];
      b += x[i];
    }
    __syncthreads();
  }
  const int k_at = (int)found[0];
  BorderIntervals out{{k_at, k_at, k_at < kIntervals ? found[3] : 0, k_at < kIntervals ? found[1] : 0}, {kIntervals, kIntervals, 0, 0}, all};
  if (f.by_sum) {
    // the weights of what top_k keeps lie between those in front of its interval and those up to its end
    const uint64_t lo = needed(f, k_at < kIntervals ? found[1] : all), hi = needed(f, k_at < kIntervals ? found[2] : all);
    uint64_t a = n_front, b = x_front;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (b < lo && b + x[i] >= lo) {
        found[4] = threadIdx.x * kOwn + i;
        found[5] = a;
        found[6] = b;
      }
      if (b < hi && b + x[i] >= hi) found[7] = threadIdx.x * kOwn + i;
      a += n[i];
      b += x[i];
    }
    __syncthreads();
    out.p = Stretch{(int)found[4], (int)found[7], found[5], found[6]};
  }
  return out;
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kSliceThreads) void collect_kernel(Params p, Scratch s) {
  __shared__ Powers powers;
  __shared__ unsigned long long sums[kMaxSlice / kStep];
  __shared__ unsigned long long tokens[kGathered];
  __shared__ unsigned int gathered, place;
  const int slice = blockIdx.x, r = blockIdx.y;
  const float t = p.temperature[r];
  const Filters f = filters_of(p, r);
  const Span span = span_of_row(s, r, f.any(), t);
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.vocab;
  const int first = slice * s.slice, end = min(p.vocab, first + s.slice);
  const Raw8<T> ahead = load_raw<T, WIDE>(row, first + threadIdx.x * 8, end);
  if (!(t > 0.f) || (uint32_t)(span.best >> 32) <= kNone) return;
  const Weights w = weights_of(span, t, &powers);
  const bool infinite = !(w.best <= 3.4028234664e38f);
  if (infinite && f.any()) {
    if (slice == 0 && threadIdx.x == 0) s.collected[r] = kCollected + 1;  // for the last kernel to look at the row
    return;
  }
  fill(powers);
  if (threadIdx.x < kMaxSlice / kStep) sums[threadIdx.x] = 0;
  if (threadIdx.x == 0) gathered = 0;
  BorderIntervals at{{kIntervals, kIntervals, 0, 0}, {kIntervals, kIntervals, 0, 0}, 0};
  if (f.any()) at = find_intervals(s, r, f);
  if (slice == 0 && threadIdx.x == 0) {
    unsigned long long* front = s.front + kFront * (size_t)r;
    auto leave = [&](unsigned long long* to, const Stretch& x) {
      to[0] = x.first;
      to[1] = x.last - x.first + 1;
      to[2] = x.tokens_front;
      to[3] = x.weight_front;
    };
    leave(front, at.k);
    leave(front + 4, at.p);
    front[8] = at.weight_all;
  }
  __syncthreads();
  const double least = (double)f.least, more_than = least - 0.5;  // of a weight not yet rounded
  // of what is surely kept, min_p - or the rounding to whole units - leaves out what is further down than this (an interval more than it has to be)
  const float i_least = (32.f * ((float)kUnit - __builtin_amdgcn_logf((float)more_than)) + 1.f) * w.finer;
  using pto_hip::block8::IntConst;
  // collected is what lies in the borders' intervals: from i_first to i_last and from i_again to i_behind
  const bool both = at.k.there() && at.p.there() && at.p.last < at.k.first;
  const float i_first = (float)min(at.k.first, at.p.first), i_sure = fminf(i_first, i_least);
  const float i_behind = fminf((float)(at.k.there() ? at.k.last + 1 : at.p.last + 1), (float)kIntervals);
  const float i_last = both ? (float)(at.p.last + 1) : i_behind, i_again = both ? (float)at.k.first : i_behind;
  const float cut = w.cut(i_behind);
  double own = kBig;  // and the weights of a step: exact
  auto take = [&](float v, int i, auto apart) __attribute__((always_inline)) {
    if (v < cut) return;  // most logits of a row with a border
    const float at_i = w.interval(v);
    if (at_i < i_sure) {
      const double x = w.scaled(w.finite_steps(v));
      own += x > more_than ? x : 0.0;
    } else if (at_i >= i_first && at_i < i_behind && (decltype(apart)::value == 0 || at_i < i_last || at_i >= i_again)) {
      const unsigned int n = atomicAdd(&gathered, 1u);
      if (n < kGathered) {
        tokens[n] = packed(v, i);
      } else {
        const unsigned int m = atomicAdd(&s.collected[r], 1u);
        if (m < kCollected) s.tokens[(size_t)r * kCollected + m] = packed(v, i);
      }
    }
  };
  // of a row without a border: nearly all of its logits weigh something, and nothing is branched around
  auto take_all = [&](float v, int) __attribute__((always_inline)) { own += w.scaled(w.finite_steps(v)); };
  auto take_heavy = [&](float v, int) __attribute__((always_inline)) {
    const double x = w.scaled(w.finite_steps(v));
    own += x > more_than ? x : 0.0;
  };
  auto take_infinite = [&](float v, int) { own += v == w.best ? (double)kOne : 0.0; };
  auto done = [&](int step) __attribute__((always_inline)) {
    const uint64_t sum = wave_sum((unsigned long long)whole(own));
    if (threadIdx.x % 64 == 0 && sum) atomicAdd(&sums[step], (unsigned long long)sum);
    own = kBig;
  };
  if (infinite) step_by_step<T, WIDE>(row, first, end, ahead, take_infinite, done);
  else if (i_first == (float)kIntervals && f.least == 1) step_by_step<T, WIDE>(row, first, end, ahead, take_all, done);  // what is below a half adds nothing
  else if (i_first == (float)kIntervals) step_by_step<T, WIDE>(row, first, end, ahead, take_heavy, done);
  else if (both) step_by_step<T, WIDE>(row, first, end, ahead, [&](float v, int i) __attribute__((always_inline)) { take(v, i, IntConst<1>{}); }, done);
  else step_by_step<T, WIDE>(row, first, end, ahead, [&](float v, int i) __attribute__((always_inline)) { take(v, i, IntConst<0>{}); }, done);
  __syncthreads();
  const int stretch = first / kStep + threadIdx.x;
  if (threadIdx.x < s.slice / kStep && stretch < s.stretches) s.sums[(size_t)r * s.stretches + stretch] = sums[threadIdx.x];
  const unsigned int n = min(gathered, (unsigned int)kGathered);
  if (n == 0) return;
  if (threadIdx.x == 0) place = atomicAdd(&s.collected[r], n);
  __syncthreads();
  for (unsigned int i = threadIdx.x; i < n; i += kSliceThreads)
    if (place + i < kCollected) s.tokens[(size_t)r * kCollected + place + i] = tokens[i];
}

constexpr int kCells = 1024;  // of the border's intervals
// A cell of so few tokens is put in order by counting those in front of each (one row of 151936 bf16 logits, hundreds of them equal to its border's: 12.6 -> 10.7 us); the
// counts grow with the square of the tokens, a bitonic order's steps with the square of their logarithm.
constexpr int kCounted = 512;
struct DrawShared {
  Powers powers;
  unsigned long long sums[kMaxVocab / kStep];
  unsigned long long found[6];
  unsigned long long waves[kWaves];
  unsigned int gathered;
  unsigned long long tokens[kCollected];  // of one cell, in order
  union {
    Shared row;
    struct {
      unsigned long long weight[kCells];
      unsigned int count[kCells];
    } cells;
  };
};

// Where the running sum of the collected tokens of a border's intervals (by_weight: of their weights), in order and from what lies in front of them on, reaches `need`: the place of
// that token and the sum of the weights up to it.  The cell that it lies in first, then the cell's tokens in order.  All threads take part; `need` is reached.
struct Reached {
  uint64_t place, weight;
};
// The intervals that they are looked for in, as the kernel in front left them: first and number.
struct Within {
  float first, behind, cells_each;
  uint64_t tokens_front, weight_front;
  __device__ __forceinline__ explicit Within(const unsigned long long* at)
      : first((float)at[0]), behind((float)(at[0] + at[1])), cells_each((float)kCells / (float)at[1]), tokens_front(at[2]), weight_front(at[3]) {}
  // the cell of a token by its interval; -1: one in front of them or behind
  __device__ __forceinline__ int cell(float interval) const {
    return interval >= first && interval < behind ? min((int)((interval - first) * cells_each), kCells - 1) : -1;
  }
};
template <typename Interval, typename Weight>
__device__ Reached reach(DrawShared& sh, const unsigned long long* tokens, int n, bool by_weight, const Within& within, uint64_t need, Interval interval, Weight weight) {
  constexpr int kOwn = kCells / kThreads;
  const uint64_t tokens_front = within.tokens_front, weight_front = within.weight_front;
  for (int i = threadIdx.x; i < kCells; i += kThreads) {
    sh.cells.weight[i] = 0;
    sh.cells.count[i] = 0;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int at = within.cell(interval(tokens[i]));
    if (at < 0) continue;
    atomicAdd(&sh.cells.count[at], 1u);
    atomicAdd(&sh.cells.weight[at], (unsigned long long)weight(tokens[i]));
  }
  __syncthreads();
  uint64_t n_own = 0, x_own = 0;
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    n_own += sh.cells.count[threadIdx.x * kOwn + u];
    x_own += sh.cells.weight[threadIdx.x * kOwn + u];
  }
  unsigned long long all;
  uint64_t n_front = tokens_front + sum_in_front<unsigned long long>(n_own, sh.waves, &all);
  uint64_t x_front = weight_front + sum_in_front<unsigned long long>(x_own, sh.waves, &all);
  if (threadIdx.x == 0) sh.gathered = 0;
#pragma unroll
  for (int u = 0; u < kOwn; ++u) {
    const uint64_t c = sh.cells.count[threadIdx.x * kOwn + u], x = sh.cells.weight[threadIdx.x * kOwn + u];
    const uint64_t front = by_weight ? x_front : n_front;
    if (front < need && front + (by_weight ? x : c) >= need) {
      sh.found[0] = threadIdx.x * kOwn + u;
      sh.found[1] = n_front;
      sh.found[2] = x_front;
    }
    n_front += c;
    x_front += x;
  }
  __syncthreads();
  const int here = (int)sh.found[0];
  const uint64_t n_cell = sh.found[1], x_cell = sh.found[2];
  for (int i = threadIdx.x; i < n; i += kThreads)
    if (within.cell(interval(tokens[i])) == here) sh.tokens[atomicAdd(&sh.gathered, 1u)] = tokens[i];
  __syncthreads();
  const int m = (int)sh.gathered;
  // in order
  if (m <= kCounted) {
    constexpr int kMine = kCounted / kThreads;
    uint64_t mine[kMine];
    int at[kMine];
#pragma unroll
    for (int u = 0; u < kMine; ++u) {
      mine[u] = threadIdx.x + u * kThreads < m ? sh.tokens[threadIdx.x + u * kThreads] : 0;
      at[u] = 0;
    }
    for (int i = 0; i < m; ++i) {
      const uint64_t other = sh.tokens[i];
#pragma unroll
      for (int u = 0; u < kMine; ++u) at[u] += other > mine[u];
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMine; ++u)
      if (threadIdx.x + u * kThreads < m) sh.tokens[at[u]] = mine[u];
    __syncthreads();
  } else {
    int size = 1;
    while (size < m) size *= 2;
    for (int i = m + threadIdx.x; i < size; i += kThreads) sh.tokens[i] = 0;  // the last places
    __syncthreads();
    for (int span = 2; span <= size; span *= 2)
      for (int gap = span / 2; gap > 0; gap /= 2) {
        for (int i = threadIdx.x; i < size / 2; i += kThreads) {
          const int a = 2 * i - (i & (gap - 1)), b = a + gap;
          const uint64_t va = sh.tokens[a], vb = sh.tokens[b];
          if ((va < vb) == ((a & span) == 0)) {
            sh.tokens[a] = vb;
            sh.tokens[b] = va;
          }
        }
        __syncthreads();
      }
  }
  // neighbouring tokens a thread
  const int per = (m + kThreads - 1) / kThreads, first = threadIdx.x * per;
  uint64_t own = 0;
  for (int u = first; u < min(first + per, m); ++u) own += weight(sh.tokens[u]);
  uint64_t x = x_cell + sum_in_front<unsigned long long>(own, sh.waves, &all);
  for (int u = first; u < min(first + per, m); ++u) {
    const uint64_t each = weight(sh.tokens[u]);
    const bool reached = by_weight ? x < need && x + each >= need : n_cell + u + 1 == need;
    x += each;
    if (reached) {
      sh.found[3] = sh.tokens[u];
      sh.found[4] = x;
    }
  }
  __syncthreads();
  return Reached{sh.found[3], sh.found[4]};
}

template <typename T, bool WIDE>
__global__ __launch_bounds__(kThreads) void draw_kernel(Params p, Scratch s) {
  __shared__ DrawShared sh;
  const int r = blockIdx.x;
  const T* row = reinterpret_cast<const T*>(p.logits) + (size_t)r * p.vocab;
  // everything that others left, asked for at once
  const float t = p.temperature[r];
  const Filters f = filters_of(p, r);
  const unsigned int collected = s.collected[r];
  const Span span = span_of_row(s, r, f.any(), t);
  for (int i = threadIdx.x; i < s.stretches; i += kThreads) sh.sums[i] = s.sums[(size_t)r * s.stretches + i];
  const uint32_t top = (uint32_t)(span.best >> 32);
  if (top <= kNone || !(t > 0.f)) {  // nothing to choose from, or no choice
    if (threadIdx.x == 0) {
      p.tokens[r] = top <= kNone ? -1 : (int32_t)~(uint32_t)span.best;
      if (p.probs) p.probs[r] = top <= kNone ? 0.f : 1.f;
    }
    return;
  }
  fill(sh.powers);
  const Weights w = weights_of(span, t, &sh.powers);
  const int n = f.any() ? (int)min(collected, (unsigned int)kCollected + 1) : 0;
  uint64_t border = (uint64_t)(kNone + 1) << 32;
  __syncthreads();
  if (n > kCollected) {
    border = border_of_row<T, WIDE>(sh.row, row, p.vocab, span.low, w, f);
    // the stretches' sums lack what the border's intervals keep
    for (int i = threadIdx.x; i < s.stretches; i += kThreads) sh.sums[i] = 0;
    __syncthreads();
    uint64_t own = 0;
    step_by_step<T, WIDE>(row, 0, p.vocab, load_raw<T, WIDE>(row, threadIdx.x * 8, p.vocab), [&](float v, int i) {
      const uint64_t x = i < p.vocab && packed(v, i) >= border ? w(v) : 0;
      own += x >= f.least ? x : 0;
    }, [&](int step) {
      const uint64_t sum = wave_sum((unsigned long long)own);
      if (threadIdx.x % 64 == 0 && sum) atomicAdd(&sh.sums[step], (unsigned long long)sum);
      own = 0;
    });
  } else if (n > 0) {
    const unsigned long long* tokens = s.tokens + (size_t)r * kCollected;
    const unsigned long long* front = s.front + kFront * (size_t)r;
    auto weight = [&](uint64_t token) { return w(value_of((uint32_t)(token >> 32))); };
    auto interval = [&](uint64_t token) { return w.interval(value_of((uint32_t)(token >> 32))); };
    uint64_t sum = front[8];
    if (front[0] < kIntervals) {
      const Reached k = reach(sh, tokens, n, false, Within(front), (uint64_t)f.k, interval, weight);
      border = k.place;
      sum = k.weight;
    }
    if (f.by_sum) {
      const Reached at = reach(sh, tokens, n, true, Within(front + 4), needed(f, sum), interval, weight);
      border = at.place > border ? at.place : border;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const uint64_t x = tokens[i] >= border ? weight(tokens[i]) : 0;
      if (x >= f.least) atomicAdd(&sh.sums[(int)~(uint32_t)tokens[i] / kStep], (unsigned long long)x);
    }
  }
  __syncthreads();
  // the stretch in which the running sum passes its share
  if (threadIdx.x < 64) {
    constexpr int kOwn = kMaxVocab / kStep / 64;
    uint64_t x[kOwn], own = 0;
#pragma unroll
    for (int u = 0; u < kOwn; ++u) {
      const int i = threadIdx.x * kOwn + u;
      x[u] = i < s.stretches ? sh.sums[i] : 0;
      own += x[u];
    }
    uint64_t to = own;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const uint64_t o = __shfl_up((unsigned long long)to, off);
      if ((int)threadIdx.x >= off) to += o;
    }
    const uint64_t sum = __shfl((unsigned long long)to, 63);
    const double u = fmin(fmax((double)p.uniform[r], 0x1p-25), 1.0 - 0x1p-24);
    const uint64_t target = (uint64_t)(u * (double)sum);
    uint64_t front = to - own;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      if (front <= target && front + x[i] > target) {
        sh.found[0] = threadIdx.x * kOwn + i;
        sh.found[1] = target;
        sh.found[2] = front;
        sh.found[3] = sum;
      }
      front += x[i];
    }
  }
  __syncthreads();
  const int first = (int)sh.found[0] * kStep, end = min(p.vocab, first + kStep);
  const uint64_t target = sh.found[1], sum = sh.found[3];
  // the thread whose eight tokens hold it, and the token among them
  const int mine = first + threadIdx.x * 8;
  float v[8];
  load8<T, WIDE>(row, mine, end, v);
  uint64_t x[8], own = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    x[e] = mine + e < end && packed(v[e], mine + e) >= border ? w(v[e]) : 0;
    x[e] = x[e] >= f.least ? x[e] : 0;
    own += x[e];
  }
  unsigned long long all;
  uint64_t front = sh.found[2] + sum_in_front<unsigned long long>(own, sh.waves, &all);
  if (front <= target && front + own > target) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (front <= target && front + x[e] > target) {
        p.tokens[r] = mine + e;
        if (p.probs) p.probs[r] = (float)(w.exact(v[e]) / ((double)sum * (1.0 / (double)kOne)));
      }
      front += x[e];
    }
  }
}

template <typename T, bool WIDE>
void launch_slices(const Params& p, const Scratch& s, hipStream_t st) {
  const dim3 grid(s.slices, p.rows), threads(kSliceThreads);
  hipLaunchKernelGGL((best_kernel<T, WIDE>), grid, threads, 0, st, p, s);
  if (p.top_k || p.top_p) hipLaunchKernelGGL((histogram_kernel<T, WIDE>), grid, threads, 0, st, p, s);
  hipLaunchKernelGGL((collect_kernel<T, WIDE>), grid, threads, 0, st, p, s);
  hipLaunchKernelGGL((draw_kernel<T, WIDE>), dim3(p.rows), dim3(kThreads), 0, st, p, s);
}

constexpr int64_t kRowsAtOnce = 1024;
template <typename T>
int launch(Params p, hipStream_t st) {
  const int64_t rows = p.rows, at_once = std::min(rows, kRowsAtOnce);
  // slices for some four workgroups a CU
  const int64_t even = (at_once * p.vocab + 4 * pto_hip::ctx().num_cu - 1) / (4 * pto_hip::ctx().num_cu);
  Scratch s{};
  s.slice = (int)std::min<int64_t>(kMaxSlice, std::max<int64_t>(kStep, (even + kStep - 1) / kStep * kStep));
  s.slices = (p.vocab + s.slice - 1) / s.slice;
  s.stretches = (p.vocab + kStep - 1) / kStep;
  const size_t per_row = 8 * ((size_t)s.slices + s.stretches + kIntervals + kCollected + kFront) + 4 * (kIntervals + 2 + (size_t)s.slices);
  void* ws = nullptr;
  const int rc = pto_hip::workspace(per_row * at_once, &ws);
  if (rc) return rc;
  s.best = reinterpret_cast<unsigned long long*>(ws);
  s.sums = s.best + at_once * s.slices;
  s.weight = s.sums + at_once * s.stretches;
  s.tokens = s.weight + at_once * kIntervals;
  s.front = s.tokens + at_once * kCollected;
  s.count = reinterpret_cast<unsigned int*>(s.front + kFront * at_once);
  s.collected = s.count + at_once * kIntervals;
  s.low = reinterpret_cast<float*>(s.collected + at_once);
  const bool wide = (uintptr_t)p.logits % 16 == 0 && (int64_t)p.vocab * sizeof(T) % 16 == 0;
  const Params whole = p;
  for (int64_t r = 0; r < rows; r += at_once) {
    p.rows = (int)std::min(at_once, rows - r);
    p.logits = reinterpret_cast<const T*>(whole.logits) + r * p.vocab;
    p.temperature = whole.temperature + r;
    p.top_k = whole.top_k ? whole.top_k + r : nullptr;
    p.top_p = whole.top_p ? whole.top_p + r : nullptr;
    p.min_p = whole.min_p ? whole.min_p + r : nullptr;
    p.uniform = whole.uniform + r;
    p.tokens = whole.tokens + r;
    p.probs = whole.probs ? whole.probs + r : nullptr;
    wide ? launch_slices<T, true>(p, s, st) : launch_slices<T, false>(p, s, st);
  }
  return PTO_HIP_OK;
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
  const int rc = logits_dtype == PTO_HIP_FP32 ? launch<float>(p, st) : logits_dtype == PTO_HIP_BF16 ? launch<__bf16>(p, st) : launch<_Float16>(p, st);
  if (rc) return rc;
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
