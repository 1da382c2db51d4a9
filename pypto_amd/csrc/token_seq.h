// Ragged batches: which sequence a token belongs to, from the rising list of the sequences' first tokens.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

namespace pto_hip {

// The device that a call's pointers belong to is the library's; the caller's current one may be another, and is again afterwards.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (hipGetDevice(&before_) != hipSuccess || before_ == device) return;
    changed_ = hipSetDevice(device) == hipSuccess;
  }
  ~DeviceScope() {
    if (changed_) (void)hipSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

struct TokenSeq {
  int seq;    // -1: the token belongs to nobody
  int first;  // the sequence's first token
  int count;  // and how many it has
};

// A start as every kernel takes it: one in front of the batch's rows or behind them counts as their end on that side, so that a sequence which passes them has the tokens that there are.
__device__ __forceinline__ int within(int start, int tokens) { return min(max(start, 0), tokens); }
// Whether there are such starts (they rise): to be reported, by one thread of a launch.
__device__ __forceinline__ bool pass_the_rows(const int32_t* starts, int batch, int tokens) { return starts[0] < 0 || starts[batch] > tokens; }

// The last sequence that starts at `token` or in front of it, looked for by a whole wavefront: 64 starts a step, so that 64 sequences take one
// trip to memory and 4096 two.  starts[0 .. batch], of a batch of `tokens` rows; whatever they hold, no other element is read and the answer lies in the batch.
__device__ __forceinline__ TokenSeq sequence_of(const int32_t* starts, int batch, int tokens, int token, int lane) {
  int lo = 0, n = batch;
  while (n > 64) {
    const int step = (n + 63) / 64;
    const int at = lo + lane * step;
    const uint64_t in_front = __ballot(lane * step < n && starts[min(at, batch)] <= token);
    const int k = max((int)__popcll(in_front) - 1, 0);  // below the number of lanes that voted: lo stays in the batch
    lo += k * step;
    n = min(step, n - k * step);
  }
  const int at = min(lo + lane, batch);
  const int start = within(starts[at], tokens), next = within(starts[min(at + 1, batch)], tokens);
  const int k = max((int)__popcll(__ballot(lane < n && start <= token)) - 1, 0);
  const int first = __shfl(start, k), end = __shfl(next, k);
  return TokenSeq{first <= token && token < end ? lo + k : -1, first, end - first};
}

// f(tokens) for the tokens of each launch of a call with parameters p: a launch holds fewer than 2^32 threads.
template <typename P, typename F>
void in_launches(P& p, int64_t threads_a_token, F f) {
  const int64_t most = std::max<int64_t>(1, (1ll << 31) / threads_a_token);
  for (int64_t t = 0; t < p.tokens; t += most) {
    p.t0 = (int)t;
    f((unsigned)std::min<int64_t>(most, p.tokens - t));
  }
}

// Sums over a wavefront without a trip through LDS: along rows of 16 lanes, then from row to row; lane 63 has all.
template <int CTRL, int ROWS>
__device__ __forceinline__ int add_from(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float add_from(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, true));
}
// The sum of the lanes up to this one (of integers: exact).
template <typename V>
__device__ __forceinline__ V wave_running_sum(V v) {
  v = add_from<0x111, 0xf>(v);
  v = add_from<0x112, 0xf>(v);
  v = add_from<0x114, 0xf>(v);
  v = add_from<0x118, 0xf>(v);
  v = add_from<0x142, 0xa>(v);
  v = add_from<0x143, 0xc>(v);
  return v;
}
template <typename V>
__device__ __forceinline__ V wave_total(V v) {
  return __builtin_bit_cast(V, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_running_sum(v)), 63));
}

}  // namespace pto_hip
