// The experts' FFN of a mixture layer on e4m3 operands with a scale for each block of 128:
//
//   out[t] = sum_j weights[t, j] * FFN_e(x[t]),  e = ids[t, j],   FFN_e(x) = (SiLU(x Wg_e) * (x Wu_e)) Wd_e
//
// The slots (t, j) are put in order of their experts, so that the rows of a tile of either product share one expert's
// matrices; the tiles of all experts are one launch.  h = SiLU(g) * u is quantised per 128 channels in the
// first product's epilogue, from 32 bits; the second product's rows stay in 32 bits until the sum over a token's experts (bf16 results: in fp16 with
// a power of two per 128 channels, see run_pass).
//
// 2048 tokens, 8 of 64 experts of 4096 x 1408, bf16: 475 to 490 us, of them the plan 11, gate/up 300 to 340, down 200, the sum 30.  Bound by memory and power
// together: 1.1 GB of weights take 215 us at the copy's rate and are read once per height of tile (1.18 GB of gate and up instead of 0.74), a tile of 256
// rows takes 87 us where it would take 63 with its weights in the caches, at a clock of 1.7 to 2.1 GHz.  40 tokens, 4 of 60 of 2048 x 1024, fp16: 78 us, the
// stream of 350 MB (68 at the copy's rate) between two kernels of 5.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block_gemm8.h"
#include "block_tiled8.h"
#include "common.h"
#include "launch_choice.h"

namespace pto_hip {
namespace block8 {

constexpr int kMaxExperts = 1024;
constexpr int kPlanThreads = 1024;
constexpr int kFewSlots = 1024, kFewThreads = 256;  // a plan of few slots and experts: 192 slots of 16 experts 2.8 us for 3.6, 1024 of 250 3.4 for 4.6
// Tokens are worked through in passes of at most so many slots (expert_pass_tokens), so that the scratch stays small and every index inside 32 bits.
constexpr int64_t kPassSlots = kExpertPassSlots;
constexpr int64_t kMostDirectSlots = 1024;

// The plan: slots by expert, and tiles of one expert each: of `height` rows, and what an expert has left in a tile of the least of height,
// height / 2 and height / 4 rows (64 at least) that holds it.  The heights lie one behind the other, n_tiles[] of each.  One workgroup, EACH
// slots a thread; a slot with a negative expert is in no tile, one with an expert that there is not is reported.  Each wavefront counts for
// itself ([wavefronts][experts] in LDS), so that the counters of a busy expert are shared by 64 lanes and not by all, and a slot's rank in its
// wavefront's count is its place.  The sorted slots are put together in LDS: written one by one, each to a line of its own, they took 5 us
// more.  The order of the ranks is that of the atomics: which row of which tile a slot becomes changes no bit of its result.
// Bound by the LDS atomics: 192 slots 2.8 us (4.8 behind a stream that has emptied the caches), 4096 6, 16384 12, 32768 16.
template <int EACH, int THREADS>
__global__ __launch_bounds__(THREADS) void plan_kernel(const int32_t* __restrict__ ids, int slots, int experts, int height,
                                                            int32_t* __restrict__ order, int4* __restrict__ tiles, int* __restrict__ n_tiles,
                                                            int* __restrict__ flag) {
  constexpr int kWaves = THREADS / 64;
  extern __shared__ int count[];  // [kWaves][experts], then the slots by expert
  uint16_t* const sorted = reinterpret_cast<uint16_t*>(count + kWaves * experts);
  __shared__ int sums[2][kWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int i = tid; i < kWaves * experts; i += THREADS) count[i] = 0;
  int place[EACH];  // the slot's expert, then with its rank behind the experts' bits; -1: none
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int s = i * THREADS + tid;
    const int id = ids[(uint32_t)min(s, slots - 1)];
    place[i] = s < slots ? id : -1;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int e = place[i];
    if (e >= experts) *flag = 1;
    int rank = 0;
    if ((unsigned)e < (unsigned)experts) rank = atomicAdd(&count[wave * experts + e], 1);
    place[i] = (unsigned)e < (unsigned)experts ? e | rank * kMaxExperts : -1;
  }
  __syncthreads();
  // thread t: expert t's rows and tiles, exclusive sums over the experts in front, then over its wavefronts
  int rows = 0, counted[kWaves];
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    counted[w] = tid < experts ? count[w * experts + tid] : 0;
    rows += counted[w];
  }
  int mine[3] = {rows / height, 0, 0};
  const int rest = rows - mine[0] * height;
  const int rest_height = height >= 256 && rest <= height / 4 ? 2 : height >= 128 && rest <= height / 2 ? 1 : 0;
#pragma unroll
  for (int q = 0; q < 3; ++q) mine[q] += rest > 0 && rest_height == q;
  // two sums in a word: rows (at most 2^15) and tiles of height / 4 (at most kMaxExperts), tiles of height and of height / 2
  const int each[2] = {rows | mine[2] << 16, mine[0] | mine[1] << 16};
  int sum[2] = {each[0], each[1]};
#pragma unroll
  for (int q = 0; q < 2; ++q) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int o = __shfl_up(sum[q], off);
      if (lane >= off) sum[q] += o;
    }
    if (lane == 63) sums[q][wave] = sum[q];
  }
  __syncthreads();
  int before[2] = {sum[0] - each[0], sum[1] - each[1]}, all[2] = {0, 0};
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      if (w < wave) before[q] += sums[q][w];
      all[q] += sums[q][w];
    }
  if (tid < experts) {
    int at = before[0] & 0xffff;
    const int full = before[1] & 0xffff, all_full = all[1] & 0xffff;
    for (int i = 0; i < rows / height; ++i) tiles[full + i] = int4{tid, at + i * height, height, 0};
    if (rest > 0) {
      const int place = rest_height == 0 ? full + rows / height : all_full + (rest_height == 1 ? before[1] >> 16 : (all[1] >> 16) + (before[0] >> 16));
      tiles[place] = int4{tid, at + rows - rest, rest, 0};
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      count[w * experts + tid] = at;
      at += counted[w];
    }
  }
  if (tid < 3) n_tiles[tid] = tid == 0 ? all[1] & 0xffff : tid == 1 ? all[1] >> 16 : all[0] >> 16;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i)
    if (place[i] >= 0)
      sorted[count[wave * experts + (unsigned)place[i] % kMaxExperts] + (unsigned)place[i] / kMaxExperts] = (uint16_t)(i * THREADS + tid);
  __syncthreads();
  for (int i = tid; i < (all[0] & 0xffff); i += THREADS) order[i] = sorted[i];
}

size_t plan_smem(int64_t slots, int experts, int threads) { return (size_t)(threads / 64) * experts * sizeof(int) + (size_t)slots * sizeof(uint16_t); }

// out[t] = sum over j of weights[t, j] * y[t * top_k + j], the slots without an expert left out.  Y _Float16: times the row's power
// of two of each 128 channels.  One workgroup per token and 2048 channels, eight a thread.  Bound by memory: 16384 rows of 4096 in fp16 30 us (140 MB
// in, 17 out: 5.2 TB/s).
template <typename Y, typename OutT>
__global__ __launch_bounds__(256) void combine_kernel(const Y* __restrict__ y, const float* __restrict__ y_scale, const int32_t* __restrict__ ids,
                                                      const float* __restrict__ weights, OutT* __restrict__ out, int hidden, int experts,
                                                      int top_k) {
  typedef __attribute__((__vector_size__(8 * sizeof(Y)))) Y vec8;
  const int col = (blockIdx.x * 256 + threadIdx.x) * 8;
  if (col >= hidden) return;
  const int64_t token = blockIdx.y;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int j = 0; j < top_k; ++j) {
    const int64_t slot = token * top_k + j;
    const int e = ids[slot];
    if (e < 0 || e >= experts) continue;
    float w = weights[slot];
    if constexpr (sizeof(Y) == 2) w *= y_scale[slot * (hidden / kBlock) + col / kBlock];
    const vec8 v = *reinterpret_cast<const vec8*>(y + slot * hidden + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] = fmaf(w, (float)v[i], sum[i]);
  }
  store_upto4(out + token * hidden + col, f32x4{sum[0], sum[1], sum[2], sum[3]}, 4);
  store_upto4(out + token * hidden + col + 4, f32x4{sum[4], sum[5], sum[6], sum[7]}, 4);
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

// ---- a few tokens: every slot reads its expert's matrices for itself, without a plan ----------------------------------------
// Bound by the stream of those matrices; the matrix unit's 16 rows are one and the same.  A workgroup has 16 channels (of gate and up),
// its wavefronts share k.  One token, 8 of 64 experts of 4096 x 1408: 32 us, of them 20.5 for the 92 MB of gate and up (4.5 TB/s) and 12.3 for the
// 46 MB of down, where the copy's rate would take 26.6.
constexpr int kDirectUp = 4, kDirectDown = 8;  // wavefronts

// h[slot, n] = SiLU(g) * u in 32 bits, 16 outputs of one slot a workgroup.
template <int NS>
__global__ __launch_bounds__(kDirectUp * 64) void direct_gate_up_kernel(Experts x, float* __restrict__ h, int* __restrict__ flag) {
  __shared__ __attribute__((aligned(16))) f32x4 red[kDirectUp][2][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, kg = lane >> 4;
  const int tiles_n = x.inter / 16;
  const int slot = blockIdx.x / tiles_n, n0 = (blockIdx.x - slot * tiles_n) * 16;
  const int expert = __builtin_amdgcn_readfirstlane(x.ids[slot]);
  if (expert < 0 || expert >= x.experts) {
    if (expert >= 0 && tid == 0) *flag = 1;
    return;
  }
  const int kb = x.hidden / kBlock, mine = (kb - wave + kDirectUp - 1) / kDirectUp;
  const size_t token = slot / x.top_k;
  const uint8_t* xp = x.x + token * x.hidden + wave * kBlock + kg * 16;
  const float* sp = x.x_scale + token * kb + wave;
  const size_t at0 = ((size_t)expert * x.inter + n0 + c) * x.hidden + wave * kBlock + kg * 16;
  const uint8_t* wp[2] = {x.gate + at0, x.up + at0};
  const size_t sat = ((size_t)expert * (x.inter / kBlock) + n0 / kBlock) * kb + wave;
  const float* wsp[2] = {x.gate_scale + sat, x.up_scale + sat};
  struct Held {
    i32x4 w[2][2], a[2];
    float sa, sw[2];
  };
  f32x4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
  auto load = [&](Held& s, int round) {  // past the last step: the first again
    const size_t step = round < mine ? (size_t)round * kDirectUp : 0, at = step * kBlock;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int q = 0; q < 2; ++q) s.w[t][q] = *reinterpret_cast<const i32x4*>(wp[t] + at + q * 64);
      s.sw[t] = wsp[t][step];
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) s.a[q] = *reinterpret_cast<const i32x4*>(xp + at + q * 64);
    s.sa = sp[step];
  };
  auto compute = [&](const Held& s) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const f32x4 part = block_product(s.w[t], s.a);
      const float scale = s.sa * s.sw[t];
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(part[e], scale, acc[t][e]);
    }
  };
  Held st[NS];
  if (mine > 0) {
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) load(st[i], i);
    int r = 0;
    for (; r + NS <= mine; r += NS) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        load(st[(i + NS - 1) % NS], r + i + NS - 1);
        compute(st[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
      if (r + i < mine) compute(st[i]);
  }
#pragma unroll
  for (int t = 0; t < 2; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  if (wave > 0) return;
  f32x4 sum[2] = {red[0][0][lane], red[0][1][lane]};
#pragma unroll
  for (int w = 1; w < kDirectUp; ++w)
#pragma unroll
    for (int t = 0; t < 2; ++t) sum[t] += red[w][t][lane];
  if (c > 0) return;
  f32x4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = silu(sum[0][e]) * sum[1][e];
  *reinterpret_cast<f32x4*>(h + (size_t)slot * x.inter + n0 + 4 * kg) = y;
}

// out[t, n] of 16 channels a workgroup: the token's rows of h are quantised into LDS, their scales times the slots' weights, and all
// its experts' products are one sum over (slot, block of k), shared by the wavefronts in turn.
template <int NS, typename OutT>
__global__ __launch_bounds__(kDirectDown * 64) void direct_down_kernel(Experts x, const float* __restrict__ h) {
  extern __shared__ __attribute__((aligned(16))) uint8_t codes[];  // [top_k][inter], then scales [top_k][inter / 128]
  __shared__ __attribute__((aligned(16))) f32x4 red[kDirectDown][64];
  __shared__ int experts[64], slots[64], count;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, kg = lane >> 4;
  const int tiles_n = x.hidden / 16;
  const int token = blockIdx.x / tiles_n, n0 = (blockIdx.x - token * tiles_n) * 16;
  const int kb = x.inter / kBlock;
  float* const scales = reinterpret_cast<float*>(codes + x.top_k * x.inter);
  if (wave == 0) {  // the slots that have an expert
    const int e = lane < x.top_k ? x.ids[(size_t)token * x.top_k + lane] : -1;
    const bool used = e >= 0 && e < x.experts;
    const uint64_t all = __ballot(used);
    if (used) {
      const int at = __popcll(all & ((1ull << lane) - 1));
      experts[at] = e;
      slots[at] = lane;
    }
    if (lane == 0) count = __popcll(all);
  }
  __syncthreads();
  const int units = count * kb, mine = (units - wave + kDirectDown - 1) / kDirectDown;  // (slot, block) pairs of this wavefront
  struct Held {
    i32x4 w[2];
    float sw;
  };
  auto load = [&](Held& s, int round) {  // past the last unit: the first again
    const int u = (round < mine ? round * kDirectDown : 0) + wave, j = u / kb, b = u - j * kb;
    const size_t expert = experts[j];
    const uint8_t* src = x.down + (expert * x.hidden + n0 + c) * x.inter + b * kBlock + kg * 16;
#pragma unroll
    for (int q = 0; q < 2; ++q) s.w[q] = *reinterpret_cast<const i32x4*>(src + q * 64);
    s.sw = x.down_scale[(expert * (x.hidden / kBlock) + n0 / kBlock) * kb + b];
  };
  // Half a wavefront quantises a group of 128 at a time, four values a lane; a round is kGroups of them, asked for at once.  The first
  // round's values are asked for ahead of the weights: loads come back in order, and the weights are then on their way meanwhile.
  constexpr int kGroups = 6;
  const int half = wave * 2 + (lane >> 5), lane32 = lane & 31;
  float4 v[kGroups];
  float weight[kGroups];
  auto ask = [&](int first) {
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int u = min(first + i * 2 * kDirectDown + half, units - 1), j = u / kb, b = u - j * kb;
      const size_t slot = (size_t)token * x.top_k + slots[j];
      v[i] = *reinterpret_cast<const float4*>(h + slot * x.inter + b * kBlock + 4 * lane32);
      weight[i] = x.weights[slot];
    }
  };
  if (units > 0) ask(0);
  Held st[NS];
  if (mine > 0) {
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) load(st[i], i);
  }
  for (int first = 0; first < units; first += kGroups * 2 * kDirectDown) {
    if (first > 0) ask(first);
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      const int u = first + i * 2 * kDirectDown + half;
      float amax = fmaxf(fmaxf(fabsf(v[i].x), fabsf(v[i].y)), fmaxf(fabsf(v[i].z), fabsf(v[i].w)));
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
      const float s = group_scale(amax);
      const GroupQuotient q(s);
      if (u < units) {  // rows and groups lie one behind the other in units' order
        *reinterpret_cast<uint32_t*>(codes + u * kBlock + 4 * lane32) = codes4(q.near(v[i].x), q.near(v[i].y), q.near(v[i].z), q.near(v[i].w));
        if (lane32 == 0) scales[u] = s * weight[i];
      }
    }
  }
  __syncthreads();
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  auto compute = [&](const Held& s, int round) {
    const int u = round * kDirectDown + wave;
    i32x4 a[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) a[q] = *reinterpret_cast<const i32x4*>(codes + u * kBlock + kg * 16 + q * 64);
    const f32x4 part = block_product(s.w, a);
    const float scale = scales[u] * s.sw;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = fmaf(part[e], scale, acc[e]);
  };
  if (mine > 0) {
    int r = 0;
    for (; r + NS <= mine; r += NS) {
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        load(st[(i + NS - 1) % NS], r + i + NS - 1);
        compute(st[i], r + i);
      }
    }
#pragma unroll
    for (int i = 0; i < NS - 1; ++i)
      if (r + i < mine) compute(st[i], r + i);
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave > 0 || c > 0) return;
  f32x4 sum = red[0][lane];
#pragma unroll
  for (int w = 1; w < kDirectDown; ++w) sum += red[w][lane];
  store_upto4(reinterpret_cast<OutT*>(x.out) + (size_t)token * x.hidden + n0 + 4 * kg, sum, 4);
}

size_t direct_smem(const Experts& x) { return (size_t)x.top_k * x.inter + (size_t)x.top_k * (x.inter / kBlock) * sizeof(float); }
constexpr size_t kDirectSmem = 48 * 1024;  // a token's rows of h as codes

template <typename OutT>
int run_direct(const Experts& x, int64_t tokens, hipStream_t st) {
  const int64_t slots = tokens * x.top_k;
  void* ws = nullptr;
  const int rc = workspace((size_t)slots * x.inter * sizeof(float), &ws);
  if (rc) return rc;
  float* const h = reinterpret_cast<float*>(ws);
  hipLaunchKernelGGL(direct_gate_up_kernel<3>, dim3((unsigned)(slots * (x.inter / 16))), dim3(kDirectUp * 64), 0, st, x, h, ctx().flags + 3);
  hipLaunchKernelGGL((direct_down_kernel<3, OutT>), dim3((unsigned)(tokens * (x.hidden / 16))), dim3(kDirectDown * 64), direct_smem(x), st, x,
                     reinterpret_cast<const float*>(h));
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

// ---- more tokens: the plan, two tiled products, the sum -------------------------------------------------------------------

// Scratch of a pass over `tokens` tokens; y_bytes: of an element of the second product's rows.
struct Scratch {
  size_t order, tiles, n_tiles, h, h_scale, y, y_scale, bytes;
  int max_tiles;
  Scratch(int64_t tokens, const Experts& x, int height, size_t y_bytes) {
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
    n_tiles = take(3 * sizeof(int));
    h = take((size_t)slots * x.inter);
    h_scale = take((size_t)slots * (x.inter / kBlock) * 4);
    y = take((size_t)slots * x.hidden * y_bytes);
    y_scale = take((size_t)slots * (x.hidden / kBlock) * 4);
    bytes = at;
  }
};

template <typename OutT>
int run_pass(const Experts& x, int64_t tokens, const Scratch& s, int height, char* ws, hipStream_t st) {
  // The first product's sums decide codes of h: on the 8-bit matrix instructions, 1.4e-5 off, one in 3000 is another one, which costs a
  // bf16 result a fifth more error (2.0e-3 against 1.7e-3) and an fp16 result five times its own rounding (1.3e-3 against 2.1e-4).  For fp16 the codes
  // are widened; for bf16 that was left out: 2048 tokens, 8 of 64 experts of 4096 x 1408, 674 us for 474, 512 tokens 296 for 263.
  // The second product's only add theirs.  Its rows go through fp16 to a bf16 result, half the bytes, which adds an eighth of that result's
  // own rounding; to an fp16 result it would add as much as that.
  constexpr bool kExactUp = !std::is_same<OutT, __bf16>::value, kExactDown = std::is_same<OutT, float>::value;
  typedef typename std::conditional<kExactUp, float, _Float16>::type Y;
  int32_t* order = reinterpret_cast<int32_t*>(ws + s.order);
  int4* tiles = reinterpret_cast<int4*>(ws + s.tiles);
  int* n_tiles = reinterpret_cast<int*>(ws + s.n_tiles);
  const int slots = (int)(tokens * x.top_k);
  auto plan = [&](auto kern, int threads) {
    hipLaunchKernelGGL(kern, dim3(1), dim3(threads), plan_smem(slots, x.experts, threads), st, x.ids, slots, x.experts, height, order, tiles, n_tiles,
                       ctx().flags + 3);
  };
  if (slots <= kFewSlots && x.experts <= kFewThreads) plan(plan_kernel<kFewSlots / kFewThreads, kFewThreads>, kFewThreads);
  else if (slots <= 8 * kPlanThreads) plan(plan_kernel<8, kPlanThreads>, kPlanThreads);
  else if (slots <= 16 * kPlanThreads) plan(plan_kernel<16, kPlanThreads>, kPlanThreads);
  else plan(plan_kernel<kPassSlots / kPlanThreads, kPlanThreads>, kPlanThreads);
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
  int rc;
  if (height == 64) rc = launch_tiled_experts<kGateUp, 64, kExactUp, uint8_t>(p, s.max_tiles, st);
  else if (height == 128 || kExactUp) rc = launch_tiled_experts<kGateUp, 128, kExactUp, uint8_t>(p, s.max_tiles, st);
  else rc = launch_tiled_experts<kGateUp, kExactUp ? 128 : 256, kExactUp, uint8_t>(p, s.max_tiles, st);
  if (rc) return rc;
  Params d = p;
  d.a = reinterpret_cast<const uint8_t*>(ws + s.h);
  d.sa = reinterpret_cast<const float*>(ws + s.h_scale);
  d.b0 = x.down;
  d.sb0 = x.down_scale;
  d.c = ws + s.y;
  d.c_scale = reinterpret_cast<float*>(ws + s.y_scale);
  d.n = x.hidden;
  d.k = x.inter;
  d.kb = x.inter / kBlock;
  if (height == 64) rc = launch_tiled_experts<kDown, 64, kExactDown, Y>(d, s.max_tiles, st);
  else if (height == 128 || kExactUp) rc = launch_tiled_experts<kDown, 128, kExactDown, Y>(d, s.max_tiles, st);
  else rc = launch_tiled_experts<kDown, kExactUp ? 128 : 256, kExactDown, Y>(d, s.max_tiles, st);
  if (rc) return rc;
  hipLaunchKernelGGL((combine_kernel<Y, OutT>), dim3((unsigned)((x.hidden + 2047) / 2048), (unsigned)tokens), dim3(256), 0, st,
                     reinterpret_cast<const Y*>(ws + s.y), reinterpret_cast<const float*>(ws + s.y_scale), x.ids, x.weights,
                     reinterpret_cast<OutT*>(x.out), x.hidden, x.experts, x.top_k);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

template <typename OutT>
int run_experts(Experts x, int64_t tokens, hipStream_t st) {
  static std::atomic<bool> attr_set{false};  // callers hold the dispatch lock
  if (!attr_set.load(std::memory_order_acquire)) {
    for (const void* kern : {reinterpret_cast<const void*>(plan_kernel<8, kPlanThreads>), reinterpret_cast<const void*>(plan_kernel<16, kPlanThreads>),
                             reinterpret_cast<const void*>(plan_kernel<kPassSlots / kPlanThreads, kPlanThreads>)})
      PTO_CHECK_HIP(hipFuncSetAttribute(kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem(kPassSlots, kMaxExperts, kPlanThreads)));
    attr_set.store(true, std::memory_order_release);
  }
  constexpr bool kExactUp = !std::is_same<OutT, __bf16>::value, kExactDown = std::is_same<OutT, float>::value;
  int height = (int)ctx().block_gemm_rows;
  const int64_t slots = tokens * x.top_k;
  const bool direct = height == 0 ? experts_direct(slots, x.experts, x.hidden, x.inter, kExactUp) : height == 16;
  if (direct && slots <= kMostDirectSlots && direct_smem(x) <= kDirectSmem) return run_direct<OutT>(x, tokens, st);
  const int64_t pass = expert_pass_tokens(tokens, x.top_k, x.hidden, x.inter, kExactUp ? 4 : 2);
  if (height < 64) height = choose_expert_rows(pass * x.top_k, x.experts, x.hidden, x.inter, kExactUp, kExactDown, ctx().num_cu);
  if (kExactUp) height = std::min(height, 128);
  const Scratch s(pass, x, height, kExactUp ? 4 : 2);
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
  {
    const int64_t hb = hidden / block8::kBlock, ib = intermediate / block8::kBlock, matrix = experts * hidden * intermediate;
    const struct {
      const void* at;
      int64_t bytes;
    } operands[] = {{x8, tokens * hidden}, {x_scale, tokens * hb * 4}, {expert_ids, tokens * top_k * 4}, {expert_weights, tokens * top_k * 4},
                    {w_gate8, matrix}, {w_up8, matrix}, {w_down8, matrix}, {w_gate_scale, experts * hb * ib * 4}, {w_up_scale, experts * hb * ib * 4},
                    {w_down_scale, experts * hb * ib * 4}};
    for (const auto& o : operands)
      PTO_CHECK_ARG(!block8::overlap(out, tokens * hidden * dtype_bytes(out_dtype), o.at, o.bytes), "experts_ffn_fp8_block: out overlaps an operand");
  }
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
