// Several new tokens per sequence: norm of every query and key head, rotation, and the rows' way into the paged cache.
//
//   q' = rope(q / sqrt(mean q^2 + eps) * gamma_q)    k' = rope(k / sqrt(mean k^2 + eps) * gamma_k)    v' = v
//   rope: y_i = x_i cos_i - x_{i+R/2} sin_i,  y_{i+R/2} = x_{i+R/2} cos_i + x_i sin_i  for i < R/2, the rest as it is
//
// at positions[t]; token i of sequence b goes to cache row (block_table[b][n / bs] * Hkv + h) * bs + n % bs with n = context_lens[b] + i.
// The form for one token per sequence is rope.hip's (examples/models/qwen3_jit/kernels/attention.py:39-102).
//
// Every row is read once and written once, eight elements a lane; a pair's other element comes from another lane.  Large batches are bound by memory: 12000 tokens of 40 + 16
// fp16 heads of 128 take 69 us, 350 MB at 5.1 TB/s, what a large copy reaches.  Small ones are bound by their chain of loads - the token's sequence, its length, its block, and
// the row's angles beside them -: one token of 32 + 16 heads 3.4 us, 408 tokens 6.2 us.  Over e4m3 caches a block's scale has to be known before its rows are coded: a workgroup takes
// all new rows of a (block, head) and reads them twice (385 tokens of 64 + 16 heads 11 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_fp8.h"
#include "common.h"
#include "token_seq.h"

namespace {

using pto_hip::in_launches;
using pto_hip::TokenSeq;

constexpr int kThreads = 256;
constexpr int64_t kMaxTokens = 1 << 20;
constexpr float kE4m3Max = 448.f;
// A workgroup takes one group of heads of a token (256 / lanes a head), or four where there are this many groups a CU: 12000 tokens of 56 heads are 97 us by one
// and 69 us by four (the row's angles and places are looked up once, four loads are on their way at once), 408 tokens of 40 heads 6.2 us and 7.1 us.
constexpr int kManyGroups = 16;

struct Params {
  const void* qkv;  // [T, (Hq + 2 Hkv) D]
  const int32_t* positions;
  const int32_t* starts;  // [B + 1]
  const int32_t* ctx_lens;
  const float* cos;  // [max_pos, rope_w]
  const float* sin;
  const float* gamma_q;
  const float* gamma_k;
  const int32_t* block_table;
  void* key_cache;
  void* value_cache;
  float* k_scale;
  float* v_scale;
  void* q_out;
  int t0;  // the launch's first token
  int tokens, batch, hq, hkv, d, bs, max_blocks, max_pos, pool_blocks;
  int rope_w;     // columns of the tables
  int rope_half;  // R / 2
  float eps;
  int* error_flag;
};

// Eight consecutive elements of a row as they lie in memory, and as fp32.
template <typename T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) * 8 / 4;
  uint32_t w[kWords];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {  // 16-byte aligned
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < Raw8<T>::kWords / 4; ++i) {
    const uint4 v = reinterpret_cast<const uint4*>(p)[i];
    r.w[4 * i] = v.x;
    r.w[4 * i + 1] = v.y;
    r.w[4 * i + 2] = v.z;
    r.w[4 * i + 3] = v.w;
  }
  return r;
}
template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T>& r, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (sizeof(T) == 4) {
      x[i] = __builtin_bit_cast(float, r.w[i]);
    } else if constexpr (std::is_same<T, __bf16>::value) {
      x[i] = __builtin_bit_cast(float, i & 1 ? r.w[i / 2] & 0xffff0000u : r.w[i / 2] << 16);
    } else {
      x[i] = (float)__builtin_bit_cast(_Float16, (uint16_t)(r.w[i / 2] >> (i & 1 ? 16 : 0)));
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&y)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = (uint32_t)__builtin_bit_cast(uint16_t, (T)y[2 * i]) | (uint32_t)__builtin_bit_cast(uint16_t, (T)y[2 * i + 1]) << 16;
  *reinterpret_cast<uint4*>(p) = uint4{w[0], w[1], w[2], w[3]};
}
__device__ __forceinline__ void load_f8(const float* p, float (&x)[8]) {  // any alignment of a float
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[i];
}

// The cosines and sines of a lane's eight elements.
struct Angles {
  float c[8], s[8];
};
__device__ __forceinline__ Angles load_angles(const Params& p, int pos, int e0) {
  Angles a{};
  if (e0 < 2 * p.rope_half) {
    // a table of one angle a pair is read at the pair's number, the reference's tables at the element's own
    const size_t at = (size_t)pos * p.rope_w + (p.rope_w == p.d || e0 < p.rope_half ? e0 : e0 - p.rope_half);
    load_f8(p.cos + at, a.c);
    load_f8(p.sin + at, a.s);
  }
  return a;
}

// Norm and rotation of one head's row by the LANES lanes that hold it, eight elements each (lanes past the row hold none): y = what
// becomes of the lane's own.  All lanes of the group take part.
template <typename In, int LANES>
__device__ __forceinline__ void turn_row(const Params& p, const Raw8<In>& raw, const float* gamma, const Angles& angles, bool turn, int e0, float (&y)[8]) {
  widen8(raw, y);
  if (!turn) return;  // a value's row
  const bool inside = e0 < p.d;
  const int half = p.rope_half;
  // the other element of each rotated pair lies `half` away, in another lane
  const bool low = e0 < half, turned = e0 < 2 * half;
  const int other_e = turned ? (low ? e0 + half : e0 - half) : e0;
  const int other_lane = other_e / 8;
  Raw8<In> other_raw;
#pragma unroll
  for (int i = 0; i < Raw8<In>::kWords; ++i) other_raw.w[i] = (uint32_t)__shfl((int)raw.w[i], other_lane, LANES);
  float x[8];
  widen8(other_raw, x);
  if (gamma) {
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum = fmaf(y[i], y[i], sum);
    sum = inside ? sum : 0.f;
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) sum += __shfl_xor(sum, off, LANES);
    const float r = 1.f / sqrtf(sum / (float)p.d + p.eps);
    if (inside) {
      float g[8];
      load_f8(gamma + e0, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = y[i] * r * g[i];
      load_f8(gamma + other_e, g);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = x[i] * r * g[i];
    }
  }
  if (inside && turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = low ? y[i] * angles.c[i] - x[i] * angles.s[i] : y[i] * angles.c[i] + x[i] * angles.s[i];
  }
}

// Where a token's row lies in the cache: the physical block and the place in it.  False, and reported, where there is none.
__device__ __forceinline__ bool cache_place(const Params& p, int seq, int number, int* block, int* place) {
  const int64_t n = (int64_t)p.ctx_lens[seq] + number;
  bool ok = n >= 0 && n / p.bs < p.max_blocks;
  if (ok) {
    *block = p.block_table[(size_t)seq * p.max_blocks + n / p.bs];
    *place = (int)(n % p.bs);
    ok = (unsigned)*block < (unsigned)p.pool_blocks;
  }
  if (!ok) *p.error_flag = 1;
  return ok;
}

// By the first workgroup of the launch with the queries' heads.
__device__ __forceinline__ void report_starts(const Params& p, int part) {
  if (p.t0 + blockIdx.x == 0 && part == 0 && threadIdx.x == 0 && pto_hip::pass_the_rows(p.starts, p.batch, p.tokens)) *p.error_flag = 1;
}

// A workgroup for GROUPS times kThreads / LANES heads of one token, LANES lanes a head, number `part` of the token.  Q_ONLY: the queries alone (beside an e4m3 cache).
template <typename In, typename T, int LANES, bool Q_ONLY, int GROUPS>
__device__ __forceinline__ void append_heads(const Params& p, int part) {
  constexpr int kHeads = kThreads / LANES;
  const int t = p.t0 + blockIdx.x, lane = threadIdx.x % 64;
  const int head0 = part * (GROUPS * kHeads) + threadIdx.x / LANES;
  const int heads = Q_ONLY ? p.hq : p.hq + 2 * p.hkv;
  const int e0 = threadIdx.x % LANES * 8;
  const int width = p.hq + 2 * p.hkv;
  Raw8<In> raw[GROUPS] = {};
#pragma unroll
  for (int g = 0; g < GROUPS; ++g)
    if (e0 < p.d && head0 + g * kHeads < heads) raw[g] = load8(reinterpret_cast<const In*>(p.qkv) + ((size_t)t * width + head0 + g * kHeads) * p.d + e0);
  const int pos = p.positions[t];
  const TokenSeq s = pto_hip::sequence_of(p.starts, p.batch, p.tokens, t, lane);
  report_starts(p, part);
  if (s.seq < 0) return;  // nobody's token
  if (pos < 0 || pos >= p.max_pos) {
    if (threadIdx.x == 0) *p.error_flag = 1;
    return;
  }
  const Angles angles = load_angles(p, pos, e0);
  int block = 0, place = 0;
  if (!cache_place(p, s.seq, t - s.first, &block, &place)) return;
#pragma unroll
  for (int g = 0; g < GROUPS; ++g) {
    const int head = head0 + g * kHeads;
    const bool is_q = head < p.hq, is_k = !is_q && head < p.hq + p.hkv;
    float y[8];
    turn_row<In, LANES>(p, raw[g], is_q ? p.gamma_q : p.gamma_k, angles, is_q || is_k, e0, y);
    if (e0 >= p.d || head >= heads) continue;
    T* dst;
    if (is_q) {
      dst = reinterpret_cast<T*>(p.q_out) + ((size_t)t * p.hq + head) * p.d;
    } else {
      const int h = head - p.hq - (is_k ? 0 : p.hkv);
      dst = reinterpret_cast<T*>(is_k ? p.key_cache : p.value_cache) + (((size_t)block * p.hkv + h) * p.bs + place) * p.d;
    }
    store8(dst + e0, y);
  }
}

template <typename In, typename T, int LANES, int GROUPS>
__global__ __launch_bounds__(kThreads) void append_kernel(Params p) {
  append_heads<In, T, LANES, false, GROUPS>(p, blockIdx.y);
}

// Any even head_dim and any tables: one wavefront a head, pair by pair.
template <typename In, typename T>
__global__ __launch_bounds__(64) void append_any_kernel(Params p) {
  const int t = p.t0 + blockIdx.x, head = blockIdx.y, lane = threadIdx.x;
  const int pos = p.positions[t];
  const TokenSeq s = pto_hip::sequence_of(p.starts, p.batch, p.tokens, t, lane);
  report_starts(p, head);
  if (s.seq < 0) return;
  if (pos < 0 || pos >= p.max_pos) {
    if (lane == 0) *p.error_flag = 1;
    return;
  }
  int block = 0, place = 0;
  if (!cache_place(p, s.seq, t - s.first, &block, &place)) return;
  const bool is_q = head < p.hq, is_k = !is_q && head < p.hq + p.hkv;
  const In* src = reinterpret_cast<const In*>(p.qkv) + ((size_t)t * (p.hq + 2 * p.hkv) + head) * p.d;
  T* dst;
  if (is_q) {
    dst = reinterpret_cast<T*>(p.q_out) + ((size_t)t * p.hq + head) * p.d;
  } else {
    const int h = head - p.hq - (is_k ? 0 : p.hkv);
    dst = reinterpret_cast<T*>(is_k ? p.key_cache : p.value_cache) + (((size_t)block * p.hkv + h) * p.bs + place) * p.d;
  }
  const float* gamma = is_q ? p.gamma_q : is_k ? p.gamma_k : nullptr;
  float r = 1.f;
  if (gamma) {
    float sum = 0.f;
    for (int i = lane; i < p.d; i += 64) sum = fmaf((float)src[i], (float)src[i], sum);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    r = 1.f / sqrtf(sum / (float)p.d + p.eps);
  }
  auto value = [&](int i) { return gamma ? (float)src[i] * r * gamma[i] : (float)src[i]; };
  const int half = is_q || is_k ? p.rope_half : 0;
  for (int i = lane; i < half; i += 64) {
    const size_t lo = (size_t)pos * p.rope_w + i, hi = p.rope_w == p.d ? lo + half : lo;
    const float a = value(i), b = value(i + half);
    dst[i] = (T)(a * p.cos[lo] - b * p.sin[lo]);
    dst[i + half] = (T)(b * p.cos[hi] + a * p.sin[hi]);
  }
  for (int i = 2 * half + lane; i < p.d; i += 64) dst[i] = (T)value(i);
}

// ---- e4m3 caches ----
__device__ __forceinline__ float saturate(float v) { return v != v ? v : fminf(fmaxf(v, -kE4m3Max), kE4m3Max); }
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d) {
  return pto_hip::block8::codes4(saturate(a), saturate(b), saturate(c), saturate(d));
}
__device__ __forceinline__ float code_value(uint32_t word, int byte) {
  switch (byte) {
    case 0: return __builtin_amdgcn_cvt_f32_fp8(word, 0);
    case 1: return __builtin_amdgcn_cvt_f32_fp8(word, 1);
    case 2: return __builtin_amdgcn_cvt_f32_fp8(word, 2);
    default: return __builtin_amdgcn_cvt_f32_fp8(word, 3);
  }
}

__device__ __forceinline__ float times(float v, double by) { return (float)((double)v * by); }

// The new rows of one block and KV head, keys or values, by one workgroup: that of the block's first new token.  Their maximum first, then their codes,
// from the rows read again; the rows in front are coded again where the scale grows.
template <typename In, int LANES>
__device__ __forceinline__ void append_codes(const Params& p, int kv_head) {
  __shared__ float wave_most[kThreads / 64];
  const int t = p.t0 + blockIdx.x, lane = threadIdx.x % 64;
  const bool is_k = kv_head < p.hkv;
  const int h = is_k ? kv_head : kv_head - p.hkv;
  const TokenSeq s = pto_hip::sequence_of(p.starts, p.batch, p.tokens, t, lane);
  if (s.seq < 0) return;
  int block = 0, place = 0;
  {
    // every new token of a block that the table does not have reports it; only the first of the others has work
    const int64_t n = (int64_t)p.ctx_lens[s.seq] + (t - s.first);
    if (n >= 0 && t > s.first && n % p.bs != 0) return;
  }
  if (!cache_place(p, s.seq, t - s.first, &block, &place)) return;
  const int rows = min(s.count - (t - s.first), p.bs - place);
  const int head = p.hq + (is_k ? 0 : p.hkv) + h, width = p.hq + 2 * p.hkv;
  const int group = threadIdx.x / LANES, e0 = threadIdx.x % LANES * 8;
  const bool inside = e0 < p.d;
  auto row = [&](int r, float (&y)[8]) -> bool {  // false: a token that is left out
    const int token = t + min(r, rows - 1);
    Raw8<In> raw{};
    if (inside) raw = load8(reinterpret_cast<const In*>(p.qkv) + ((size_t)token * width + head) * p.d + e0);
    const int pos = p.positions[token];
    const bool ok = r < rows && pos >= 0 && pos < p.max_pos;
    if (r < rows && !ok) *p.error_flag = 1;
    turn_row<In, LANES>(p, raw, p.gamma_k, is_k ? load_angles(p, ok ? pos : 0, e0) : Angles{}, is_k, e0, y);
    return ok;
  };
  constexpr int kGroups = kThreads / LANES;
  float most = 0.f;
  for (int r = group; r - group < rows; r += kGroups) {
    float y[8];
    if (row(r, y) && inside) {
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, pto_hip::block8::finite_size(y[i]));
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off));
  if (lane == 0) wave_most[threadIdx.x / 64] = most;
  __syncthreads();
  most = wave_most[0];
#pragma unroll
  for (int w = 1; w < kThreads / 64; ++w) most = fmaxf(most, wave_most[w]);

  uint8_t* base = reinterpret_cast<uint8_t*>(is_k ? p.key_cache : p.value_cache) + ((size_t)block * p.hkv + h) * p.bs * p.d;
  float* slot = (is_k ? p.k_scale : p.v_scale) + (size_t)block * p.hkv + h;
  const float before = *slot;
  float scale = pto_hip::block8::group_scale(most);
  // Quotients are taken by the exact scale, most / 448, in 64 bits: a 16-bit value is often a tie between two codes, which the rounded scale would push to either
  // side, and never so near one that 2^-52 matters.
  double inverse = scale == 1.f || scale == 0x1p-126f ? 1.0 / (double)scale : (double)kE4m3Max / (double)most;
  if (place > 0) {
    scale = fmaxf(before, most / kE4m3Max);
    if (!(scale > before)) {
      inverse = scale > 0.f ? 1.0 / (double)scale : 0.0;
    } else {
      inverse = (double)kE4m3Max / (double)most;
      const double ratio = (double)before * inverse;
      uint32_t* words = reinterpret_cast<uint32_t*>(base);
      for (size_t w = threadIdx.x; w < (size_t)place * p.d / 4; w += kThreads) {
        const uint32_t c = words[w];
        words[w] = codes4(times(code_value(c, 0), ratio), times(code_value(c, 1), ratio), times(code_value(c, 2), ratio),
                          times(code_value(c, 3), ratio));
      }
    }
  }
  for (int r = group; r - group < rows; r += kGroups) {
    float y[8];
    if (row(r, y) && inside) {
      uint32_t* dst = reinterpret_cast<uint32_t*>(base + (size_t)(place + r) * p.d + e0);
      dst[0] = codes4(times(y[0], inverse), times(y[1], inverse), times(y[2], inverse), times(y[3], inverse));
      dst[1] = codes4(times(y[4], inverse), times(y[5], inverse), times(y[6], inverse), times(y[7], inverse));
    }
  }
  __syncthreads();  // everybody has read the scale of before
  if (threadIdx.x == 0) *slot = scale;
}

// Workgroups for both: a token's key and value heads, which take longest, then its queries.
template <typename In, typename T, int LANES, int GROUPS>
__global__ __launch_bounds__(kThreads) void append_fp8_kernel(Params p) {
  if ((int)blockIdx.y < 2 * p.hkv) append_codes<In, LANES>(p, blockIdx.y);
  else append_heads<In, T, LANES, true, GROUPS>(p, blockIdx.y - 2 * p.hkv);
}

template <int N>
using Lanes = pto_hip::block8::IntConst<N>;
// f(lanes) with the number of lanes that hold a row of d elements, eight each.
template <typename F>
void with_lanes(int d, F f) {
  if (d <= 64) f(Lanes<8>{});
  else if (d <= 128) f(Lanes<16>{});
  else if (d <= 256) f(Lanes<32>{});
  else f(Lanes<64>{});
}

template <typename In, typename T>
void launch(Params& p, bool fp8, bool wide, hipStream_t st) {
  const int heads = p.hq + 2 * p.hkv;
  if (!wide) {
    in_launches(p, 64 * heads, [&](unsigned n) { hipLaunchKernelGGL((append_any_kernel<In, T>), dim3(n, heads), dim3(64), 0, st, p); });
    return;
  }
  with_lanes(p.d, [&](auto lanes) {
    constexpr int L = decltype(lanes)::value, kHeads = kThreads / L;
    const int groups = ((fp8 ? p.hq : heads) + kHeads - 1) / kHeads;
    auto of = [&](auto per) {
      constexpr int G = decltype(per)::value;
      const int y = (groups + G - 1) / G + (fp8 ? 2 * p.hkv : 0);
      in_launches(p, (int64_t)kThreads * y, [&](unsigned n) {
        if (fp8) hipLaunchKernelGGL((append_fp8_kernel<In, T, L, G>), dim3(n, y), dim3(kThreads), 0, st, p);
        else hipLaunchKernelGGL((append_kernel<In, T, L, G>), dim3(n, y), dim3(kThreads), 0, st, p);
      });
    };
    if ((int64_t)p.tokens * groups >= kManyGroups * pto_hip::ctx().num_cu) of(Lanes<4>{});
    else of(Lanes<1>{});
  });
}

}  // namespace

extern "C" int pto_hip_rope_append_tokens(const PtoHipRopeAppendArgs* args, void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  PTO_CHECK_ARG(args != nullptr, "rope_append_tokens: null arguments");
  const PtoHipRopeAppendArgs& a = *args;
  const bool fp8 = a.kv_dtype == PTO_HIP_FP8E4M3FN;
  PTO_CHECK_ARG(a.tokens >= 0 && a.batch >= 0, "rope_append_tokens: negative extent");
  PTO_CHECK_ARG(a.num_heads > 0 && a.kv_head_num > 0 && a.num_heads + 2 * a.kv_head_num < 65536, "rope_append_tokens: bad head counts %lld / %lld",
                (long long)a.num_heads, (long long)a.kv_head_num);
  PTO_CHECK_ARG(a.head_dim > 0 && a.head_dim % 2 == 0 && a.head_dim <= 65536, "rope_append_tokens: head_dim %lld must be even, at most 65536",
                (long long)a.head_dim);
  PTO_CHECK_ARG(a.dtype == PTO_HIP_BF16 || a.dtype == PTO_HIP_FP16, "rope_append_tokens: cache/query dtype %s not in {BF16, FP16}", dtype_name(a.dtype));
  PTO_CHECK_ARG(a.kv_dtype == 0 || a.kv_dtype == a.dtype || fp8, "rope_append_tokens: caches of %s beside queries of %s", dtype_name(a.kv_dtype),
                dtype_name(a.dtype));
  PTO_CHECK_ARG(a.qkv_dtype == PTO_HIP_FP32 || a.qkv_dtype == PTO_HIP_BF16 || a.qkv_dtype == PTO_HIP_FP16,
                "rope_append_tokens: qkv dtype %s not in {FP32, BF16, FP16}", dtype_name(a.qkv_dtype));
  PTO_CHECK_ARG((a.gamma_q == nullptr) == (a.gamma_k == nullptr), "rope_append_tokens: gamma_q and gamma_k come together");
  const int64_t width = a.rope_table_width == 0 ? a.head_dim / 2 : a.rope_table_width;
  PTO_CHECK_ARG(width > 0 && (width <= a.head_dim / 2 || width == a.head_dim),
                "rope_append_tokens: rope tables must be [max_pos, at most %lld] or [max_pos, %lld], got width %lld", (long long)a.head_dim / 2,
                (long long)a.head_dim, (long long)width);
  const int64_t half = width == a.head_dim ? a.head_dim / 2 : width;
  PTO_CHECK_ARG(a.block_size > 0 && a.max_num_blocks_per_req > 0 && a.max_pos > 0 && a.pool_blocks > 0, "rope_append_tokens: non-positive extent");
  PTO_CHECK_ARG(a.block_size < 1ll << 31 && a.max_num_blocks_per_req < 1ll << 31 && a.max_pos < 1ll << 31 && a.pool_blocks < 1ll << 31 &&
                    a.batch < 1ll << 30,
                "rope_append_tokens: extent beyond 2^31");
  const bool eights = a.head_dim % 8 == 0 && half % 8 == 0 && a.head_dim <= 512;
  if (fp8 && !eights)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "rope_append_tokens: FP8E4M3FN caches need a head_dim of a multiple of 8, at most 512, with rope tables of a "
                "multiple of 8 angles, got %lld and %lld", (long long)a.head_dim, (long long)half);
  if (a.tokens > kMaxTokens)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "rope_append_tokens: at most %lld tokens, got %lld", (long long)kMaxTokens, (long long)a.tokens);
  if (a.tokens == 0 || a.batch == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(a.qkv && a.positions && a.token_starts && a.context_lens && a.rope_cos && a.rope_sin && a.block_table && a.key_cache &&
                    a.value_cache && a.q_out && (!fp8 || (a.k_scale && a.v_scale)),
                "rope_append_tokens: null tensor pointer");
  const int esz = dtype_bytes(a.dtype), in_esz = dtype_bytes(a.qkv_dtype);
  PTO_CHECK_ARG(((uintptr_t)a.positions | (uintptr_t)a.token_starts | (uintptr_t)a.context_lens | (uintptr_t)a.rope_cos | (uintptr_t)a.rope_sin |
                 (uintptr_t)a.gamma_q | (uintptr_t)a.gamma_k | (uintptr_t)a.block_table | (uintptr_t)a.k_scale | (uintptr_t)a.v_scale) % 4 == 0 &&
                    (uintptr_t)a.qkv % in_esz == 0 && (uintptr_t)a.q_out % esz == 0 &&
                    ((uintptr_t)a.key_cache | (uintptr_t)a.value_cache) % (fp8 ? 8 : esz) == 0,
                "rope_append_tokens: misaligned operand");
  const bool aligned = (uintptr_t)a.qkv % 16 == 0 && (uintptr_t)a.q_out % 16 == 0 && (fp8 || ((uintptr_t)a.key_cache | (uintptr_t)a.value_cache) % 16 == 0);
  PTO_CHECK_ARG(aligned || !fp8, "rope_append_tokens: qkv and q_out beside FP8E4M3FN caches must start at multiples of 16 bytes");
  {
    using block8::overlap;
    const int64_t heads = a.num_heads + 2 * a.kv_head_num, rows = a.pool_blocks * a.kv_head_num * a.block_size;
    const int64_t scales = a.pool_blocks * a.kv_head_num * 4, table = a.max_pos * width * 4;
    struct Span { const void* at; int64_t bytes; };
    const Span outs[5] = {{a.q_out, a.tokens * a.num_heads * a.head_dim * esz},
                          {a.key_cache, rows * a.head_dim * (fp8 ? 1 : esz)},
                          {a.value_cache, rows * a.head_dim * (fp8 ? 1 : esz)},
                          {fp8 ? a.k_scale : nullptr, scales},
                          {fp8 ? a.v_scale : nullptr, scales}};
    const Span ins[9] = {{a.qkv, a.tokens * heads * a.head_dim * in_esz}, {a.positions, a.tokens * 4}, {a.token_starts, (a.batch + 1) * 4},
                         {a.context_lens, a.batch * 4}, {a.rope_cos, table}, {a.rope_sin, table}, {a.gamma_q, a.head_dim * 4},
                         {a.gamma_k, a.head_dim * 4}, {a.block_table, a.batch * a.max_num_blocks_per_req * 4}};
    for (int i = 0; i < 5; ++i) {
      for (const Span& in : ins) PTO_CHECK_ARG(!overlap(outs[i].at, outs[i].bytes, in.at, in.bytes), "rope_append_tokens: an output overlaps an input");
      for (int j = 0; j < i; ++j)
        PTO_CHECK_ARG(!overlap(outs[i].at, outs[i].bytes, outs[j].at, outs[j].bytes), "rope_append_tokens: two outputs overlap");
    }
  }
  Params p{};
  p.qkv = a.qkv;
  p.positions = a.positions;
  p.starts = a.token_starts;
  p.ctx_lens = a.context_lens;
  p.cos = a.rope_cos;
  p.sin = a.rope_sin;
  p.gamma_q = a.gamma_q;
  p.gamma_k = a.gamma_k;
  p.block_table = a.block_table;
  p.key_cache = a.key_cache;
  p.value_cache = a.value_cache;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.q_out = a.q_out;
  p.tokens = (int)a.tokens;
  p.batch = (int)a.batch;
  p.hq = (int)a.num_heads;
  p.hkv = (int)a.kv_head_num;
  p.d = (int)a.head_dim;
  p.bs = (int)a.block_size;
  p.max_blocks = (int)a.max_num_blocks_per_req;
  p.max_pos = (int)a.max_pos;
  p.pool_blocks = (int)a.pool_blocks;
  p.rope_w = (int)width;
  p.rope_half = (int)half;
  p.eps = a.eps;
  p.error_flag = ctx().flags + 4;
  const DeviceScope scope(ctx().device);
  hipStream_t st = (hipStream_t)stream;
  const bool wide = eights && aligned;
  auto with_out = [&](auto in) {
    typedef decltype(in) In;
    if (a.dtype == PTO_HIP_BF16) launch<In, __bf16>(p, fp8, wide, st);
    else launch<In, _Float16>(p, fp8, wide, st);
  };
  if (a.qkv_dtype == PTO_HIP_FP32) with_out(float{});
  else if (a.qkv_dtype == PTO_HIP_BF16) with_out(__bf16{});
  else with_out(_Float16{});
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
