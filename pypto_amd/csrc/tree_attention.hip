// Attention of several new tokens per sequence over a paged cache and over each other, by a mask: a step that verifies drafted tokens.
//
//   out[t, h] = sum_n p_n v_n / sum_n p_n,   p_n = exp(scale q k_n - max),   n over the keys that row t sees:
//   n < context_lens[b], and n = context_lens[b] + j for the new tokens j of its sequence whose bit is set in tree_mask[t]
//
// The form for one token per sequence is paged_attention.hip's (examples/models/04_paged_attention.py:62-227).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_fp8.h"
#include "common.h"
#include "token_seq.h"

namespace {

using pto_hip::TokenSeq;

constexpr int64_t kMaxTokens = 1 << 20;
constexpr int kMaxWords = 32;
constexpr int kMaxD = 256;

struct Params {
  const void* q;  // [T, Hq, D]
  const void* kc;
  const void* vc;
  const float* k_scale;  // [pool_blocks, Hkv] with an e4m3 cache
  const float* v_scale;
  const int32_t* block_table;
  const int32_t* ctx_lens;
  const int32_t* starts;  // [B + 1]
  const uint32_t* mask;   // [T, words]
  void* out;
  int t0;  // the launch's first token
  int tokens, batch, hq, hkv, group, d, bs, max_blocks, pool_blocks, words;
  float scale;
  int* error_flag;
};

// element i of a row of the cache or the query, as fp32
template <typename E>
__device__ __forceinline__ float elem(const void* base, size_t i) {
  if constexpr (std::is_same<E, uint8_t>::value) return __builtin_amdgcn_cvt_f32_fp8((int)reinterpret_cast<const uint8_t*>(base)[i], 0);
  else return (float)reinterpret_cast<const E*>(base)[i];
}

// The keys of a sequence: those in the cache, those that its tokens see at most, and whether lengths or tables are not as they should be.
struct KeyRange {
  int ctx, end;
  bool bad;
};
__device__ __forceinline__ KeyRange key_range(const Params& p, const TokenSeq& s) {
  const int64_t room = (int64_t)p.max_blocks * p.bs;
  const int64_t ctx = p.ctx_lens[s.seq];
  const int64_t seen = min(s.count, 32 * p.words);
  const int64_t from = min(max(ctx, (int64_t)0), room), to = min(from + seen, room);
  return KeyRange{(int)from, (int)to, ctx < 0 || ctx + s.count > room || s.count > 32 * p.words};
}

// Any shape: one wavefront for each query head of a token.  64 keys at a time, a lane each for the scores, a lane per channel for the values.
template <typename T, typename E>
__global__ __launch_bounds__(64) void tree_any_kernel(Params p) {
  __shared__ float qs[kMaxD];
  const int t = p.t0 + blockIdx.x, hq = blockIdx.y, h = hq / p.group, lane = threadIdx.x;
  const int d = p.d, bs = p.bs;
  const TokenSeq s = pto_hip::sequence_of(p.starts, p.batch, t, lane);
  if (s.seq < 0) return;
  const size_t row = (size_t)t * p.hq + hq;
  for (int i = lane; i < d; i += 64) qs[i] = (float)reinterpret_cast<const T*>(p.q)[row * d + i] * p.scale;
  __syncthreads();
  const KeyRange keys = key_range(p, s);
  bool bad = keys.bad;
  float o[kMaxD / 64] = {0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  for (int n0 = 0; n0 < keys.end; n0 += 64) {
    const int n = n0 + lane, j = n - keys.ctx;
    const bool sees = n < keys.end && (j < 0 || (p.mask[(size_t)t * p.words + j / 32] >> (j % 32) & 1));
    int block = n < keys.end ? p.block_table[(size_t)s.seq * p.max_blocks + n / bs] : 0;
    if ((unsigned)block >= (unsigned)p.pool_blocks) {
      bad = true;
      block = 0;
    }
    const size_t at = ((size_t)block * p.hkv + h) * bs + n % bs;
    float ks = 1.f, vs = 1.f, score = -INFINITY;
    if constexpr (std::is_same<E, uint8_t>::value) {
      ks = p.k_scale[(size_t)block * p.hkv + h];
      vs = p.v_scale[(size_t)block * p.hkv + h];
    }
    if (sees) {
      float sum = 0.f;
      for (int i = 0; i < d; ++i) sum = fmaf(qs[i], elem<E>(p.kc, at * d + i), sum);
      score = sum * ks;
    }
    float most = score;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off));
    const float m_new = fmaxf(m, most);
    if (m_new == -INFINITY && __ballot(sees) == 0) continue;  // nobody of these is seen
    const float keep = m == m_new ? 1.f : expf(m - m_new);
    m = m_new;
    const float prob = sees ? (score == m ? 1.f : expf(score - m)) : 0.f;
    float sum = prob;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
    l = l * keep + sum;
#pragma unroll
    for (int u = 0; u < kMaxD / 64; ++u) o[u] *= keep;
    for (uint64_t left = __ballot(sees); left; left &= left - 1) {  // keys that are not seen have no part, whatever they hold
      const int from = __builtin_ctzll(left);
      const float pn = __shfl(prob, from) * __shfl(vs, from);
      const size_t vrow = (size_t)__shfl((unsigned long long)at, from);
#pragma unroll
      for (int u = 0; u < kMaxD / 64; ++u)
        if (lane + 64 * u < d) o[u] = fmaf(pn, elem<E>(p.vc, vrow * d + lane + 64 * u), o[u]);
    }
  }
  if (bad) *p.error_flag = 1;
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
  for (int u = 0; u < kMaxD / 64; ++u)
    if (lane + 64 * u < d) reinterpret_cast<T*>(p.out)[row * d + lane + 64 * u] = (T)(o[u] * inv);
}

template <typename T, typename E>
void launch_any(Params& p, hipStream_t st) {
  const int64_t most = std::max<int64_t>(1, (1ll << 31) / (64 * p.hq));  // a launch holds fewer than 2^32 threads
  for (int64_t t = 0; t < p.tokens; t += most) {
    p.t0 = (int)t;
    hipLaunchKernelGGL((tree_any_kernel<T, E>), dim3((unsigned)std::min<int64_t>(most, p.tokens - t), p.hq), dim3(64), 0, st, p);
  }
}

}  // namespace

extern "C" int pto_hip_tree_attention(const PtoHipTreeAttentionArgs* args, void* stream) {
  PTO_DISPATCH_LOCK();
  using namespace pto_hip;
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  PTO_CHECK_ARG(args != nullptr, "tree_attention: null arguments");
  const PtoHipTreeAttentionArgs& a = *args;
  const bool fp8 = a.kv_dtype == PTO_HIP_FP8E4M3FN;
  PTO_CHECK_ARG(a.tokens >= 0 && a.batch >= 0, "tree_attention: negative extent");
  PTO_CHECK_ARG(a.num_heads > 0 && a.kv_head_num > 0 && a.num_heads < 65536 && a.num_heads % a.kv_head_num == 0,
                "tree_attention: %lld query heads do not divide over %lld KV heads", (long long)a.num_heads, (long long)a.kv_head_num);
  PTO_CHECK_ARG(a.head_dim > 0 && a.block_size > 0 && a.max_num_blocks_per_req > 0 && a.pool_blocks > 0 && a.mask_words > 0,
                "tree_attention: non-positive extent");
  PTO_CHECK_ARG(a.block_size < 1ll << 31 && a.max_num_blocks_per_req < 1ll << 31 && a.pool_blocks < 1ll << 31 && a.batch < 1ll << 30 &&
                    a.block_size * a.max_num_blocks_per_req < 1ll << 30,
                "tree_attention: extent beyond 2^31, or a table of 2^30 tokens and more");
  PTO_CHECK_ARG(a.dtype == PTO_HIP_BF16 || a.dtype == PTO_HIP_FP16, "tree_attention: query dtype %s not in {BF16, FP16}", dtype_name(a.dtype));
  PTO_CHECK_ARG(a.kv_dtype == 0 || a.kv_dtype == a.dtype || fp8, "tree_attention: caches of %s under queries of %s", dtype_name(a.kv_dtype),
                dtype_name(a.dtype));
  PTO_CHECK_ARG(a.scale == a.scale && a.scale - a.scale == 0.f, "tree_attention: scale must be finite");
  if (a.head_dim > kMaxD)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "tree_attention: head_dim at most %d, got %lld", kMaxD, (long long)a.head_dim);
  if (a.tokens > kMaxTokens || a.mask_words > kMaxWords)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "tree_attention: at most %lld tokens and %d mask words, got %lld and %lld", (long long)kMaxTokens, kMaxWords,
                (long long)a.tokens, (long long)a.mask_words);
  if (a.tokens == 0 || a.batch == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(a.query && a.key_cache && a.value_cache && a.block_table && a.context_lens && a.token_starts && a.tree_mask && a.out &&
                    (!fp8 || (a.k_scale && a.v_scale)),
                "tree_attention: null tensor pointer");
  const int esz = dtype_bytes(a.dtype), csz = fp8 ? 1 : esz;
  PTO_CHECK_ARG(((uintptr_t)a.block_table | (uintptr_t)a.context_lens | (uintptr_t)a.token_starts | (uintptr_t)a.tree_mask | (uintptr_t)a.k_scale |
                 (uintptr_t)a.v_scale) % 4 == 0 &&
                    ((uintptr_t)a.query | (uintptr_t)a.out | (uintptr_t)a.key_cache | (uintptr_t)a.value_cache) % 16 == 0,
                "tree_attention: misaligned operand (query, out and the caches start at multiples of 16 bytes)");
  {
    using block8::overlap;
    const int64_t rows = a.tokens * a.num_heads * a.head_dim * esz, cache = a.pool_blocks * a.kv_head_num * a.block_size * a.head_dim * csz;
    const int64_t scales = fp8 ? a.pool_blocks * a.kv_head_num * 4 : 0;
    PTO_CHECK_ARG(!overlap(a.out, rows, a.query, rows) && !overlap(a.out, rows, a.key_cache, cache) && !overlap(a.out, rows, a.value_cache, cache) &&
                      !overlap(a.out, rows, a.k_scale, scales) && !overlap(a.out, rows, a.v_scale, scales) &&
                      !overlap(a.out, rows, a.block_table, a.batch * a.max_num_blocks_per_req * 4) &&
                      !overlap(a.out, rows, a.context_lens, a.batch * 4) && !overlap(a.out, rows, a.token_starts, (a.batch + 1) * 4) &&
                      !overlap(a.out, rows, a.tree_mask, a.tokens * a.mask_words * 4),
                  "tree_attention: out overlaps an operand");
  }
  Params p{};
  p.q = a.query;
  p.kc = a.key_cache;
  p.vc = a.value_cache;
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.block_table = a.block_table;
  p.ctx_lens = a.context_lens;
  p.starts = a.token_starts;
  p.mask = reinterpret_cast<const uint32_t*>(a.tree_mask);
  p.out = a.out;
  p.tokens = (int)a.tokens;
  p.batch = (int)a.batch;
  p.hq = (int)a.num_heads;
  p.hkv = (int)a.kv_head_num;
  p.group = (int)(a.num_heads / a.kv_head_num);
  p.d = (int)a.head_dim;
  p.bs = (int)a.block_size;
  p.max_blocks = (int)a.max_num_blocks_per_req;
  p.pool_blocks = (int)a.pool_blocks;
  p.words = (int)a.mask_words;
  p.scale = a.scale;
  p.error_flag = ctx().flags + 5;
  const DeviceScope scope(ctx().device);
  hipStream_t st = (hipStream_t)stream;
  if (a.dtype == PTO_HIP_BF16) fp8 ? launch_any<__bf16, uint8_t>(p, st) : launch_any<__bf16, __bf16>(p, st);
  else fp8 ? launch_any<_Float16, uint8_t>(p, st) : launch_any<_Float16, _Float16>(p, st);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
