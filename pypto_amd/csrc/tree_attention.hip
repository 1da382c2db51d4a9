// Attention of several new tokens per sequence over a paged cache and over each other, by a mask: a step that verifies drafted tokens.
//
//   out[t, h] = sum_n p_n v_n / sum_n p_n,   p_n = exp(scale q k_n - max),   n over the keys that row t sees:
//   n < context_lens[b], and n = context_lens[b] + j for the new tokens j of its sequence whose bit is set in tree_mask[t]
//
// The form for one token per sequence is paged_attention.hip's (examples/models/04_paged_attention.py:62-227).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_merge.h"
#include "attn_tile.h"
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
  // matrix form
  float scale_log2e;
  int target;         // workgroups that the keys are cut for
  int least;          // fewest keys of a part
  int slots;          // partial results that there is room for, in tokens
  float* part_o;      // [slots * Hq, D]
  float* part_ml;     // [slots * Hq, 2]: running maximum in units of log 2, sum
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

// ---------------------------------------------------------------------------------------------
// Matrix form.  A workgroup of NW wavefronts has up to ROWS = NW * GT * 16 query rows of one sequence and KV head - row = token number * group + head of
// the group - and walks a part of the sequence's keys, 32 at a time: its threads bring a chunk of K and V rows to LDS together, and every wavefront multiplies
// them with its own GT tiles of 16 rows.  S^T = K Q^T and O^T = V^T P^T, so that the probabilities stay in the accumulators' layout on their way into the
// second product.  Maxima and sums per row run along (online softmax); parts are joined by a second kernel.
//
// The parts are cut on the device, where the lengths are known: with `total` keys times row blocks over all sequences and KV heads, a part has total / target
// keys (a multiple of 64, at least `least`), so that target workgroups and at most one more per row block have work that lasts alike.
// ---------------------------------------------------------------------------------------------
using pto_hip::attn::f32x4;
using pto_hip::attn::fp8x8_widen;
using pto_hip::attn::kMinMax;
using pto_hip::attn::mfma16;
using pto_hip::attn::round_pack;
using pto_hip::attn::u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;

constexpr int kChunk = 32;

// A sequence of the plan, as one lane holds it.
struct Work {
  int first, count;  // its tokens
  int ctx, end;      // keys in front of its new ones, and all
  int blocks;        // row blocks
};
__device__ __forceinline__ Work work_of(const Params& p, int b, int rows) {
  Work w{};
  if (b < p.batch) {
    const int first = p.starts[b], next = p.starts[b + 1];
    const int ctx = p.ctx_lens[b];
    const bool sound = first >= 0 && next > first && next <= p.tokens;
    const int64_t room = (int64_t)p.max_blocks * p.bs;
    w.first = first;
    w.count = sound ? next - first : 0;
    w.ctx = (int)min(max((int64_t)ctx, (int64_t)0), room);
    w.end = sound ? (int)min((int64_t)w.ctx + min(w.count, 32 * p.words), room) : 0;
    w.blocks = sound ? (w.count * p.group + rows - 1) / rows : 0;
  }
  return w;
}
__device__ __forceinline__ int64_t wave_total(int64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor((long long)v, off);
  return v;
}
// Sum of the lanes up to this one.
__device__ __forceinline__ int64_t wave_scan(int64_t v, int lane) {
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t o = __shfl_up((long long)v, off);
    if (lane >= off) v += o;
  }
  return v;
}
// Keys of a part (wave-uniform).
__device__ __forceinline__ int part_keys(const Params& p, int rows, int lane, const Work& first64) {
  int64_t total = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    total += (int64_t)w.end * w.blocks;
  }
  total = wave_total(total) * p.hkv;
  const int64_t even = (total / p.target + 64) & ~63ll;
  return (int)min(max(even, (int64_t)p.least), (int64_t)1 << 30);
}
__device__ __forceinline__ int parts_of(const Work& w, int keys) { return w.blocks ? max(1, (w.end + keys - 1) / keys) : 0; }

struct Share {
  int seq;  // -1: nothing to do
  int first, count, ctx, end;
  int parts, part, block, h;
  int64_t slot;  // of the sequence's first token in its first part
};
__device__ __forceinline__ int64_t from_lane(int64_t v, int lane) { return __shfl((long long)v, lane); }
// What workgroup `id` does.  Parts of a sequence follow each other, in each the row blocks, in each the KV heads: the blocks that read the same keys are a
// multiple of the KV heads apart, on one XCD where these are a multiple of eight.
__device__ __forceinline__ Share share_of(const Params& p, int rows, int64_t id, int lane) {
  const Work first64 = work_of(p, lane, rows);
  const int keys = part_keys(p, rows, lane, first64);
  int64_t ids = 0, slots = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    const int parts = parts_of(w, keys);
    const int64_t mine = (int64_t)parts * w.blocks * p.hkv, held = parts > 1 ? (int64_t)parts * w.count : 0;
    const int64_t to = ids + wave_scan(mine, lane), slot_to = slots + wave_scan(held, lane);
    const uint64_t behind = __ballot(to > id);
    if (behind) {
      const int k = __builtin_ctzll(behind);
      Share s;
      s.seq = b0 + k;
      s.first = __shfl(w.first, k);
      s.count = __shfl(w.count, k);
      s.ctx = __shfl(w.ctx, k);
      s.end = __shfl(w.end, k);
      s.parts = __shfl(parts, k);
      s.slot = from_lane(slot_to - held, k);
      const int blocks = __shfl(w.blocks, k);
      int at = (int)(id - from_lane(to - mine, k));
      s.h = at % p.hkv;
      at /= p.hkv;
      s.block = at % blocks;
      s.part = at / blocks;
      if (s.parts > 1 && s.slot + (int64_t)s.parts * s.count > p.slots) s.seq = -1;  // only where the starts do not rise
      return s;
    }
    ids = from_lane(to, 63);
    slots = from_lane(slot_to, 63);
  }
  Share none{};
  none.seq = -1;
  return none;
}

// LDS of a stage: K rows and V rows, 16 bytes apart from each other beyond their length, so that 16 rows read at one column lie in different banks.
template <int D, bool FP8>
struct Stage {
  static constexpr int kRow = FP8 ? D : 2 * D;
  static constexpr int kPitch = kRow + 16;
  static constexpr int kBytes = 2 * kChunk * kPitch;
  static constexpr int kItems = kChunk * kRow / 16;  // 16-byte pieces of K, and of V
};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Whether any of a piece's values is infinite or NaN.
template <bool BF16, bool FP8>
__device__ __forceinline__ bool any_unbounded(u32x4 v) {
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (FP8) {
#pragma unroll
      for (int k = 0; k < 4; ++k) bad |= (v[i] >> (8 * k) & 0x7fu) == 0x7fu;
    } else {
      constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
      bad |= (v[i] & e) == e || (v[i] >> 16 & e) == e;
    }
  }
  return bad;
}
template <bool BF16>
__device__ __forceinline__ uint32_t drop_unbounded(uint32_t v) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  if ((v & e) == e) v &= 0xffff0000u;
  if ((v >> 16 & e) == e) v &= 0xffffu;
  return v;
}

template <int D, bool BF16, bool FP8, int NW, int GT>
__global__ __launch_bounds__(NW * 64) void tree_kernel(Params p) {
  typedef Stage<D, FP8> S;
  constexpr int kThreads = NW * 64, kRows = NW * GT * 16;
  constexpr int kPieces = (S::kItems + kThreads - 1) / kThreads;  // of K, and of V, a thread brings
  constexpr int kEpl = D >= 128 ? 8 : D / 16;    // V elements of a lane and token
  constexpr int kSets = D >= 128 ? D / 128 : 1;  // ... in so many groups of 16 lanes' worth
  constexpr int kEsz = FP8 ? 1 : 2;
  typedef typename std::conditional<BF16, __bf16, _Float16>::type T;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // of chunk n in place n % 3: new tokens whose values hold infinities or NaN, as bits.  A place is read while the next is written and the one
  // behind it cleared.
  __shared__ unsigned int odd_keys[3];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, j = lane >> 4;
  const Share s = share_of(p, kRows, blockIdx.x, lane);
  if (s.seq < 0) return;
  const int seq = __builtin_amdgcn_readfirstlane(s.seq), h = __builtin_amdgcn_readfirstlane(s.h);
  const int ctx = __builtin_amdgcn_readfirstlane(s.ctx), count = __builtin_amdgcn_readfirstlane(s.count);
  const int token0 = __builtin_amdgcn_readfirstlane(s.first);
  const int parts = __builtin_amdgcn_readfirstlane(s.parts), part = __builtin_amdgcn_readfirstlane(s.part);
  const int all = __builtin_amdgcn_readfirstlane(s.end);
  // even parts of whole chunks
  const int chunks = (all + kChunk - 1) / kChunk;
  const int tok_first = (int)((int64_t)chunks * part / parts) * kChunk;
  const int tok_end = min((int)((int64_t)chunks * (part + 1) / parts) * kChunk, all);
  const int row0 = (__builtin_amdgcn_readfirstlane(s.block) * NW + wave) * GT * 16;  // first row of this wavefront
  const int rows = count * p.group;
  const bool active = row0 < rows;
  if (threadIdx.x == 0) {
    odd_keys[0] = odd_keys[1] = odd_keys[2] = 0;
    const int64_t raw = p.ctx_lens[seq];
    if (raw < 0 || raw + count > (int64_t)p.max_blocks * p.bs || count > 32 * p.words) *p.error_flag = 1;
  }

  // Query fragments (B operand): column = row c of the tile; k-group j of step u holds elements (u*4+j)*8..+8, or beside e4m3 keys, of which 16 bytes are
  // two steps, ((u/2)*4+j)*16 + (u%2)*8..+8.
  u32x4 qf[GT][D / 32];
  int node[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const int r = row0 + t * 16 + c;
    const bool there = r < rows;
    node[t] = there ? r / p.group : 0;
    const int g = there ? r % p.group : 0;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + ((size_t)(token0 + node[t]) * p.hq + h * p.group + g) * D;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      const int el = FP8 ? ((u >> 1) * 4 + j) * 16 + (u & 1) * 8 : (u * 4 + j) * 8;
      const u32x4 z = {0u, 0u, 0u, 0u};
      qf[t][u] = there ? *reinterpret_cast<const u32x4*>(q + el) : z;
    }
  }
  f32x4 acc[GT][kSets][kEpl];
  float m_run[GT], l_run[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) {
#pragma unroll
    for (int a = 0; a < kSets; ++a)
#pragma unroll
      for (int i = 0; i < kEpl; ++i) acc[t][a][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[t] = kMinMax;
    l_run[t] = 0.f;
  }

  // Block-table window: lane i holds the physical block (and the scales) of logical block win_base + i.
  const int32_t* table = p.block_table + (size_t)seq * p.max_blocks;
  int win_base = 0, win_blk = 0;
  float win_ks = 1.f, win_vs = 1.f;
  bool bad_entry = false;
  auto load_window = [&](int first_block) {
    win_base = first_block;
    const bool used = (int64_t)(first_block + lane) * p.bs < tok_end;
    win_blk = used ? table[first_block + lane] : 0;
    if ((unsigned)win_blk >= (unsigned)p.pool_blocks) {
      bad_entry = true;
      win_blk = 0;
    }
    if constexpr (FP8) {
      win_ks = used ? p.k_scale[(size_t)win_blk * p.hkv + h] : 1.f;
      win_vs = used ? p.v_scale[(size_t)win_blk * p.hkv + h] : 1.f;
    }
  };
  auto slot_of = [&](int tok) {  // window slot of a token's block (uniform)
    const int lb = tok / p.bs;
    if (lb < win_base || lb >= win_base + 64) load_window(lb);
    return lb - win_base;
  };

  u32x4 kr[kPieces], vr[kPieces];  // a chunk on its way to LDS
  float k_mul_next = p.scale_log2e, v_unit_next = 1.f;
  auto request = [&](int tok) {
    if (tok >= tok_end) return;
    int slot0 = slot_of(tok);
    const int tok1 = min(tok + 16, tok_end - 1);
    const int lb1 = tok1 / p.bs;
    if (lb1 >= win_base + 64) {  // the chunk's halves in two windows
      load_window(tok / p.bs);
      slot0 = 0;
    }
    const int slot1 = lb1 - win_base;
    const int blk0 = __builtin_amdgcn_readlane(win_blk, slot0), blk1 = __builtin_amdgcn_readlane(win_blk, slot1);
    if constexpr (FP8) {  // a chunk lies in one block
      k_mul_next = p.scale_log2e * __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, win_ks), slot0));
      v_unit_next = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, win_vs), slot0));
    }
    const size_t at0 = (((size_t)blk0 * p.hkv + h) * p.bs + tok % p.bs) * S::kRow;
    const size_t at1 = (((size_t)blk1 * p.hkv + h) * p.bs + (tok + 16) % p.bs) * S::kRow;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int item = threadIdx.x + i * kThreads;
      const int row = item * 16 / S::kRow;
      // rows from tok_end on are zeros: what lies there has no part in anything
      const bool there = (S::kItems % kThreads == 0 || item < S::kItems) && tok + row < tok_end;
      const size_t at = (row < 16 ? at0 : at1 - 16 * S::kRow) + (size_t)item * 16;
      const u32x4 z = {0u, 0u, 0u, 0u};
      kr[i] = there ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p.kc) + at)) : z;
      vr[i] = there ? __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(p.vc) + at)) : z;
    }
  };
  auto park = [&](int stage, int odd_place, int tok) {
    char* base = lds + stage * S::kBytes;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int item = threadIdx.x + i * kThreads;
      if (S::kItems % kThreads != 0 && item >= S::kItems) continue;
      const int row = item * 16 / S::kRow, col = item * 16 % S::kRow;
      *reinterpret_cast<u32x4*>(base + row * S::kPitch + col) = kr[i];
      *reinterpret_cast<u32x4*>(base + (kChunk + row) * S::kPitch + col) = vr[i];
      if (tok + kChunk > ctx) {
        if (tok + row >= ctx && any_unbounded<BF16, FP8>(vr[i])) atomicOr(&odd_keys[odd_place], 1u << row);
      }
    }
  };

  float k_mul = p.scale_log2e, v_unit = 1.f;
  load_window(tok_first / p.bs);
  request(tok_first);
  if constexpr (FP8) {
    k_mul = k_mul_next;
    v_unit = v_unit_next;
  }
  lds_barrier();  // the flags are cleared
  if (tok_first < tok_end) park(0, 0, tok_first);
  request(tok_first + kChunk);
  lds_barrier();
  int stage = 0, odd_place = 0;
  for (int tok = tok_first; tok < tok_end; tok += kChunk) {
    const float k_next = k_mul_next, v_next = v_unit_next;
    if (tok + kChunk < tok_end) {
      park(stage ^ 1, odd_place == 2 ? 0 : odd_place + 1, tok + kChunk);
      request(tok + 2 * kChunk);
    }
    const char* kbase = lds + stage * S::kBytes;
    const char* vbase = kbase + kChunk * S::kPitch;
    if (active) {
      const bool masked = tok + kChunk > ctx;
      const unsigned int odd = masked ? odd_keys[odd_place] : 0u;
      // S^T: rows = keys, columns = query rows
      f32x4 s0[GT], s1[GT];
#pragma unroll
      for (int t = 0; t < GT; ++t) s0[t] = s1[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < S::kRow / 64; ++u) {
        const u32x4 a0 = *reinterpret_cast<const u32x4*>(kbase + c * S::kPitch + (u * 4 + j) * 16);
        const u32x4 a1 = *reinterpret_cast<const u32x4*>(kbase + (16 + c) * S::kPitch + (u * 4 + j) * 16);
        if constexpr (FP8) {
          const u32x4 lo0 = fp8x8_widen<BF16>(a0[0], a0[1]), hi0 = fp8x8_widen<BF16>(a0[2], a0[3]);
          const u32x4 lo1 = fp8x8_widen<BF16>(a1[0], a1[1]), hi1 = fp8x8_widen<BF16>(a1[2], a1[3]);
#pragma unroll
          for (int t = 0; t < GT; ++t) {
            s0[t] = mfma16<BF16>(lo0, qf[t][2 * u], s0[t]);
            s1[t] = mfma16<BF16>(lo1, qf[t][2 * u], s1[t]);
            s0[t] = mfma16<BF16>(hi0, qf[t][2 * u + 1], s0[t]);
            s1[t] = mfma16<BF16>(hi1, qf[t][2 * u + 1], s1[t]);
          }
        } else {
#pragma unroll
          for (int t = 0; t < GT; ++t) {
            s0[t] = mfma16<BF16>(a0, qf[t][u], s0[t]);
            s1[t] = mfma16<BF16>(a1, qf[t][u], s1[t]);
          }
        }
      }
      // online softmax, a column of lanes a row
      u32x4 pf[GT];
      uint32_t bits[GT];
#pragma unroll
      for (int t = 0; t < GT; ++t) {
        float sv[8] = {s0[t][0], s0[t][1], s0[t][2], s0[t][3], s1[t][0], s1[t][1], s1[t][2], s1[t][3]};
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[e] *= k_mul;
        bits[t] = 0xffffffffu;
        if (masked) {
          // the 32 keys from tok on, as this row sees them
          const uint32_t* words = p.mask + (size_t)(token0 + node[t]) * p.words;
          const int j0 = tok - ctx;
          if (j0 < 0) {
            bits[t] = (words[0] << -j0) | ((1u << -j0) - 1u);
          } else {
            const int w = j0 >> 5, sh = j0 & 31;
            const uint32_t lo = w < p.words ? words[w] : 0u, hi = w + 1 < p.words ? words[w + 1] : 0u;
            bits[t] = (uint32_t)(((uint64_t)hi << 32 | lo) >> sh);
          }
          if (tok + kChunk > all) bits[t] &= (1u << (all - tok)) - 1u;
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (!(bits[t] >> ((e >> 2) * 16 + j * 4 + (e & 3)) & 1u)) sv[e] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(sv[0], sv[1]), fmaxf(sv[2], sv[3])), fmaxf(fmaxf(sv[4], sv[5]), fmaxf(sv[6], sv[7])));
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        if (__builtin_amdgcn_ballot_w64(mx > m_run[t]) != 0) {
          const float m_new = fmaxf(m_run[t], mx);
          const float alpha = __builtin_amdgcn_exp2f(m_run[t] - m_new);
          m_run[t] = m_new;
          l_run[t] *= alpha;
#pragma unroll
          for (int a = 0; a < kSets; ++a)
#pragma unroll
            for (int i = 0; i < kEpl; ++i) acc[t][a][i] *= alpha;
        }
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float ra, rb;
          pf[t][e >> 1] = round_pack<BF16>(__builtin_amdgcn_exp2f(sv[e] - m_run[t]), __builtin_amdgcn_exp2f(sv[e + 1] - m_run[t]), ra, rb);
          sum += ra + rb;
        }
        l_run[t] += sum;
      }
      // O^T += V^T P^T: a lane's 8 tokens x kEpl elements, transposed in registers
#pragma unroll
      for (int a = 0; a < kSets; ++a) {
        u32x4 vw[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const char* src = vbase + ((e >> 2) * 16 + j * 4 + (e & 3)) * S::kPitch + (a * 16 + c) * kEpl * kEsz;
          if constexpr (FP8) {
            if constexpr (kEpl == 8) {
              const u32x2 w = *reinterpret_cast<const u32x2*>(src);
              vw[e] = fp8x8_widen<BF16>(w[0], w[1]);
            } else {
              vw[e] = fp8x8_widen<BF16>(*reinterpret_cast<const uint32_t*>(src), 0u);
            }
          } else if constexpr (kEpl == 8) {
            vw[e] = *reinterpret_cast<const u32x4*>(src);
          } else {
            const u32x2 w = *reinterpret_cast<const u32x2*>(src);
            vw[e] = u32x4{w[0], w[1], 0u, 0u};
          }
        }
        if (odd) {
          // Values of new tokens that are infinite or NaN are left out of the product, where they would meet the zero probabilities of rows that do not see
          // them, and added for the rows that do.
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if (!(odd >> ((e >> 2) * 16 + j * 4 + (e & 3)) & 1u)) continue;
#pragma unroll
            for (int i = 0; i < kEpl / 2; ++i) vw[e][i] = drop_unbounded<BF16>(vw[e][i]);
          }
          for (unsigned int left = odd; left; left &= left - 1) {
            const int key = __builtin_ctz(left);
            const int e_key = (key >> 4) * 4 + (key & 3), from = ((key >> 2) & 3) * 16 + c;
#pragma unroll
            for (int t = 0; t < GT; ++t) {
              const uint32_t pair = (uint32_t)(e_key < 4 ? (e_key < 2 ? __shfl((int)pf[t][0], from) : __shfl((int)pf[t][1], from))
                                                         : (e_key < 6 ? __shfl((int)pf[t][2], from) : __shfl((int)pf[t][3], from)));
              const uint16_t half = (uint16_t)(e_key & 1 ? pair >> 16 : pair);
              const float prob = (float)__builtin_bit_cast(T, half);
              if (!(bits[t] >> key & 1u)) continue;
#pragma unroll
              for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int i = 0; i < kEpl; ++i) {
                  const int el = (a * 16 + j * 4 + r) * kEpl + i;
                  float v;
                  if constexpr (FP8) v = __builtin_amdgcn_cvt_f32_fp8((int)*reinterpret_cast<const uint8_t*>(vbase + key * S::kPitch + el), 0);
                  else v = (float)reinterpret_cast<const T*>(vbase + key * S::kPitch)[el];
                  if (!(fabsf(v) <= 3.4e38f)) acc[t][a][i][r] = fmaf(prob, v, acc[t][a][i][r]);
                }
            }
          }
        }
#pragma unroll
        for (int i = 0; i < kEpl; ++i) {
          const uint32_t sel = (i & 1) ? 0x07060302u : 0x05040100u;
          u32x4 vt;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) vt[kk] = __builtin_amdgcn_perm(vw[2 * kk + 1][i >> 1], vw[2 * kk][i >> 1], sel);
#pragma unroll
          for (int t = 0; t < GT; ++t) acc[t][a][i] = mfma16<BF16>(vt, pf[t], acc[t][a][i]);
        }
      }
    }
    if constexpr (FP8) {
      // the next chunk may be another block's: the accumulators go on in its values' scale
      if (tok + kChunk < tok_end) {
        if (v_next != v_unit) {
          const float ratio = v_unit / v_next;
#pragma unroll
          for (int t = 0; t < GT; ++t)
#pragma unroll
            for (int a = 0; a < kSets; ++a)
#pragma unroll
              for (int i = 0; i < kEpl; ++i) acc[t][a][i] *= ratio;
          v_unit = v_next;
        }
        k_mul = k_next;
      }
    }
    if (threadIdx.x == 0) odd_keys[odd_place == 0 ? 2 : odd_place - 1] = 0;
    lds_barrier();
    stage ^= 1;
    odd_place = odd_place == 2 ? 0 : odd_place + 1;
  }
  if (bad_entry) *p.error_flag = 1;
  if (!active) return;
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    float l = l_run[t];
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    const int r = row0 + t * 16 + c;
    if (r >= rows) continue;
    const int head = h * p.group + r % p.group;
    if (parts == 1) {
      const float mul = l > 0.f || l != l ? v_unit / l : 0.f;
      T* out = reinterpret_cast<T*>(p.out) + ((size_t)(token0 + node[t]) * p.hq + head) * D;
#pragma unroll
      for (int a = 0; a < kSets; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[kEpl / 2];
#pragma unroll
          for (int i = 0; i < kEpl; i += 2)
            w[i / 2] = (uint32_t)__builtin_bit_cast(uint16_t, (T)(acc[t][a][i][u] * mul)) |
                       (uint32_t)__builtin_bit_cast(uint16_t, (T)(acc[t][a][i + 1][u] * mul)) << 16;
          T* dst = out + (a * 16 + j * 4 + u) * kEpl;
          if constexpr (kEpl == 8) *reinterpret_cast<u32x4*>(dst) = u32x4{w[0], w[1], w[2], w[3]};
          else *reinterpret_cast<u32x2*>(dst) = u32x2{w[0], w[1]};
        }
    } else {
      const size_t slot = ((size_t)(s.slot + (int64_t)part * count + node[t])) * p.hq + head;
#pragma unroll
      for (int a = 0; a < kSets; ++a)
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < kEpl; i += 4)
            *reinterpret_cast<f32x4*>(p.part_o + slot * D + (a * 16 + j * 4 + u) * kEpl + i) =
                f32x4{acc[t][a][i][u] * v_unit, acc[t][a][i + 1][u] * v_unit, acc[t][a][i + 2][u] * v_unit, acc[t][a][i + 3][u] * v_unit};
      if (j == 0) {
        p.part_ml[slot * 2] = m_run[t];
        p.part_ml[slot * 2 + 1] = l;
      }
    }
  }
}

// Joins a row's parts: one wavefront each, lane i the channels i, i + 64, ...
template <int D, typename T>
__global__ __launch_bounds__(256) void tree_join_kernel(Params p, int rows) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)p.tokens * p.hq) return;
  const int token = (int)(row / p.hq), head = (int)(row % p.hq);
  const Work first64 = work_of(p, lane, rows);
  const int keys = part_keys(p, rows, lane, first64);
  int64_t slots = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    const int parts = parts_of(w, keys);
    const int64_t held = parts > 1 ? (int64_t)parts * w.count : 0;
    const int64_t slot_to = slots + wave_scan(held, lane);
    const uint64_t own = __ballot(w.count > 0 && w.first <= token && token < w.first + w.count);
    if (own) {
      const int k = __builtin_ctzll(own);
      const int np = __shfl(parts, k), count = __shfl(w.count, k);
      const int64_t slot = from_lane(slot_to - held, k);
      if (np <= 1 || slot + (int64_t)np * count > p.slots) return;
      const size_t first = ((size_t)slot + (token - __shfl(w.first, k))) * p.hq + head, step = (size_t)count * p.hq;
      float m = kMinMax, l = 0.f, o[D / 64];
#pragma unroll
      for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
      for (int q0 = 0; q0 < np; q0 += 64) {
        const int q = min(q0 + lane, np - 1);
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + (first + q * step) * 2);
        const bool there = q0 + lane < np;
        float most = there ? ml.x : kMinMax;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off));
        const float m_new = fmaxf(m, most), keep = __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        const float weight = there ? __builtin_amdgcn_exp2f(ml.x - m) : 0.f;
        l = l * keep;
        float sum = there ? weight * ml.y : 0.f;
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
        l += sum;
#pragma unroll
        for (int i = 0; i < D / 64; ++i) o[i] *= keep;
        const int n = min(64, np - q0);
        constexpr int kBatch = 8;
        for (int u0 = 0; u0 < n; u0 += kBatch) {
          float v[kBatch][D / 64];
#pragma unroll
          for (int u = 0; u < kBatch; ++u)
#pragma unroll
            for (int i = 0; i < D / 64; ++i) v[u][i] = p.part_o[(first + min(q0 + u0 + u, np - 1) * step) * D + i * 64 + lane];
#pragma unroll
          for (int u = 0; u < kBatch; ++u) {
            const float wgt = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), min(u0 + u, 63)));
#pragma unroll
            for (int i = 0; i < D / 64; ++i) o[i] = u0 + u < n ? fmaf(wgt, v[u][i], o[i]) : o[i];
          }
        }
      }
      const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
#pragma unroll
      for (int i = 0; i < D / 64; ++i) reinterpret_cast<T*>(p.out)[((size_t)token * p.hq + head) * D + i * 64 + lane] = (T)(o[i] * inv);
      return;
    }
    slots = from_lane(slot_to, 63);
  }
}

template <int D, bool BF16, bool FP8, int NW, int GT>
int launch_tiles(Params& p, hipStream_t st) {
  typedef typename std::conditional<BF16, __bf16, _Float16>::type T;
  constexpr int kRows = NW * GT * 16;
  constexpr int kLds = 2 * Stage<D, FP8>::kBytes;
  static bool allowed = false;
  if (!allowed && kLds > 64 * 1024) {
    PTO_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(&tree_kernel<D, BF16, FP8, NW, GT>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    allowed = true;
  }
  // wavefronts of 256 registers: two to a SIMD; LDS may hold fewer workgroups
  const int by_waves = std::max(1, 8 / NW), by_lds = std::max(1, (160 * 1024) / (kLds + 64));
  p.target = pto_hip::ctx().num_cu * std::min(by_waves, by_lds);
  p.least = std::max(64, kRows);
  const int64_t blocks = (int64_t)p.tokens * p.group / kRows + std::min(p.batch, p.tokens);
  const int64_t grid = p.target + blocks * p.hkv;
  const int64_t slots = ((int64_t)p.target * kRows + p.hq - 1) / p.hq + p.tokens + 1;
  PTO_CHECK_ARG(grid < 1ll << 24 && slots * p.hq * D < 1ll << 33, "tree_attention: %d tokens of %d heads are more than one call takes", p.tokens, p.hq);
  const size_t o_bytes = (size_t)slots * p.hq * D * 4, ml_bytes = (size_t)slots * p.hq * 8;
  void* ws = nullptr;
  const int rc = pto_hip::workspace(o_bytes + ml_bytes, &ws);
  if (rc) return rc;
  p.slots = (int)slots;
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + o_bytes);
  hipLaunchKernelGGL((tree_kernel<D, BF16, FP8, NW, GT>), dim3((unsigned)grid), dim3(NW * 64), kLds, st, p);
  hipLaunchKernelGGL((tree_join_kernel<D, T>), dim3((unsigned)(((int64_t)p.tokens * p.hq + 3) / 4)), dim3(256), 0, st, p, kRows);
  return PTO_HIP_OK;
}

template <int D, bool BF16, bool FP8>
int launch_rows(Params& p, hipStream_t st) {
  const int64_t rows = (int64_t)std::min<int64_t>((p.tokens + p.batch - 1) / p.batch, 32 * p.words) * p.group;  // of a sequence, on average
  if (rows <= 32) return launch_tiles<D, BF16, FP8, 2, 1>(p, st);
  if (rows <= 64) return launch_tiles<D, BF16, FP8, 4, 1>(p, st);
  if constexpr (D == 256) {  // two tiles' accumulators of a wavefront would leave no room for a second one on its SIMD
    return launch_tiles<D, BF16, FP8, 8, 1>(p, st);
  } else {
    if (rows <= 128) return launch_tiles<D, BF16, FP8, 4, 2>(p, st);
    return launch_tiles<D, BF16, FP8, 8, 2>(p, st);
  }
}
template <int D>
int launch_matrix(Params& p, bool bf16, bool fp8, hipStream_t st) {
  if (bf16) return fp8 ? launch_rows<D, true, true>(p, st) : launch_rows<D, true, false>(p, st);
  return fp8 ? launch_rows<D, false, true>(p, st) : launch_rows<D, false, false>(p, st);
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
  p.scale_log2e = a.scale * 1.4426950408889634f;
  if ((a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && a.block_size % (fp8 ? 32 : 16) == 0) {
    const bool bf16 = a.dtype == PTO_HIP_BF16;
    const int rc = a.head_dim == 64 ? launch_matrix<64>(p, bf16, fp8, st) : a.head_dim == 128 ? launch_matrix<128>(p, bf16, fp8, st)
                                                                                              : launch_matrix<256>(p, bf16, fp8, st);
    if (rc) return rc;
    PTO_CHECK_HIP(hipGetLastError());
    return PTO_HIP_OK;
  }
  if (a.dtype == PTO_HIP_BF16) fp8 ? launch_any<__bf16, uint8_t>(p, st) : launch_any<__bf16, __bf16>(p, st);
  else fp8 ? launch_any<_Float16, uint8_t>(p, st) : launch_any<_Float16, _Float16>(p, st);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
