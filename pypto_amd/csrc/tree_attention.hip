// Attention of several new tokens per sequence over a paged cache and over each other, by a mask: a step that verifies drafted tokens.
//
//   out[t, h] = sum_n p_n v_n / sum_n p_n,   p_n = exp(scale q k_n - max),   n over the keys that row t sees:
//   n < context_lens[b], and n = context_lens[b] + j for the new tokens j of its sequence whose bit is set in tree_mask[t]
//
// The form for one token per sequence is paged_attention.hip's (examples/models/04_paged_attention.py:62-227).
//
// With few rows a sequence the caches' bytes bound it, with many the products: 16 sequences of 512 to 4096 bf16 keys and 1 to 40 new tokens, 32 heads over 8: 54 us (158 MB;
// 30 us at the 5.2 TB/s of a large copy), 32 sequences of 2000 to 16000 e4m3 keys and 4 to 8 tokens, 64 heads over 8: 146 to 152 us (596 MB, 115 us), 4 sequences of 20000 to 32000 fp16 keys and
// 64 tokens, 64 heads: 261 to 274 us (218 GFLOP, 182 us at the 1.2 PFLOP/s of a large product), one sequence of 4096 keys and 16 tokens: 18 us (14 and the join's 4), a chain of the
// plan, the first loads, some 8 chunks and the join.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "attn_merge.h"
#include "attn_tile.h"
#include "block_fp8.h"
#include "common.h"
#include "token_seq.h"

namespace {

using pto_hip::in_launches;
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
  float per_target;   // 1 / target
  float least;        // fewest chunks of a part
  int slots;          // partial results that there is room for, in tokens
  uint32_t block_bytes;  // of a cache's block, all KV heads
  int4* joins;        // [T] of each token: parts, slot of its first part, tokens of its sequence
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

// A score below it weighs nothing, by either form: where the running maximum, of the matrix form in units of log 2, starts.
constexpr float kLeastScore = pto_hip::attn::kMinMax * 0.69314718f;

// Any shape: one wavefront for each query head of a token.  64 keys at a time, a lane each for the scores, a lane per channel for the values.
template <typename T, typename E>
__global__ __launch_bounds__(64) void tree_any_kernel(Params p) {
  __shared__ float qs[kMaxD];
  const int t = p.t0 + blockIdx.x, hq = blockIdx.y, h = hq / p.group, lane = threadIdx.x;
  const int d = p.d, bs = p.bs;
  const TokenSeq s = pto_hip::sequence_of(p.starts, p.batch, p.tokens, t, lane);
  if (t == 0 && hq == 0 && lane == 0 && pto_hip::pass_the_rows(p.starts, p.batch, p.tokens)) *p.error_flag = 1;
  if (s.seq < 0) return;
  const size_t row = (size_t)t * p.hq + hq;
  for (int i = lane; i < d; i += 64) qs[i] = (float)reinterpret_cast<const T*>(p.q)[row * d + i] * p.scale;
  __syncthreads();
  const KeyRange keys = key_range(p, s);
  bool bad = keys.bad;
  float o[kMaxD / 64] = {0.f, 0.f, 0.f, 0.f};
  float m = kLeastScore, l = 0.f;
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
    if (__ballot(sees) == 0) continue;  // nobody of these is seen
    const float keep = expf(m - m_new);
    m = m_new;
    const float prob = sees ? expf(score - m) : 0.f;
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
// keys or somewhat more (at least `least`), so that the workgroups that a GPU holds at once have work that lasts alike.
// ---------------------------------------------------------------------------------------------
using pto_hip::attn::f32x4;
using pto_hip::attn::fp8x8_widen;
using pto_hip::attn::kMinMax;
using pto_hip::attn::mfma16;
using pto_hip::attn::u32x4;
typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;

constexpr int kChunk = 32;

// a / b of numbers below 2^26 whose quotient is below 2^20 (a division of integers is some 40 instructions).
__device__ __forceinline__ int quotient(int a, int b) {
  const int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));  // off by one at most
  const int r = a - q * b;
  return q + (r >= b) - (r < 0);
}

// A sequence of the plan, as one lane holds it.
struct Work {
  int first, count;  // its tokens
  int ctx, end;      // keys in front of its new ones, and all
  int blocks;        // row blocks
};
__device__ __forceinline__ int chunks_of(const Work& w) { return (w.end + kChunk - 1) / kChunk; }
__device__ __forceinline__ Work work_of(const Params& p, int b, int rows) {
  const int at = min(b, p.batch - 1);
  const int first = pto_hip::within(p.starts[at], p.tokens), next = pto_hip::within(p.starts[at + 1], p.tokens), ctx = p.ctx_lens[at];
  const bool sound = b < p.batch && next > first;
  const int room = p.max_blocks * p.bs;  // below 2^29
  Work w;
  w.first = first;
  w.count = sound ? next - first : 0;
  w.ctx = min(max(ctx, 0), room);
  w.end = sound ? min(w.ctx + min(w.count, 32 * p.words), room) : 0;
  w.blocks = (int)(((uint32_t)w.count * (uint32_t)p.group + (uint32_t)rows - 1) / (uint32_t)rows);
  return w;
}
__device__ __forceinline__ int parts_of(const Work& w, int part) { return w.blocks ? max(1, quotient(chunks_of(w) + part - 1, part)) : 0; }
// Chunks of a part (wave-uniform): total / target, or a few eighths more, the least with which the workgroups are no more than target; twice as many where none of
// these will do, as with short sequences.
__device__ __forceinline__ int part_chunks(const Params& p, int rows, int lane, const Work& first64) {
  using pto_hip::wave_total;
  float total = 0.f;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    total += wave_total((float)chunks_of(w) * (float)w.blocks);
  }
  total *= (float)p.hkv * 1.0001f * p.per_target;  // not below the exact quotient: the grid and the room for partial results count on it
  constexpr int kTries = 8;
  float part[kTries], count[kTries];
#pragma unroll
  for (int i = 0; i < kTries; ++i) {
    part[i] = fmaxf(floorf(fminf(total * (1.f + 0.125f * i), 0x1p25f)) + 1.f, p.least);  // 2^25 chunks: of no sequence more than one part
    count[i] = 0.f;
  }
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    const float chunks = (float)chunks_of(w), blocks = (float)w.blocks;
#pragma unroll
    for (int i = 0; i < kTries; ++i) count[i] += wave_total(fmaxf(ceilf(chunks * __builtin_amdgcn_rcpf(part[i])), 1.f) * blocks);
  }
  float found = part[kTries - 1];
#pragma unroll
  for (int i = kTries - 2; i >= 0; --i) found = count[i] * (float)p.hkv <= (float)p.target ? part[i] : found;
  return (int)found;
}

struct Share {
  int seq;  // -1: nothing to do
  Work w;
  int parts, part, block, h;
  int slot;  // of the sequence's first token in its first part
};
// A sequence's partial results, in tokens: none where it has one part.  No more than there can be room for, so that sums over 64 of them stay in 32 bits.
__device__ __forceinline__ int held_of(const Params& p, const Work& w, int parts) {
  return parts > 1 ? (int)fminf((float)parts * (float)w.count, (float)(p.slots + 1)) : 0;
}
__device__ __forceinline__ Work work_in_lane(const Work& w, int k) {
  return Work{__builtin_amdgcn_readlane(w.first, k), __builtin_amdgcn_readlane(w.count, k), __builtin_amdgcn_readlane(w.ctx, k),
              __builtin_amdgcn_readlane(w.end, k), __builtin_amdgcn_readlane(w.blocks, k)};
}
// What workgroup `id` does.  Parts of a sequence follow each other, in each the row blocks, in each the KV heads: the blocks that read the same keys are a
// multiple of the KV heads apart, on one XCD where these are a multiple of eight.
__device__ __forceinline__ Share share_of(const Params& p, int rows, int id, int lane) {
  const Work first64 = work_of(p, lane, rows);
  const int part = part_chunks(p, rows, lane, first64);
  int ids = 0, slots = 0;
  Share s{};
  s.seq = -1;
  for (int b0 = 0; b0 < p.batch; b0 += 64) {
    const Work w = b0 == 0 ? first64 : work_of(p, b0 + lane, rows);
    const int parts = parts_of(w, part);
    const int mine = parts * w.blocks * p.hkv, held = held_of(p, w, parts);
    const int to = pto_hip::wave_running_sum(mine) + ids, slot_to = pto_hip::wave_running_sum(held) + slots;
    const uint64_t behind = __ballot(to > id);
    if (behind) {
      const int k = __builtin_ctzll(behind);
      s.seq = b0 + k;
      s.w = work_in_lane(w, k);
      s.parts = __builtin_amdgcn_readlane(parts, k);
      s.slot = __builtin_amdgcn_readlane(slot_to - held, k);
      const int at = id - __builtin_amdgcn_readlane(to - mine, k);
      const int per_head = quotient(at, p.hkv);
      s.h = at - per_head * p.hkv;
      s.part = quotient(per_head, s.w.blocks);
      s.block = per_head - s.part * s.w.blocks;
      if (s.parts > 1 && (s.slot < 0 || (int64_t)s.slot + (int64_t)s.parts * s.w.count > p.slots)) {  // only where the starts do not rise
        s.seq = -1;
        for (int i = lane; i < s.w.count; i += 64) p.joins[s.w.first + i] = int4{0, 0, 0, 0};
      }
      return s;
    }
    ids = __builtin_amdgcn_readlane(to, 63);
    slots = min(__builtin_amdgcn_readlane(slot_to, 63), p.slots + 1);
  }
  return s;
}

// LDS of a stage: K rows and V rows as 16-bit values, 32 bytes apart from each other beyond their length: eight rows read 16 bytes wide at one column lie in
// different banks, and so do four rows read 32 bytes wide.
template <int D>
struct Stage {
  static constexpr int kRow = 2 * D;
  static constexpr int kPitch = kRow + 32;
  static constexpr int kBytes = 2 * kChunk * kPitch;
};

__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Zeros in the place of those of eight 16-bit values that are infinite or NaN; whether there were any.
template <bool BF16>
__device__ __forceinline__ bool drop_unbounded(u32x4& v) {
  constexpr uint32_t e = BF16 ? 0x7f80u : 0x7c00u;
  bool any = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const bool low = (v[i] & e) == e, high = (v[i] >> 16 & e) == e;
    v[i] = (low ? 0u : v[i] & 0xffffu) | (high ? 0u : v[i] & 0xffff0000u);
    any |= low || high;
  }
  return any;
}
// Two fp32 rounded to the 16-bit type, nearest even, the first in the low half.
template <bool BF16>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  typedef typename std::conditional<BF16, __bf16, _Float16>::type T;
  typedef T T2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), T2));
}
// The largest over the four lanes c, c + 16, c + 32, c + 48.
__device__ __forceinline__ float column_max(float v) {
  auto both = [](auto r) { return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1])); };
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const uint32_t w = __builtin_bit_cast(uint32_t, both(__builtin_amdgcn_permlane16_swap(u, u, false, false)));
  return both(__builtin_amdgcn_permlane32_swap(w, w, false, false));
}
// Four rows of 16 16-bit values each, from LDS: the 16 lanes of a group give the addresses of a row's quarters, four lanes a row, and lane c has column c.
__device__ __forceinline__ u32x2 read_columns(const char* p) {
  typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p)));
}

// A row's maximum may fall behind by so much (in powers of two) before sums and accumulators are brought up to it.  At 0, with every rise followed: 65 us for 55 over 16 sequences,
// 317 us for 273 over four long ones.
constexpr int kSlack = 6;
constexpr int kLarge = 12;

// Whether a wavefront shares its SIMD with three others: with one tile of rows, over e4m3 caches, whose rows on their way are half as long (32 sequences of 4 to 8 drafts, 64 heads:
// 190 -> 179 us by the kernel).  128 registers hold all that the loop over cached keys needs (with 128 channels 20 values lie in scratch, of the chunks with new tokens and of the end); one
// reload in that loop waits for every row on its way (157 -> 180 us).  16-bit caches need 178.
template <int D, bool FP8, int GT>
constexpr bool lean() { return GT == 1 && FP8 && D <= 128; }

template <int D, bool BF16, bool FP8, int NW, int GT, int AHEAD>
__global__ __launch_bounds__(NW * 64, (lean<D, FP8, GT>() ? 4 : 2)) void tree_kernel(Params p) {
  typedef Stage<D> S;
  constexpr int kThreads = NW * 64, kRows = NW * GT * 16;
  constexpr int kEsz = FP8 ? 1 : 2;
  constexpr int kRowBytes = D * kEsz;                     // of a cache row
  constexpr int kItems = kChunk * kRowBytes / 16;         // 16-byte pieces of a chunk's K, and of its V
  constexpr int kPieces = (kItems + kThreads - 1) / kThreads;  // ... a thread brings
  typedef typename std::conditional<BF16, __bf16, _Float16>::type T;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  // Chunk n lies in stage n % kStages.  Between two barriers the wavefronts multiply AHEAD chunks and bring the AHEAD behind those, each at its own pace: held
  // together at every chunk, the two of a SIMD would be at the same kind of work all along.
  constexpr int kStages = 2 * AHEAD;
  // Of chunk n in place n % kPlaces: new tokens whose values hold infinities or NaN, as bits.  A place is read between two barriers, cleared between the next two
  // and written again behind those.
  constexpr int kPlaces = 3 * AHEAD;
  __shared__ unsigned int odd_keys[kPlaces];
  __shared__ float2 chunk_scale[kStages];  // e4m3 caches: of the chunk's keys and values
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, j = lane >> 4;
  const Share s = share_of(p, kRows, blockIdx.x, lane);
  if (blockIdx.x == 0 && threadIdx.x == 0 && pto_hip::pass_the_rows(p.starts, p.batch, p.tokens)) *p.error_flag = 1;
  if (s.seq < 0) return;
  const int seq = s.seq, h = s.h, ctx = s.w.ctx, count = s.w.count, token0 = s.w.first, parts = s.parts, part = s.part, all = s.w.end;
  // even parts of whole chunks
  const int chunks = chunks_of(s.w), each = quotient(chunks, parts), more = chunks - each * parts;
  const int tok_first = (part * each + min(part, more)) * kChunk;
  const int tok_end = min(tok_first + (each + (part < more)) * kChunk, all);
  const int row0 = (s.block * NW + wave) * GT * 16;  // first row of this wavefront
  const int rows = count * p.group;
  const bool active = row0 < rows;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kPlaces; ++i) odd_keys[i] = 0;
    const int64_t raw = p.ctx_lens[seq];
    if (raw < 0 || raw + count > (int64_t)p.max_blocks * p.bs || count > 32 * p.words) *p.error_flag = 1;
  }

  if (part == 0 && s.block == 0 && h == 0)
    for (int i = threadIdx.x; i < count; i += kThreads) p.joins[token0 + i] = int4{parts, s.slot + i, count, 0};

  // Query fragments (B operand): column = row c of the tile; k-group j of step u holds elements (u*4+j)*8..+8.  A negative scale changes their sign, so that
  // the largest product is the largest score.
  const uint32_t flip = p.scale_log2e < 0.f ? 0x80008000u : 0u;
  const float scale = fabsf(p.scale_log2e);
  u32x4 qf[GT][D / 32];
  int node[GT];
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const int r = row0 + t * 16 + c;
    const bool there = r < rows;
    node[t] = there ? quotient(r, p.group) : 0;
    const int g = there ? r - node[t] * p.group : 0;
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p.q) + ((size_t)(token0 + node[t]) * p.hq + h * p.group + g) * D;
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      const u32x4 z = {0u, 0u, 0u, 0u};
      qf[t][u] = there ? *reinterpret_cast<const u32x4*>(q + (u * 4 + j) * 8) ^ flip : z;
    }
  }
  // acc[t][i][r]: row c of tile t, channel 16 i + 4 j + r; sum[t]: its probabilities' sum, in every lane of the column
  f32x4 acc[GT][D / 16], sum[GT];
  float m_run[GT];
  const uint32_t one = BF16 ? 0x3f803f80u : 0x3c003c00u;
  const u32x4 ones = {one, one, one, one};
#pragma unroll
  for (int t = 0; t < GT; ++t) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[t][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    sum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[t] = kMinMax;
  }

  // Block-table window: lane i holds the physical block (and the scales) of logical block win_base + i.
  const int32_t* table = p.block_table + (size_t)seq * p.max_blocks;
  int win_base = 0, win_blk = 0;
  float win_ks = 1.f, win_vs = 1.f;
  bool bad_entry = false;
  auto load_window = [&](int first_block) __attribute__((always_inline)) {
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
      asm volatile("" : "+v"(win_ks), "+v"(win_vs));
    }
    // the wait for these loads belongs here, on a branch rarely taken: left to their first use it would become one for every load in flight, each chunk
    asm volatile("" : "+v"(win_blk));
  };
  // The next 16 tokens to be asked for: logical block and place in it (a block is a multiple of 16 tokens).
  int lb = tok_first / p.bs, off = tok_first % p.bs;

  const char* k_head = reinterpret_cast<const char*>(p.kc) + (size_t)h * p.bs * kRowBytes;
  const char* v_head = reinterpret_cast<const char*>(p.vc) + (size_t)h * p.bs * kRowBytes;
  // two chunks on their way to LDS, and the scales of their keys and values
  u32x4 kr[2][kPieces], vr[2][kPieces];
  float k_units[2] = {1.f, 1.f}, v_units[2] = {1.f, 1.f};
  // Every request is as many loads, with nothing to skip them, so that the number in flight at each wait is known to the compiler.  Where no tokens are left the
  // window's blocks are block 0, whose rows lie in the cache as any block's.
  auto request = [&](auto set, int tok) __attribute__((always_inline)) {
    constexpr int SET = decltype(set)::value;
    // a chunk's halves lie in one block where blocks are a multiple of it, and a wavefront's piece in one half
    int lb1 = lb, off1 = off + 16;
    lb1 += off1 == p.bs;
    off1 = off1 == p.bs ? 0 : off1;
    if (lb1 >= win_base + 64) load_window(lb);
    const int slot = lb - win_base;
    const uint32_t blk0 = __builtin_amdgcn_readlane(win_blk, slot), blk1 = __builtin_amdgcn_readlane(win_blk, lb1 - win_base);
    if constexpr (FP8) {  // a chunk lies in one block
      k_units[SET] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, win_ks), slot));
      v_units[SET] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, win_vs), slot));
    }
    const uint64_t at0 = (uint64_t)blk0 * p.block_bytes + (uint32_t)(off * kRowBytes);
    const uint64_t at1 = (uint64_t)blk1 * p.block_bytes + (uint32_t)(off1 * kRowBytes) - 16 * kRowBytes;
    off = off1 + 16;
    lb = lb1 + (off == p.bs);
    off = off == p.bs ? 0 : off;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      if constexpr (kItems % kThreads == 0 && kThreads * 16 >= 16 * kRowBytes) {
        // every piece of the workgroup's lies in one half, or the wavefront's in one
        const bool second = (wave * 64 + i * kThreads) * 16 >= 16 * kRowBytes;
        const uint64_t at = (second ? at1 : at0) + (uint32_t)(i * kThreads * 16);
        kr[SET][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k_head + at + threadIdx.x * 16));
        vr[SET][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v_head + at + threadIdx.x * 16));
      } else {
        int item = threadIdx.x + i * kThreads;
        if constexpr (kItems % kThreads != 0) item = min(item, kItems - 1);
        const uint64_t at = (item * 16 / kRowBytes < 16 ? at0 : at1) + (uint32_t)(item * 16);
        kr[SET][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(k_head + at));
        vr[SET][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(v_head + at));
      }
    }
  };
  auto park = [&](auto set, int stage, int odd_place, int tok) __attribute__((always_inline)) {
    constexpr int SET = decltype(set)::value;
    char* base = lds + stage * S::kBytes;
    if constexpr (FP8) {
      if (threadIdx.x == 0) {
        // of an infinite or NaN value scale: rows that see one of the keys are NaN by their scores, the others have no part in it
        const bool bounded = fabsf(v_units[SET]) <= 3.4028234664e38f;
        chunk_scale[stage] = float2{bounded ? scale * k_units[SET] : __builtin_nanf(""), bounded ? v_units[SET] : 0.f};
      }
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int item = threadIdx.x + i * kThreads;
      if (kItems % kThreads != 0 && item >= kItems) continue;
      const int row = item * 16 / kRowBytes, col = item * 16 % kRowBytes * (2 / kEsz);
      char* k = base + row * S::kPitch + col;
      char* v = k + kChunk * S::kPitch;
      // rows from tok_end on are zeros: what lies there has no part in anything
      const bool there = tok + row < tok_end;
      const u32x4 z = {0u, 0u, 0u, 0u};
      const u32x4 kx = there ? kr[SET][i] : z, vx = there ? vr[SET][i] : z;
      u32x4 v0 = vx, v1 = z;
      if constexpr (FP8) {  // widened once for all wavefronts; exact
        v0 = fp8x8_widen<BF16>(vx[0], vx[1]);
        v1 = fp8x8_widen<BF16>(vx[2], vx[3]);
      }
      if (tok + kChunk > ctx) {
        if (tok + row >= ctx) {
          bool odd = drop_unbounded<BF16>(v0);
          if constexpr (FP8) odd |= drop_unbounded<BF16>(v1);
          if (odd) atomicOr(&odd_keys[odd_place], 1u << row);
        }
      }
      if constexpr (FP8) {
        *reinterpret_cast<u32x4*>(k) = fp8x8_widen<BF16>(kx[0], kx[1]);
        *reinterpret_cast<u32x4*>(k + 16) = fp8x8_widen<BF16>(kx[2], kx[3]);
        *reinterpret_cast<u32x4*>(v + 16) = v1;
      } else {
        *reinterpret_cast<u32x4*>(k) = kx;
      }
      *reinterpret_cast<u32x4*>(v) = v0;
    }
  };

  float k_mul = scale, v_unit = 1.f, v_top = 0.f;
  // A chunk's products from stage base `kbase`.  MASKED: some of its keys may be new tokens, or lie behind the last one.
  auto multiply = [&](const char* kbase, int tok, unsigned int odd, auto masked) __attribute__((always_inline)) {
    constexpr bool MASKED = decltype(masked)::value;
    const char* vbase = kbase + kChunk * S::kPitch;
    // S^T: rows = keys, columns = query rows
    f32x4 s0[GT], s1[GT];
#pragma unroll
    for (int t = 0; t < GT; ++t) s0[t] = s1[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int u = 0; u < D / 32; ++u) {
      const u32x4 a0 = *reinterpret_cast<const u32x4*>(kbase + c * S::kPitch + (u * 4 + j) * 16);
      const u32x4 a1 = *reinterpret_cast<const u32x4*>(kbase + (16 + c) * S::kPitch + (u * 4 + j) * 16);
#pragma unroll
      for (int t = 0; t < GT; ++t) {
        s0[t] = mfma16<BF16>(a0, qf[t][u], s0[t]);
        s1[t] = mfma16<BF16>(a1, qf[t][u], s1[t]);
      }
    }
    // The values' fragments are asked for in front of the softmax (as many as there are registers for): lane (c, j) has channel 16 i + c of the tokens whose
    // probabilities it will have.
    const char* vlane = vbase + (j * 4 + (c >> 2)) * S::kPitch + (c & 3) * 8;
    constexpr int kHeld = lean<D, FP8, GT>() ? 4 : D <= 128 ? D / 16 : 8;
    u32x4 vt[kHeld];
    auto fetch_values = [&](int from) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const u32x2 lo = read_columns(vlane + (from + i) * 32), hi = read_columns(vlane + 16 * S::kPitch + (from + i) * 32);
        vt[i] = u32x4{lo[0], lo[1], hi[0], hi[1]};
      }
    };
    fetch_values(0);
    asm volatile("" ::: "memory");  // not put off behind it
    // Online softmax, a column of lanes a row.  The probabilities are taken against the maximum so far first: as long as none passes 2^kSlack - each lane looks at its
    // own - there is no need to know the chunk's maximum, nor to bring sums and accumulators to it.
    u32x4 pf[GT];
    uint32_t bits[GT];
    float pv[GT][8];
    bool risen = false;
    // Against a maximum of this chunk's own the product is rounded first, as the maximum was: none passes 1, where scores are so large that what a product is rounded by is more than an
    // exponential holds (from 2^30 on).  Rows whose maximum passes 2^kLarge always take this way, so that equal scores weigh the same; below, the difference is 2^-13 at most.
    auto probabilities = [&](int t, auto own) __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma clang fp contract(off)
        const float s = e < 4 ? s0[t][e] : s1[t][e - 4];
        pv[t][e] = __builtin_amdgcn_exp2f(decltype(own)::value ? s * k_mul - m_run[t] : fmaf(s, k_mul, -m_run[t]));
        if constexpr (MASKED) pv[t][e] = bits[t] >> ((e >> 2) * 16 + j * 4 + (e & 3)) & 1u ? pv[t][e] : 0.f;
      }
    };
#pragma unroll
    for (int t = 0; t < GT; ++t) {
      if constexpr (MASKED) {
        // the 32 keys from tok on, as this row sees them
        const uint32_t* words = p.mask + (size_t)(token0 + node[t]) * p.words;
        const int j0 = tok - ctx;
        if (j0 <= -kChunk) {
          bits[t] = 0xffffffffu;
        } else if (j0 < 0) {
          bits[t] = (words[0] << -j0) | ((1u << -j0) - 1u);
        } else {
          const int w = j0 >> 5, sh = j0 & 31;
          const uint32_t lo = w < p.words ? words[w] : 0u, hi = w + 1 < p.words ? words[w + 1] : 0u;
          bits[t] = (uint32_t)(((uint64_t)hi << 32 | lo) >> sh);
        }
        if (tok + kChunk > all) bits[t] &= (1u << (all - tok)) - 1u;
      }
      probabilities(t, std::false_type{});
      risen |= fabsf(m_run[t]) > (float)(1 << kLarge);
      risen |= fmaxf(fmaxf(fmaxf(pv[t][0], pv[t][1]), fmaxf(pv[t][2], pv[t][3])), fmaxf(fmaxf(pv[t][4], pv[t][5]), fmaxf(pv[t][6], pv[t][7]))) >
               (float)(1 << kSlack);
    }
    if (__builtin_amdgcn_ballot_w64(risen) != 0) {
#pragma unroll
      for (int t = 0; t < GT; ++t) {
        float top = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = e < 4 ? s0[t][e] : s1[t][e - 4];
          bool seen = true;
          if constexpr (MASKED) seen = bits[t] >> ((e >> 2) * 16 + j * 4 + (e & 3)) & 1u;
          top = fmaxf(top, seen ? x : -INFINITY);
        }
        const float m_new = fmaxf(m_run[t], column_max(top) * k_mul);
        const float alpha = __builtin_amdgcn_exp2f(m_run[t] - m_new);
        m_run[t] = m_new;
        sum[t] *= alpha;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) acc[t][i] *= alpha;
        probabilities(t, std::true_type{});
      }
    }
#pragma unroll
    for (int t = 0; t < GT; ++t) {
#pragma unroll
      // 16 bits are what the matrix instruction takes: half a step of each probability, which in the mean over the keys leaves the result 1.4 times as far from the exact one as its own
      // rounding does (2.3e-3 and 1.7e-3 of its size in bfloat16).  A second product of what the rounding leaves would double the instructions of this half.
      for (int e = 0; e < 8; e += 2) pf[t][e >> 1] = round_pair<BF16>(pv[t][e], pv[t][e + 1]);
      sum[t] = mfma16<BF16>(ones, pf[t], sum[t]);  // of the probabilities as rounded
    }
    // O^T += V^T P^T
#pragma unroll
    for (int i0 = 0; i0 < D / 16; i0 += kHeld) {
      if (i0) fetch_values(i0);
#pragma unroll
      for (int n = 0; n < kHeld; ++n) {
        const int i = i0 + n;
#pragma unroll
        for (int t = 0; t < GT; ++t) acc[t][i] = mfma16<BF16>(vt[n], pf[t], acc[t][i]);
      }
    }
    if constexpr (MASKED) {
      // Values of new tokens that are infinite or NaN are zeros in LDS, where they would meet the zero probabilities of rows that do not see them, and are
      // added here, from the cache, for the rows that do.
      for (unsigned int left = odd; left; left &= left - 1) {
        const int key = __builtin_ctz(left), n = tok + key;
        const int e_key = (key >> 4) * 4 + (key & 3), from = ((key >> 2) & 3) * 16 + c;
        int block = table[n / p.bs];
        if ((unsigned)block >= (unsigned)p.pool_blocks) block = 0;
        const size_t row = (((size_t)block * p.hkv + h) * p.bs + n % p.bs) * D;
#pragma unroll
        for (int t = 0; t < GT; ++t) {
          const uint32_t pair = (uint32_t)(e_key < 4 ? (e_key < 2 ? __shfl((int)pf[t][0], from) : __shfl((int)pf[t][1], from))
                                                     : (e_key < 6 ? __shfl((int)pf[t][2], from) : __shfl((int)pf[t][3], from)));
          const float prob = (float)__builtin_bit_cast(T, (uint16_t)(e_key & 1 ? pair >> 16 : pair));
          if (!(bits[t] >> key & 1u)) continue;
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float v = elem<typename std::conditional<FP8, uint8_t, T>::type>(p.vc, row + i * 16 + j * 4 + r);
              if (!(fabsf(v) <= 3.4e38f)) acc[t][i][r] = fmaf(prob, v, acc[t][i][r]);
            }
        }
      }
    }
  };

  using pto_hip::block8::IntConst;
  load_window(lb);
  request(IntConst<0>{}, tok_first);
  request(IntConst<1>{}, tok_first + kChunk);
  lds_barrier();  // the flags are cleared
  int stage = 0, place = 0, until_barrier = AHEAD;  // of the chunk to be multiplied
  auto behind = [](int i, int by, int n) { return i + by >= n ? i + by - n : i + by; };
  // Chunk number n = PARITY modulo 2, of the tokens from `tok` on.  The AHEAD-th behind it goes to its stage, the second behind that is asked for.
  auto step = [&](auto parity, int tok, auto masked) __attribute__((always_inline)) {
    constexpr int SET = (decltype(parity)::value + AHEAD) & 1;
    park(IntConst<SET>{}, behind(stage, AHEAD, kStages), behind(place, AHEAD, kPlaces), tok + AHEAD * kChunk);
    request(IntConst<SET>{}, tok + (AHEAD + 2) * kChunk);
    if constexpr (FP8) {
      const float2 s = chunk_scale[stage];
      k_mul = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s.x)));
      float v_now = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, s.y)));
      // The chunk may be another block's than the one in front: the accumulators go on in its values' scale.  One below 2^-60 of the largest counts as that (its values are
      // off by 2^-51 of that scale at most), and 0 as the smallest number at least, so that they stay finite.
      v_top = fmaxf(v_top, v_now);
      const float v_least = fmaxf(v_top * 0x1p-60f, 0x1p-149f);
      v_now = v_now < v_least ? v_least : v_now;
      if (v_now != v_unit) {
        const float ratio = tok == tok_first ? 1.f : v_unit / v_now;
#pragma unroll
        for (int t = 0; t < GT; ++t)
#pragma unroll
          for (int i = 0; i < D / 16; ++i) acc[t][i] *= ratio;
        v_unit = v_now;
      }
    }
    if (active) multiply(lds + stage * S::kBytes, tok, decltype(masked)::value ? odd_keys[place] : 0u, masked);
    if (threadIdx.x == 0) odd_keys[behind(place, kPlaces - AHEAD, kPlaces)] = 0;
    if (--until_barrier == 0) {
      lds_barrier();
      until_barrier = AHEAD;
    }
    stage = behind(stage, 1, kStages);
    place = behind(place, 1, kPlaces);
  };
  if (tok_first < tok_end) {
#pragma unroll
    for (int i = 0; i < AHEAD; i += 2) {
      park(IntConst<0>{}, i, i, tok_first + i * kChunk);
      request(IntConst<0>{}, tok_first + (i + 2) * kChunk);
      if (i + 1 < AHEAD) {
        park(IntConst<1>{}, i + 1, i + 1, tok_first + (i + 1) * kChunk);
        request(IntConst<1>{}, tok_first + (i + 3) * kChunk);
      }
    }
    lds_barrier();
    // chunks that lie in the cache as it was, two at a time, then the others
    int tok = tok_first;
    const int plain_end = min(tok_end, ctx);
    for (; tok + 2 * kChunk <= plain_end; tok += 2 * kChunk) {
      step(IntConst<0>{}, tok, std::false_type{});
      step(IntConst<1>{}, tok + kChunk, std::false_type{});
    }
    for (; tok < tok_end; tok += 2 * kChunk) {
      step(IntConst<0>{}, tok, std::true_type{});
      if (tok + kChunk < tok_end) step(IntConst<1>{}, tok + kChunk, std::true_type{});
    }
  }
  if (bad_entry) *p.error_flag = 1;
  if (!active) return;
#pragma unroll
  for (int t = 0; t < GT; ++t) {
    const float l = sum[t][0];
    const int r = row0 + t * 16 + c;
    if (r >= rows) continue;
    const int head = h * p.group + r - node[t] * p.group;
    if (parts == 1) {
      const float mul = l > 0.f || l != l ? v_unit / l : 0.f;
      T* out = reinterpret_cast<T*>(p.out) + ((size_t)(token0 + node[t]) * p.hq + head) * D + j * 4;
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        *reinterpret_cast<u32x2*>(out + i * 16) =
            u32x2{round_pair<BF16>(acc[t][i][0] * mul, acc[t][i][1] * mul), round_pair<BF16>(acc[t][i][2] * mul, acc[t][i][3] * mul)};
    } else {
      const size_t slot = (size_t)(s.slot + part * count + node[t]) * p.hq + head;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(p.part_o + slot * D + i * 16 + j * 4) = acc[t][i] * v_unit;
      if (j == 0) {
        p.part_ml[slot * 2] = m_run[t];
        p.part_ml[slot * 2 + 1] = l;
      }
    }
  }
}

// Joins a row's parts: one wavefront each, lane i the channels i, i + 64, ...
template <int D, typename T>
__global__ __launch_bounds__(256) void tree_join_kernel(Params p) {
  const int lane = threadIdx.x & 63;
  const int token = p.t0 + blockIdx.x, head = blockIdx.y * 4 + (threadIdx.x >> 6);
  if (head >= p.hq) return;
  const int from = p.starts[0], to = p.starts[p.batch];
  const int4 join = p.joins[token];  // by the kernel in front, for every token that a sequence has
  const int np = join.x, count = join.z;
  if (token < from || token >= to || np <= 1) return;
  if (join.y < 0 || count < 1 || (int64_t)join.y + (int64_t)(np - 1) * count >= p.slots) return;  // only where the starts do not rise
  const size_t first = (size_t)join.y * p.hq + head, step = (size_t)count * p.hq;
  const float2* part_ml = reinterpret_cast<const float2*>(p.part_ml) + first;
  const float* part_o = p.part_o + first * D + lane;
  constexpr int kBatch = 8;
  float ahead[kBatch][D / 64];  // the first parts' values, on their way while their weights are made
#pragma unroll
  for (int u = 0; u < kBatch; ++u)
#pragma unroll
    for (int i = 0; i < D / 64; ++i) ahead[u][i] = part_o[min(u, np - 1) * step * D + i * 64];
  float m = kMinMax, l = 0.f, o[D / 64];
#pragma unroll
  for (int i = 0; i < D / 64; ++i) o[i] = 0.f;
  for (int q0 = 0; q0 < np; q0 += 64) {
    const int q = min(q0 + lane, np - 1);
    const float2 ml = part_ml[q * step];
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
    for (int u0 = 0; u0 < n; u0 += kBatch) {
      float v[kBatch][D / 64];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
#pragma unroll
        for (int i = 0; i < D / 64; ++i) v[u][i] = ahead[u][i];
      if (q0 + u0 + kBatch < np) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
#pragma unroll
          for (int i = 0; i < D / 64; ++i) ahead[u][i] = part_o[min(q0 + u0 + kBatch + u, np - 1) * step * D + i * 64];
      }
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
}

// Every workgroup makes the plan of all sequences, which grows with the square of their number: one token each, 64 heads over 8 of 64 channels, contexts of 8 to 15 (250 to 500) keys: 1024
// sequences 272 (383) us by the matrix form and 87 (1618) by the plain one, 4096 3.4 (3.9) and 0.3 (6.2) ms, 16384 52 (54) and 1.5 (24) ms, 65536 824 (831) and 6.1 (96) ms.  The host does not know the
// contexts; from the most on that this form takes it is behind with those of a few thousand too.
constexpr int kMaxSequences = 1 << 15;
constexpr int64_t kMaxGrid = 1 << 22;
constexpr int kOtherForm = -1;  // no status: what this form does not take

template <int D, bool BF16, bool FP8, int NW, int GT, int AHEAD>
int launch_tiles(Params& p, hipStream_t st) {
  typedef typename std::conditional<BF16, __bf16, _Float16>::type T;
  constexpr int kRows = NW * GT * 16;
  constexpr int kLds = 2 * AHEAD * Stage<D>::kBytes;
  static int resident = 0, asked = -1;  // workgroups that a CU holds, of the device that was asked (calls take turns: PTO_DISPATCH_LOCK)
  if (asked != pto_hip::ctx().device) {
    const void* kernel = reinterpret_cast<const void*>(&tree_kernel<D, BF16, FP8, NW, GT, AHEAD>);
    if (kLds > 64 * 1024) PTO_CHECK_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, kLds));
    int n = 0;
    PTO_CHECK_HIP(hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, NW * 64, kLds));
    resident = std::max(1, n);
    asked = pto_hip::ctx().device;
  }
  p.target = pto_hip::ctx().num_cu * resident;
  p.per_target = 1.f / (float)p.target;
  // parts of 256 keys at least: one sequence of 4096 keys takes 18.6 us, by parts of 64 keys 24.7, of 512 21.7 (what one launch saves the join takes, and the other way round)
  p.least = (float)(std::max(256, kRows) / kChunk);
  p.block_bytes = (uint32_t)((int64_t)p.hkv * p.bs * D * (FP8 ? 1 : 2));
  const int64_t blocks = (int64_t)p.tokens * p.group / kRows + std::min(p.batch, p.tokens);
  const int64_t grid = p.target + blocks * p.hkv;
  // Partial results, in tokens of all heads.  parts * blocks * hkv, over the sequences, is at most target + blocks * hkv: target * rows and the tokens themselves.  And with P chunks
  // a part a sequence that is cut has over P of them, so that its parts are fewer than 2 chunks / P: no more than 2 target row blocks, however many tokens.
  const int64_t slots = std::min<int64_t>(((int64_t)p.target * kRows + p.hq - 1) / p.hq + p.tokens, (2ll * p.target * kRows + p.hq - 1) / p.hq) + 1;
  if (grid >= kMaxGrid) return kOtherForm;
  const size_t o_bytes = (size_t)slots * p.hq * D * 4, ml_bytes = (size_t)slots * p.hq * 8;
  void* ws = nullptr;
  const int rc = pto_hip::workspace(o_bytes + ml_bytes + 16 + (size_t)p.tokens * sizeof(int4), &ws);
  if (rc) return rc;
  p.slots = (int)slots;
  p.joins = reinterpret_cast<int4*>(reinterpret_cast<char*>(ws) + o_bytes + (ml_bytes + 15) / 16 * 16);
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(ws) + o_bytes);
  hipLaunchKernelGGL((tree_kernel<D, BF16, FP8, NW, GT, AHEAD>), dim3((unsigned)grid), dim3(NW * 64), kLds, st, p);
  const unsigned heads = (p.hq + 3) / 4;
  in_launches(p, 256 * heads, [&](unsigned n) { hipLaunchKernelGGL((tree_join_kernel<D, T>), dim3(n, heads), dim3(256), 0, st, p); });
  return PTO_HIP_OK;
}

template <int D, bool BF16, bool FP8>
int launch_rows(Params& p, hipStream_t st) {
  const int64_t rows = (int64_t)std::min<int64_t>((p.tokens + p.batch - 1) / p.batch, 32 * p.words) * p.group;  // of a sequence, on average
  if constexpr (D == 256) {  // four wavefronts would bring twice as much each: 13 to 46 registers of 16-bit caches' form lie in scratch then
    return launch_tiles<D, BF16, FP8, 8, 1, 2>(p, st);
  } else {
    // A sequence's rows in one workgroup as long as they fit: its keys are read once.  16 sequences of 4096 keys, 8 KV heads of 128 in bf16 (e4m3), by four wavefronts of one tile of
    // rows / four of two / eight of two: 64 rows 62 / 66 / 71 us (60 / 67 / 87), 128 rows 85 / 76 / 81 (85 / 75 / 100), 256 rows 137 / 128 / 119 (145 / 126 / 119); 8 rows 54 / 57 / 64, and 58 by two
    // wavefronts.  More tiles also want more chunks between barriers: the wavefronts of a SIMD drift apart, one in its products while the other is in its softmax.
    if (rows <= 64) return launch_tiles<D, BF16, FP8, 4, 1, 1>(p, st);
    if (rows <= 128) return launch_tiles<D, BF16, FP8, 4, 2, 2>(p, st);
    return launch_tiles<D, BF16, FP8, 8, 2, 4>(p, st);
  }
}
template <int D>
int launch_matrix(Params& p, bool bf16, bool fp8, hipStream_t st) {
  if (bf16) return fp8 ? launch_rows<D, true, true>(p, st) : launch_rows<D, true, false>(p, st);
  return fp8 ? launch_rows<D, false, true>(p, st) : launch_rows<D, false, false>(p, st);
}

template <typename T, typename E>
void launch_any(Params& p, hipStream_t st) {
  in_launches(p, 64 * p.hq, [&](unsigned n) { hipLaunchKernelGGL((tree_any_kernel<T, E>), dim3(n, p.hq), dim3(64), 0, st, p); });
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
                    a.block_size * a.max_num_blocks_per_req < 1ll << 29,
                "tree_attention: extent beyond 2^31, or a table of 2^29 tokens and more");
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
  if ((a.head_dim == 64 || a.head_dim == 128 || a.head_dim == 256) && a.block_size % (fp8 ? 32 : 16) == 0 &&
      a.kv_head_num * a.block_size * a.head_dim * csz < 1ll << 31 && a.tokens * p.group < 1ll << 24 && a.batch <= kMaxSequences) {
    const bool bf16 = a.dtype == PTO_HIP_BF16;
    const int rc = a.head_dim == 64 ? launch_matrix<64>(p, bf16, fp8, st) : a.head_dim == 128 ? launch_matrix<128>(p, bf16, fp8, st)
                                                                                              : launch_matrix<256>(p, bf16, fp8, st);
    if (rc != kOtherForm) {
      if (rc) return rc;
      PTO_CHECK_HIP(hipGetLastError());
      return PTO_HIP_OK;
    }
  }
  if (a.dtype == PTO_HIP_BF16) fp8 ? launch_any<__bf16, uint8_t>(p, st) : launch_any<__bf16, __bf16>(p, st);
  else fp8 ? launch_any<_Float16, uint8_t>(p, st) : launch_any<_Float16, _Float16>(p, st);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}
