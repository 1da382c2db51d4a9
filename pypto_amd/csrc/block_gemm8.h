// Products of e4m3 operands with a scale for each block of 128:
//
//   c[m, n] = sum_kb  sa[m, kb] * sb[n / 128, kb] * sum_{k in kb} a8[m, k] * b8[n, k]
//
// Codes are k-contiguous on both sides.  The sum over a block of 128 is made by the matrix unit in fresh registers, the sum over
// blocks an fp32 fused multiply-add of them with the blocks' scales.
//
// The matrix unit's 8-bit instructions do not add in 32 bits: of every eight products they drop what lies 2^-13 below the
// largest (448 * 448 + 7 / 256 is 448 * 448, and random products of 128 codes are 1.4e-5 off in norm).  That is below
// bf16's half step by 140, but not below fp32's, and it moves one code in 3000 of a quantised result.  So the forms here, for few rows, and the
// tiles whose results are fp32 or are quantised for fp16 and fp32 ones (EXACT in block_tiled8.h) widen the codes to bf16, which holds every one of
// them exactly, and use the 16-bit instruction (1e-8 off).  The tiles of 16-bit results multiply the codes as they are, at twice the rate: 2048 rows of
// 4096 x 11008 96 us, widened (fp32 results) 187.
#pragma once

#include <hip/hip_runtime.h>

#include "block_fp8.h"
#include "common.h"

namespace pto_hip {
namespace block8 {

struct Params {
  const uint8_t* a;   // [rows, k] codes
  const float* sa;    // [rows, kb]
  const uint8_t* b0;  // [n, k] codes, one row per output channel (experts: one matrix behind the other)
  const float* sb0;   // [ceil(n / 128), kb]
  const uint8_t* b1;  // gate/up pass: the up weights
  const float* sb1;
  void* c;       // [rows, n]
  float* c_scale;  // [rows, n / 128] where c is codes (gate/up pass) or scaled fp16 (down pass)
  int m, n, k, kb;
  // Tiled form: the blocks of k cut into ranges of this many, each a workgroup's own, whose sums go to slabs [range][m, n] in c (0: whole)
  int per_split;
  // Experts: the rows of a tile belong to one expert and are listed by the plan (experts.hip).
  const int4* tiles;       // {expert, first place, rows, 0}
  const int* n_tiles;      // of each height
  const int32_t* order;    // slot (token * top_k + j) of each place
  int top_k;
};

enum RowMap { kPlain = 0, kGateUp = 1, kDown = 2 };

// A tile's rows: row r of it is row a_row(r) of the activations.  `at`: its first row, experts: its index.
template <int MAP>
struct Tile {
  int expert, first, rows;
  const int32_t* order;
  int top_k;
  __device__ __forceinline__ Tile(const Params& p, int at, int height) : order(p.order), top_k(p.top_k) {
    if constexpr (MAP == kPlain) {
      expert = 0;
      first = at;
      rows = min(height, p.m - first);
    } else {
      const int4 t = p.tiles[at];
      expert = t.x;
      first = t.y;
      rows = t.z;
    }
  }
  __device__ __forceinline__ int a_row(int r) const { return MAP == kGateUp ? order[first + r] / top_k : first + r; }
};

// SiLU with the hardware's 1-ulp reciprocal (as the other e4m3 FFN's).
__device__ __forceinline__ float silu(float g) { return g * __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

template <typename T>
__device__ __forceinline__ void store_upto4(T* dst, const f32x4& v, int count) {
  if (count >= 4) {
    typedef __attribute__((__vector_size__(4 * sizeof(T)))) T vec4;
    const vec4 all = {(T)v[0], (T)v[1], (T)v[2], (T)v[3]};
    __builtin_memcpy(dst, &all, sizeof(all));  // one store, at any element
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < count) dst[e] = (T)v[e];
  }
}

// A lane's share of a step of 128 codes of one row: the 16 from k = 16 kg and the 16 from 64 + 16 kg (kg = lane / 16).  Any
// assignment of k to lanes gives the product as long as both operands share it; this one has four lanes read 64 consecutive bytes.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 widen8(int a, int b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  union {
    bf16x2 pair[4];
    bf16x8 all;
  } u;
  u.pair[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)a, 1.0f, false);
  u.pair[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)a, 1.0f, true);
  u.pair[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)b, 1.0f, false);
  u.pair[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((uint32_t)b, 1.0f, true);
  return u.all;
}
// The product of one block of 128 k: 16 channels of w with 16 rows of x.
__device__ __forceinline__ f32x4 block_product(const i32x4 (&w)[2], const i32x4 (&x)[2]) {
  f32x4 part = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int q = 0; q < 2; ++q)
#pragma unroll
    for (int d = 0; d < 4; d += 2)
      part = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(w[q][d], w[q][d + 1]), widen8(x[q][d], x[q][d + 1]), part, 0, 0, 0);
  return part;
}

// Up to 16 rows a tile: 16 rows x 16 CT channels, both operands straight from memory to registers; the workgroup's KW wavefronts take
// the steps of 128 codes in turn, NS of them in flight, and sum through LDS in wavefront order.  Bound by the stream of the weights and what
// starts it: 25 MB of 4096 x 6144 at one row 8.0 us a call (an empty call 6.8, the stream 4.8), 45 MB of 11008 x 4096 10.
template <int CT, int KW, int NS, typename OutT>
__global__ __launch_bounds__(KW * 64) void narrow_kernel(Params p, int tiles_n) {
  __shared__ __attribute__((aligned(16))) f32x4 red[KW][CT][64];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, kg = lane >> 4;
  const int tn = blockIdx.x % tiles_n, tm = blockIdx.x / tiles_n;
  const int m0 = tm * 16, rows = min(16, p.m - m0);
  const int n0 = tn * 16 * CT;
  const int mine = (p.kb - wave + KW - 1) / KW;  // steps of this wavefront

  const size_t a_row = m0 + min(c, rows - 1);
  const uint8_t* xp = p.a + a_row * p.k + wave * kBlock + kg * 16;
  const float* sp = p.sa + a_row * p.kb + wave;
  const uint8_t* wp[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) wp[i] = p.b0 + (size_t)min(n0 + 16 * i + c, p.n - 1) * p.k + wave * kBlock + kg * 16;
  const float* wsp = p.sb0 + (size_t)(n0 / kBlock) * p.kb + wave;  // 16 CT divides 128: one block

  struct Held {
    i32x4 w[CT][2], x[2];
    float sx, sw;
  };
  f32x4 acc[CT];
#pragma unroll
  for (int i = 0; i < CT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  // Past its last step a wavefront asks for its first again (the requests in flight stay known at compile time).
  auto load = [&](Held& s, int round) {
    const size_t step = round < mine ? (size_t)round * KW : 0, at = step * kBlock;
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int q = 0; q < 2; ++q) s.w[i][q] = *reinterpret_cast<const i32x4*>(wp[i] + at + q * 64);
    s.sw = wsp[step];
#pragma unroll
    for (int q = 0; q < 2; ++q) s.x[q] = *reinterpret_cast<const i32x4*>(xp + at + q * 64);
    s.sx = sp[step];
  };
  auto compute = [&](const Held& s) {
    const float scale = s.sx * s.sw;
#pragma unroll
    for (int i = 0; i < CT; ++i) {  // weights first: a lane then holds four consecutive channels of a row
      const f32x4 part = block_product(s.w[i], s.x);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(part[e], scale, acc[i][e]);
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
  for (int i = 0; i < CT; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int u = tid; u < CT * 64; u += KW * 64) {
    const int l = u & 63, i = u >> 6;
    const int row = l & 15, col = n0 + 16 * i + 4 * (l >> 4);
    if (row >= rows || col >= p.n) continue;
    f32x4 sum = red[0][i][l];
#pragma unroll
    for (int w = 1; w < KW; ++w) sum += red[w][i][l];
    store_upto4(reinterpret_cast<OutT*>(p.c) + (size_t)(m0 + row) * p.n + col, sum, p.n - col);
  }
}

}  // namespace block8
}  // namespace pto_hip
