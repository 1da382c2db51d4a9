// Block-scaled e4m3 products of many rows (block_gemm8.h has the operands and the form for few).
//
// A workgroup of eight wavefronts, two per SIMD, computes BM rows x 256 channels (gate/up pass: 128 gate and the 128 up channels of the same
// outputs, one group of h) or, where that would leave CUs without work, fewer.  Wavefront (wm, wn) of the 2 x 4 grid has BM / 2 rows x 64 channels as
// accumulators of 32 x 32.  A block of
// 128 k is summed by the matrix unit in fresh registers and then added to the accumulators with its scale by fused
// multiply-adds: 16 of them for each 32 x 32 block, next to 128 clocks of matrix instructions (8-bit form; twice that widened).  While one
// wavefront of a SIMD adds, the other has the matrix unit.
//
// The operand tiles of a block of k go global -> LDS directly, 1 KB per wavefront and request (8 rows), RING blocks ahead; the hardware fixes
// where a lane's 16 bytes land, so instead of padding, the lane whose bytes land in slot s of row r fetches logical chunk s ^ ((r / 2) % 8)
// and the fragment reads apply the same XOR (16 consecutive rows of one chunk then hit all 64 banks).  The rows are worked through in two
// halves: with the first half's barrier the weights (held in registers by then) and that half's slots are free and requested again, so
// that a request has one and a half blocks' time to land.  Waits count the requests in flight and never drain them.
//
// Row scales come the same way, eight blocks of k ahead: a request's 64 lanes bring 8 rows x 8 scales, 264 bytes apart in LDS so that
// 32 rows lie in different banks.  The weights' scales of the tile's two blocks of channels, all of k, are fetched at the start.
//
// What bounds it: 2048 rows of 4096 x 11008, bf16 results, 99 us (1.87 PFLOP/s; the library's product with one scale a tensor 92), the matrix
// pipes busy in 50 % of the clocks at 2.1 GHz: for a block of 128 k of a 256-row tile LDS takes in 64 KB and gives out 192 KB, 1500 clocks
// beside 2048 of matrix instructions, and the accumulators' fused multiply-adds share the issue.  Four wavefronts of 128 x 128 would read a third
// less, but half of their 256 accumulator registers would be out of the vector unit's reach.  333 rows of 5120 x 5003 (64 x 128 tiles)
// 18.8 us: what a CU takes in, 1 MB a tile.  48 rows of 4096 x 14336 (64 x 64) 14.3: the stream of 59 MB, start and end of one round.
// Experts' products: experts.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block_gemm8.h"
#include "lds_load.h"

namespace pto_hip {
namespace block8 {

typedef __attribute__((__vector_size__(16 * sizeof(float)))) float f32x16;
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) char lds_char;
typedef __attribute__((address_space(3))) const i32x4 lds_ci32x4;
typedef __attribute__((address_space(3))) float lds_float;
typedef __attribute__((address_space(3))) int lds_int;

constexpr int kXcds = 8;
// Consecutive logical ids to one XCD: workgroups are dealt to the XCDs in turn.
__device__ __forceinline__ int xcd_remap(int pid, int nwg) {
  const int x = pid % kXcds, local = pid / kXcds;
  const int full = nwg / kXcds, rem = nwg % kXcds;
  const int base = x < rem ? x * (full + 1) : rem * (full + 1) + (x - rem) * full;
  return base + local;
}

// BM rows x BN channels; with BN below 256 the wavefronts are KG groups of 2 x (BN / 64), which take the blocks of k in turn (a stage
// is KG blocks) and are summed at the end.
template <int BM_, int BN_>
struct TiledShape {
  static constexpr int BM = BM_, BN = BN_;
  static constexpr int WN = BN / 64, KG = 4 / WN;
  static constexpr int MF = BM / 64;             // 32-row fragments of a wavefront
  static constexpr int PH = MF > 1 ? 2 : 1;      // row halves
  static constexpr int HF = MF / PH;             // fragments of a half
  static constexpr int kBlockBytes = (BM + BN) * kBlock, kStage = KG * kBlockBytes;
  static constexpr int RING = kStage > 48 * 1024 ? 2 : 3;
  static constexpr int NA = BM / PH / 64, NB = BN / 64;  // requests of a wavefront for a half of the rows of a block, for its channels
  static constexpr int NS = BM / 64;                     // ... for eight blocks' row scales
  static constexpr int kScaleRow8 = 264;                 // bytes of a request of those
  static constexpr int kScaleBuf = BM / 8 * kScaleRow8;
  static constexpr int kScales = RING * kStage, kRows = kScales + 2 * kScaleBuf, kChannelScales = kRows + BM * 4;
  static constexpr size_t smem(int kb) { return (size_t)kChannelScales + 2 * (size_t)((kb + 63) / 64 * 64) * sizeof(float); }
  static_assert(KG == 1 || PH == 1, "groups along k have one half of rows");
};

// A workgroup's place among the tiles: bands of eight row tiles, rows first, so that an XCD's 32 consecutive ids are 8 row tiles x 4
// column tiles.
struct Place {
  int tm, tn;
  __device__ __forceinline__ Place(int logical, int tiles_m, int tiles_n) {
    const int per_band = 8 * tiles_n;
    const int band = logical / per_band, idx = logical - band * per_band;
    const int band_rows = min(8, tiles_m - band * 8);
    tn = idx / band_rows, tm = band * 8 + (idx - tn * band_rows);
  }
};

// STREAM: the weights are read with the non-temporal hint.
template <int MAP, int BM, int BN, bool EXACT, bool STREAM, typename OutT>
__device__ __forceinline__ void work_tile(const Params& p, int at, int tn, int range, uint8_t* smem) {
  typedef TiledShape<BM, BN> S;
  constexpr bool GATE = MAP == kGateUp;
  static_assert(!GATE || BN == 256, "a gate/up tile holds whole groups of h");
  lds_char* const lds0 = (lds_char*)smem;

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave & 1, wn = (wave >> 1) % S::WN, kg = (wave >> 1) / S::WN;
  constexpr bool SPLIT = MAP == kPlain && std::is_same<OutT, float>::value;
  const int k0 = range * p.per_split;  // first block of k
  const Tile<MAP> tile(p, at, BM);
  const int n0 = tn * (GATE ? kBlock : BN);
  const int nk = SPLIT && p.per_split ? min(p.per_split, p.kb - k0) : p.kb;

  // ---- the channels' scales, all of k: two blocks of channels, or gate and up ----
  const int nk64 = (nk + 63) / 64 * 64;  // a request brings 64
  lds_float* const s_cols = (lds_float*)(lds0 + S::kChannelScales);  // [2][nk64]
  const uint32_t lds_base = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)lds0);
  {
    const int blocks_n = (p.n + kBlock - 1) / kBlock, first = tile.expert * blocks_n;
    const float* c0 = p.sb0 + (size_t)(first + n0 / kBlock) * p.kb + k0;
    const float* c1 = (GATE ? p.sb1 : p.sb0) + (size_t)(first + (GATE ? n0 / kBlock : min(n0 / kBlock + 1, blocks_n - 1))) * p.kb + k0;
    for (int i = (wave >> 1) * 64; i < nk; i += 256)
      to_lds_dword((uint32_t)min(i + lane, nk - 1) * 4u, wave & 1 ? c1 : c0, lds_base + S::kChannelScales + ((wave & 1) * nk64 + i) * 4);
  }

  // ---- down pass: where the rows go, for the epilogue (asked for there, between the stores, they took 3 us a tile) ----
  lds_int* const s_rows = (lds_int*)(lds0 + S::kRows);
  if constexpr (MAP == kDown) {
    if (wave < BM / 64)
      to_lds_dword((uint32_t)min(wave * 64 + lane, tile.rows - 1) * 4u, p.order + tile.first, lds_base + S::kRows + wave * 256);
  }
  auto c_row = [&](int r) { return (size_t)(MAP == kDown ? s_rows[r] : tile.first + r); };

  // ---- requests: instruction e of a part brings its rows 64 e + 8 wave + lane / 8; rows and channels past the end are clamped
  // (their products are not stored) ----
  const int q_row = wave * 8 + (lane >> 3);
  const int chunk = (lane & 7) ^ ((q_row >> 1) & 7);  // logical chunk whose slot this lane fills
  const uint8_t* base_a = p.a + (size_t)k0 * kBlock;
  const float* base_s = p.sa + k0;
  if (MAP == kPlain) {
    base_a += (size_t)tile.first * p.k;
    base_s += (size_t)tile.first * p.kb;
  }
  auto row_at = [&](int r) { return (uint32_t)(MAP == kPlain ? min(r, tile.rows - 1) : tile.a_row(min(r, tile.rows - 1))); };
  uint32_t va[S::PH][S::NA], vb[S::NB], vs[S::NS];
#pragma unroll
  for (int h = 0; h < S::PH; ++h)
#pragma unroll
    for (int e = 0; e < S::NA; ++e) va[h][e] = row_at(h * (BM / S::PH) + e * 64 + q_row) * (uint32_t)p.k + chunk * 16;
  const uint8_t* base_b = (GATE && wave >= 4 ? p.b1 : p.b0) + ((size_t)tile.expert * p.n + n0) * p.k + (size_t)k0 * kBlock;
#pragma unroll
  for (int e = 0; e < S::NB; ++e) {
    // gate/up: of each 64 rows of the tile 32 are gate channels (wavefronts 0 to 3 bring them), then their up channels
    const int ch = GATE ? e * 32 + (wave & 3) * 8 + (lane >> 3) : e * 64 + q_row;
    vb[e] = (uint32_t)min(ch, p.n - 1 - n0) * (uint32_t)p.k + chunk * 16;
  }
  // scales: request e of wavefront w brings rows 8 (e * 8 + w) .. +8, block lane % 8 of eight
#pragma unroll
  for (int e = 0; e < S::NS; ++e) vs[e] = row_at((e * 8 + wave) * 8 + (lane >> 3)) * (uint32_t)p.kb;
  const uint32_t lds_w = lds_base + wave * 1024;
  // the first half (all, if there is one) or the second of the rows, and the channels, of stage t (past the last one: the last block)
  auto request_a = [&](auto half_c, int t, uint32_t slot) {
    constexpr int H = decltype(half_c)::value, AT = H * (BM / S::PH) * kBlock;
#pragma unroll
    for (int g = 0; g < S::KG; ++g) {
      const uint8_t* src = base_a + min(t * S::KG + g, nk - 1) * kBlock;
      to_lds<AT>(va[H][0], src, lds_w + slot + g * S::kBlockBytes);
      if constexpr (S::NA > 1) to_lds<AT + 8192>(va[H][S::NA - 1], src, lds_w + slot + g * S::kBlockBytes);
    }
  };
  auto request_b = [&](int t, uint32_t slot) {
#pragma unroll
    for (int g = 0; g < S::KG; ++g) {
      const uint8_t* src = base_b + min(t * S::KG + g, nk - 1) * kBlock;
      const uint32_t dst = lds_w + slot + g * S::kBlockBytes;
      to_lds<BM * kBlock, STREAM>(vb[0], src, dst);
      if constexpr (S::NB > 1) to_lds<BM * kBlock + 8192, STREAM>(vb[1], src, dst);
      if constexpr (S::NB > 2) {
        to_lds<BM * kBlock + 16384, STREAM>(vb[2], src, dst);
        to_lds<BM * kBlock + 24576, STREAM>(vb[3], src, dst);
      }
    }
  };
  auto request_scales = [&](int t8) {  // of blocks t8 .. t8 + 7
    const uint32_t dst = lds_base + S::kScales + ((t8 >> 3) & 1) * S::kScaleBuf + wave * S::kScaleRow8;
    const uint32_t kb = (uint32_t)min(t8 + (lane & 7), nk - 1);
#pragma unroll
    for (int e = 0; e < S::NS; ++e) to_lds_dword((vs[e] + kb) * 4u, base_s, dst + e * 8 * S::kScaleRow8);
  };
  typedef IntConst<0> C0;
  typedef IntConst<S::PH - 1> C1;

  // ---- fragments: lane l holds row / channel l % 32, logical chunks 4 ks + 2 (l / 32) and the next of either half of a block ----
  const int hi = lane >> 5;
  uint32_t off[4];
#pragma unroll
  for (int cc = 0; cc < 4; ++cc) off[cc] = (lane & 31) * kBlock + (((4 * (cc >> 1) + 2 * hi + (cc & 1)) ^ ((lane >> 1) & 7)) << 4);
  const uint32_t a_wave = kg * S::kBlockBytes + wm * (BM / S::PH / 2) * kBlock, b_wave = kg * S::kBlockBytes + BM * kBlock + wn * 64 * kBlock;
  // this lane's scale of fragment i in buffer 0: row r of the tile lies in request r / 8
  uint32_t s_off = S::kScales + (lane & 7) * 32 + ((lane & 31) >> 3) * S::kScaleRow8;

  f32x16 acc[S::MF][2];
#pragma unroll
  for (int i = 0; i < S::MF; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  // ---- one fragment of rows: its products with both channel fragments into part[0] and part[1], and those added to the accumulators
  // with their scales.  part[0] is added while part[1] is being made, part[1] while the next fragment's part[0] is, so that a
  // wavefront keeps the matrix unit busy by itself; the next fragment, and behind a block's last one the next block's channels, are
  // read over the registers that the matrix unit has just taken. ----
  f32x16 part[2];
  float scale1 = 0.f;  // of part[1], which is added one fragment later
#pragma unroll
  for (int r = 0; r < 16; ++r) part[1][r] = 0.f;
  auto add = [&](f32x16& to, const f32x16& from, float scale) {
#pragma unroll
    for (int r = 0; r < 16; ++r) to[r] = fmaf(from[r], scale, to[r]);
  };
  f32x16 zero;
#pragma unroll
  for (int r = 0; r < 16; ++r) zero[r] = 0.f;
  auto read_chunk = [&](uint32_t at, int cc) { return *reinterpret_cast<lds_ci32x4*>(lds0 + at + off[cc]); };
  i32x4 a[4], b[2][4];      // 8-bit form: the fragment and the channels
  bf16x8 aw[8], bw[2][8];   // widened form: the same
  auto fragment = [&](auto i_c, uint32_t next_a, uint32_t next_b, float sa, float s0, float s1) {
    constexpr int I = decltype(i_c)::value, PREV = (I + S::MF - 1) % S::MF;
    constexpr bool LAST = I == S::MF - 1;
    if constexpr (EXACT) {
      i32x4 v[4], w[4];
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) {
        if constexpr (LAST) w[cc] = read_chunk(next_b, cc);
        v[cc] = read_chunk(next_a, cc);
      }
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        part[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[0][ks], aw[ks], ks ? part[0] : zero, 0, 0, 0);
        if (ks == 0) {
          __builtin_amdgcn_sched_barrier(0);
          add(acc[PREV][1], part[1], scale1);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (LAST) bw[0][ks] = widen8(w[ks >> 1][2 * (ks & 1)], w[ks >> 1][2 * (ks & 1) + 1]);
        if constexpr (LAST) {
          if (ks & 1) w[ks >> 1] = read_chunk(next_b + 32 * kBlock, ks >> 1);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        part[1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(bw[1][ks], aw[ks], ks ? part[1] : zero, 0, 0, 0);
        if (ks == 0) {
          __builtin_amdgcn_sched_barrier(0);
          add(acc[I][0], part[0], sa * s0);
          __builtin_amdgcn_sched_barrier(0);
        }
        aw[ks] = widen8(v[ks >> 1][2 * (ks & 1)], v[ks >> 1][2 * (ks & 1) + 1]);
        if constexpr (LAST) bw[1][ks] = widen8(w[ks >> 1][2 * (ks & 1)], w[ks >> 1][2 * (ks & 1) + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
    } else {
      auto product = [&](int j, int ks, const f32x16& from) {
        const v8i rows = __builtin_shufflevector(a[2 * ks], a[2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        const v8i channels = __builtin_shufflevector(b[j][2 * ks], b[j][2 * ks + 1], 0, 1, 2, 3, 4, 5, 6, 7);
        part[j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(channels, rows, from, 0, 0, 0, 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      };
      auto next_channels = [&](int j, int ks) {
        if constexpr (LAST) {
          b[j][2 * ks] = read_chunk(next_b + j * 32 * kBlock, 2 * ks);
          b[j][2 * ks + 1] = read_chunk(next_b + j * 32 * kBlock, 2 * ks + 1);
        }
      };
      auto next_rows = [&](int ks) {
        a[2 * ks] = read_chunk(next_a, 2 * ks);
        a[2 * ks + 1] = read_chunk(next_a, 2 * ks + 1);
        __builtin_amdgcn_sched_barrier(0);
      };
      product(0, 0, zero);
      next_channels(0, 0);
      add(acc[PREV][1], part[1], scale1);
      __builtin_amdgcn_sched_barrier(0);
      product(1, 0, zero);
      next_channels(1, 0);
      next_rows(0);
      product(0, 1, part[0]);
      next_channels(0, 1);
      product(1, 1, part[1]);
      next_channels(1, 1);
      next_rows(1);
      add(acc[I][0], part[0], sa * s0);
      __builtin_amdgcn_sched_barrier(0);
    }
    scale1 = sa * (GATE ? s1 : s0);
  };

  // ---- prologue ----
  request_scales(0);
#pragma unroll
  for (int t = 0; t < S::RING; ++t) {
    request_a(C0{}, t, t * S::kStage);
    request_b(t, t * S::kStage);
    if constexpr (S::PH == 2) request_a(C1{}, t, t * S::kStage);
  }
  constexpr int kTile = S::KG * (S::PH * S::NA + S::NB);  // requests of a stage
  // A half of a block is waited for one fragment ahead of its first use (by the barrier in front of the last fragment of the half before
  // it): at that point the newest kAhead requests may be in flight.
  constexpr int kAhead = S::PH == 2 ? (S::RING - 1) * kTile : (S::RING - 2) * kTile;
  constexpr int kFirst = (S::RING - 1) * kTile + (S::PH == 2 ? S::NA : 0);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kFirst) : "memory");
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int cc = 0; cc < 4; ++cc) {
    a[cc] = read_chunk(a_wave, cc);
#pragma unroll
    for (int j = 0; j < 2; ++j) b[j][cc] = read_chunk(b_wave + j * 32 * kBlock, cc);
  }
  if constexpr (EXACT) {
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      aw[ks] = widen8(a[ks >> 1][2 * (ks & 1)], a[ks >> 1][2 * (ks & 1) + 1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) bw[j][ks] = widen8(b[j][ks >> 1][2 * (ks & 1)], b[j][ks >> 1][2 * (ks & 1) + 1]);
    }
  }

  uint32_t slot = 0;
  for (int t = 0; t * S::KG < nk; ++t) {
    const uint32_t next_slot = slot + S::kStage == S::RING * S::kStage ? 0 : slot + S::kStage;
    // A group without a block of its own in the last stage has the last block once more, with scales of zero (a code or sum that is
    // not finite has made the same results NaN already).
    const int block = S::KG == 1 ? t : min(t * S::KG + kg, nk - 1);
    const bool spare = S::KG > 1 && t * S::KG + kg >= nk;
    float s0 = s_cols[(GATE ? 0 : wn / 2) * nk64 + block], s1 = GATE ? s_cols[nk64 + block] : 0.f;
    const uint32_t s_at = s_off + ((block >> 3) & 1) * S::kScaleBuf + (block & 7) * 4;
    auto one = [&](auto i_c) {
      constexpr int I = decltype(i_c)::value, H = I / S::HF, ROW = H * (BM / S::PH) + (I % S::HF) * 32;
      constexpr int N = (I + 1) % S::MF, NEXT_ROW = (N / S::HF) * (BM / S::PH) + (N % S::HF) * 32;
      float sa = *(lds_float*)(lds0 + s_at + (ROW / 8 + wm * (BM / S::PH / 16)) * S::kScaleRow8);
      if (spare) sa = s0 = 0.f;
      if constexpr (I % S::HF == S::HF - 1) {
        // the next half has landed; everybody has read all of this one (and behind its first half the block's channels too)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kAhead) : "memory");
        __builtin_amdgcn_sched_barrier(0);
        request_a(IntConst<H>{}, t + S::RING, slot);
        if constexpr (H == 0) {
          request_b(t + S::RING, slot);
          if ((t * S::KG & 7) == 0 && t * S::KG + 8 < nk) request_scales(t * S::KG + 8);  // over those of the eight blocks before this one
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      fragment(i_c, (I == S::MF - 1 ? next_slot : slot) + a_wave + NEXT_ROW * kBlock, next_slot + b_wave, sa, s0, s1);
    };
    one(IntConst<0>{});
    if constexpr (S::MF > 1) one(IntConst<1>{});
    if constexpr (S::MF > 2) {
      one(IntConst<2>{});
      one(IntConst<3>{});
    }
    slot = next_slot;
  }
  add(acc[S::MF - 1][1], part[1], scale1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // nothing may land in LDS after this
  __syncthreads();

  if constexpr (S::KG > 1) {
    // the groups' sums in the order of the groups
    float* const sums = reinterpret_cast<float*>(smem);  // [KG - 1][2 WN wavefronts][32 values][64 lanes]
    if (kg > 0) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[((wave - 2 * S::WN) * 32 + j * 16 + r) * 64 + lane] = acc[0][j][r];
    }
    __syncthreads();
    if (kg == 0) {
#pragma unroll
      for (int g = 0; g < S::KG - 1; ++g)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[0][j][r] += sums[((g * 2 * S::WN + wave) * 32 + j * 16 + r) * 64 + lane];
    }
    __syncthreads();
  }

  // ---- epilogue: acc[i][j][r] is row r0 + lane % 32 of the tile, channel 32 j + (r / 4) * 8 + hi * 4 + r % 4 of the wavefront's 64 ----
  auto row_of = [&](int i) { return (i / S::HF) * (BM / S::PH) + wm * (BM / S::PH / 2) + (i % S::HF) * 32 + (lane & 31); };
  if constexpr (GATE) {
    // the wavefront's 32 outputs of a row, the largest of the row's 128 through LDS, codes staged there for whole rows' stores
    constexpr int PITCH = kBlock + 16;  // bytes; with rows of 128 the 32 lanes of a store were in one bank, 4 us of a 256-row tile
    lds_float* const top = (lds_float*)(lds0 + S::kScales);  // [4][BM]
    f32x16 y[S::MF];
#pragma unroll
    for (int i = 0; i < S::MF; ++i) {
      float amax = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        y[i][r] = silu(acc[i][0][r]) * acc[i][1][r];
        amax = fmaxf(amax, fabsf(y[i][r]));
      }
      amax = fmaxf(amax, __shfl_xor(amax, 32));
      if (hi == 0) top[wn * BM + row_of(i)] = amax;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < S::MF; ++i) {
      const int row = row_of(i);
      const float s = group_scale(fmaxf(fmaxf(top[row], top[BM + row]), fmaxf(top[2 * BM + row], top[3 * BM + row])));
      const GroupQuotient q(s);
#pragma unroll
      for (int v = 0; v < 4; ++v)
        *reinterpret_cast<uint32_t*>(smem + row * PITCH + wn * 32 + v * 8 + hi * 4) =
            codes4(q.near(y[i][4 * v]), q.near(y[i][4 * v + 1]), q.near(y[i][4 * v + 2]), q.near(y[i][4 * v + 3]));
      if (wn == 0 && hi == 0 && row < tile.rows) p.c_scale[c_row(row) * (p.n / kBlock) + tn] = s;
    }
    __syncthreads();
    uint8_t* const codes = reinterpret_cast<uint8_t*>(p.c);
    for (int u = tid; u < tile.rows * 8; u += 512) {
      const int row = u >> 3;
      *reinterpret_cast<i32x4*>(codes + c_row(row) * p.n + n0 + (u & 7) * 16) = *reinterpret_cast<const i32x4*>(smem + row * PITCH + (u & 7) * 16);
    }
  } else {
    // Rows go through LDS, a half of them at a time, so that they are written in whole lines: straight from the accumulators a wavefront's
    // store has 16 bytes of each of 32 rows.
    constexpr bool SCALED = MAP == kDown && std::is_same<OutT, _Float16>::value;
    constexpr int ROWS = BM / S::PH, PITCH = BN * (int)sizeof(OutT) + 16;  // bytes; the padding spreads rows over the banks
    static_assert(ROWS * PITCH <= (SCALED ? (int)S::kScales : (int)S::kRows), "a half of the rows fits");
    int e[S::MF];  // SCALED: rows for the sum over a token's experts, fp16 with a power of two per row and 128 channels that puts the largest below 2^15
#pragma unroll
    for (int i = 0; i < S::MF; ++i) e[i] = 0;
    if constexpr (SCALED) {
      lds_float* const top = (lds_float*)(lds0 + S::kScales);  // [4][BM]
#pragma unroll
      for (int i = 0; i < S::MF; ++i) {
        float amax = 0.f;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int r = 0; r < 16; ++r) amax = fmaxf(amax, fabsf(acc[i][j][r]));
        if (__builtin_expect(__ballot(!(amax <= 3.4028234664e38f)) != 0, 0)) {  // infinities aside
          amax = 0.f;
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) amax = fmaxf(amax, finite_size(acc[i][j][r]));
        }
        amax = fmaxf(amax, __shfl_xor(amax, 32));
        if (hi == 0) top[wn * BM + row_of(i)] = amax;
      }
      __syncthreads();
      const int group = n0 / kBlock + wn / 2;
#pragma unroll
      for (int i = 0; i < S::MF; ++i) {
        const int row = row_of(i);
        e[i] = half_exponent(fmaxf(top[(wn & ~1) * BM + row], top[(wn | 1) * BM + row]));
        if ((wn & 1) == 0 && hi == 0 && row < tile.rows && group * kBlock < p.n)
          p.c_scale[c_row(row) * (p.n / kBlock) + group] = __builtin_ldexpf(1.f, e[i]);
      }
    }
    OutT* const c = reinterpret_cast<OutT*>(p.c) + (size_t)range * p.m * p.n + n0;
    const int cols = min(BN, p.n - n0);
#pragma unroll
    for (int h = 0; h < S::PH; ++h) {
      if (kg == 0) {
#pragma unroll
        for (int f = 0; f < S::HF; ++f) {
          const int i = h * S::HF + f;
          uint8_t* const dst = smem + (row_of(i) - h * ROWS) * PITCH + (wn * 64 + hi * 4) * (int)sizeof(OutT);
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              typedef __attribute__((__vector_size__(4 * sizeof(OutT)))) OutT vec4;
              vec4 y;
#pragma unroll
              for (int r = 0; r < 4; ++r) y[r] = (OutT)(SCALED ? __builtin_ldexpf(acc[i][j][4 * v + r], -e[i]) : acc[i][j][4 * v + r]);
              *reinterpret_cast<vec4*>(dst + (j * 32 + v * 8) * (int)sizeof(OutT)) = y;
            }
        }
      }
      __syncthreads();
      const int rows = min(ROWS, tile.rows - h * ROWS);
      constexpr int VEC = 16 / (int)sizeof(OutT), PER_ROW = BN / VEC;
      for (int u = tid; u < rows * PER_ROW; u += 512) {
        const int row = u / PER_ROW, at = u % PER_ROW * VEC;
        OutT* const dst = c + c_row(h * ROWS + row) * p.n + at;
        const i32x4 v = *reinterpret_cast<const i32x4*>(smem + row * PITCH + at * (int)sizeof(OutT));
        if (at + VEC <= cols) {
          __builtin_memcpy(dst, &v, 16);  // (rows may start at any element)
        } else {
          for (int i = 0; at + i < cols; ++i) dst[i] = reinterpret_cast<const OutT*>(smem + row * PITCH)[at + i];
        }
      }
      if (h + 1 < S::PH) __syncthreads();
    }
  }
}

// The rows of a product in tiles of one height of 64 or 128 channels, groups of wavefronts along k.
template <int BN, bool EXACT, typename OutT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void tiled_kernel(Params p, int tiles_m, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int tiles = tiles_m * tiles_n;
  int logical = xcd_remap(blockIdx.x, (int)gridDim.x);
  const int range = std::is_same<OutT, float>::value ? logical / tiles : 0;
  logical -= range * tiles;
  const Place at(logical, tiles_m, tiles_n);
  work_tile<kPlain, 64, BN, EXACT, false, OutT>(p, at.tm * 64, at.tn, range, smem);
}

// Tiles of 256 channels and up to three heights: `high` row tiles of BM rows, then `half` of BM / 2 and the rest of BM / 4 (64 at least).
// Each height is dealt to the XCDs by itself, the highest first, so that the lower ones fill up what the higher leave.
template <int BM, bool EXACT, typename OutT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void tiled_rows_kernel(Params p, int high, int half, int quarter, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int ranges = std::is_same<OutT, float>::value && p.per_split ? (p.kb + p.per_split - 1) / p.per_split : 1;
  int id = blockIdx.x, first = 0;
  auto work = [&](auto height_c, int tiles_m) {
    constexpr int H = decltype(height_c)::value;
    const int tiles = tiles_m * tiles_n;
    if (id < tiles * ranges) {
      int logical = xcd_remap(id, tiles * ranges);
      const int range = logical / tiles;
      logical -= range * tiles;
      const Place at(logical, tiles_m, tiles_n);
      work_tile<kPlain, H, 256, EXACT, false, OutT>(p, first + at.tm * H, at.tn, range, smem);
      return true;
    }
    id -= tiles * ranges;
    first += tiles_m * H;
    return false;
  };
  if (work(IntConst<BM>{}, high)) return;
  if constexpr (BM >= 128) {
    if (work(IntConst<BM / 2>{}, half)) return;
  }
  if constexpr (BM >= 256) work(IntConst<BM / 4>{}, quarter);
}

// The same for tiles of experts, which lie in the plan's list by height, p.n_tiles[] of each.  With tiles of 64 rows most
// experts have one, whose weights nobody else reads: with the non-temporal hint gate and up of 128 tokens for 8 of 64 experts of 4096 x 1408
// took 129 us for 140, of 40 tokens for 4 of 60 of 2048 x 1024 41 for 45; with 512 tokens of the former, several tiles an expert, 186 for 182.
// (A projection's weights are left to the caches: 48 rows of 4096 x 14336 that the last-level cache holds 14.3 us for 17.2, from memory 18.5
// for 17.5.)
template <int MAP, int BM, bool EXACT, typename OutT>
__global__ __launch_bounds__(512) __attribute__((amdgpu_waves_per_eu(2, 2))) void tiled_experts_kernel(Params p, int tiles_n) {
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  int id = blockIdx.x, first = 0;
  auto work = [&](auto height_c, int which) {
    constexpr int H = decltype(height_c)::value;
    const int tiles = __builtin_amdgcn_readfirstlane(p.n_tiles[which]);
    if (id < tiles * tiles_n) {
      const Place at(xcd_remap(id, tiles * tiles_n), tiles, tiles_n);
      work_tile<MAP, H, 256, EXACT, BM == 64, OutT>(p, first + at.tm, at.tn, 0, smem);
      return true;
    }
    id -= tiles * tiles_n;
    first += tiles;
    return false;
  };
  if (work(IntConst<BM>{}, 0)) return;
  if constexpr (BM >= 128) {
    if (work(IntConst<BM / 2>{}, 1)) return;
  }
  if constexpr (BM >= 256) work(IntConst<BM / 4>{}, 2);
}

template <typename K, typename... Args>
int launch_tiles_of(K kern, std::atomic<bool>& attr_set, int most_smem, int64_t wgs, size_t smem, hipStream_t st, const Params& p, Args... args) {
  if (!attr_set.load(std::memory_order_acquire)) {  // callers hold the dispatch lock
    PTO_CHECK_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, most_smem));
    attr_set.store(true, std::memory_order_release);
  }
  if (wgs >= (1 << 23)) return fail(PTO_HIP_ERR_UNSUPPORTED, "a product of %lld tiles is more than one launch holds", (long long)wgs);
  hipLaunchKernelGGL(kern, dim3((unsigned)wgs), dim3(512), smem, st, p, args...);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

template <int BM>
constexpr size_t mixed_smem(int kb) {
  return std::max(TiledShape<BM, 256>::smem(kb), std::max(TiledShape<std::max(BM / 2, 64), 256>::smem(kb), TiledShape<64, 256>::smem(kb)));
}

inline int64_t ranges_of(const Params& p) { return p.per_split ? (p.kb + p.per_split - 1) / p.per_split : 1; }

template <int BN, bool EXACT, typename OutT>
int launch_tiled(const Params& p, hipStream_t st) {
  typedef TiledShape<64, BN> S;
  static std::atomic<bool> attr_set{false};  // per instantiation
  const int tiles_m = (p.m + 63) / 64, tiles_n = (p.n + BN - 1) / BN;
  return launch_tiles_of(tiled_kernel<BN, EXACT, OutT>, attr_set, (int)S::smem(kMaxK / kBlock), tiles_m * ranges_of(p) * tiles_n, S::smem(p.kb), st, p,
                         tiles_m, tiles_n);
}

// tiles: of BM, BM / 2 and BM / 4 rows
template <int BM, bool EXACT, typename OutT>
int launch_tiled_rows(const Params& p, const int (&tiles)[3], hipStream_t st) {
  static std::atomic<bool> attr_set{false};
  const int tiles_n = (p.n + 255) / 256;
  return launch_tiles_of(tiled_rows_kernel<BM, EXACT, OutT>, attr_set, (int)mixed_smem<BM>(kMaxK / kBlock),
                         ((int64_t)tiles[0] + tiles[1] + tiles[2]) * ranges_of(p) * tiles_n, mixed_smem<BM>(p.kb), st, p, tiles[0], tiles[1], tiles[2],
                         tiles_n);
}

// most_tiles: as many row tiles as the plan may have.
template <int MAP, int BM, bool EXACT, typename OutT>
int launch_tiled_experts(const Params& p, int most_tiles, hipStream_t st) {
  static std::atomic<bool> attr_set{false};
  const int tiles_n = MAP == kGateUp ? p.n / kBlock : (p.n + 255) / 256;
  return launch_tiles_of(tiled_experts_kernel<MAP, BM, EXACT, OutT>, attr_set, (int)mixed_smem<BM>(kMaxK / kBlock),
                         (int64_t)most_tiles * tiles_n, mixed_smem<BM>(p.kb), st, p, tiles_n);
}

}  // namespace block8
}  // namespace pto_hip
