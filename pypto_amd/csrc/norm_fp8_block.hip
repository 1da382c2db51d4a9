// RMSNorm with the residual's addition in front and an e4m3 output with a scale per 128 columns behind, one pass:
//
//   s = x + residual      n = s * rsqrt(mean s^2 + eps) * gamma      scale = amax_group |n| / 448      codes = e4m3(n / scale)
//
// and, where asked for, s (the next residual) and n in the 16-bit type of x.  s and n stay in 32 bits from the loads to the
// outputs, so that each output is rounded once: the codes are those of n itself, not of its 16-bit copy.  n / scale is 448 t / max t with
// t = s gamma: the row's statistic cancels, and the quotient's 32-bit roundings (2^-22) matter only next to a border between two codes.
// There, 13 values in a million, the group is done again in 64 bits: the codes are the exact rows' (a plain evaluation in 32 bits has one in a
// million wrong).
// Without the norm the same kernel is the quantiser of activations that come from elsewhere.
//
// Bound by memory: 2 bytes an element for x and for each of residual, sum and normed, 1 for the codes.  One workgroup holds a row in
// registers; a group of 128 columns is 16 lanes of 8 columns, its maximum four lane exchanges.
// Outputs larger than the eight L2s together (kStreamBytes) are written with the non-temporal hint, as they would only displace what
// is still to be read; smaller ones stay there for who reads them next.  All outputs of bf16 rows, us without / with it, and with a
// product of the codes behind: 4096 x 8192 63.3 / 54.3 (302 MB: 5.6 TB/s) and 113.5 / 108.5, 2048 x 5120 25.8 / 16.8 and 45.0 / 39.5, 8192 x
// 2048 31.6 / 25.7 and 44.2 / 38.5; but 1024 x 4096 9.3 / 8.2 and 20.9 / 22.4, 512 x 4096 8.3 / 7.6 and 18.8 / 20.7.
// With the weights asked for ahead of the row's statistic 4096 x 8192 takes 50 us in a loop of its own (6.1 TB/s), 4096 x 16384 95.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_fp8.h"
#include "common.h"

namespace {

using pto_hip::block8::codes4;
using pto_hip::block8::group_scale;
using pto_hip::block8::GroupQuotient;
using pto_hip::block8::kBlock;

constexpr int kThreads = 256;
constexpr int kVecs = 8;  // most groups of eight columns a thread holds
constexpr int64_t kStreamBytes = 32 << 20;
constexpr int64_t kLaunchRows = 1 << 23;  // a launch holds fewer than 2^32 threads

template <bool STREAM, typename V>
__device__ __forceinline__ void store(V* to, const V& v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, to);
  else *to = v;
}

// A group in 64 bits: its quotients s g inv / scale, rounded to 32 so that they stay on their side of every border between two codes (to
// zero, the last bit set where anything is lost).  wide: s g may lie outside of what fp32 holds well, and its largest value and n are made here
// as well.  top: the group's largest |n|; all lanes of the group take part.
__device__ __forceinline__ void exact_group(const float (&s)[8], const float (&g)[8], float inv, bool wide, float& top, float& scale, float (&n)[8],
                                            float (&q)[8]) {
  double amax = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmax(amax, fabs((double)s[e] * (double)g[e]));
#pragma unroll
  for (int off = 8; off > 0; off >>= 1) amax = fmax(amax, __shfl_xor(amax, off));
  if (wide) {
    top = (float)(amax * (double)inv);
    scale = group_scale(top);
#pragma unroll
    for (int e = 0; e < 8; ++e) n[e] = (float)((double)s[e] * (double)g[e] * (double)inv);
  }
  // (no scale but 1 for a row normalised to zeros, none below the smallest normal number)
  const bool least = top < 448.f * 0x1p-126f;
  // 448 s g has at most 51 bits: a quotient that is a tie between two codes is one here too, as it is divided last
  const double factor = !(top > 0.f) ? (double)inv * 0.0 : least ? (double)inv : 448.0, over = !(top > 0.f) ? 1.0 : least ? (double)scale : amax;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const double v = (double)s[e] * (double)g[e] * factor / over;
    const float f = __double2float_rz(v);
    q[e] = (double)f == v || !(v == v) ? f : __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, f) | 1u);
  }
}

// sum_out and normed_out may be x or residual themselves: a thread writes the columns that it alone has read.
template <typename T, bool NORM, bool STREAM, int VECS>
__global__ __launch_bounds__(kThreads) void norm_fp8_block_kernel(const T* x, const T* residual, const float* __restrict__ gamma,
                                                                  T* sum_out, T* normed_out, uint8_t* __restrict__ codes,
                                                                  float* __restrict__ scale, int cols, float eps) {
  typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec8;
  __shared__ float red[kThreads / 64];
  const int64_t row = blockIdx.x;
  const int nvec = cols / 8, groups = (cols + kBlock - 1) / kBlock;
  const vec8* xr = reinterpret_cast<const vec8*>(x + row * cols);
  const vec8* rr = residual ? reinterpret_cast<const vec8*>(residual + row * cols) : nullptr;
  vec8 in[VECS], res[VECS];
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = threadIdx.x + u * kThreads;
    if (i < nvec) {
      in[u] = xr[i];
      if (rr) res[u] = rr[i];
    }
  }
  float s[VECS][8];
  float ss = 0.f;
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const bool live = (int)threadIdx.x + u * kThreads < nvec;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      s[u][e] = !live ? 0.f : rr ? (float)in[u][e] + (float)res[u][e] : (float)in[u][e];
      ss += s[u][e] * s[u][e];
    }
  }
  if (sum_out) {
    vec8* out = reinterpret_cast<vec8*>(sum_out + row * cols);
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int i = threadIdx.x + u * kThreads;
      vec8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)s[u][e];
      if (i < nvec) store<STREAM>(out + i, v);
    }
  }
  float inv = 1.f, g[VECS][8];  // NORM: the columns' weights
  if constexpr (NORM) {
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int i = threadIdx.x + u * kThreads;
#pragma unroll
      for (int e = 0; e < 8; ++e) g[u][e] = 1.f;
      if (gamma && i < nvec) {
        *reinterpret_cast<float4*>(&g[u][0]) = reinterpret_cast<const float4*>(gamma)[2 * i];
        *reinterpret_cast<float4*>(&g[u][4]) = reinterpret_cast<const float4*>(gamma)[2 * i + 1];
      }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) ss += __shfl_xor(ss, off);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = ss;
    __syncthreads();
    float tot = red[0];
#pragma unroll
    for (int w = 1; w < kThreads / 64; ++w) tot += red[w];
    inv = rsqrtf(tot / (float)cols + eps);
  }
  typedef __attribute__((__vector_size__(2 * sizeof(uint32_t)))) uint32_t u32x2;
  u32x2* crow = reinterpret_cast<u32x2*>(codes + row * cols);
  float* srow = scale + row * groups;
#pragma unroll
  for (int u = 0; u < VECS; ++u) {
    const int i = threadIdx.x + u * kThreads;
    float t[8], q[8], amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      t[e] = NORM ? s[u][e] * g[u][e] : s[u][e];
      amax = fmaxf(amax, fabsf(t[e]));
    }
    auto store_normed = [&](const float (&n)[8], float times) {
      vec8 v;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (T)(n[e] * times);
      if (i < nvec) store<STREAM>(reinterpret_cast<vec8*>(normed_out + row * cols) + i, v);
    };
    if (NORM && normed_out) store_normed(t, inv);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) amax = fmaxf(amax, __shfl_xor(amax, off));
    float top = NORM ? amax * inv : amax, sc = group_scale(top);
    if constexpr (NORM) {
      // n / scale is 448 t / max t: the row's statistic cancels
      const float r = amax > 0.f ? 448.f * GroupQuotient(amax).r : inv * 0.f;  // (a statistic that is not finite: NaN)
      const bool wide = amax > 0.f && !(amax > 0x1p-90f && amax < 0x1p90f);
      bool exact = amax > 0.f && (wide || !(top >= 448.f * 0x1p-126f));
      // Within 6 steps of the 24-bit format of a border between two codes: the roundings so far, 2^-22 together, are up to 4.  A border lies
      // where the last 20 bits are 0x80000; below 2^-6, where codes lie 2^-9 apart, of 32 |q| + 1/2 (larger ones are 1 there: no border).
      constexpr uint32_t kReach = 6;
      auto past = [](float v) { return (__builtin_bit_cast(uint32_t, v) << 12) - ((0x80000u - kReach) << 12); };
      uint32_t nearest = ~0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] = t[e] * r;
        nearest = min(nearest, min(past(q[e]), past(__builtin_amdgcn_fmed3f(fmaf(fabsf(q[e]), 32.f, 0.5f), 0.f, 1.f))));
      }
      exact |= nearest <= (2 * kReach) << 12;
      if (__builtin_expect(__ballot(exact) != 0, 0)) {
        exact_group(s[u], g[u], inv, wide, top, sc, t, q);
        if (normed_out && wide) store_normed(t, 1.f);  // over the one above
      }
    } else {
      const GroupQuotient quotient(sc);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = quotient(t[e]);
    }
    if (i < nvec) {
      store<STREAM>(crow + i, u32x2{codes4(q[0], q[1], q[2], q[3]), codes4(q[4], q[5], q[6], q[7])});
      if (i % 16 == 0) srow[i / 16] = sc;
    }
  }
}

template <typename T, bool NORM, bool STREAM>
int launch(const void* x, const void* residual, const float* gamma, void* sum_out, void* normed_out, void* codes, float* scale,
           int64_t rows, int64_t cols, float eps, hipStream_t st) {
  auto go = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3((unsigned)rows), dim3(kThreads), 0, st, reinterpret_cast<const T*>(x),
                       reinterpret_cast<const T*>(residual), gamma, reinterpret_cast<T*>(sum_out), reinterpret_cast<T*>(normed_out),
                       reinterpret_cast<uint8_t*>(codes), scale, (int)cols, eps);
  };
  const int64_t vecs = (cols / 8 + kThreads - 1) / kThreads;
  if (vecs <= 1) go(norm_fp8_block_kernel<T, NORM, STREAM, 1>);
  else if (vecs <= 2) go(norm_fp8_block_kernel<T, NORM, STREAM, 2>);
  else if (vecs <= 4) go(norm_fp8_block_kernel<T, NORM, STREAM, 4>);
  else go(norm_fp8_block_kernel<T, NORM, STREAM, kVecs>);
  PTO_CHECK_HIP(hipGetLastError());
  return PTO_HIP_OK;
}

int run(const char* what, bool norm, const void* x, const void* residual, const float* gamma, void* sum_out, void* normed_out, void* codes,
        float* scale, int64_t rows, int64_t cols, float eps, int x_dtype, hipStream_t st) {
  using namespace pto_hip;
  PTO_CHECK_ARG(rows >= 0 && cols > 0 && rows < (1ll << 31), "%s: bad shape [%lld, %lld]", what, (long long)rows, (long long)cols);
  PTO_CHECK_ARG(x_dtype == PTO_HIP_BF16 || x_dtype == PTO_HIP_FP16, "%s: dtype %s not in {BF16, FP16}", what, dtype_name(x_dtype));
  if (cols % 8 != 0 || cols > 8 * kThreads * kVecs)
    return fail(PTO_HIP_ERR_UNSUPPORTED, "%s: %lld columns; rows must be a multiple of 8 and at most %d long", what, (long long)cols,
                8 * kThreads * kVecs);
  if (!ctx().initialized) return fail(PTO_HIP_ERR_NOT_INITIALIZED, "pto_hip_init has not been called");
  if (rows == 0) return PTO_HIP_OK;
  PTO_CHECK_ARG(x && codes && scale, "%s: null tensor pointer", what);
  PTO_CHECK_ARG(((uintptr_t)x | (uintptr_t)residual | (uintptr_t)gamma | (uintptr_t)sum_out | (uintptr_t)normed_out) % 16 == 0 &&
                    (uintptr_t)codes % 8 == 0 && (uintptr_t)scale % 4 == 0,
                "%s: misaligned operand", what);
  {
    using block8::overlap;
    const int64_t row_bytes = 2 * rows * cols, scale_bytes = rows * ((cols + kBlock - 1) / kBlock) * 4, gamma_bytes = cols * 4;
    auto apart = [&](const void* o, int64_t bytes, bool in_place) {  // an output from the inputs; in_place: it may be one of the rows themselves
      return !overlap(o, bytes, gamma, gamma_bytes) && ((in_place && o == x) || !overlap(o, bytes, x, row_bytes)) &&
             ((in_place && o == residual) || !overlap(o, bytes, residual, row_bytes));
    };
    PTO_CHECK_ARG(apart(sum_out, row_bytes, true) && apart(normed_out, row_bytes, true) && apart(codes, rows * cols, false) &&
                      apart(scale, scale_bytes, false),
                  "%s: an output overlaps an input (sum_out and normed_out may be x or residual as a whole)", what);
    PTO_CHECK_ARG(!overlap(sum_out, row_bytes, normed_out, row_bytes) && !overlap(codes, rows * cols, scale, scale_bytes) &&
                      !overlap(codes, rows * cols, sum_out, row_bytes) && !overlap(codes, rows * cols, normed_out, row_bytes) &&
                      !overlap(scale, scale_bytes, sum_out, row_bytes) && !overlap(scale, scale_bytes, normed_out, row_bytes),
                  "%s: two outputs overlap", what);
  }
  const bool stream = rows * cols * (1 + 2 * (sum_out != nullptr) + 2 * (normed_out != nullptr)) > kStreamBytes;
  auto go = [&](auto type, auto norm_c, auto stream_c) {
    auto from = [&](auto* p, int64_t bytes) { return p ? reinterpret_cast<decltype(p)>((uintptr_t)p + bytes) : nullptr; };
    for (int64_t r = 0; r < rows; r += kLaunchRows) {
      const int64_t at = r * cols;
      const int rc = launch<decltype(type), decltype(norm_c)::value, decltype(stream_c)::value>(
          from(x, 2 * at), from(residual, 2 * at), gamma, from(sum_out, 2 * at), from(normed_out, 2 * at), from(codes, at),
          scale + r * ((cols + block8::kBlock - 1) / block8::kBlock), std::min(kLaunchRows, rows - r), cols, eps, st);
      if (rc) return rc;
    }
    return (int)PTO_HIP_OK;
  };
  auto typed = [&](auto type) {
    if (norm) return stream ? go(type, std::true_type{}, std::true_type{}) : go(type, std::true_type{}, std::false_type{});
    return stream ? go(type, std::false_type{}, std::true_type{}) : go(type, std::false_type{}, std::false_type{});
  };
  return x_dtype == PTO_HIP_BF16 ? typed(__bf16{}) : typed(_Float16{});
}

}  // namespace

extern "C" int pto_hip_rms_norm_fp8_block(const void* x, const void* residual, const float* gamma, void* sum_out, void* normed_out,
                                          void* codes, float* scale, int64_t rows, int64_t cols, float eps, int x_dtype, void* stream) {
  PTO_DISPATCH_LOCK();
  return run("rms_norm_fp8_block", true, x, residual, gamma, sum_out, normed_out, codes, scale, rows, cols, eps, x_dtype,
             (hipStream_t)stream);
}

extern "C" int pto_hip_quantize_fp8_block(const void* x, void* codes, float* scale, int64_t rows, int64_t cols, int x_dtype,
                                          void* stream) {
  PTO_DISPATCH_LOCK();
  return run("quantize_fp8_block", false, x, nullptr, nullptr, nullptr, nullptr, codes, scale, rows, cols, 0.f, x_dtype,
             (hipStream_t)stream);
}
