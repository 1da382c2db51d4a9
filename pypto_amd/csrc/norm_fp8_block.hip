// RMSNorm with the residual's addition in front and an e4m3 output with a scale per 128 columns behind, one pass:
//
//   s = x + residual      n = s * rsqrt(mean s^2 + eps) * gamma      scale = amax_group |n| / 448      codes = e4m3(n / scale)
//
// and, where asked for, s (the next residual) and n in the 16-bit type of x.  s and n stay in 32 bits from the loads to the
// outputs, so that each output is rounded once: the codes are those of n itself, not of its 16-bit copy.  n / scale is 448 t / max t with
// t = s gamma: the row's statistic cancels, and the quotient's 32-bit roundings (7 * 2^-24) matter only next to a border between two codes.
// There, some 15 values in a million, the group is done again in 64 bits from its inputs, read once more: the codes are the exact rows' (a plain evaluation
// in 32 bits has one in a million wrong), but in groups whose scale is the least there is, 2^-126, where the statistic does not cancel.
// Without the norm the same kernel is the quantiser of activations that come from elsewhere.
//
// Bound by memory: 2 bytes an element for x and for each of residual, sum and normed, 1 for the codes.  One workgroup holds a row in
// registers; a group of 128 columns is 16 lanes of 8 columns, its maximum four lane exchanges.
// Outputs larger than the eight L2s together (kStreamBytes) are written with the non-temporal hint, as they would only displace what
// is still to be read; smaller ones stay there for who reads them next.  All outputs of bf16 rows, us without / with it, and with a
// product of the codes behind: 4096 x 8192 63.3 / 54.3 (302 MB: 5.6 TB/s) and 113.5 / 108.5, 2048 x 5120 25.8 / 16.8 and 45.0 / 39.5, 8192 x
// 2048 31.6 / 25.7 and 44.2 / 38.5; but 1024 x 4096 9.3 / 8.2 and 20.9 / 22.4, 512 x 4096 8.3 / 7.6 and 18.8 / 20.7.
// With the weights asked for ahead of the row's statistic 4096 x 8192 takes 49 us in a loop of its own (6.1 TB/s), 4096 x 16384 99.
// Rows of up to 4096 columns have 64 registers, so that a SIMD holds eight of their wavefronts: 2048 x 4096 12.8 us, with 70 of them 13.9.
// Where every weight is the same, ties are common and most wavefronts go through the 64 bits: 4096 x 8192 53 us.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "block_fp8.h"
#include "common.h"

namespace {

using pto_hip::block8::codes4;
using pto_hip::block8::group_scale;
using pto_hip::block8::GroupQuotient;
using pto_hip::block8::i32x4;
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

// v of the lane N further round in the 16 that hold a group.
template <int N>
__device__ __forceinline__ uint32_t rotated(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x120 + N, 0xf, 0xf, true);
}
template <int N>
__device__ __forceinline__ float rotated(float v) {
  return __builtin_bit_cast(float, rotated<N>(__builtin_bit_cast(uint32_t, v)));
}
template <int N>
__device__ __forceinline__ double rotated(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)rotated<N>((uint32_t)(b >> 32)) << 32 | rotated<N>((uint32_t)b));
}
// The group's largest value, in all of its lanes.
template <typename V>
__device__ __forceinline__ V group_max(V v) {
  v = fmax(v, rotated<8>(v));
  v = fmax(v, rotated<4>(v));
  v = fmax(v, rotated<2>(v));
  return fmax(v, rotated<1>(v));
}

// The codes of a group of p inv / scale, p = s gamma, in 64 bits, from its inputs (x + residual may not fit 32).  A quotient 448 p / max p is first made in 32 bits;
// which side of the border between the two codes around it the exact one lies on, or whether on the border itself, is the sign of
// 448 p - border max p, exact where s has 24 bits.  wide: p may lie outside of what fp32 holds well, and the group's largest |n| and its scale are
// made here as well.  All lanes of the group take part.
// Products are made for each use: whatever is held here are registers of the whole kernel.
template <typename T>
__device__ __forceinline__ void exact_codes(i32x4 x, i32x4 residual, bool add, const float (&g)[8], float inv, bool wide, float& top, float& scale,
                                            uint32_t (&codes)[2]) {
  auto product = [&](int e) {
    typedef __attribute__((__vector_size__(8 * sizeof(T)))) T vec8;
    const double a = (double)(float)__builtin_bit_cast(vec8, x)[e], b = (double)(float)__builtin_bit_cast(vec8, residual)[e];
    float weight = g[e];
    asm volatile("" : "+v"(weight));
    return (add ? a + b : a) * (double)weight;
  };
  double amax = 0.0;
#pragma unroll
  for (int e = 0; e < 8; ++e) amax = fmax(amax, fabs(product(e)));
  amax = group_max(amax);
  if (wide) {
    float by = inv;
    asm volatile("" : "+v"(by));
    top = (float)(amax * (double)by);
    scale = group_scale(top);
  }
  auto encode = [&](auto quotient) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      asm volatile("" : "+v"(x), "+v"(residual));
      const float q0 = quotient(4 * h), q1 = quotient(4 * h + 1), q2 = quotient(4 * h + 2), q3 = quotient(4 * h + 3);
      codes[h] = codes4(q0, q1, q2, q3);
    }
  };
  // a row that is normalised to zeros or to NaN, and one that is divided by the least scale that there is
  const bool none = !(top > 0.f) || amax > 0x1.fffffffffffffp1023, special = none || top < 448.f * 0x1p-126f;
  if (!special) {
    const int exponent = __builtin_amdgcn_frexp_exp(amax);
    amax = ldexp(amax, -exponent);  // 1/2 to 1
    const float r = 448.f * GroupQuotient((float)amax).r;
    encode([&](int e) {
      const double v = product(e), size = ldexp(fabs(v), -exponent);
      const float near = (float)size * r;
      const bool low = near < 0x1p-6f;  // (there 32 |q| + 1/2 has the borders where larger ones have them)
      float border = low ? fminf(fmaf(near, 32.f, 0.5f), 0x1.fffffep-1f) : near;
      border = __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, border) & ~0xfffffu) | 0x80000u);
      border = low ? (border - 0.5f) * 0x1p-5f : border;
      const double past = fma(448.0, size, -((double)border * amax));
      const uint32_t side = __builtin_bit_cast(uint32_t, border) + (uint32_t)(past > 0.0) - (uint32_t)(past < 0.0);
      return copysignf(__builtin_bit_cast(float, side), (float)v);
    });
  } else {
    const float times = none ? inv * 0.f : inv;
    encode([&](int e) {
      float by = times;
      asm volatile("" : "+v"(by));
      return (float)(ldexp(product(e), 126) * (double)by);
    });
  }
}

// sum_out and normed_out may be x or residual themselves: a thread writes the columns that it alone reads, behind its last use of them.
template <typename T, bool NORM, bool STREAM, int VECS>
__global__ __launch_bounds__(kThreads, VECS <= 2 ? 8 : 2) void norm_fp8_block_kernel(const T* x, const T* residual, const float* __restrict__ gamma,
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
  auto store_sum = [&](int u) {
    const int i = threadIdx.x + u * kThreads;
    vec8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)s[u][e];
    if (i < nvec) store<STREAM>(reinterpret_cast<vec8*>(sum_out + row * cols) + i, v);
  };
  const bool in_place = sum_out == x || sum_out == residual;  // the exact codes read both again
  if (NORM && sum_out && !in_place) {
#pragma unroll
    for (int u = 0; u < VECS; ++u) store_sum(u);
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
    amax = group_max(amax);
    float top = NORM ? amax * inv : amax, sc = group_scale(top);
    uint32_t word[2];
    if constexpr (NORM) {
      // n / scale is 448 t / max t: the row's statistic cancels
      const float r = amax > 0.f ? 448.f * GroupQuotient(amax).r : inv * 0.f;  // (a statistic that is not finite: NaN)
      const bool wide = amax > 0.f && !(amax > 0x1p-90f && amax < 0x1p90f);
      bool exact = amax > 0.f && (wide || !(top >= 448.f * 0x1p-126f));
      // Within 7 steps of the 24-bit format of a border between two codes: the roundings so far, seven of 2^-24, are less.  A border lies
      // where the last 20 bits are 0x80000; below 2^-6, where codes lie 2^-9 apart, of 32 |q| + 1/2 (larger ones are 1 there: no border).
      constexpr uint32_t kReach = 7;
      auto past = [](float v) { return (__builtin_bit_cast(uint32_t, v) << 12) - ((0x80000u - kReach) << 12); };
      uint32_t nearest = ~0u;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        q[e] = t[e] * r;
        nearest = min(nearest, min(past(q[e]), past(__builtin_amdgcn_fmed3f(fmaf(fabsf(q[e]), 32.f, 0.5f), 0.f, 1.f))));
      }
      exact |= nearest <= (2 * kReach) << 12;
      word[0] = codes4(q[0], q[1], q[2], q[3]), word[1] = codes4(q[4], q[5], q[6], q[7]);
      if (__builtin_expect(__ballot(exact) != 0, 0)) {
        const vec8 *xa = xr, *ra = rr;
        asm volatile("" : "+s"(xa), "+s"(ra));  // (read again: kept since the start they would be registers of the whole kernel)
        vec8 a = {}, b = {};
        if (i < nvec) {
          a = xa[i];
          if (ra) b = ra[i];
        }
        exact_codes<T>(__builtin_bit_cast(i32x4, a), __builtin_bit_cast(i32x4, b), rr != nullptr, g[u], inv, wide, top, sc, word);
      }
      if (normed_out) {
        vec8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          asm volatile("" : "+v"(s[u][e]));  // (not held over the branch)
          v[e] = (T)(s[u][e] * g[u][e] * inv);
        }
        if (__builtin_expect(__ballot(wide) != 0, 0)) {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = wide ? (T)(float)((double)s[u][e] * (double)inv * (double)g[u][e]) : v[e];
        }
        if (i < nvec) store<STREAM>(reinterpret_cast<vec8*>(normed_out + row * cols) + i, v);
      }
    } else {
      const GroupQuotient quotient(sc);
#pragma unroll
      for (int e = 0; e < 8; ++e) q[e] = quotient(t[e]);
      word[0] = codes4(q[0], q[1], q[2], q[3]), word[1] = codes4(q[4], q[5], q[6], q[7]);
    }
    if (NORM && sum_out && in_place) store_sum(u);
    if (i < nvec) {
      store<STREAM>(crow + i, u32x2{word[0], word[1]});
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
