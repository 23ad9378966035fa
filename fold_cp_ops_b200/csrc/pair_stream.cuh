// Shared pieces of the pair-stream kernels (pair_norm.cu, pair_norm_grad.cu, pair_embed.cu): groups of eight
// channels in registers, the row walk over strided (b, i, j, d) tensors, and the dropout's generator.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/pair_stream_sm100.h"

namespace trimul {
int report_error(int code, const char* fmt, ...);  // sets trimul_sm100_last_error() and returns `code`
int current_device_sms();
}  // namespace trimul

namespace pair {

// ---------------------------------------------------------------------------------------------
// eight channels of one row
// ---------------------------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Raw storage of eight elements: 16 bytes for the 16-bit types, 32 for fp32.
template <typename T>
struct alignas(16) Oct {
  T e[8];
};

// `kWide`: the address is 16-byte aligned and all eight channels exist (one or two 16-byte accesses); otherwise the
// first n channels are moved one by one.  Loads carry the streaming hint: every activation is read once.
template <bool kWide, typename T>
__device__ __forceinline__ Oct<T> load_oct(const T* p, int n) {
  Oct<T> o;
  if constexpr (kWide) {
    uint4* w = reinterpret_cast<uint4*>(&o);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(o) / 16); ++k) w[k] = __ldcs(reinterpret_cast<const uint4*>(p) + k);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k) o.e[k] = k < n ? p[k] : from_f32<T>(0.f);
  }
  return o;
}

template <bool kWide, typename T>
__device__ __forceinline__ void store_oct(T* p, const Oct<T>& o, int n) {
  if constexpr (kWide) {
    const uint4* w = reinterpret_cast<const uint4*>(&o);
#pragma unroll
    for (int k = 0; k < static_cast<int>(sizeof(o) / 16); ++k) __stcs(reinterpret_cast<uint4*>(p) + k, w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (k < n) p[k] = o.e[k];
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const Oct<T>& o, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = to_f32(o.e[k]);
}

template <typename T>
__device__ __forceinline__ Oct<T> pack(const float (&f)[8]) {
  Oct<T> o;
#pragma unroll
  for (int k = 0; k < 8; ++k) o.e[k] = from_f32<T>(f[k]);
  return o;
}

template <typename T>
__device__ __forceinline__ Oct<T> zero_oct() {
  Oct<T> o;
#pragma unroll
  for (int k = 0; k < 8; ++k) o.e[k] = from_f32<T>(0.f);
  return o;
}

// One value of a tensor whose type is known at run time only (gains: read once per CTA).
__device__ __forceinline__ float load_any(const void* p, int64_t at, int dtype) {
  if (dtype == PAIR_FP32) return static_cast<const float*>(p)[at];
  if (dtype == PAIR_FP16) return __half2float(static_cast<const __half*>(p)[at]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[at]);
}
__device__ __forceinline__ void store_any(void* p, int64_t at, int dtype, float v) {
  if (dtype == PAIR_FP32)
    static_cast<float*>(p)[at] = v;
  else if (dtype == PAIR_FP16)
    static_cast<__half*>(p)[at] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[at] = __float2bfloat16_rn(v);
}

inline int type_bytes(int dtype) { return dtype == PAIR_FP32 ? 4 : 2; }

// ---------------------------------------------------------------------------------------------
// rows of a strided tensor
// ---------------------------------------------------------------------------------------------
// Quotient by a divisor fixed at launch: with l = ceil(log2 d) and m = ceil(2^(31+l) / d) < 2^32 the product n m
// exceeds n 2^(31+l) / d by less than n d / d <= 2^31 <= 2^(31+l) / d, so floor(n m / 2^(31+l)) = floor(n / d) for
// 0 <= n < 2^31.
struct FastDiv {
  uint32_t m, shift, d;
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * m) >> shift);
  }
};
inline FastDiv make_fast_div(uint32_t d) {
  uint32_t l = 0;
  while ((1ull << l) < d) ++l;
  return FastDiv{static_cast<uint32_t>(((1ull << (31 + l)) + d - 1) / d), 31 + l, d};
}

// Where a row lies: row = (b * I + i) * J + j.
struct RowWalk {
  FastDiv by_j, by_i;
  __device__ __forceinline__ void at(uint32_t row, uint32_t& b, uint32_t& i, uint32_t& j) const {
    const uint32_t line = by_j.div(row);
    j = row - line * by_j.d;
    b = by_i.div(line);
    i = line - b * by_i.d;
  }
};

template <typename T>
struct Strided {
  const T* p;
  int64_t sb, si, sj;
  __device__ __forceinline__ const T* row(uint32_t b, uint32_t i, uint32_t j) const {
    return p + (static_cast<int64_t>(b) * sb + static_cast<int64_t>(i) * si + static_cast<int64_t>(j) * sj);
  }
};

template <typename T>
inline Strided<T> strided(const pair_tensor_t* t) {
  if (t == nullptr) return Strided<T>{nullptr, 0, 0, 0};
  return Strided<T>{static_cast<const T*>(t->data), t->stride_b, t->stride_i, t->stride_j};
}

// ---------------------------------------------------------------------------------------------
// dropout
// ---------------------------------------------------------------------------------------------
struct Dropout {
  uint32_t key0, key1, offset, keep;
  const uint64_t* device_seed;
  int shared;
  uint32_t b0, i0, j0;
  float gain;  // 65536 / keep
};

inline Dropout make_dropout(const pair_dropout_t& d) {
  Dropout o;
  o.key0 = static_cast<uint32_t>(d.seed);
  o.key1 = static_cast<uint32_t>(d.seed >> 32);
  o.offset = d.offset;
  o.keep = d.keep;
  o.device_seed = d.device_seed;
  o.shared = d.shared;
  o.b0 = static_cast<uint32_t>(d.origin_b);
  o.i0 = static_cast<uint32_t>(d.origin_i);
  o.j0 = static_cast<uint32_t>(d.origin_j);
  o.gain = d.keep == 0 ? 0.f : 65536.f / static_cast<float>(d.keep);
  return o;
}

// A seed that lives in device memory is read by the kernel, so that a replayed graph draws a new mask.
__device__ __forceinline__ void resolve_seed(Dropout& d) {
  if (d.device_seed != nullptr) {
    const uint64_t seed = d.device_seed[0];
    d.key0 = static_cast<uint32_t>(seed);
    d.key1 = static_cast<uint32_t>(seed >> 32);
    d.offset = static_cast<uint32_t>(d.device_seed[1]);
  }
}

// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011): 128 bits of a
// 128-bit counter.  One call serves eight channels, 16 bits each: a keep probability is a multiple of 2^-16 and the
// gain is its exact reciprocal, so the expectation stays what it was.
__device__ __forceinline__ uint4 philox(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0, uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = static_cast<uint64_t>(c0) * 0xD2511F53u;
    const uint64_t p1 = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(p1 >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(p1);
    c2 = static_cast<uint32_t>(p0 >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(p0);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

// A dropped element becomes 0 whatever it was (an infinity or NaN included): selected, not multiplied.
__device__ __forceinline__ void apply_dropout(const Dropout& d, uint32_t b, uint32_t i, uint32_t j, uint32_t oct,
                                              float (&f)[8]) {
  const uint32_t ci = d.shared == PAIR_SHARED_ROWS ? 0u : i + d.i0;
  const uint32_t cj = d.shared == PAIR_SHARED_COLUMNS ? 0u : j + d.j0;
  const uint4 r = philox(((b + d.b0) << 16) | oct, cj, ci, d.offset, d.key0, d.key1);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    f[2 * k] = (w[k] & 0xffffu) < d.keep ? f[2 * k] * d.gain : 0.f;
    f[2 * k + 1] = (w[k] >> 16) < d.keep ? f[2 * k + 1] * d.gain : 0.f;
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the lanes that share a row
// ---------------------------------------------------------------------------------------------
constexpr int kThreads = 256;

// kGroup <= 32: lanes of one warp; kGroup == kThreads: the CTA.  Every lane of the warp takes part, every lane gets
// the result.  `buf` holds 2 x 8 x kN floats for the CTA form and alternates with `parity`, so one barrier per call
// is enough: a warp can only be one call ahead of another.
template <int kGroup, int kN>
__device__ __forceinline__ void group_sum(float (&v)[kN], float* buf, int parity) {
  constexpr int kLanes = kGroup < 32 ? kGroup : 32;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < kN; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
  if constexpr (kGroup > 32) {
    float* b = buf + parity * 8 * kN;
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int n = 0; n < kN; ++n) b[warp * kN + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < kThreads / 32; ++w) s += b[w * kN + n];
      v[n] = s;
    }
  }
}

template <int kGroup>
__device__ __forceinline__ float group_max(float v, float* buf, int parity) {
  constexpr int kLanes = kGroup < 32 ? kGroup : 32;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  if constexpr (kGroup > 32) {
    float* b = buf + parity * 8;
    if ((threadIdx.x & 31) == 0) b[threadIdx.x >> 5] = v;
    __syncthreads();
    v = b[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) v = fmaxf(v, b[w]);
  }
  return v;
}

// Host-side checks shared by the entry points.
int check_norm_desc(const pair_norm_desc_t* d, const char* who);
int check_dtype(int dtype, const char* what, const char* who);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// every row of the tensor starts on a 16-byte boundary
inline bool rows_aligned(const pair_tensor_t* t, int bytes) {
  if (t == nullptr || t->data == nullptr) return true;
  const int64_t m = 16 / bytes;
  return aligned16(t->data) && t->stride_b % m == 0 && t->stride_i % m == 0 && t->stride_j % m == 0;
}

}  // namespace pair
