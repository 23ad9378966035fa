// Shared pieces of the pair-stream kernels (pair_norm.cu, pair_norm_grad.cu, pair_embed.cu): groups of eight
// channels in registers, the row walk over strided (b, i, j, d) tensors, and the dropout's generator.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "../../include/pair_stream_sm100.h"

namespace trimul {
int report_error(int code, const char* fmt, ...);  // sets trimul_sm100_last_error() and returns `code`
int current_device_sms();
}  // namespace trimul

namespace pair {

// ---------------------------------------------------------------------------------------------
// units: the channels that one memory access of a lane moves
// ---------------------------------------------------------------------------------------------
// Rows that start on 16-byte boundaries and have whole octs are moved in units of eight channels (16 bytes of a 16-bit
// type, 32 of fp32).  All others are moved in units of two 16-bit channels where rows start on 4-byte boundaries, of four fp32 where the
// addition alone finds 16-byte ones, else of one channel: a warp's accesses are then still contiguous, where groups of eight at odd
// addresses would make each access of a warp touch every line of the row.  Such rows are bound by the instructions that move them:
// the norm of 80000 fp16 rows with a residual takes 11 us at 128 channels, 22 at 130 and at 131 (alone 9, 19 and 18); of fp32 rows 28 and 36.
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

template <typename T, int kU>
struct alignas(sizeof(T) * kU < 16 ? sizeof(T) * kU : 16) Unit {
  T e[kU];
};

// Loads carry the streaming hint: every activation is read once.
template <typename T, int kU>
__device__ __forceinline__ Unit<T, kU> load_unit(const T* p) {
  Unit<T, kU> o;
  constexpr int kBytes = sizeof(T) * kU;
  if constexpr (kBytes == 32) {
    // (the alignment of a row is 16 bytes)
    uint4* w = reinterpret_cast<uint4*>(&o);
    w[0] = __ldcs(reinterpret_cast<const uint4*>(p));
    w[1] = __ldcs(reinterpret_cast<const uint4*>(p) + 1);
  } else if constexpr (kBytes == 16) {
    *reinterpret_cast<uint4*>(&o) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else if constexpr (kBytes == 4) {
    *reinterpret_cast<uint32_t*>(&o) = __ldcs(reinterpret_cast<const uint32_t*>(p));
  } else {
    static_assert(kBytes == 2, "a unit is 2, 4, 16 or 32 bytes");
    *reinterpret_cast<uint16_t*>(&o) = __ldcs(reinterpret_cast<const uint16_t*>(p));
  }
  return o;
}

template <typename T, int kU>
__device__ __forceinline__ void store_unit(T* p, const Unit<T, kU>& o) {
  constexpr int kBytes = sizeof(T) * kU;
  if constexpr (kBytes >= 16) {
    const uint4* w = reinterpret_cast<const uint4*>(&o);
#pragma unroll
    for (int k = 0; k < kBytes / 16; ++k) __stcs(reinterpret_cast<uint4*>(p) + k, w[k]);
  } else if constexpr (kBytes == 4) {
    __stcs(reinterpret_cast<uint32_t*>(p), *reinterpret_cast<const uint32_t*>(&o));
  } else {
    __stcs(reinterpret_cast<uint16_t*>(p), *reinterpret_cast<const uint16_t*>(&o));
  }
}

// Asynchronous copies of a lane's own units into its own slots of shared memory, read back by the same lane: bytes in flight that
// cost no registers, and no barrier (cp.async groups complete per thread).
template <typename T, int kU>
__device__ __forceinline__ void stage_unit(void* slot, const T* p) {
  constexpr int kBytes = sizeof(T) * kU;
  static_assert(kBytes == 4 || kBytes == 16, "cp.async moves 4 or 16 bytes here");
  const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(slot));
  if constexpr (kBytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(p) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(p) : "memory");
}
template <typename T, int kU>
__device__ __forceinline__ Unit<T, kU> staged_unit(const void* slot) {
  return *static_cast<const Unit<T, kU>*>(slot);
}
__device__ __forceinline__ void stage_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kPending>
__device__ __forceinline__ void stage_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kPending) : "memory"); }

// Which rows travel that way: not octs of fp32, whose two 16-byte halves would each touch every sector of the row, where direct loads
// find the second half in L1 (131072 rows of 256 channels: 95 against 126 us), nor 2-byte units, which cp.async does not know
// (copying the 4-byte words under them takes more instructions than the loads do: 80000 rows of 131 channels without a residual 26 against 17 us).
template <typename T, int kU, int kGroup, int kUnits>
struct Rows {
  static constexpr int kWide = kGroup <= 32 ? 256 : kGroup;  // threads of the CTA
  static constexpr int kBytes = sizeof(T) * kU;
  static constexpr bool kStaged = kBytes == 4 || kBytes == 16;
  static constexpr int kStage = kStaged ? kUnits * kWide * kBytes : 0;  // shared memory of one row of every group

  // Begins to copy this lane's units of a row into a stage.
  static __device__ __forceinline__ void fetch(char* stage, const T* row, int d) {
    if constexpr (kStaged) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int c = (threadIdx.x % kGroup + k * kGroup) * kU;
        if (c < d) stage_unit<T, kU>(stage + k * kWide * kBytes + threadIdx.x * kBytes, row + c);
      }
    }
  }
  static __device__ __forceinline__ Unit<T, kU> read(const char* stage, int k) {
    return staged_unit<T, kU>(stage + k * kWide * kBytes + threadIdx.x * kBytes);
  }
};

template <typename T, int kU>
__device__ __forceinline__ Unit<T, kU> zero_unit() {
  Unit<T, kU> o;
#pragma unroll
  for (int k = 0; k < kU; ++k) o.e[k] = from_f32<T>(0.f);
  return o;
}

// The fp32 values of all units of a lane in pairs, for the packed fp32 instructions (one issue slot for two operations): channels
// of a unit, or, of one-channel units, two steps' units.
template <int kU, int kUnits>
struct Lane {
  static constexpr int kPairs = kU * kUnits / 2;
  static_assert(kU * kUnits % 2 == 0, "one-channel units come in even numbers");
  float2 p[kPairs];
};

template <typename T, int kU, int kUnits>
__device__ __forceinline__ Lane<kU, kUnits> unpack_all(const Unit<T, kU> (&u)[kUnits]) {
  Lane<kU, kUnits> v;
#pragma unroll
  for (int n = 0; n < v.kPairs; ++n) {
    v.p[n].x = to_f32(u[2 * n / kU].e[2 * n % kU]);
    v.p[n].y = to_f32(u[(2 * n + 1) / kU].e[(2 * n + 1) % kU]);
  }
  return v;
}

template <typename T, int kU, int kUnits>
__device__ __forceinline__ void pack_all(const Lane<kU, kUnits>& v, Unit<T, kU> (&u)[kUnits]) {
#pragma unroll
  for (int n = 0; n < v.kPairs; ++n) {
    if constexpr (sizeof(T) == 2 && kU > 1) {
      if constexpr (__is_same(T, __half))
        reinterpret_cast<__half2*>(&u[2 * n / kU])[n % (kU / 2)] = __float22half2_rn(v.p[n]);
      else
        reinterpret_cast<__nv_bfloat162*>(&u[2 * n / kU])[n % (kU / 2)] = __float22bfloat162_rn(v.p[n]);
    } else {
      u[2 * n / kU].e[2 * n % kU] = from_f32<T>(v.p[n].x);
      u[(2 * n + 1) / kU].e[(2 * n + 1) % kU] = from_f32<T>(v.p[n].y);
    }
  }
}

// One oct.
template <typename T>
__device__ __forceinline__ Lane<8, 1> unpack(const Unit<T, 8>& o) {
  const Unit<T, 8> u[1] = {o};
  return unpack_all<T, 8, 1>(u);
}
template <typename T>
__device__ __forceinline__ Unit<T, 8> pack(const Lane<8, 1>& v) {
  Unit<T, 8> u[1];
  pack_all<T, 8, 1>(v, u);
  return u[0];
}

// The library is built to flush fp32 subnormals.  What becomes the stream (sums, kept elements, embeddings) keeps them, in packed
// pairs like the rest; what is computed from it (statistics, norms, gradients' sums) does not.
__device__ __forceinline__ float2 add_whole(float2 a, float2 b) {
  float2 r;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 mul_whole(float2 a, float2 b) {
  float2 r;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)));
  return r;
}
__device__ __forceinline__ float2 fma_whole(float2 a, float2 b, float2 c) {
  float2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(r))
      : "l"(reinterpret_cast<const uint64_t&>(a)), "l"(reinterpret_cast<const uint64_t&>(b)), "l"(reinterpret_cast<const uint64_t&>(c)));
  return r;
}
__device__ __forceinline__ float add_whole(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float mul_whole(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float fma_whole(float a, float b, float c) {
  float r;
  asm("fma.rn.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// a + b in the unit's type, rounded once: for 16-bit pairs the packed addition, which rounds the exact sum.
template <typename T, int kU>
__device__ __forceinline__ Unit<T, kU> add_units(const Unit<T, kU>& a, const Unit<T, kU>& b) {
  Unit<T, kU> o;
  if constexpr (sizeof(T) == 2 && kU > 1) {
#pragma unroll
    for (int k = 0; k < kU / 2; ++k) {
      if constexpr (__is_same(T, __half))
        reinterpret_cast<__half2*>(&o)[k] = __hadd2_rn(reinterpret_cast<const __half2*>(&a)[k], reinterpret_cast<const __half2*>(&b)[k]);
      else
        reinterpret_cast<__nv_bfloat162*>(&o)[k] =
            __hadd2_rn(reinterpret_cast<const __nv_bfloat162*>(&a)[k], reinterpret_cast<const __nv_bfloat162*>(&b)[k]);
    }
  } else {
#pragma unroll
    for (int k = 0; k < kU; ++k) o.e[k] = from_f32<T>(add_whole(to_f32(a.e[k]), to_f32(b.e[k])));
  }
  return o;
}

__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

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

// The gain's values of a lane's channels; 0 behind the row's end.
template <int kU, int kGroup, int kUnits>
__device__ __forceinline__ Lane<kU, kUnits> load_gain(const void* weight, int dtype, int lane, int units) {
  Lane<kU, kUnits> w;
#pragma unroll
  for (int c = 0; c < kU * kUnits; ++c) {
    const int n = lane + c / kU * kGroup;
    const float f = n < units ? load_any(weight, n * kU + c % kU, dtype) : 0.f;
    (c & 1 ? w.p[c / 2].y : w.p[c / 2].x) = f;
  }
  return w;
}

// ---------------------------------------------------------------------------------------------
// rows of a strided tensor
// ---------------------------------------------------------------------------------------------
// Quotient by a divisor fixed at launch: with l = ceil(log2 d) and m = ceil(2^(31+l) / d) < 2^32 the product n m
// exceeds n 2^(31+l) / d by less than n d / d <= 2^31 <= 2^(31+l) / d, so floor(n m / 2^(31+l)) = floor(n / d) for
// 0 <= n < 2^31.
struct FastDiv {
  uint32_t m, shift, d;
  __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
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
  // rows of a tensor whose b, i and j axes collapse into one
  __device__ __forceinline__ const T* flat(uint32_t row) const { return p + static_cast<int64_t>(row) * sj; }
  __device__ __forceinline__ const T* row(uint32_t b, uint32_t i, uint32_t j) const {
    return p + (static_cast<int64_t>(b) * sb + static_cast<int64_t>(i) * si + static_cast<int64_t>(j) * sj);
  }
};

template <typename T>
inline Strided<T> strided(const pair_tensor_t* t) {
  if (t == nullptr) return Strided<T>{nullptr, 0, 0, 0};
  return Strided<T>{static_cast<const T*>(t->data), t->stride_b, t->stride_i, t->stride_j};
}

// A tensor as the kernels and the rules below take it.  An axis of one entry is never stepped along, and what its stride holds (a slice
// keeps that of the whole tensor) says nothing about alignment: it becomes the stride that lets rows lie one behind another.
inline pair_tensor_t canonical(const pair_tensor_t* t, int bb, int ii, int jj) {
  if (t == nullptr || t->data == nullptr) return pair_tensor_t{nullptr, 0, 0, 0};
  pair_tensor_t c = *t;
  if (jj == 1) c.stride_j = ii != 1 ? c.stride_i : bb != 1 ? c.stride_b : 0;
  if (ii == 1) c.stride_i = c.stride_j * jj;
  if (bb == 1) c.stride_b = c.stride_i * ii;
  return c;
}

// Whether row * stride_j reaches every row of a canonical tensor.
inline bool collapses(const pair_tensor_t* t, int ii, int jj) {
  return t->data == nullptr || (t->stride_i == t->stride_j * jj && t->stride_b == t->stride_i * ii);
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

// The four words of oct `oct` (channels 8 oct ...) of position (b, i, j) of this block.
__device__ __forceinline__ uint4 draw_oct(const Dropout& d, uint32_t b, uint32_t i, uint32_t j, uint32_t oct) {
  const uint32_t ci = d.shared == PAIR_SHARED_ROWS ? 0u : i + d.i0;
  const uint32_t cj = d.shared == PAIR_SHARED_COLUMNS ? 0u : j + d.j0;
  return philox(((b + d.b0) << 16) | oct, cj, ci, d.offset, d.key0, d.key1);
}

// Dropout of the eight channels of an oct, four pairs.  `line` is keep << 16: the high half of a word is below keep exactly when
// the word is below that, the low half when the word shifted up is (keep is at most 65535 here).  A dropped element becomes
// 0 whatever it was (an infinity or NaN included): it is selected, and what is kept is multiplied.
__device__ __forceinline__ void drop_oct(const uint4 r, uint32_t line, float gain, float2* p) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    p[k].x = (w[k] << 16) < line ? p[k].x : 0.f;
    p[k].y = w[k] < line ? p[k].y : 0.f;
    p[k] = mul_whole(p[k], both(gain));
  }
}

// What an oct keeps, one bit per channel.
__device__ __forceinline__ uint32_t keep_bits(const uint4 r, uint32_t line) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  uint32_t bits = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    bits |= (((w[k] << 16) < line ? 1u : 0u) | (w[k] < line ? 2u : 0u)) << (2 * k);
  return bits;
}

// Narrow units: unit n of a row lies in oct n kU / 8, so the lanes of a warp would draw every oct 8 / kU times.  Instead they
// draw each oct of the warp's units once and hand the bits around.  `first` is the warp's first unit of step 0, step k begins
// kStep units further; afterwards the bits of unit (first + lane + k kStep) come from `narrow_bits`.
template <int kU, int kUnits>
struct NarrowMask {
  static constexpr int kPer = 4 * kU;                             // octs of a warp's 32 units
  static constexpr int kSlots = (kUnits * kPer + 31) / 32;        // octs a lane draws
  uint32_t bits[(kSlots + 3) / 4];
};

template <int kU, int kUnits, int kStep>
__device__ __forceinline__ NarrowMask<kU, kUnits> draw_narrow(const Dropout& d, uint32_t line, uint32_t b, uint32_t i, uint32_t j,
                                                              int first, int octs) {
  NarrowMask<kU, kUnits> m;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 0; s < (m.kSlots + 3) / 4; ++s) m.bits[s] = 0;
#pragma unroll
  for (int s = 0; s < m.kSlots; ++s) {
    const int q = lane + 32 * s;
    const int oct = (first + q / m.kPer * kStep) * kU / 8 + q % m.kPer;
    if (q < kUnits * m.kPer && oct < octs) m.bits[s / 4] |= keep_bits(draw_oct(d, b, i, j, oct), line) << (8 * (s & 3));
  }
  return m;
}

// The bits of the lane's unit of step k, lowest channel first.  Every lane of the warp takes part.
template <int kU, int kUnits>
__device__ __forceinline__ uint32_t narrow_bits(const NarrowMask<kU, kUnits>& m, int k) {
  const int lane = threadIdx.x & 31;
  const int q = m.kPer * k + lane * kU / 8;  // kPer is 4, 8 or 16, so all lanes share the slot q / 32
  const int slot = m.kPer * k / 32;
  const uint32_t byte = (__shfl_sync(0xffffffffu, m.bits[slot / 4], q & 31) >> (8 * (slot & 3))) & 0xffu;
  return byte >> (lane * kU % 8);
}

// Dropout of all units of a lane.  `lane` is the lane of its group; every lane of the warp takes part.
template <int kU, int kGroup, int kUnits>
__device__ __forceinline__ void drop_all(const Dropout& d, uint32_t line, uint32_t b, uint32_t i, uint32_t j, int lane, int octs,
                                         Lane<kU, kUnits>& v) {
  if constexpr (kU == 8) {
#pragma unroll
    for (int k = 0; k < kUnits; ++k) drop_oct(draw_oct(d, b, i, j, lane + k * kGroup), line, d.gain, v.p + 4 * k);
  } else {
    const auto mask = draw_narrow<kU, kUnits, kGroup>(d, line, b, i, j, lane & ~31, octs);
#pragma unroll
    for (int n = 0; n < v.kPairs; ++n) {
      const uint32_t x = narrow_bits<kU, kUnits>(mask, 2 * n / kU) >> (2 * n % kU);
      const uint32_t y = kU > 1 ? x >> 1 : narrow_bits<kU, kUnits>(mask, 2 * n + 1);
      // one by one: packed, the compiler joins this product and the residual's addition, and rows on other boundaries would round otherwise
      v.p[n].x = x & 1u ? mul_whole(v.p[n].x, d.gain) : 0.f;
      v.p[n].y = y & 1u ? mul_whole(v.p[n].y, d.gain) : 0.f;
    }
  }
}

// ---------------------------------------------------------------------------------------------
// sums over the lanes that share a row
// ---------------------------------------------------------------------------------------------
// A row has kGroup lanes: 8, 16 or 32 of a warp, or a CTA of its own of 64 to 1024 threads.
constexpr int kThreads = 256;
__host__ __device__ constexpr int threads_of(int group) { return group <= 32 ? kThreads : group; }

template <bool kMax>
__device__ __forceinline__ float merge(float a, float b) { return kMax ? fmaxf(a, b) : a + b; }

// Sums (or maxima) of kN values over the lanes of a row; every lane of the warp takes part, every lane gets the results.
// `buf` holds 2 x 32 x kN floats for the CTA form and alternates with `parity`, so that one barrier per call is enough: a
// warp that writes one half again has passed the barrier of the call between, and so have the readers of that half.
template <int kGroup, int kN, bool kMax>
__device__ __forceinline__ void group_merge(float (&v)[kN], float* buf, int parity) {
  constexpr int kLanes = kGroup < 32 ? kGroup : 32;
#pragma unroll
  for (int o = kLanes / 2; o > 0; o >>= 1)
#pragma unroll
    for (int n = 0; n < kN; ++n) v[n] = merge<kMax>(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
  if constexpr (kGroup > 32) {
    constexpr int kWarps = kGroup / 32;
    float* b = buf + parity * 32 * kN;
    const int lane = threadIdx.x & 31;
    if (lane == 0)
#pragma unroll
      for (int n = 0; n < kN; ++n) b[(threadIdx.x >> 5) * kN + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < kN; ++n) v[n] = b[(lane % kWarps) * kN + n];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
#pragma unroll
      for (int n = 0; n < kN; ++n) v[n] = merge<kMax>(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
  }
}

template <int kGroup, int kN>
__device__ __forceinline__ void group_sum(float (&v)[kN], float* buf, int parity) {
  group_merge<kGroup, kN, false>(v, buf, parity);
}
template <int kGroup, int kN>
__device__ __forceinline__ void group_max(float (&v)[kN], float* buf, int parity) {
  group_merge<kGroup, kN, true>(v, buf, parity);
}

// Launches.  The kernels of one call follow one another: each but the last says at its start that the next may be set up while it
// runs (next_may_start), and the next waits at its start for it to end, its results included (behind_previous).  That hides the
// launch of all but the first.  The last says nothing: what follows the call sees an ordinary kernel.
// A kernel that waits here may be running while the kernels before it still write, and a chain may write a buffer twice: what they write is
// read by ordinary loads (or __ldcg) behind the wait, never by __ldg, which is for memory that nobody writes while the kernel lives
// and which the compiler may move above the wait.
__device__ __forceinline__ void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void behind_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <bool kBehind, typename K, typename... A>
cudaError_t launch_kernel(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = stream;
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &early;
  c.numAttrs = kBehind ? 1 : 0;
  return cudaLaunchKernelEx(&c, kernel, args...);
}
template <typename K, typename... A>
cudaError_t launch(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, A... args) {
  return launch_kernel<false>(kernel, grid, threads, smem, stream, args...);
}
// Behind a kernel of the same call; the kernel begins with behind_previous().
template <typename K, typename... A>
cudaError_t launch_behind(K kernel, dim3 grid, unsigned threads, size_t smem, cudaStream_t stream, A... args) {
  return launch_kernel<true>(kernel, grid, threads, smem, stream, args...);
}

// CTAs of a kernel that an SM holds at once (at least one).
template <typename K>
int resident_ctas(K kernel, int threads, int smem) {
  int n = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, smem) != cudaSuccess) {
    cudaGetLastError();
    n = 1;
  }
  return n < 1 ? 1 : n;
}

// The grid of a kernel whose CTAs walk over `need` steps in all: one wave of the `resident` CTAs an SM that fit, or as many whole waves
// as leave each CTA about `steps` steps.  A single wave of equal shares ends with its slowest SM (a profile of one showed the others
// idle for a fifth of the time); CTAs of a later wave go where one is done.
inline unsigned walk_grid(uint64_t need, int sms, int resident, uint32_t steps) {
  const uint64_t wave = static_cast<uint64_t>(sms) * resident;
  if (need <= wave) return static_cast<unsigned>(need);
  const uint64_t waves = (need / steps + wave / 2) / wave;
  return static_cast<unsigned>(waves > 1 ? waves * wave : wave);
}

// Host-side checks shared by the entry points.
int check_norm_desc(const pair_norm_desc_t* d, const char* who);
int check_dtype(int dtype, const char* what, const char* who);

inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
// every row of the tensor starts on a multiple of `bytes`
inline bool rows_aligned(const pair_tensor_t* t, int type_size, int bytes) {
  if (t == nullptr || t->data == nullptr) return true;
  const int64_t m = bytes / type_size;
  return aligned(t->data, bytes) && t->stride_b % m == 0 && t->stride_i % m == 0 && t->stride_j % m == 0;
}

// Whether every tensor of a call starts (and every row of a strided one) on a multiple of its elements.
inline bool elements_aligned(int type_size, std::initializer_list<const pair_tensor_t*> strided, std::initializer_list<const void*> flat) {
  for (const pair_tensor_t* t : strided)
    if (t != nullptr && !aligned(t->data, type_size)) return false;
  for (const void* p : flat)
    if (!aligned(p, type_size)) return false;
  return true;
}

// Whether every row of a call's tensors can be moved in units of so many channels.
inline bool units_fit(int unit, int d, int type_size, std::initializer_list<const pair_tensor_t*> strided,
                      std::initializer_list<const void*> flat) {
  const int bytes = unit * type_size < 16 ? unit * type_size : 16;
  if (d % unit != 0) return false;
  for (const pair_tensor_t* t : strided)
    if (!rows_aligned(t, type_size, bytes)) return false;
  for (const void* p : flat)
    if (!aligned(p, bytes)) return false;
  return true;
}

// Channels per memory access that every tensor of a call allows: 8, 2 (16-bit types) or 1.
inline int unit_of(int d, int type_size, std::initializer_list<const pair_tensor_t*> strided, std::initializer_list<const void*> flat) {
  if (units_fit(8, d, type_size, strided, flat)) return 8;
  return type_size == 2 && units_fit(2, d, type_size, strided, flat) ? 2 : 1;
}

}  // namespace pair
