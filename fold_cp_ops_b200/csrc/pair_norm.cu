// z = residual + dropout(update) and y = rms_norm(z), in one pass over the rows of the pair stream.
//
// Mathematics.  u = keep ? x * 65536 / keep16 : 0;  z = round(r + u);  s = 1 / sqrt(mean_c z^2 + eps);
// y = z s w.  The norm reads the STORED z (rounded to the activations' type): y is then exactly what a later norm
// of the stream would give, and the gradient needs nothing but z.  The sum of squares and s are fp32.
// e4m3 output: a = max |y| over a group of channels, scale = a / 448, q = e4m3(y / scale) (see Quotient).
//
// Bound.  HBM: update and residual are read, z and y written once; nothing else moves.  Behind it come the issue slots: an SM has
// about 8 of them while the 48 to 64 bytes of a 16-bit oct move, for each of its lanes' shares, so the arithmetic is in packed
// fp32 pairs (and in packed 16-bit additions where there is no dropout).
// Split.  A row of up to 256 channels is one oct (eight channels, 16 bytes of a 16-bit type) per lane of 8, 16 or 32 lanes, so
// that the reductions stay inside a warp; up to 384 it is three octs of 16 lanes, up to 512 two of 32; wider rows take a CTA with
// one oct per thread.  CTAs walk over the rows, 64 channels a lane or one wave of CTAs (walk_grid); while one row of a lane is at hand
// the next is on its way through shared memory.
// Measured (of the 6457 GB/s of a copy): 1024 x 1024 rows of 256 bf16 channels to e4m3 293 us, 100 % (333 with one wave of CTAs); the
// addition alone with an elementwise dropout 267 us, 93 % (282); 512 x 512 fp32 rows of 256 169 us, 98 % (193); 384 x 384
// rows of 128 with dropout 31 us, 75 %: there the tensors are small and the fill and drain of the one wave or two show.
#include "pair_stream.cuh"

namespace pair {
namespace {

constexpr float kE4m3Max = 448.f;
// Channels that a lane of the norm takes, where there are enough for several waves: eight rows of an oct, three of three octs.  (To e4m3, 96 x 768
// rows of 384 take 37 us with two to four rows a lane and 40 with eight; 256 x 512 rows of 256 45 with three, 42 with eight.)
constexpr uint32_t kLaneChannels = 64;

enum Mode { kNorm = 0, kNormE4m3 = 1 };

template <typename T>
struct NormArgs {
  Strided<T> update, residual;
  const void* weight;
  T* stream;
  void* y;
  float* scales;
  RowWalk walk;
  Dropout drop;
  uint32_t rows;
  int d, octs;
  int weight_dtype;
  int scales_per_row;
  int scale_shift;  // log2 of the octs per scale; -1: the row has one scale
  int flat;   // the rows of update and residual lie at a constant distance
  float eps, inv_d;
};

__device__ __forceinline__ uint32_t e4m3x2(float2 v) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(v.y), "f"(v.x));
  return r;
}

// The e4m3 output.  With p = z w, exact for 16-bit z and w, y = p s; so scale = max|p| s / 448 and y / scale = p (448 / max|p|), from
// which s has gone.  Random bf16 rows have one quotient in some 2500 that lies exactly between two e4m3 values, and roundings
// before it would send it to either side.  448 / max|p| is held as the sum of an approximation and of what a fused product shows it to lack, good to
// 2^-44: a quotient that fp32 holds, as every tie is, then comes out exactly, every other within 2^-24 of it.  (1024 x 1024 rows of 256
// take 324 us, 321 with a product by an approximate 1 / scale, which misses ties, and 365 with divisions.)
struct Quotient {
  float scale, factor, lack;
  __device__ __forceinline__ float2 operator()(float2 p) const { return __ffma2_rn(p, both(factor), __fmul2_rn(p, both(lack))); }
};
__device__ __forceinline__ Quotient quotient_near(float top, float rstd) {
  const float inverse = 1.f / (top * (1.f / kE4m3Max));
  return Quotient{top * rstd * (1.f / kE4m3Max), inverse, __fmaf_rn(-inverse, top, kE4m3Max) * (inverse * (1.f / kE4m3Max))};
}
// Not for sizes far from 1, rows of zeros and rows without a norm.  (What is below 2^-126 beside a largest |p| of 2^-90 is 0 in e4m3.)
__device__ __forceinline__ bool is_near(float top, float rstd) { return top >= 0x1p-90f && top <= 3.4e38f && top * rstd >= 0x1p-100f; }

// The same for every size, from p = (z 2^k) w with s = 2^k rest, 1/2 <= rest < 1 (p is not flushed before y is): y / scale = p rest / scale,
// within 2^-21.
struct Parts {
  float power, rest;
};
__device__ __forceinline__ Parts parts_of(float rstd) {
  if (!(rstd > 0.f)) return Parts{rstd, 1.f};   // an infinity's row, a NaN's
  const uint32_t bits = __float_as_uint(rstd);  // normal: eps is
  return Parts{__uint_as_float((bits & 0x7f800000u) + 0x00800000u), __uint_as_float((bits & 0x007fffffu) | 0x3f000000u)};
}
__device__ __forceinline__ Quotient quotient_far(float top, float rest) {
  const float most = top * rest;
  const float scale = most > 0.f ? fmaxf(most * (1.f / kE4m3Max), 1.17549435e-38f) : 1.f;
  return Quotient{scale, 1.f / scale * rest, 0.f};
}

// round(r + dropout(u)) of one oct.
template <typename T>
__device__ __forceinline__ Unit<T, 8> drop_and_add(const Dropout& d, uint32_t line, uint32_t b, uint32_t i, uint32_t j, uint32_t oct,
                                                   const Unit<T, 8>& u, const Unit<T, 8>& r, bool has_residual) {
  Lane<8, 1> v = unpack(u);
  drop_oct(draw_oct(d, b, i, j, oct), line, d.gain, v.p);
  if (has_residual) {
    const Lane<8, 1> x = unpack(r);
#pragma unroll
    for (int e = 0; e < 4; ++e) v.p[e] = add_whole(v.p[e], x.p[e]);
  }
  return pack<T>(v);
}

// kU channels per access, kGroup lanes per row, kUnits units per lane.
template <typename T, int kU, int kGroup, int kUnits, int kMode>
__global__ void __launch_bounds__(threads_of(kGroup), (kUnits * kU > 16 ? 768 : 1024) / threads_of(kGroup)) add_norm_kernel(const __grid_constant__ NormArgs<T> a) {
  __shared__ float sums[2 * 32];
  __shared__ float tops[2 * 32];
  extern __shared__ uint4 ring[];
  constexpr int kWide = threads_of(kGroup);
  constexpr int kRows = kWide / kGroup;  // rows a CTA holds side by side
  constexpr int kPairs = kU * kUnits / 2;
  using In = Rows<T, kU, kGroup, kUnits>;
  const int lane = threadIdx.x % kGroup;
  const int units = a.d / kU;
  const bool dropping = a.drop.keep < 65536u;
  const bool has_residual = a.residual.p != nullptr;
  const uint32_t line = a.drop.keep << 16;
  Dropout drop = a.drop;
  if (dropping) resolve_seed(drop);

  const Lane<kU, kUnits> w = load_gain<kU, kGroup, kUnits>(a.weight, a.weight_dtype, lane, units);

  const uint32_t span = gridDim.x * kRows;
  const uint32_t mine = blockIdx.x * kRows + threadIdx.x / kGroup;  // this group's first row
  // rows at a constant distance are reached step by step, others by their (b, i, j)
  const T *next_u = a.update.flat(mine), *next_r = a.residual.flat(mine);
  const int64_t step_u = span * a.update.sj, step_r = span * a.residual.sj;
  auto next_rows = [&](uint32_t row, const T*& up, const T*& rp) {
    if (a.flat) {
      up = next_u, rp = next_r;
      next_u += step_u, next_r += step_r;
    } else if (row < a.rows) {
      uint32_t b, i, j;
      a.walk.at(row, b, i, j);
      up = a.update.row(b, i, j);
      rp = a.residual.row(b, i, j);
    }
  };
  // Two stages, one at hand and one on its way; each holds the update's row of every group, then the residual's.  (More are slower:
  // with one wave of CTAs 1024 x 1024 rows of 256 to e4m3 take 334 us with two, 357 with three or four.)
  const int stage_bytes = In::kStage * (has_residual ? 2 : 1);
  auto fetch = [&](uint32_t row, int stage) {
    const T *up, *rp;
    next_rows(row, up, rp);
    if (row < a.rows) {
      char* to = reinterpret_cast<char*>(ring) + stage * stage_bytes;
      In::fetch(to, up, a.d);
      if (has_residual) In::fetch(to + In::kStage, rp, a.d);
    }
    stage_commit();
  };
  if constexpr (In::kStaged) fetch(mine, 0);

  int parity = 0;
  const int64_t out_step = static_cast<int64_t>(span) * a.d, scale_step = static_cast<int64_t>(span) * a.scales_per_row;
  int64_t out = static_cast<int64_t>(mine) * a.d + lane * kU;  // the lane's first channel
  int64_t scale_row = static_cast<int64_t>(mine) * a.scales_per_row;
  // the bound is the CTA's first row: lanes whose row lies behind the end still take part in the reductions
  uint32_t row = mine;
  for (uint32_t first = blockIdx.x * kRows; first < a.rows;
       first += span, row += span, parity ^= 1, out += out_step, scale_row += scale_step) {
    const bool valid = row < a.rows;
    // octs are not cleared where a lane has none: their sums are left out instead
    constexpr bool kClear = kU < 8 || !In::kStaged;
    Unit<T, kU> u[kUnits], r[kUnits];
    if constexpr (In::kStaged) {
      fetch(row + span, parity ^ 1);
      stage_wait<1>();
      const char* from = reinterpret_cast<const char*>(ring) + parity * stage_bytes;
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const bool on = !kClear || (valid && lane + k * kGroup < units);
        u[k] = on ? In::read(from, k) : zero_unit<T, kU>();
        r[k] = on && has_residual ? In::read(from + In::kStage, k) : zero_unit<T, kU>();
      }
    } else {
      const T *up = nullptr, *rp = nullptr;
      next_rows(row, up, rp);
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int n = lane + k * kGroup;
        const bool on = valid && n < units;
        u[k] = on ? load_unit<T, kU>(up + n * kU) : zero_unit<T, kU>();
        r[k] = on && has_residual ? load_unit<T, kU>(rp + n * kU) : zero_unit<T, kU>();
      }
    }

    if (dropping) {
      uint32_t b, i, j;
      a.walk.at(valid ? row : 0, b, i, j);
      if constexpr (kU == 8) {  // oct by oct: fewer values at a time
#pragma unroll
        for (int k = 0; k < kUnits; ++k) u[k] = drop_and_add<T>(drop, line, b, i, j, lane + k * kGroup, u[k], r[k], has_residual);
      } else {
        Lane<kU, kUnits> v = unpack_all<T, kU, kUnits>(u);
        drop_all<kU, kGroup, kUnits>(drop, line, b, i, j, lane, a.octs, v);
        const Lane<kU, kUnits> x = unpack_all<T, kU, kUnits>(r);
#pragma unroll
        for (int n = 0; n < kPairs; ++n) v.p[n] = add_whole(v.p[n], x.p[n]);
        pack_all<T, kU, kUnits>(v, u);
      }
    } else if (has_residual) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) u[k] = add_units(u[k], r[k]);
    }
    if (a.stream != nullptr && valid) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
        if (lane + k * kGroup < units) store_unit<T, kU>(a.stream + out + k * kGroup * kU, u[k]);
    }
    Lane<kU, kUnits> v = unpack_all<T, kU, kUnits>(u);
    float ss[1] = {0.f};
    if constexpr (kClear) {
      float2 s = both(0.f);
#pragma unroll
      for (int n = 0; n < kPairs; ++n) s = __ffma2_rn(v.p[n], v.p[n], s);
      ss[0] = s.x + s.y;
    } else {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        float2 s = __fmul2_rn(v.p[4 * k], v.p[4 * k]);
#pragma unroll
        for (int n = 1; n < 4; ++n) s = __ffma2_rn(v.p[4 * k + n], v.p[4 * k + n], s);
        ss[0] += valid && lane + k * kGroup < units ? s.x + s.y : 0.f;
      }
    }
    group_sum<kGroup, 1>(ss, sums, parity);
    const float rstd = rsqrtf(ss[0] * a.inv_d + a.eps);
    const auto gain = [&](float by) {
#pragma unroll
      for (int n = 0; n < kPairs; ++n) v.p[n] = __fmul2_rn(__fmul2_rn(v.p[n], both(by)), w.p[n]);
    };

    if constexpr (kMode == kNorm) {
      gain(rstd);
      T* yp = static_cast<T*>(a.y) + out;
      pack_all<T, kU, kUnits>(v, u);
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
        if (valid && lane + k * kGroup < units) store_unit<T, kU>(yp + k * kGroup * kU, u[k]);
    } else if constexpr (kMode == kNormE4m3) {
      const bool whole = kU < 8 || a.scale_shift < 0;  // the only form of narrow units
      float top[kUnits];
      const auto find_top = [&] {
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          top[k] = 0.f;
#pragma unroll
          for (int e = 0; e < kU; ++e) {
            const float2 x = v.p[(k * kU + e) / 2];
            top[k] = fmaxf(top[k], fabsf((k * kU + e) & 1 ? x.y : x.x));
          }
          if constexpr (!kClear) top[k] = valid && lane + k * kGroup < units ? top[k] : 0.f;
        }
        if (whole) {
          float m[1] = {top[0]};
#pragma unroll
          for (int k = 1; k < kUnits; ++k) m[0] = fmaxf(m[0], top[k]);
          group_max<kGroup, 1>(m, tops, parity);
#pragma unroll
          for (int k = 0; k < kUnits; ++k) top[k] = m[0];
        } else {
          // 32, 64 or 128 channels are 4, 8 or 16 neighbouring lanes
#pragma unroll
          for (int o = 0; o < 4; ++o)
            if (o < a.scale_shift) {
#pragma unroll
              for (int k = 0; k < kUnits; ++k) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], 1 << o));
            }
        }
      };
      // One oct a lane: p = z w, and the long way, a warp or all that share one scale together, where that will not do.  More channels a
      // lane have no registers for both ways and take the long one (96 x 768 rows of 384: 38.7 us, with both 40.9).
      bool far = true;
      if constexpr (kU == 8 && kUnits == 1) {
#pragma unroll
        for (int n = 0; n < kPairs; ++n) v.p[n] = __fmul2_rn(v.p[n], w.p[n]);
        find_top();
        far = __any_sync(0xffffffffu, !is_near(top[0], rstd) && (whole || lane < units));
        if (far) {
          v = unpack_all<T, kU, kUnits>(u);
          if (kGroup > 32 && whole) __syncthreads();  // the first maxima have been read
        }
      }
      float rest = rstd;
      if (far) {
        const Parts parts = parts_of(rstd);
        rest = parts.rest;
        gain(parts.power);
        find_top();
      }
      if (!valid) continue;
      uint8_t* yp = static_cast<uint8_t*>(a.y) + out;
      float* sp = a.scales + scale_row;
      if constexpr (kU == 8) {
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
          const int n = lane + k * kGroup;
          if (n >= units) continue;
          const Quotient by = !far || is_near(top[k], rest) ? quotient_near(top[k], rest) : quotient_far(top[k], rest);
          if (whole ? n == 0 : (n & ((1 << a.scale_shift) - 1)) == 0) sp[whole ? 0 : n >> a.scale_shift] = by.scale;
          uint32_t q[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) q[e] = e4m3x2(by(v.p[4 * k + e]));
          __stcs(reinterpret_cast<uint2*>(yp + k * kGroup * 8), make_uint2(q[0] | (q[1] << 16), q[2] | (q[3] << 16)));
        }
      } else {
        const Quotient by = is_near(top[0], rest) ? quotient_near(top[0], rest) : quotient_far(top[0], rest);
        if (lane == 0) sp[0] = by.scale;
#pragma unroll
        for (int m = 0; m < kPairs; ++m) {
          const uint32_t q = e4m3x2(by(v.p[m]));  // a unit of two channels, or two units
          constexpr int kStep = 2 / kU;
          const int n = lane + m * kStep * kGroup;
          if constexpr (kU == 2) {
            if (n < units) *reinterpret_cast<uint16_t*>(yp + m * kGroup * 2) = static_cast<uint16_t>(q);
          } else {
            if (n < units) yp[2 * m * kGroup] = static_cast<uint8_t>(q);
            if (n + kGroup < units) yp[(2 * m + 1) * kGroup] = static_cast<uint8_t>(q >> 8);
          }
        }
      }
    }
  }
}

// The addition alone, of whole octs: no reduction, kFlight octs per thread and step.
template <typename T, int kFlight>
__global__ void __launch_bounds__(kThreads) add_octs_kernel(const __grid_constant__ NormArgs<T> a, const FastDiv by_octs) {
  Dropout drop = a.drop;
  const bool dropping = drop.keep < 65536u;
  const bool has_residual = a.residual.p != nullptr;
  const uint32_t line = drop.keep << 16;
  if (dropping) resolve_seed(drop);
  const int64_t total = static_cast<int64_t>(a.rows) * a.octs;
  const int64_t span = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t n0 = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; n0 < total; n0 += kFlight * span) {
    Unit<T, 8> u[kFlight], r[kFlight];
    uint32_t b[kFlight], i[kFlight], j[kFlight], oct[kFlight];
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int64_t n = n0 + f * span;
      if (n < total) {
        uint32_t row;
        if (total <= 0x7fffffff) {
          row = by_octs.div(static_cast<uint32_t>(n));
          oct[f] = static_cast<uint32_t>(n) - row * by_octs.d;
        } else {
          row = static_cast<uint32_t>(n / a.octs);
          oct[f] = static_cast<uint32_t>(n - static_cast<int64_t>(row) * a.octs);
        }
        if (dropping || !a.flat) a.walk.at(row, b[f], i[f], j[f]);
        u[f] = load_unit<T, 8>((a.flat ? a.update.flat(row) : a.update.row(b[f], i[f], j[f])) + oct[f] * 8);
        if (has_residual) r[f] = load_unit<T, 8>((a.flat ? a.residual.flat(row) : a.residual.row(b[f], i[f], j[f])) + oct[f] * 8);
      }
    }
#pragma unroll
    for (int f = 0; f < kFlight; ++f) {
      const int64_t n = n0 + f * span;
      if (n >= total) break;
      if (dropping) {
        u[f] = drop_and_add<T>(drop, line, b[f], i[f], j[f], oct[f], u[f], r[f], has_residual);
      } else if (has_residual) {
        u[f] = add_units(u[f], r[f]);
      }
      store_unit<T, 8>(a.stream + n * 8, u[f]);
    }
  }
}

// The addition alone, of other rows: a warp takes 256 channels of a row at a time, in units of kU channels per access.  Each
// lane draws one of the piece's octs.
template <typename T, int kU>
__global__ void __launch_bounds__(kThreads) add_pieces_kernel(const __grid_constant__ NormArgs<T> a, const FastDiv by_pieces) {
  constexpr int kUnits = 8 / kU;  // units of a lane
  Dropout drop = a.drop;
  const bool dropping = drop.keep < 65536u;
  const bool has_residual = a.residual.p != nullptr;
  const uint32_t line = drop.keep << 16;
  if (dropping) resolve_seed(drop);
  const int lane = threadIdx.x & 31;
  const int64_t total = static_cast<int64_t>(a.rows) * by_pieces.d;
  const int64_t span = static_cast<int64_t>(gridDim.x) * (kThreads / 32);
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5); n < total; n += span) {
    uint32_t row, piece, b = 0, i = 0, j = 0;
    if (total <= 0x7fffffff) {
      row = by_pieces.div(static_cast<uint32_t>(n));
      piece = static_cast<uint32_t>(n) - row * by_pieces.d;
    } else {
      row = static_cast<uint32_t>(n / by_pieces.d);
      piece = static_cast<uint32_t>(n - static_cast<int64_t>(row) * by_pieces.d);
    }
    if (dropping || !a.flat) a.walk.at(row, b, i, j);
    const int c0 = piece * 256 + lane * kU;  // the lane's first channel
    const T* up = (a.flat ? a.update.flat(row) : a.update.row(b, i, j)) + c0;
    const T* rp = (a.flat ? a.residual.flat(row) : a.residual.row(b, i, j)) + c0;
    Unit<T, kU> u[kUnits], r[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const bool on = c0 + k * 32 * kU < a.d;
      u[k] = on ? load_unit<T, kU>(up + k * 32 * kU) : zero_unit<T, kU>();
      r[k] = on && has_residual ? load_unit<T, kU>(rp + k * 32 * kU) : zero_unit<T, kU>();
    }
    if (dropping) {
      Lane<kU, kUnits> v = unpack_all<T, kU, kUnits>(u);
      drop_all<kU, 32, kUnits>(drop, line, b, i, j, piece * (256 / kU) + lane, a.octs, v);
      const Lane<kU, kUnits> x = unpack_all<T, kU, kUnits>(r);
#pragma unroll
      for (int k = 0; k < v.kPairs; ++k) v.p[k] = add_whole(v.p[k], x.p[k]);
      pack_all<T, kU, kUnits>(v, u);
    } else if (has_residual) {
#pragma unroll
      for (int k = 0; k < kUnits; ++k) u[k] = add_units(u[k], r[k]);
    }
    T* zp = a.stream + static_cast<int64_t>(row) * a.d + c0;
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
      if (c0 + k * 32 * kU < a.d) store_unit<T, kU>(zp + k * 32 * kU, u[k]);
  }
}

template <typename T, int kU>
cudaError_t launch_pieces(const NormArgs<T>& a, int sms, cudaStream_t s) {
  auto kernel = add_pieces_kernel<T, kU>;
  static const int resident = resident_ctas(kernel, kThreads, 0);
  const uint32_t pieces = (a.d + 255) / 256;
  const uint64_t need = (static_cast<uint64_t>(a.rows) * pieces + kThreads / 32 - 1) / (kThreads / 32);
  return launch(kernel, walk_grid(need, sms, resident, 4), kThreads, 0, s, a, make_fast_div(pieces));
}

template <typename T>
cudaError_t launch_add(const NormArgs<T>& a, int unit, int sms, cudaStream_t s) {
  if (unit == 8) {
    constexpr int kFlight = sizeof(T) == 2 ? 2 : 1;
    auto kernel = add_octs_kernel<T, kFlight>;
    static const int resident = resident_ctas(kernel, kThreads, 0);
    const uint64_t need = (static_cast<uint64_t>(a.rows) * a.octs + kThreads - 1) / kThreads;
    return launch(kernel, walk_grid(need, sms, resident, 4 * kFlight), kThreads, 0, s, a, make_fast_div(a.octs));
  }
  if constexpr (sizeof(T) == 2)
    if (unit == 2) return launch_pieces<T, 2>(a, sms, s);
  if constexpr (sizeof(T) == 4)
    if (unit == 4) return launch_pieces<T, 4>(a, sms, s);
  return launch_pieces<T, 1>(a, sms, s);
}

template <typename T, int kU, int kGroup, int kUnits, int kMode>
cudaError_t launch_rows(const NormArgs<T>& a, int sms, cudaStream_t stream) {
  constexpr uint32_t kWide = threads_of(kGroup), kRows = kWide / kGroup;
  auto kernel = add_norm_kernel<T, kU, kGroup, kUnits, kMode>;
  const bool has_residual = a.residual.p != nullptr;
  constexpr int kStages = 2 * Rows<T, kU, kGroup, kUnits>::kStage;  // of one tensor
  const int smem = kStages * (has_residual ? 2 : 1);
  if (2 * kStages > 47 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * kStages);
    if (e != cudaSuccess) return e;
  }
  // what is resident without and with a residual's stages
  static const int resident[2] = {resident_ctas(kernel, kWide, kStages), resident_ctas(kernel, kWide, 2 * kStages)};
  const uint32_t need = (a.rows + kRows - 1) / kRows;
  return pair::launch(kernel, walk_grid(need, sms, resident[has_residual], (kLaneChannels + kU * kUnits / 2) / (kU * kUnits)), kWide, smem, stream, a);
}

// Octs.
template <typename T, int kMode>
cudaError_t wide_rows(const NormArgs<T>& a, int sms, cudaStream_t s) {
  const int o = a.octs;
  if (o <= 8) return launch_rows<T, 8, 8, 1, kMode>(a, sms, s);
  if (o <= 16) return launch_rows<T, 8, 16, 1, kMode>(a, sms, s);
  if (o <= 32) return launch_rows<T, 8, 32, 1, kMode>(a, sms, s);
  if (o <= 48) return launch_rows<T, 8, 16, 3, kMode>(a, sms, s);
  if (o <= 64) return launch_rows<T, 8, 32, 2, kMode>(a, sms, s);
  if (o <= 128) return launch_rows<T, 8, 128, 1, kMode>(a, sms, s);
  if (o <= 256) return launch_rows<T, 8, 256, 1, kMode>(a, sms, s);
  if (o <= 512) return launch_rows<T, 8, 512, 1, kMode>(a, sms, s);
  return launch_rows<T, 8, 1024, 1, kMode>(a, sms, s);
}

// Units of one or two channels: four to eight channels per lane of a warp, then eight per thread of a CTA (four of twice the threads
// take up to 1.5 times as long: fewer rows are at hand on an SM).
template <typename T, int kU, int kMode>
cudaError_t narrow_rows(const NormArgs<T>& a, int sms, cudaStream_t s) {
  if (a.d <= 128) return launch_rows<T, kU, 32, 4 / kU, kMode>(a, sms, s);
  if constexpr (kU == 1)
    if (a.d <= 192) return launch_rows<T, kU, 32, 6, kMode>(a, sms, s);
  if (a.d <= 256) return launch_rows<T, kU, 32, 8 / kU, kMode>(a, sms, s);
  if (a.d <= 512) return launch_rows<T, kU, 64, 8 / kU, kMode>(a, sms, s);
  if (a.d <= 1024) return launch_rows<T, kU, 128, 8 / kU, kMode>(a, sms, s);
  if (a.d <= 2048) return launch_rows<T, kU, 256, 8 / kU, kMode>(a, sms, s);
  if (a.d <= 4096) return launch_rows<T, kU, 512, 8 / kU, kMode>(a, sms, s);
  return launch_rows<T, kU, 1024, 8 / kU, kMode>(a, sms, s);
}

template <typename T, int kMode>
cudaError_t by_unit(const NormArgs<T>& a, int unit, int sms, cudaStream_t s) {
  if (unit == 8) return wide_rows<T, kMode>(a, sms, s);
  if constexpr (sizeof(T) == 2)
    if (unit == 2) return narrow_rows<T, 2, kMode>(a, sms, s);
  return narrow_rows<T, 1, kMode>(a, sms, s);
}

template <typename T>
cudaError_t run(const pair_norm_desc_t* d, const pair_tensor_t* update, const pair_tensor_t* residual, const void* weight,
                void* stream, void* y, float* scales, int unit, int sms, cudaStream_t s) {
  NormArgs<T> a;
  a.update = strided<T>(update);
  a.residual = strided<T>(residual);
  a.weight = weight;
  a.stream = static_cast<T*>(stream);
  a.y = y;
  a.scales = scales;
  a.walk = RowWalk{make_fast_div(d->j), make_fast_div(d->i)};
  a.drop = make_dropout(d->dropout);
  a.rows = static_cast<uint32_t>(d->b) * d->i * d->j;
  a.d = d->d;
  a.octs = (d->d + 7) / 8;
  a.weight_dtype = d->weight_dtype;
  a.scales_per_row = d->group != 0 ? d->d / d->group : 0;
  a.scale_shift = d->group == d->d ? -1 : d->group == 32 ? 2 : d->group == 64 ? 3 : 4;
  a.flat = collapses(update, d->i, d->j) && collapses(residual, d->i, d->j);
  a.eps = d->eps;
  a.inv_d = 1.f / static_cast<float>(d->d);
  if (y == nullptr) return launch_add<T>(a, unit, sms, s);
  return d->group != 0 ? by_unit<T, kNormE4m3>(a, unit, sms, s) : by_unit<T, kNorm>(a, unit, sms, s);
}

}  // namespace

int check_dtype(int dtype, const char* what, const char* who) {
  if (dtype == PAIR_BF16 || dtype == PAIR_FP16 || dtype == PAIR_FP32) return TRIMUL_OK;
  return trimul::report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: %s has the unknown type %d", who, what, dtype);
}

int check_norm_desc(const pair_norm_desc_t* d, const char* who) {
  using trimul::report_error;
  if (d == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: desc is NULL", who);
  if (d->b < 0 || d->i < 0 || d->j < 0 || d->d < 1)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: shape (%d, %d, %d, %d) is not a pair tensor's", who, d->b, d->i, d->j, d->d);
  if (d->d > PAIR_MAX_WIDTH)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: width d=%d is above %d", who, d->d, PAIR_MAX_WIDTH);
  // (b * i) * j cannot pass 2^63: each factor is below 2^31 and the partial product is checked first
  const int64_t lines = static_cast<int64_t>(d->b) * d->i;
  if (lines > 0x7fffffffLL || lines * d->j > 0x7fffffffLL)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: %d x %d x %d rows are above 2^31 - 1", who, d->b, d->i, d->j);
  if (int rc = check_dtype(d->dtype, "the activation", who)) return rc;
  if (int rc = check_dtype(d->weight_dtype, "the weight", who)) return rc;
  // smaller values are subnormal and would be flushed to 0, where a row of zeros has no norm
  if (!(d->eps >= 1.17549435e-38f && d->eps <= 3.4e38f))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: eps must be a normal number > 0; got %g", who, d->eps);
  const pair_dropout_t& p = d->dropout;
  if (p.keep > 65536u) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: dropout.keep=%u is above 65536", who, p.keep);
  if (p.shared < PAIR_SHARED_NONE || p.shared > PAIR_SHARED_COLUMNS)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: dropout.shared=%d is none of 0, 1, 2", who, p.shared);
  if (p.origin_b < 0 || p.origin_i < 0 || p.origin_j < 0)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: dropout origin (%d, %d, %d) must not be negative", who, p.origin_b, p.origin_i, p.origin_j);
  if (p.keep < 65536u && static_cast<int64_t>(p.origin_b) + d->b > PAIR_MAX_BATCH)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: dropout numbers at most %d batch entries", who, PAIR_MAX_BATCH);
  return TRIMUL_OK;
}

}  // namespace pair

extern "C" int pair_sm100_add_norm(const pair_norm_desc_t* desc, const pair_tensor_t* update, const pair_tensor_t* residual,
                                   const void* weight, void* stream, void* y, float* scales, trimul_stream_t cuda_stream) {
  using namespace pair;
  using trimul::report_error;
  const char* who = "pair_sm100_add_norm";
  if (int rc = check_norm_desc(desc, who)) return rc;
  const int g = desc->group;
  if (g != 0 && g != desc->d && g != 32 && g != 64 && g != 128)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: group=%d is none of 32, 64, 128, d", who, g);
  if (g != 0 && desc->d % g != 0)
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: group=%d does not divide d=%d", who, g, desc->d);
  // an empty tensor has nothing to point at
  if (static_cast<int64_t>(desc->b) * desc->i * desc->j == 0) return TRIMUL_OK;
  if ((weight == nullptr) != (y == nullptr))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: weight and y come together", who);
  if (y == nullptr && stream == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: no output", who);
  if (g != 0 && (y == nullptr || scales == nullptr))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: an e4m3 output needs y and scales", who);
  if (update == nullptr || update->data == nullptr)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: update is NULL", who);
  const pair_tensor_t u = canonical(update, desc->b, desc->i, desc->j), r = canonical(residual, desc->b, desc->i, desc->j);
  update = &u, residual = &r;
  const int size = type_bytes(desc->dtype);
  if (!elements_aligned(size, {update, residual}, {stream, g == 0 ? y : nullptr}) || !aligned(scales, 4) ||
      !aligned(weight, type_bytes(desc->weight_dtype)) || !aligned(desc->dropout.device_seed, 8))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", who);
  int unit = unit_of(desc->d, size, {update, residual}, {stream, g == 0 ? y : nullptr});
  if (y == nullptr && unit == 1 && size == 4 && units_fit(4, desc->d, size, {update, residual}, {stream})) unit = 4;
  if (g != 0 && g != desc->d && (unit != 8 || !aligned(y, 8)))
    return report_error(TRIMUL_ERR_UNSUPPORTED_SHAPE, "%s: scales per group need rows that start on 16-byte boundaries", who);
  if (g != 0 && !aligned(y, unit)) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: an e4m3 output starts on an 8-byte boundary", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  cudaError_t e;
  if (desc->dtype == PAIR_FP32)
    e = run<float>(desc, update, residual, weight, stream, y, scales, unit, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = run<__half>(desc, update, residual, weight, stream, y, scales, unit, sms, cuda_stream);
  else
    e = run<__nv_bfloat16>(desc, update, residual, weight, stream, y, scales, unit, sms, cuda_stream);
  if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return TRIMUL_OK;
}
