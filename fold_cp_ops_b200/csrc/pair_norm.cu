// z = residual + dropout(update) and y = rms_norm(z), in one pass over the rows of the pair stream.
//
// Mathematics.  u = keep ? x * 65536 / keep16 : 0;  z = round(r + u);  s = 1 / sqrt(mean_c z^2 + eps);
// y = z s w.  The norm reads the STORED z (rounded to the activations' type): y is then exactly what a later norm
// of the stream would give, and the gradient needs nothing but z.  The sum of squares and s are fp32.
// e4m3 output: a = max |y| over a group of channels, scale = a / 448, q = e4m3(y / scale).
//
// Bound.  HBM: update and residual are read, z and y written once; nothing else moves.
// Split.  A row of up to 256 channels is one oct (eight channels, 16 bytes of a 16-bit type) per lane of 8, 16 or 32
// lanes, so that the reductions stay inside a warp; up to 1024 channels it is two or four octs per lane of a warp;
// wider rows take a CTA.
#include "pair_stream.cuh"

namespace pair {
namespace {

constexpr float kE4m3Max = 448.f;

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
  int group;  // channels per scale
  float eps;
};

__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

template <typename T, int kGroup, int kOcts, bool kWide, int kMode>
__global__ void __launch_bounds__(kThreads) add_norm_kernel(const __grid_constant__ NormArgs<T> a) {
  __shared__ float sums[2 * 8];
  __shared__ float tops[2 * 8];
  constexpr int kRows = kThreads / kGroup;  // rows a CTA holds at a time
  const int lane = threadIdx.x % kGroup;
  Dropout drop = a.drop;
  if (drop.keep < 65536u) resolve_seed(drop);

  float w[kOcts][8];
#pragma unroll
  for (int k = 0; k < kOcts; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = (lane + k * kGroup) * 8 + e;
      w[k][e] = c < a.d ? load_any(a.weight, c, a.weight_dtype) : 0.f;
    }

  int parity = 0;
  // the bound is the CTA's first row: lanes whose row lies behind the end still take part in the reductions
  for (uint32_t first = blockIdx.x * kRows; first < a.rows; first += gridDim.x * kRows, parity ^= 1) {
    const uint32_t row = first + threadIdx.x / kGroup;
    const bool valid = row < a.rows;
    uint32_t b, i, j;
    a.walk.at(valid ? row : 0, b, i, j);
    const T* up = a.update.row(b, i, j);
    const T* rp = a.residual.p != nullptr ? a.residual.row(b, i, j) : nullptr;
    const int64_t out_row = static_cast<int64_t>(row) * a.d;

    Oct<T> u[kOcts], r[kOcts];
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int v = lane + k * kGroup;
      const bool on = valid && v < a.octs;
      u[k] = on ? load_oct<kWide>(up + v * 8, a.d - v * 8) : zero_oct<T>();
      r[k] = on && rp != nullptr ? load_oct<kWide>(rp + v * 8, a.d - v * 8) : zero_oct<T>();
    }

    float ss[1] = {0.f};
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int v = lane + k * kGroup;
      float f[8], g[8];
      unpack(u[k], f);
      if (drop.keep < 65536u) apply_dropout(drop, b, i, j, v, f);
      if (rp != nullptr) {
        unpack(r[k], g);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] += g[e];
      }
      u[k] = pack<T>(f);
      if (valid && v < a.octs) {
        if (a.stream != nullptr) store_oct<kWide>(a.stream + out_row + v * 8, u[k], a.d - v * 8);
        unpack(u[k], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss[0] += (kWide || v * 8 + e < a.d) ? f[e] * f[e] : 0.f;
      }
    }
    group_sum<kGroup, 1>(ss, sums, parity);
    const float rstd = rsqrtf(ss[0] / static_cast<float>(a.d) + a.eps);

    if constexpr (kMode == kNorm) {
      T* yp = static_cast<T*>(a.y) + out_row;
#pragma unroll
      for (int k = 0; k < kOcts; ++k) {
        const int v = lane + k * kGroup;
        float f[8];
        unpack(u[k], f);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= rstd * w[k][e];
        if (valid && v < a.octs) store_oct<kWide>(yp + v * 8, pack<T>(f), a.d - v * 8);
      }
    } else {
      uint8_t* yp = static_cast<uint8_t*>(a.y) + out_row;
      float top[kOcts];
#pragma unroll
      for (int k = 0; k < kOcts; ++k) {
        const int v = lane + k * kGroup;
        float f[8];
        unpack(u[k], f);
        top[k] = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (kWide || v * 8 + e < a.d) top[k] = fmaxf(top[k], fabsf(f[e] * (rstd * w[k][e])));
      }
      const int per = a.group >> 3;  // octs per scale
      if (a.group == a.d) {
        float m = 0.f;
#pragma unroll
        for (int k = 0; k < kOcts; ++k) m = fmaxf(m, top[k]);
        m = group_max<kGroup>(m, tops, parity);
#pragma unroll
        for (int k = 0; k < kOcts; ++k) top[k] = m;
      } else {
        // a group of 32, 64 or 128 channels is 4, 8 or 16 neighbouring lanes
        for (int o = 1; o < per; o <<= 1)
#pragma unroll
          for (int k = 0; k < kOcts; ++k) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], o));
      }
#pragma unroll
      for (int k = 0; k < kOcts; ++k) {
        const int v = lane + k * kGroup;
        const float scale = top[k] > 0.f ? fmaxf(top[k] / kE4m3Max, 1.17549435e-38f) : 1.f;
        if (valid && v < a.octs) {
          if (a.group == a.d) {
            if (v == 0) a.scales[row] = scale;
          } else if (v % per == 0) {
            a.scales[static_cast<int64_t>(row) * (a.d / a.group) + v / per] = scale;
          }
          const float inv = 1.f / scale;
          float f[8];
          unpack(u[k], f);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] *= rstd * w[k][e];
          uint2 q;
          q.x = e4m3x2(f[0] * inv, f[1] * inv) | (e4m3x2(f[2] * inv, f[3] * inv) << 16);
          q.y = e4m3x2(f[4] * inv, f[5] * inv) | (e4m3x2(f[6] * inv, f[7] * inv) << 16);
          if constexpr (kWide) {
            __stcs(reinterpret_cast<uint2*>(yp + v * 8), q);
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (v * 8 + e < a.d) yp[v * 8 + e] = static_cast<uint8_t>((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
          }
        }
      }
    }
  }
}

// The addition alone: no reduction, one oct per thread and step.
template <typename T, bool kWide>
__global__ void __launch_bounds__(kThreads) add_kernel(const __grid_constant__ NormArgs<T> a, const FastDiv by_octs) {
  Dropout drop = a.drop;
  if (drop.keep < 65536u) resolve_seed(drop);
  const int64_t total = static_cast<int64_t>(a.rows) * a.octs;
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t n = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; n < total; n += step) {
    uint32_t row, v;
    if (total <= 0x7fffffff) {
      row = by_octs.div(static_cast<uint32_t>(n));
      v = static_cast<uint32_t>(n) - row * by_octs.d;
    } else {
      row = static_cast<uint32_t>(n / a.octs);
      v = static_cast<uint32_t>(n - static_cast<int64_t>(row) * a.octs);
    }
    uint32_t b, i, j;
    a.walk.at(row, b, i, j);
    const int left = a.d - static_cast<int>(v) * 8;
    const Oct<T> u = load_oct<kWide>(a.update.row(b, i, j) + v * 8, left);
    Oct<T> r;
    if (a.residual.p != nullptr) r = load_oct<kWide>(a.residual.row(b, i, j) + v * 8, left);
    float f[8], g[8];
    unpack(u, f);
    if (drop.keep < 65536u) apply_dropout(drop, b, i, j, v, f);
    if (a.residual.p != nullptr) {
      unpack(r, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] += g[e];
    }
    store_oct<kWide>(a.stream + static_cast<int64_t>(row) * a.d + v * 8, pack<T>(f), left);
  }
}

template <typename T, int kGroup, int kOcts, bool kWide, int kMode>
cudaError_t launch(const NormArgs<T>& a, int sms, cudaStream_t stream) {
  constexpr uint32_t kRows = kThreads / kGroup;
  const uint32_t need = (a.rows + kRows - 1) / kRows;
  const uint32_t most = static_cast<uint32_t>(sms) * 8;
  add_norm_kernel<T, kGroup, kOcts, kWide, kMode><<<need < most ? need : most, kThreads, 0, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, bool kWide, int kMode>
cudaError_t by_width(const NormArgs<T>& a, int sms, cudaStream_t s) {
  const int o = a.octs;
  if (o <= 8) return launch<T, 8, 1, kWide, kMode>(a, sms, s);
  if (o <= 16) return launch<T, 16, 1, kWide, kMode>(a, sms, s);
  if (o <= 32) return launch<T, 32, 1, kWide, kMode>(a, sms, s);
  if (o <= 64) return launch<T, 32, 2, kWide, kMode>(a, sms, s);
  if (o <= 128) return launch<T, 32, 4, kWide, kMode>(a, sms, s);
  if (o <= 256) return launch<T, 256, 1, kWide, kMode>(a, sms, s);
  if (o <= 512) return launch<T, 256, 2, kWide, kMode>(a, sms, s);
  return launch<T, 256, 4, kWide, kMode>(a, sms, s);
}

template <typename T>
cudaError_t run(const pair_norm_desc_t* d, const pair_tensor_t* update, const pair_tensor_t* residual, const void* weight,
                void* stream, void* y, float* scales, int sms, cudaStream_t s) {
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
  a.group = d->group;
  a.eps = d->eps;
  const bool wide = d->d % 8 == 0 && rows_aligned(update, sizeof(T)) && rows_aligned(residual, sizeof(T)) &&
                    aligned16(stream) && aligned16(y);
  if (y == nullptr) {
    const int64_t total = static_cast<int64_t>(a.rows) * a.octs;
    const int64_t need = (total + kThreads - 1) / kThreads, most = static_cast<int64_t>(sms) * 8;
    const unsigned grid = static_cast<unsigned>(need < most ? need : most);
    const FastDiv by_octs = make_fast_div(a.octs);
    if (wide)
      add_kernel<T, true><<<grid, kThreads, 0, s>>>(a, by_octs);
    else
      add_kernel<T, false><<<grid, kThreads, 0, s>>>(a, by_octs);
    return cudaGetLastError();
  }
  if (d->group != 0) return wide ? by_width<T, true, kNormE4m3>(a, sms, s) : by_width<T, false, kNormE4m3>(a, sms, s);
  return wide ? by_width<T, true, kNorm>(a, sms, s) : by_width<T, false, kNorm>(a, sms, s);
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
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  cudaError_t e;
  if (desc->dtype == PAIR_FP32)
    e = run<float>(desc, update, residual, weight, stream, y, scales, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = run<__half>(desc, update, residual, weight, stream, y, scales, sms, cuda_stream);
  else
    e = run<__nv_bfloat16>(desc, update, residual, weight, stream, y, scales, sms, cuda_stream);
  if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return TRIMUL_OK;
}
