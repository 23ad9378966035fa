// Gradients of y = z s w, s = 1 / sqrt(mean_c z^2 + eps), z = residual + dropout(update).
//
// Mathematics.  With t = w dy:   g = dz + s t - z s^3 mean_c(t z);   d_residual = g;
// d_update = keep ? g * 65536 / keep16 : 0 (the mask is drawn again);   d_w = sum over rows of dy z s.
// s is recomputed: z has to be read for g anyway, and both reductions of a row, sum z^2 and sum t z, share their
// shuffles.
//
// Bound.  HBM: z, dy and dz are read, one gradient (two with dropout) is written.
// Split.  Rows as in the forward kernel.  CTAs stay resident and walk over rows, so that a lane keeps the gain's
// gradient of its own channels in registers; every kFold rows it is added to a sum in 64 bits in shared memory (fp32
// sums of 32 terms lose about 2^-23, where sums of thousands would lose ten times that), the CTA's rows are
// joined there and each CTA leaves one row of sums in the workspace.  A second kernel adds those in a fixed order:
// no atomics, the same bits every time.
#include "pair_stream.cuh"

namespace pair {
namespace {

constexpr int kFold = 32;

template <typename T>
struct GradArgs {
  Strided<T> z, dy, dz;
  const void* weight;
  T* d_stream;
  T* d_update;
  double* partial;  // (grid, d); nullptr when the gain's gradient is not wanted
  RowWalk walk;
  Dropout drop;
  uint32_t rows;
  int d, octs;
  int weight_dtype;
  int flat;  // the rows of z, dy and dz lie at a constant distance
  float eps, inv_d;
};

// As add_norm_kernel: kU channels per access, kGroup lanes per row, kUnits units per lane.
template <typename T, int kU, int kGroup, int kUnits>
__global__ void __launch_bounds__(threads_of(kGroup)) norm_grad_kernel(const __grid_constant__ GradArgs<T> a) {
  __shared__ float sums[2 * 32 * 2];
  extern __shared__ double fold[];  // [unit of the lane][channel of the unit][thread]
  constexpr int kWide = threads_of(kGroup);
  constexpr int kRows = kWide / kGroup;
  constexpr int kPairs = (kU + 1) / 2;
  const int lane = threadIdx.x % kGroup;
  const int units = a.d / kU;
  const bool dropping = a.drop.keep < 65536u && a.d_update != nullptr;
  const uint32_t line = a.drop.keep << 16;
  Dropout drop = a.drop;
  if (dropping) resolve_seed(drop);

  Vals<kU> w[kUnits], dw[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    float f[kPairs * 2];
#pragma unroll
    for (int e = 0; e < kPairs * 2; ++e) {
      const int n = lane + k * kGroup;
      f[e] = n < units && e < kU ? load_any(a.weight, n * kU + e, a.weight_dtype) : 0.f;
      if (e < kU && a.partial != nullptr) fold[(k * kU + e) * kWide + threadIdx.x] = 0.0;
    }
#pragma unroll
    for (int e = 0; e < kPairs; ++e) {
      w[k].p[e] = make_float2(f[2 * e], f[2 * e + 1]);
      dw[k].p[e] = both(0.f);
    }
  }
  auto carry = [&] {
#pragma unroll
    for (int k = 0; k < kUnits; ++k)
#pragma unroll
      for (int e = 0; e < kU; ++e) {
        fold[(k * kU + e) * kWide + threadIdx.x] += e & 1 ? dw[k].p[e / 2].y : dw[k].p[e / 2].x;
        (e & 1 ? dw[k].p[e / 2].y : dw[k].p[e / 2].x) = 0.f;
      }
  };

  int parity = 0, held = 0;
  for (uint32_t first = blockIdx.x * kRows; first < a.rows; first += gridDim.x * kRows, parity ^= 1) {
    const uint32_t row = first + threadIdx.x / kGroup;
    const bool valid = row < a.rows;
    uint32_t b = 0, i = 0, j = 0;
    if (valid && (dropping || !a.flat)) a.walk.at(row, b, i, j);
    const T* zp = a.flat ? a.z.flat(row) : a.z.row(b, i, j);
    const T* yp = a.flat ? a.dy.flat(row) : a.dy.row(b, i, j);
    const T* gp = a.flat ? a.dz.flat(row) : a.dz.row(b, i, j);

    Unit<T, kU> z[kUnits], dy[kUnits], dz[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int n = lane + k * kGroup;
      const bool on = valid && n < units;
      z[k] = on ? load_unit<T, kU>(zp + n * kU) : zero_unit<T, kU>();
      dy[k] = on && a.dy.p != nullptr ? load_unit<T, kU>(yp + n * kU) : zero_unit<T, kU>();
      dz[k] = on && a.dz.p != nullptr ? load_unit<T, kU>(gp + n * kU) : zero_unit<T, kU>();
    }

    float2 zz = both(0.f), tz = both(0.f);
#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const Vals<kU> vz = unpack(z[k]), vy = unpack(dy[k]);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        zz = __ffma2_rn(vz.p[e], vz.p[e], zz);
        tz = __ffma2_rn(__fmul2_rn(vy.p[e], w[k].p[e]), vz.p[e], tz);
      }
    }
    float s[2] = {zz.x + zz.y, tz.x + tz.y};
    group_sum<kGroup, 2>(s, sums, parity);
    const float rstd = rsqrtf(s[0] * a.inv_d + a.eps);
    // in this order a row of zeros gives 0 even where rstd^3 would overflow
    const float back = -rstd * (rstd * (rstd * (s[1] * a.inv_d)));
    const int64_t out_row = static_cast<int64_t>(row) * a.d;
    NarrowMask<kU < 8 ? kU : 1, kUnits> mask;
    if constexpr (kU < 8)
      if (dropping) mask = draw_narrow<kU, kUnits, kGroup>(drop, line, b, i, j, lane & ~31, a.octs);

#pragma unroll
    for (int k = 0; k < kUnits; ++k) {
      const int n = lane + k * kGroup;
      const bool on = valid && n < units;
      const Vals<kU> vz = unpack(z[k]), vy = unpack(dy[k]);
      Vals<kU> g = unpack(dz[k]);
#pragma unroll
      for (int e = 0; e < kPairs; ++e) {
        const float2 y = __fmul2_rn(vy.p[e], both(rstd));
        g.p[e] = __ffma2_rn(vz.p[e], both(back), __ffma2_rn(w[k].p[e], y, g.p[e]));
        dw[k].p[e] = __ffma2_rn(vz.p[e], y, dw[k].p[e]);
      }
      if (on && a.d_stream != nullptr) store_unit<T, kU>(a.d_stream + out_row + n * kU, pack<T, kU>(g));
      if (a.d_update != nullptr) {
        if (dropping) {
          if constexpr (kU == 8) {
            drop_oct(draw_oct(drop, b, i, j, n), line, drop.gain, g);
          } else {
            const uint32_t bits = narrow_bits<kU, kUnits>(mask, k);
            g.p[0].x = bits & 1u ? g.p[0].x * drop.gain : 0.f;
            if constexpr (kU > 1) g.p[0].y = bits & 2u ? g.p[0].y * drop.gain : 0.f;
          }
        }
        if (on) store_unit<T, kU>(a.d_update + out_row + n * kU, pack<T, kU>(g));
      }
    }
    if (a.partial != nullptr && ++held == kFold) {
      held = 0;
      carry();
    }
  }

  if (a.partial == nullptr) return;
  carry();
  __syncthreads();
  // channel c is part of unit c / kU: lane (c / kU) % kGroup, unit (c / kU) / kGroup of every row the CTA holds
  for (int c = threadIdx.x; c < a.d; c += kWide) {
    const int n = c / kU;
    const double* f = fold + (n / kGroup * kU + c % kU) * kWide + n % kGroup;
    double sum = 0.0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) sum += f[r * kGroup];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.d + c] = sum;
  }
}

// d_w[c] = sum over the CTAs' sums: 16 channels and 64 rows of sums per CTA, four rows of a thread in flight.
constexpr int kJoinChannels = 16, kJoinRows = 64;
__global__ void __launch_bounds__(kJoinChannels* kJoinRows) join_weight_kernel(const double* partial, int parts, int d,
                                                                              void* d_weight, int dtype) {
  behind_previous();
  __shared__ double s[kJoinRows][kJoinChannels + 1];
  const int x = threadIdx.x % kJoinChannels, y = threadIdx.x / kJoinChannels;
  const int c = blockIdx.x * kJoinChannels + x;
  double sum = 0.0;
  if (c < d) {
    const double* p = partial + c;
#pragma unroll 4
    for (int r = y; r < parts; r += kJoinRows) sum += p[static_cast<int64_t>(r) * d];
  }
  s[y][x] = sum;
#pragma unroll
  for (int half = kJoinRows / 2; half > 0; half /= 2) {
    __syncthreads();
    if (y < half) s[y][x] += s[y + half][x];
  }
  if (y == 0 && c < d) store_any(d_weight, c, dtype, static_cast<float>(s[0][x]));
}

// Lanes per row and channels per lane, by unit (8, 2 or 1 channels) and width.
struct Shape {
  int group, channels;
};
inline Shape shape_of(int unit, int d) {
  if (unit == 8) {
    if (d <= 64) return {8, 8};
    if (d <= 128) return {16, 8};
    if (d <= 256) return {32, 8};
    if (d <= 512) return {32, 16};
    return {d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024, 8};
  }
  if (d <= 128) return {32, 4};
  if (d <= 256) return {32, 8};
  return {d <= 512 ? 128 : d <= 1024 ? 256 : d <= 2048 ? 512 : 1024, d <= 4096 ? 4 : 8};
}

// CTAs of the gradient kernel: what 64 registers a thread let be resident (half of that for 16 channels a lane), or one
// per group of rows.
inline uint32_t grid_of(uint32_t rows, Shape w, int sms) {
  const uint32_t threads = threads_of(w.group), held = threads / w.group;
  const uint32_t need = (rows + held - 1) / held;
  const uint32_t most = static_cast<uint32_t>(sms) * ((w.channels == 16 ? 512 : 1024) / threads);
  return need < most ? need : most;
}

template <typename T, int kU, int kGroup, int kUnits>
cudaError_t launch_rows(const GradArgs<T>& a, uint32_t grid, cudaStream_t stream) {
  constexpr int kWide = threads_of(kGroup);
  const int smem = a.partial != nullptr ? kUnits * kU * kWide * static_cast<int>(sizeof(double)) : 0;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(norm_grad_kernel<T, kU, kGroup, kUnits>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  norm_grad_kernel<T, kU, kGroup, kUnits><<<grid, kWide, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, int kU>
cudaError_t by_shape(const GradArgs<T>& a, Shape w, uint32_t grid, cudaStream_t s) {
  if constexpr (kU == 8) {
    if (w.group == 8) return launch_rows<T, 8, 8, 1>(a, grid, s);
    if (w.group == 16) return launch_rows<T, 8, 16, 1>(a, grid, s);
    if (w.group == 32 && w.channels == 8) return launch_rows<T, 8, 32, 1>(a, grid, s);
    if (w.group == 32) return launch_rows<T, 8, 32, 2>(a, grid, s);
    if (w.group == 128) return launch_rows<T, 8, 128, 1>(a, grid, s);
    if (w.group == 256) return launch_rows<T, 8, 256, 1>(a, grid, s);
    if (w.group == 512) return launch_rows<T, 8, 512, 1>(a, grid, s);
    return launch_rows<T, 8, 1024, 1>(a, grid, s);
  } else {
    if (w.group == 32 && w.channels == 4) return launch_rows<T, kU, 32, 4 / kU>(a, grid, s);
    if (w.group == 32) return launch_rows<T, kU, 32, 8 / kU>(a, grid, s);
    if (w.group == 128) return launch_rows<T, kU, 128, 4 / kU>(a, grid, s);
    if (w.group == 256) return launch_rows<T, kU, 256, 4 / kU>(a, grid, s);
    if (w.group == 512) return launch_rows<T, kU, 512, 4 / kU>(a, grid, s);
    if (w.channels == 4) return launch_rows<T, kU, 1024, 4 / kU>(a, grid, s);
    return launch_rows<T, kU, 1024, 8 / kU>(a, grid, s);
  }
}

template <typename T>
cudaError_t run(const pair_norm_desc_t* d, const pair_tensor_t* z, const pair_tensor_t* dy, const pair_tensor_t* dz,
                const void* weight, void* d_stream, void* d_update, void* d_weight, void* workspace, int sms,
                cudaStream_t s) {
  GradArgs<T> a;
  a.z = strided<T>(z);
  a.dy = strided<T>(dy);
  a.dz = strided<T>(dz);
  a.weight = weight;
  a.d_stream = static_cast<T*>(d_stream);
  a.d_update = static_cast<T*>(d_update);
  a.partial = d_weight != nullptr ? static_cast<double*>(workspace) : nullptr;
  a.walk = RowWalk{make_fast_div(d->j), make_fast_div(d->i)};
  a.drop = make_dropout(d->dropout);
  a.rows = static_cast<uint32_t>(d->b) * d->i * d->j;
  a.d = d->d;
  a.octs = (d->d + 7) / 8;
  a.weight_dtype = d->weight_dtype;
  a.flat = collapses(z, d->b, d->i, d->j) && collapses(dy, d->b, d->i, d->j) && collapses(dz, d->b, d->i, d->j);
  a.eps = d->eps;
  a.inv_d = 1.f / static_cast<float>(d->d);
  const int unit = unit_of(d->d, sizeof(T), {z, dy, dz}, {d_stream, d_update});
  const Shape w = shape_of(unit, d->d);
  const uint32_t grid = grid_of(a.rows, w, sms);
  cudaError_t e = cudaSuccess;
  if (unit == 8) {
    e = by_shape<T, 8>(a, w, grid, s);
  } else {
    if constexpr (sizeof(T) == 2) {
      if (unit == 2) e = by_shape<T, 2>(a, w, grid, s);
    }
    if (unit == 1) e = by_shape<T, 1>(a, w, grid, s);
  }
  if (e != cudaSuccess || d_weight == nullptr) return e;
  return launch_behind(join_weight_kernel, (a.d + kJoinChannels - 1) / kJoinChannels, kJoinChannels * kJoinRows, 0, s,
                       static_cast<const double*>(a.partial), static_cast<int>(grid), a.d, d_weight, static_cast<int>(d->weight_dtype));
}

}  // namespace
}  // namespace pair

extern "C" int pair_sm100_add_norm_grad_workspace(const pair_norm_desc_t* desc, uint64_t* bytes) {
  using namespace pair;
  const char* who = "pair_sm100_add_norm_grad_workspace";
  if (int rc = check_norm_desc(desc, who)) return rc;
  if (bytes == nullptr) return trimul::report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: bytes is NULL", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return trimul::report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  const uint32_t rows = static_cast<uint32_t>(desc->b) * desc->i * desc->j;
  // the unit depends on addresses that are not known here: room for the largest grid
  uint32_t most = 0;
  for (int unit : {8, 2}) {
    const uint32_t grid = grid_of(rows, shape_of(unit, desc->d), sms);
    most = grid > most ? grid : most;
  }
  *bytes = static_cast<uint64_t>(most) * desc->d * sizeof(double);
  return TRIMUL_OK;
}

extern "C" int pair_sm100_add_norm_grad(const pair_norm_desc_t* desc, const pair_tensor_t* stream, const pair_tensor_t* dy,
                                        const pair_tensor_t* dz, const void* weight, void* d_stream, void* d_update,
                                        void* d_weight, void* workspace, trimul_stream_t cuda_stream) {
  using namespace pair;
  using trimul::report_error;
  const char* who = "pair_sm100_add_norm_grad";
  if (int rc = check_norm_desc(desc, who)) return rc;
  if (static_cast<int64_t>(desc->b) * desc->i * desc->j == 0) {
    if (d_weight == nullptr) return TRIMUL_OK;
    cudaError_t e = cudaMemsetAsync(d_weight, 0, static_cast<size_t>(desc->d) * type_bytes(desc->weight_dtype), cuda_stream);
    if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
    return TRIMUL_OK;
  }
  if (weight == nullptr) return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: weight is NULL", who);
  if (d_stream == nullptr && d_update == nullptr && d_weight == nullptr)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: no output", who);
  if (stream == nullptr || stream->data == nullptr)
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: stream is NULL", who);
  if (d_weight != nullptr && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7) != 0))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: the weight's gradient needs an 8-byte aligned workspace", who);
  const int sms = trimul::current_device_sms();
  if (sms <= 0) return report_error(TRIMUL_ERR_CUDA, "%s: cannot query the current device", who);
  cudaError_t e;
  if (desc->dtype == PAIR_FP32)
    e = run<float>(desc, stream, dy, dz, weight, d_stream, d_update, d_weight, workspace, sms, cuda_stream);
  else if (desc->dtype == PAIR_FP16)
    e = run<__half>(desc, stream, dy, dz, weight, d_stream, d_update, d_weight, workspace, sms, cuda_stream);
  else
    e = run<__nv_bfloat16>(desc, stream, dy, dz, weight, d_stream, d_update, d_weight, workspace, sms, cuda_stream);
  if (e != cudaSuccess) return report_error(TRIMUL_ERR_CUDA, "%s: %s", who, cudaGetErrorString(e));
  return TRIMUL_OK;
}
