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
// Measured (of the 6457 GB/s of a copy; with gradients of both outputs and of the gain): 1024 x 1024 rows of 256 bf16 channels 328 us, 101 %,
// with dropout 440, 95 % (346 and 452 with one wave of CTAs); 700 x 700 fp32 rows of 256 303 and 405 us, 102 and 96 %; 384 x 384 bf16
// rows of 128 29 and 39 us, 81 and 74 %: one wave, whose fill, drain and joining kernel show.
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

// Shared memory of a CTA: the gain's sums, and the stages of three rows where both fit an SM (all but rows of 4097 to 8192 channels
// in one-channel units of fp32, which are loaded directly).
template <typename T, int kU, int kGroup, int kUnits>
struct Shared {
  using In = Rows<T, kU, kGroup, kUnits>;
  static constexpr int kSums = kUnits * kU * In::kWide * static_cast<int>(sizeof(double));
  static constexpr bool kStaged = In::kStaged && kSums + 2 * 3 * In::kStage <= 224 * 1024;
  static constexpr int kStages = kStaged ? 2 * 3 * In::kStage : 0;
};

// As add_norm_kernel: kU channels per access, kGroup lanes per row, kUnits units per lane.
template <typename T, int kU, int kGroup, int kUnits>
__global__ void __launch_bounds__(threads_of(kGroup), (kU * kUnits > 8 ? 512 : 1024) / threads_of(kGroup)) norm_grad_kernel(const __grid_constant__ GradArgs<T> a) {
  __shared__ float sums[2 * 32 * 2];
  extern __shared__ double fold[];  // [unit of the lane][channel of the unit][thread], then the stages of the rows
  constexpr int kWide = threads_of(kGroup);
  constexpr int kRows = kWide / kGroup;
  using In = Rows<T, kU, kGroup, kUnits>;
  constexpr bool kStaged = Shared<T, kU, kGroup, kUnits>::kStaged;
  if (a.partial != nullptr) next_may_start();  // the kernel that joins the sums
  constexpr int kPairs = kU * kUnits / 2;
  const int lane = threadIdx.x % kGroup;
  const int units = a.d / kU;
  const bool dropping = a.drop.keep < 65536u && a.d_update != nullptr;
  const uint32_t line = a.drop.keep << 16;
  Dropout drop = a.drop;
  if (dropping) resolve_seed(drop);

  const Lane<kU, kUnits> w = load_gain<kU, kGroup, kUnits>(a.weight, a.weight_dtype, lane, units);
  Lane<kU, kUnits> dw;
#pragma unroll
  for (int n = 0; n < kPairs; ++n) dw.p[n] = both(0.f);
  if (a.partial != nullptr)
#pragma unroll
    for (int c = 0; c < 2 * kPairs; ++c) fold[c * kWide + threadIdx.x] = 0.0;
  auto carry = [&] {
#pragma unroll
    for (int n = 0; n < kPairs; ++n) {
      fold[2 * n * kWide + threadIdx.x] += dw.p[n].x;
      fold[(2 * n + 1) * kWide + threadIdx.x] += dw.p[n].y;
      dw.p[n] = both(0.f);
    }
  };

  const uint32_t span = gridDim.x * kRows;
  auto rows_of = [&](uint32_t row, const T*& zp, const T*& yp, const T*& gp) {
    if (a.flat) {
      zp = a.z.flat(row), yp = a.dy.flat(row), gp = a.dz.flat(row);
    } else {
      uint32_t b, i, j;
      a.walk.at(row, b, i, j);
      zp = a.z.row(b, i, j), yp = a.dy.row(b, i, j), gp = a.dz.row(b, i, j);
    }
  };
  char* const stages = reinterpret_cast<char*>(fold + (a.partial != nullptr ? kUnits * kU * kWide : 0));
  auto fetch = [&](uint32_t row, char* to) {
    if (row < a.rows) {
      const T *zp, *yp, *gp;
      rows_of(row, zp, yp, gp);
      In::fetch(to, zp, a.d);
      if (a.dy.p != nullptr) In::fetch(to + In::kStage, yp, a.d);
      if (a.dz.p != nullptr) In::fetch(to + 2 * In::kStage, gp, a.d);
    }
    stage_commit();
  };
  const uint32_t mine = threadIdx.x / kGroup;
  if constexpr (kStaged) fetch(blockIdx.x * kRows + mine, stages);

  int parity = 0, held = 0;
  for (uint32_t first = blockIdx.x * kRows; first < a.rows; first += span, parity ^= 1) {
    const uint32_t row = first + mine;
    const bool valid = row < a.rows;
    uint32_t b = 0, i = 0, j = 0;
    if (valid && dropping) a.walk.at(row, b, i, j);

    Unit<T, kU> z[kUnits], dy[kUnits], dz[kUnits];
    if constexpr (kStaged) {
      // two stages: one at hand, one on its way (a third is no faster)
      fetch(row + span, stages + (parity ^ 1) * 3 * In::kStage);
      stage_wait<1>();
      const char* from = stages + parity * 3 * In::kStage;
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const bool on = valid && lane + k * kGroup < units;
        z[k] = on ? In::read(from, k) : zero_unit<T, kU>();
        dy[k] = on && a.dy.p != nullptr ? In::read(from + In::kStage, k) : zero_unit<T, kU>();
        dz[k] = on && a.dz.p != nullptr ? In::read(from + 2 * In::kStage, k) : zero_unit<T, kU>();
      }
    } else {
      const T *zp = nullptr, *yp = nullptr, *gp = nullptr;
      if (valid) rows_of(row, zp, yp, gp);
#pragma unroll
      for (int k = 0; k < kUnits; ++k) {
        const int n = lane + k * kGroup;
        const bool on = valid && n < units;
        z[k] = on ? load_unit<T, kU>(zp + n * kU) : zero_unit<T, kU>();
        dy[k] = on && a.dy.p != nullptr ? load_unit<T, kU>(yp + n * kU) : zero_unit<T, kU>();
        dz[k] = on && a.dz.p != nullptr ? load_unit<T, kU>(gp + n * kU) : zero_unit<T, kU>();
      }
    }
    const int64_t at = static_cast<int64_t>(row) * a.d + lane * kU;  // the lane's first channel

    const Lane<kU, kUnits> vz = unpack_all<T, kU, kUnits>(z), vy = unpack_all<T, kU, kUnits>(dy);
    float2 zz = both(0.f), tz = both(0.f);
#pragma unroll
    for (int n = 0; n < kPairs; ++n) {
      zz = __ffma2_rn(vz.p[n], vz.p[n], zz);
      tz = __ffma2_rn(__fmul2_rn(vy.p[n], w.p[n]), vz.p[n], tz);
    }
    float s[2] = {zz.x + zz.y, tz.x + tz.y};
    group_sum<kGroup, 2>(s, sums, parity);
    const float rstd = rsqrtf(s[0] * a.inv_d + a.eps);
    // in this order a row of zeros gives 0 even where rstd^3 would overflow
    const float2 back = both(-rstd * (rstd * (rstd * (s[1] * a.inv_d))));
    Lane<kU, kUnits> g = unpack_all<T, kU, kUnits>(dz);
#pragma unroll
    for (int n = 0; n < kPairs; ++n) {
      const float2 y = __fmul2_rn(vy.p[n], both(rstd));
      g.p[n] = __ffma2_rn(vz.p[n], back, __ffma2_rn(w.p[n], y, g.p[n]));
      dw.p[n] = __ffma2_rn(vz.p[n], y, dw.p[n]);
    }
    Unit<T, kU> out[kUnits];
    if (a.d_stream != nullptr) {
      pack_all<T, kU, kUnits>(g, out);
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
        if (valid && lane + k * kGroup < units) store_unit<T, kU>(a.d_stream + at + k * kGroup * kU, out[k]);
    }
    if (a.d_update != nullptr) {
      if (dropping) drop_all<kU, kGroup, kUnits>(drop, line, b, i, j, lane, a.octs, g);
      pack_all<T, kU, kUnits>(g, out);
#pragma unroll
      for (int k = 0; k < kUnits; ++k)
        if (valid && lane + k * kGroup < units) store_unit<T, kU>(a.d_update + at + k * kGroup * kU, out[k]);
    }
    if (a.partial != nullptr && ++held == kFold) {
      held = 0;
      carry();
    }
  }

  if (a.partial == nullptr) return;
  carry();
  __syncthreads();
  // channel c is part of unit c / kU: lane (c / kU) % kGroup, value (c / kU) / kGroup * kU + c % kU of every row the CTA holds
  for (int c = threadIdx.x; c < a.d; c += kWide) {
    const int n = c / kU;
    const double* f = fold + (n / kGroup * kU + c % kU) * kWide + n % kGroup;
    double sum = 0.0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) sum += f[r * kGroup];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.d + c] = sum;
  }
}

// d_w[c] = sum over the CTAs' sums: 16 channels and 64 rows of sums per CTA, eight rows of a thread in flight.
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
#pragma unroll 8
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
  if (unit == 1 && d <= 192) return {32, 6};
  if (d <= 256) return {32, 8};
  return {d <= 512 ? 64 : d <= 1024 ? 128 : d <= 2048 ? 256 : d <= 4096 ? 512 : 1024, 8};
}

// CTAs of the gradient kernel, from the sizes alone: what 64 registers a thread let be resident (half of that for 16 channels a lane),
// or more where each still has 32 rows a lane and 256 rows in all: a CTA costs a row of sums.
inline uint32_t grid_of(uint32_t rows, Shape w, int sms) {
  const uint32_t threads = threads_of(w.group), held = threads / w.group;
  const uint32_t need = (rows + held - 1) / held;
  const uint32_t resident = (w.channels == 16 ? 512 : 1024) / threads, least = held < 8 ? 256 / held : 32;
  const uint32_t eighth = need / (8 * static_cast<uint32_t>(sms) * resident);  // at most eight waves: one thread adds up every 64th CTA's sums
  return walk_grid(need, sms, resident, least > eighth ? least : eighth);
}

template <typename T, int kU, int kGroup, int kUnits>
cudaError_t launch_rows(const GradArgs<T>& a, uint32_t grid, cudaStream_t stream) {
  constexpr int kWide = threads_of(kGroup);
  constexpr int kSums = Shared<T, kU, kGroup, kUnits>::kSums, kStages = Shared<T, kU, kGroup, kUnits>::kStages;
  auto kernel = norm_grad_kernel<T, kU, kGroup, kUnits>;
  if (kSums + kStages > 47 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSums + kStages);
    if (e != cudaSuccess) return e;
  }
  return pair::launch(kernel, grid, kWide, kStages + (a.partial != nullptr ? kSums : 0), stream, a);
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
    if constexpr (kU == 1)
      if (w.group == 32 && w.channels == 6) return launch_rows<T, kU, 32, 6>(a, grid, s);
    if (w.group == 32) return launch_rows<T, kU, 32, 8 / kU>(a, grid, s);
    if (w.group == 64) return launch_rows<T, kU, 64, 8 / kU>(a, grid, s);
    if (w.group == 128) return launch_rows<T, kU, 128, 8 / kU>(a, grid, s);
    if (w.group == 256) return launch_rows<T, kU, 256, 8 / kU>(a, grid, s);
    if (w.group == 512) return launch_rows<T, kU, 512, 8 / kU>(a, grid, s);
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
  a.flat = collapses(z, d->i, d->j) && collapses(dy, d->i, d->j) && collapses(dz, d->i, d->j);
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
  for (int unit : {8, 2, 1}) {
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
  const pair_tensor_t z = canonical(stream, desc->b, desc->i, desc->j), y = canonical(dy, desc->b, desc->i, desc->j),
                      g = canonical(dz, desc->b, desc->i, desc->j);
  stream = &z, dy = &y, dz = &g;
  const int weight_size = type_bytes(desc->weight_dtype);
  if (!elements_aligned(type_bytes(desc->dtype), {stream, dy, dz}, {d_stream, d_update}) || !aligned(weight, weight_size) ||
      !aligned(d_weight, weight_size) || !aligned(desc->dropout.device_seed, 8))
    return report_error(TRIMUL_ERR_INVALID_ARGUMENT, "%s: a buffer is not aligned to its elements", who);
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
