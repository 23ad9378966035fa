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
  float eps;
};

template <typename T, int kGroup, int kOcts, bool kWide>
__global__ void __launch_bounds__(kThreads) norm_grad_kernel(const __grid_constant__ GradArgs<T> a) {
  __shared__ float sums[2 * 8 * 2];
  extern __shared__ double fold[];  // [oct of the lane][channel of the oct][thread]
  constexpr int kRows = kThreads / kGroup;
  const int lane = threadIdx.x % kGroup;
  Dropout drop = a.drop;
  if (drop.keep < 65536u) resolve_seed(drop);

  float w[kOcts][8], dw[kOcts][8];
#pragma unroll
  for (int k = 0; k < kOcts; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = (lane + k * kGroup) * 8 + e;
      w[k][e] = c < a.d ? load_any(a.weight, c, a.weight_dtype) : 0.f;
      dw[k][e] = 0.f;
      if (a.partial != nullptr) fold[(k * 8 + e) * kThreads + threadIdx.x] = 0.0;
    }

  const float inv_d = 1.f / static_cast<float>(a.d);
  int parity = 0, held = 0;
  for (uint32_t first = blockIdx.x * kRows; first < a.rows; first += gridDim.x * kRows, parity ^= 1) {
    const uint32_t row = first + threadIdx.x / kGroup;
    const bool valid = row < a.rows;
    uint32_t b, i, j;
    a.walk.at(valid ? row : 0, b, i, j);
    const T* zp = a.z.row(b, i, j);
    const T* yp = a.dy.p != nullptr ? a.dy.row(b, i, j) : nullptr;
    const T* gp = a.dz.p != nullptr ? a.dz.row(b, i, j) : nullptr;

    Oct<T> z[kOcts], dy[kOcts], dz[kOcts];
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int v = lane + k * kGroup;
      const bool on = valid && v < a.octs;
      z[k] = on ? load_oct<kWide>(zp + v * 8, a.d - v * 8) : zero_oct<T>();
      dy[k] = on && yp != nullptr ? load_oct<kWide>(yp + v * 8, a.d - v * 8) : zero_oct<T>();
      dz[k] = on && gp != nullptr ? load_oct<kWide>(gp + v * 8, a.d - v * 8) : zero_oct<T>();
    }

    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      float fz[8], fy[8];
      unpack(z[k], fz);
      unpack(dy[k], fy);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s[0] += fz[e] * fz[e];
        s[1] += fy[e] * w[k][e] * fz[e];
      }
    }
    group_sum<kGroup, 2>(s, sums, parity);
    const float rstd = rsqrtf(s[0] * inv_d + a.eps);
    // in this order a row of zeros gives 0 even where rstd^3 would overflow
    const float back = rstd * (rstd * (rstd * (s[1] * inv_d)));
    const int64_t out_row = static_cast<int64_t>(row) * a.d;

#pragma unroll
    for (int k = 0; k < kOcts; ++k) {
      const int v = lane + k * kGroup;
      float fz[8], fy[8], g[8];
      unpack(z[k], fz);
      unpack(dy[k], fy);
      unpack(dz[k], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        g[e] += rstd * (w[k][e] * fy[e]) - fz[e] * back;
        dw[k][e] += valid ? fy[e] * (fz[e] * rstd) : 0.f;
      }
      if (valid && v < a.octs) {
        if (a.d_stream != nullptr) store_oct<kWide>(a.d_stream + out_row + v * 8, pack<T>(g), a.d - v * 8);
        if (a.d_update != nullptr) {
          if (drop.keep < 65536u) apply_dropout(drop, b, i, j, v, g);
          store_oct<kWide>(a.d_update + out_row + v * 8, pack<T>(g), a.d - v * 8);
        }
      }
    }
    if (a.partial != nullptr && ++held == kFold) {
      held = 0;
#pragma unroll
      for (int k = 0; k < kOcts; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          fold[(k * 8 + e) * kThreads + threadIdx.x] += dw[k][e];
          dw[k][e] = 0.f;
        }
    }
  }

  if (a.partial == nullptr) return;
#pragma unroll
  for (int k = 0; k < kOcts; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) fold[(k * 8 + e) * kThreads + threadIdx.x] += dw[k][e];
  __syncthreads();
  // channel c belongs to lane (c / 8) % kGroup, oct (c / 8) / kGroup of every row the CTA holds
  for (int c = threadIdx.x; c < a.d; c += kThreads) {
    const int v = c >> 3;
    const double* f = fold + (v / kGroup * 8 + (c & 7)) * kThreads + v % kGroup;
    double sum = 0.0;
#pragma unroll
    for (int r = 0; r < kRows; ++r) sum += f[r * kGroup];
    a.partial[static_cast<int64_t>(blockIdx.x) * a.d + c] = sum;
  }
}

// d_w[c] = sum over the CTAs' sums: 32 channels per CTA, eight rows of sums at a time.
__global__ void __launch_bounds__(kThreads) join_weight_kernel(const double* partial, int parts, int d, void* d_weight,
                                                               int dtype) {
  __shared__ double s[8][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
  double sum = 0.0;
  if (c < d)
    for (int p = y; p < parts; p += 8) sum += partial[static_cast<int64_t>(p) * d + c];
  s[y][threadIdx.x & 31] = sum;
  __syncthreads();
  if (y == 0 && c < d) {
    for (int k = 1; k < 8; ++k) sum += s[k][threadIdx.x & 31];
    store_any(d_weight, c, dtype, static_cast<float>(sum));
  }
}

struct Width {
  int group, octs;
};
inline Width width_of(int octs) {
  if (octs <= 8) return {8, 1};
  if (octs <= 16) return {16, 1};
  if (octs <= 32) return {32, 1};
  if (octs <= 64) return {32, 2};
  if (octs <= 128) return {32, 4};
  if (octs <= 256) return {256, 1};
  if (octs <= 512) return {256, 2};
  return {256, 4};
}

// CTAs of the gradient kernel: what stays resident beside the shared sums (16, 32 or 64 KB a CTA), or one per row.
inline uint32_t grid_of(uint32_t rows, int octs, int sms) {
  const Width w = width_of(octs);
  const uint32_t held = kThreads / w.group;
  const uint32_t need = (rows + held - 1) / held;
  const uint32_t most = static_cast<uint32_t>(sms) * (w.octs == 1 ? 4 : w.octs == 2 ? 3 : 2);
  return need < most ? need : most;
}

template <typename T, int kGroup, int kOcts, bool kWide>
cudaError_t launch(const GradArgs<T>& a, uint32_t grid, cudaStream_t stream) {
  const int smem = a.partial != nullptr ? kOcts * 8 * kThreads * static_cast<int>(sizeof(double)) : 0;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(norm_grad_kernel<T, kGroup, kOcts, kWide>,
                                         cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  norm_grad_kernel<T, kGroup, kOcts, kWide><<<grid, kThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

template <typename T, bool kWide>
cudaError_t by_width(const GradArgs<T>& a, uint32_t grid, cudaStream_t s) {
  const int o = a.octs;
  if (o <= 8) return launch<T, 8, 1, kWide>(a, grid, s);
  if (o <= 16) return launch<T, 16, 1, kWide>(a, grid, s);
  if (o <= 32) return launch<T, 32, 1, kWide>(a, grid, s);
  if (o <= 64) return launch<T, 32, 2, kWide>(a, grid, s);
  if (o <= 128) return launch<T, 32, 4, kWide>(a, grid, s);
  if (o <= 256) return launch<T, 256, 1, kWide>(a, grid, s);
  if (o <= 512) return launch<T, 256, 2, kWide>(a, grid, s);
  return launch<T, 256, 4, kWide>(a, grid, s);
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
  a.eps = d->eps;
  const uint32_t grid = grid_of(a.rows, a.octs, sms);
  const bool wide = d->d % 8 == 0 && rows_aligned(z, sizeof(T)) && rows_aligned(dy, sizeof(T)) &&
                    rows_aligned(dz, sizeof(T)) && aligned16(d_stream) && aligned16(d_update);
  cudaError_t e = wide ? by_width<T, true>(a, grid, s) : by_width<T, false>(a, grid, s);
  if (e != cudaSuccess || d_weight == nullptr) return e;
  join_weight_kernel<<<(a.d + 31) / 32, kThreads, 0, s>>>(a.partial, static_cast<int>(grid), a.d, d_weight,
                                                        d->weight_dtype);
  return cudaGetLastError();
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
  *bytes = static_cast<uint64_t>(grid_of(rows, (desc->d + 7) / 8, sms)) * desc->d * sizeof(double);
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
