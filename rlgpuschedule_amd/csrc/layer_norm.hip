// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / D, var = sum (x - mean)^2 / D, r = 1 / sqrt(var + eps)
//   n = (x - mean) r,  y = n w + b
//   g = dy w,  dx = r (g - mean(g) - n mean(g n))
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Statistics and sums are held in 32 bits; y, dx, dw and db are rounded to
// their types once.
#include "seq_api.h"
#include "seq_common.h"

namespace {
using namespace seq;

struct NormFwd {
  const void* x;
  const void* w;  // null: ones
  const void* b;  // null: zeros
  void* y;
  float* mean;
  float* rstd;
  int64_t rows, dim, x_stride;
  float eps;
};

struct NormBwd {
  const void* dy;
  const void* x;
  const void* w;
  const float* mean;
  const float* rstd;
  void* dx;        // null: not asked for
  float* partial;  // [parts, 2, D] sums of dy n and dy; null: not asked for
  int64_t rows, dim, x_stride, dy_stride;
  int parts;
};

struct NormSum {
  const float* partial;
  void* dw;
  void* db;
  int64_t dim;
  int parts;
};

__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = group_sum(v);
  const int wave = threadIdx.x / kWave, waves = blockDim.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[wave] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < waves; ++i) v += lds[i];
  return v;
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_fwd_kernel(NormFwd a) {
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    T* y = (T*)a.y + row * a.dim;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) s += (float)x[i];
    const float mean = block_sum(s, lds) / (float)a.dim;
    s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) {
      const float d = (float)x[i] - mean;
      s += d * d;
    }
    const float r = 1.f / sqrtf(block_sum(s, lds) / (float)a.dim + a.eps);
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) {
      const float w = a.w ? (float)((const W*)a.w)[i] : 1.f;
      const float b = a.b ? (float)((const W*)a.b)[i] : 0.f;
      y[i] = (T)(((float)x[i] - mean) * r * w + b);
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[row] = mean;
      if (a.rstd) a.rstd[row] = r;
    }
  }
}

template <typename T, typename W>
__global__ __launch_bounds__(256) void norm_dx_kernel(NormBwd a) {
  __shared__ float lds[4];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* dy = (const T*)a.dy + row * a.dy_stride;
    T* dx = (T*)a.dx + row * a.dim;
    const float mean = a.mean[row], r = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) {
      const float g = (float)dy[i] * (a.w ? (float)((const W*)a.w)[i] : 1.f);
      s1 += g;
      s2 += g * ((float)x[i] - mean) * r;
    }
    s1 = block_sum(s1, lds) / (float)a.dim;
    s2 = block_sum(s2, lds) / (float)a.dim;
    for (int64_t i = threadIdx.x; i < a.dim; i += 256) {
      const float g = (float)dy[i] * (a.w ? (float)((const W*)a.w)[i] : 1.f);
      const float n = ((float)x[i] - mean) * r;
      dx[i] = (T)(r * (g - s1 - n * s2));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_dw_kernel(NormBwd a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += a.parts) {
    const float dy = (float)((const T*)a.dy)[row * a.dy_stride + i];
    const float x = (float)((const T*)a.x)[row * a.x_stride + i];
    dw += dy * (x - a.mean[row]) * a.rstd[row];
    db += dy;
  }
  a.partial[(2 * (int64_t)blockIdx.y) * a.dim + i] = dw;
  a.partial[(2 * (int64_t)blockIdx.y + 1) * a.dim + i] = db;
}

template <typename W>
__global__ __launch_bounds__(256) void norm_sum_kernel(NormSum a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
  for (int p = 0; p < a.parts; ++p) {
    dw += a.partial[(2 * (int64_t)p) * a.dim + i];
    db += a.partial[(2 * (int64_t)p + 1) * a.dim + i];
  }
  if (a.dw) ((W*)a.dw)[i] = (W)dw;
  if (a.db) ((W*)a.db)[i] = (W)db;
}

template <typename T, typename W>
hipError_t fwd(const NormFwd& a, hipStream_t s) {
  if (a.rows == 0) return hipSuccess;
  const int64_t grid = a.rows < 65536 ? a.rows : 65536;
  return launch(norm_fwd_kernel<T, W>, dim3(grid), dim3(256), 0, s, a);
}

template <typename T, typename W>
hipError_t bwd(const NormBwd& a, const NormSum& z, hipStream_t s) {
  hipError_t e = hipSuccess;
  if (a.dx && a.rows > 0) {
    const int64_t grid = a.rows < 65536 ? a.rows : 65536;
    e = launch(norm_dx_kernel<T, W>, dim3(grid), dim3(256), 0, s, a);
  }
  if (e == hipSuccess && a.partial) {
    const int cols = (int)((a.dim + 255) / 256);
    e = launch(norm_dw_kernel<T>, dim3(cols, a.parts), dim3(256), 0, s, a);
    if (e == hipSuccess)
      e = launch(norm_sum_kernel<W>, dim3(cols), dim3(256), 0, s, z);
  }
  return e;
}

}  // namespace

extern "C" int rlsched_norm_fwd(int device, void* stream, const void* x,
                                const void* w, const void* b, void* y,
                                float* mean, float* rstd, int64_t rows,
                                int64_t dim, int64_t x_stride, double eps,
                                int type, int wtype) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const NormFwd a = {x, w, b, y, mean, rstd, rows, dim, x_stride, (float)eps};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32 && wtype == F32) return fwd<float, float>(a, s);
  if (type == BF16 && wtype == F32) return fwd<bf16, float>(a, s);
  if (type == BF16 && wtype == BF16) return fwd<bf16, bf16>(a, s);
  if (type == F16 && wtype == F32) return fwd<f16, float>(a, s);
  if (type == F16 && wtype == F16) return fwd<f16, f16>(a, s);
  return hipErrorInvalidValue;
}

// Row groups whose sums of dy n and dy the backward pass keeps apart: its
// scratch holds 2 * parts * dim floats.
extern "C" int64_t rlsched_norm_parts(int64_t rows, int64_t dim) {
  (void)dim;
  const int64_t p = (rows + 31) / 32;
  return p < 1 ? 1 : p < 128 ? p : 128;
}

extern "C" int rlsched_norm_bwd(int device, void* stream, const void* dy,
                                const void* x, const void* w,
                                const float* mean, const float* rstd, void* dx,
                                void* dw, void* db, float* partial,
                                int64_t rows, int64_t dim, int64_t x_stride,
                                int64_t dy_stride, int type, int wtype) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const int parts = (int)rlsched_norm_parts(rows, dim);
  const NormBwd a = {dy,      x,    w,   mean,     rstd,      dx,
                     partial, rows, dim, x_stride, dy_stride, parts};
  const NormSum z = {partial, dw, db, dim, parts};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32 && wtype == F32) return bwd<float, float>(a, z, s);
  if (type == BF16 && wtype == F32) return bwd<bf16, float>(a, z, s);
  if (type == BF16 && wtype == BF16) return bwd<bf16, bf16>(a, z, s);
  if (type == F16 && wtype == F32) return bwd<f16, float>(a, z, s);
  if (type == F16 && wtype == F16) return bwd<f16, f16>(a, z, s);
  return hipErrorInvalidValue;
}

// Build provenance: ops/build.py embeds a prefix of the sources' sha256 and
// checks it at load.
#ifndef RLS_SOURCE_HASH
#define RLS_SOURCE_HASH "unset"
#endif
extern "C" const char* rlsched_source_hash() {
  return "RLSHASH:" RLS_SOURCE_HASH;
}
