// Layer norm over the last dimension, forward and backward.
//
//   mean = sum x / D, var = sum (x - mean)^2 / D, r = 1 / sqrt(var + eps)
//   n = (x - mean) r,  y = n w + b
//   g = dy w,  dx = r (g - mean(g) - n mean(g n))
//   dw = sum over rows of dy n,  db = sum over rows of dy
//
// Statistics and sums are held in 32 bits; y, dx, dw and db are rounded to
// their types once.
//
// Bound by memory: of rows of up to 2048 vectors of 16 bytes x is read once by
// each pass and held in registers between the sums and what needs them, dy
// likewise. On an MI355X, whose large copy runs at 4.9 TB/s, 131072 x 256 bf16
// takes 30.5 us forward (4.4 TB/s) and 34 + 4 us backward (the last sum of dw
// and db apart; 5.3 TB/s, partly from the cache), 8192 x 4096 fp16 34 and 40 +
// 4 us; 256 x 256 fp32 takes 3.2 us, a launch's time. Longer rows are walked by
// a block, an element a lane, x three times forward, x and dy three times
// backward: 2048 x 8192 fp32 takes 26 and 38 us, 2048 x 8200 40 and 82, 1024 x
// 16384 41 and 72.
#include "seq_api.h"
#include "seq_common.h"

namespace {
using namespace seq;

struct NormFwd {
  const void* x;
  const void* w;  // null: ones
  const void* b;  // null: zeros
  void* y;
  float* mean;  // null: not kept
  float* rstd;
  int64_t rows, dim, x_stride;
  float eps;
  bool w32;  // w and b hold 32 bits, else x's type
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
  bool w32;
};

struct NormSum {
  const float* partial;
  void* dw;  // null: not asked for
  void* db;
  int64_t dim;
  int parts;
};

template <typename T>
constexpr int kVec = 16 / sizeof(T);

// ---- rows of up to G * N vectors, in registers: lane l of G has the vectors
// l, l + G, ... of each of its rows. A row's last vector begins early enough
// to end with it: the first `skip` of its elements are the vector's before,
// computed twice to the same bits and counted once.
template <typename T>
struct Place {
  int from, skip;
  bool some;
  __device__ __forceinline__ Place(int64_t dim, int j) {
    const int D = (int)dim, V = kVec<T>, base = j * V;
    some = base < D;
    from = D < V || base < D - V ? base : D - V;
    skip = base - from;
  }
};

template <typename T>
__device__ __forceinline__ void store_at(T* p, int dim, const Place<T>& at,
                                         const float (&f)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if (dim >= V) {
    store<T, V>(p + at.from, f);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < dim) p[e] = (T)f[e];
  }
}

template <typename T>
__device__ __forceinline__ void load_param(const void* p, bool w32, int dim,
                                           const Place<T>& at, float none,
                                           float (&f)[kVec<T>]) {
  constexpr int V = kVec<T>;
#pragma unroll
  for (int e = 0; e < V; ++e) f[e] = none;
  if (!p || !at.some) return;
  if (dim >= V) {
    if (w32) {
      load<float, V>((const float*)p + at.from, f);
    } else {
      load<T, V>((const T*)p + at.from, f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < dim) f[e] = w32 ? ((const float*)p)[e] : (float)((const T*)p)[e];
  }
}

// Sums over the G lanes of a row; over waves through `lds`, of which the
// caller takes another half each time, so one barrier is enough.
template <int G, int K>
__device__ __forceinline__ void row_sum(float (&v)[K],
                                        float (*lds)[K][G / kWave + 1]) {
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = group_sum<G < kWave ? G : kWave>(v[k]);
  if constexpr (G > kWave) {
    constexpr int W = G / kWave;
    const int wave = threadIdx.x / kWave;
    if (threadIdx.x % kWave == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) (*lds)[k][wave] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[k] += (*lds)[k][w];
    }
  }
}

template <int G>
constexpr int kBlock = G > kWave ? G : 512;  // rows share a block, not a barrier

template <typename T, int G, int N>
__global__ __launch_bounds__(kBlock<G>) void norm_fwd_kernel(NormFwd p) {
  constexpr int V = kVec<T>, R = kBlock<G> / G;
  __shared__ float lds[2][1][G / kWave + 1];
  const int l = threadIdx.x % G, dim = (int)p.dim;
  const float over = 1.f / (float)dim;
  Vec<T, V> x[N];
  auto read = [&](int64_t row) {
    const T* xr = (const T*)p.x + row * p.x_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
      if (dim >= V) {
        x[i] = load<T, V>(xr + at.from);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) x[i].v[e] = e < dim ? xr[e] : (T)0.f;
      }
    }
  };
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G;
  if (row < p.rows) read(row);
  float w[N][V], b[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const Place<T> at(dim, l + G * i);
    load_param<T>(p.w, p.w32, dim, at, 1.f, w[i]);
    load_param<T>(p.b, p.w32, dim, at, 0.f, b[i]);
  }
  for (; row < p.rows; row += step) {
    float f[N][V], s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[i][e] = (float)x[i].v[e];
        s[0] += e < at.skip ? 0.f : f[i][e];
      }
    }
    if (row + step < p.rows) read(row + step);  // while this one is summed
    row_sum<G>(s, &lds[0]);
    const float mean = s[0] * over;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        f[i][e] -= mean;
        const bool in = e >= at.skip && at.from + e < dim;
        s[0] += in ? f[i][e] * f[i][e] : 0.f;
      }
    }
    row_sum<G>(s, &lds[1]);
    const float r = 1.f / sqrtf(s[0] * over + p.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = f[i][e] * r * w[i][e] + b[i][e];
      store_at<T>((T*)p.y + row * p.dim, dim, at, f[i]);
    }
    if (p.mean && l == 0) {
      p.mean[row] = mean;
      p.rstd[row] = r;
    }
  }
}

// dx of a block's rows, and the rows' share of dw and db: the lanes keep
// theirs in registers over all rows, then the block's row groups are added.
// No atomics: the order of the sums is the same each time. A share is written
// and read once more, 4 us of 131072 x 256's 37.
template <typename T, int G, int N>
__global__ __launch_bounds__(kBlock<G>) void norm_bwd_kernel(NormBwd p) {
  constexpr int V = kVec<T>, R = kBlock<G> / G;
  __shared__ float lds[2][2][G / kWave + 1];
  const int l = threadIdx.x % G, group = threadIdx.x / G, dim = (int)p.dim;
  const float over = 1.f / (float)dim;
  float w[N][V], dw[N][V] = {}, db[N][V] = {};
#pragma unroll
  for (int i = 0; i < N; ++i)
    load_param<T>(p.w, p.w32, dim, Place<T>(dim, l + G * i), 1.f, w[i]);
  Vec<T, V> x[N], dy[N];
  float mean = 0.f, r = 0.f;
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t row = (int64_t)blockIdx.x * R + group;
  auto read = [&](int64_t at_row) {
    const T* xr = (const T*)p.x + at_row * p.x_stride;
    const T* dr = (const T*)p.dy + at_row * p.dy_stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
      if (dim >= V) {
        x[i] = load<T, V>(xr + at.from);
        dy[i] = load<T, V>(dr + at.from);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[i].v[e] = e < dim ? xr[e] : (T)0.f;
          dy[i].v[e] = e < dim ? dr[e] : (T)0.f;
        }
      }
    }
    mean = p.mean[at_row];
    r = p.rstd[at_row];
  };
  if (row < p.rows) read(row);
  int turn = 0;
  for (; row < p.rows; row += step, turn ^= 1) {
    float n[N][V], g[N][V], s[2] = {0.f, 0.f};
    const float rr = r;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = (float)dy[i].v[e];
        n[i][e] = ((float)x[i].v[e] - mean) * rr;
        g[i][e] = d * w[i][e];
        dw[i][e] += d * n[i][e];
        db[i][e] += d;
        const float own = e < at.skip ? 0.f : g[i][e];
        s[0] += own;
        s[1] += own * n[i][e];
      }
    }
    if (row + step < p.rows) read(row + step);  // while this one is summed
    if (!p.dx) continue;
    row_sum<G>(s, &lds[turn]);
    s[0] *= over;
    s[1] *= over;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
#pragma unroll
      for (int e = 0; e < V; ++e)
        g[i][e] = rr * (g[i][e] - s[0] - n[i][e] * s[1]);
      store_at<T>((T*)p.dx + row * p.dim, dim, at, g[i]);
    }
  }
  if (!p.partial) return;
  float* out = p.partial + 2 * (int64_t)blockIdx.x * p.dim;
  if constexpr (R > 1) {
    // in the order of the groups, through LDS
    __shared__ float sums[R][V * G];
#pragma unroll
    for (int k = 0; k < 2 * N; ++k) {
      const int i = k % N, which = k / N;
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e)
        sums[group][e * G + l] = which ? db[i][e] : dw[i][e];
      __syncthreads();
      for (int c = threadIdx.x; c < V * G; c += kBlock<G>) {
        const Place<T> at(dim, c % G + G * i);
        const int e = c / G;
        if (!at.some || at.from + e >= dim) continue;
        float v = 0.f;
#pragma unroll
        for (int q = 0; q < R; ++q) v += sums[q][c];
        out[which * p.dim + at.from + e] = v;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const Place<T> at(dim, l + G * i);
      if (!at.some) continue;
      store<float, V>(out + at.from, dw[i]);
      store<float, V>(out + p.dim + at.from, db[i]);
    }
  }
}

// ---- rows of any length: a block walks them, and reads them again
__device__ __forceinline__ float block_sum(float v, float* lds) {
  v = group_sum(v);
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < (int)(blockDim.x / kWave); ++i) v += lds[i];
  return v;
}

template <typename T>
__device__ __forceinline__ float param(const void* p, bool w32, int64_t i,
                                       float none) {
  if (!p) return none;
  return w32 ? ((const float*)p)[i] : (float)((const T*)p)[i];
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_long_fwd_kernel(NormFwd a) {
  __shared__ float lds[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    T* y = (T*)a.y + row * a.dim;
    float s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) s += (float)x[i];
    const float mean = block_sum(s, lds) / (float)a.dim;
    s = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float d = (float)x[i] - mean;
      s += d * d;
    }
    const float r = 1.f / sqrtf(block_sum(s, lds) / (float)a.dim + a.eps);
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024)
      y[i] = (T)(((float)x[i] - mean) * r * param<T>(a.w, a.w32, i, 1.f) +
                 param<T>(a.b, a.w32, i, 0.f));
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = r;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(1024) void norm_long_dx_kernel(NormBwd a) {
  __shared__ float lds[16];
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* dy = (const T*)a.dy + row * a.dy_stride;
    T* dx = (T*)a.dx + row * a.dim;
    const float mean = a.mean[row], r = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float g = (float)dy[i] * param<T>(a.w, a.w32, i, 1.f);
      s1 += g;
      s2 += g * (((float)x[i] - mean) * r);
    }
    s1 = block_sum(s1, lds) / (float)a.dim;
    s2 = block_sum(s2, lds) / (float)a.dim;
    for (int64_t i = threadIdx.x; i < a.dim; i += 1024) {
      const float g = (float)dy[i] * param<T>(a.w, a.w32, i, 1.f);
      dx[i] = (T)(r * (g - s1 - ((float)x[i] - mean) * r * s2));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void norm_long_dw_kernel(NormBwd a) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= a.dim) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += a.parts) {
    const float dy = (float)((const T*)a.dy)[row * a.dy_stride + i];
    const float x = (float)((const T*)a.x)[row * a.x_stride + i];
    dw += dy * ((x - a.mean[row]) * a.rstd[row]);
    db += dy;
  }
  a.partial[(2 * (int64_t)blockIdx.y) * a.dim + i] = dw;
  a.partial[(2 * (int64_t)blockIdx.y + 1) * a.dim + i] = db;
}

// ---- dw and db from the blocks' shares: 32 columns a block, its 32 lanes a
// column take every 32nd share, then are added in their order
constexpr int kSumLanes = 32;

template <typename W>
__global__ __launch_bounds__(32 * kSumLanes) void norm_sum_kernel(NormSum a) {
  __shared__ float lds[kSumLanes][32];
  const int lane = threadIdx.x % 32, part = threadIdx.x / 32;
  for (int64_t c0 = (int64_t)blockIdx.x * 32; c0 < 2 * a.dim;
       c0 += (int64_t)gridDim.x * 32) {
    const int64_t c = c0 + lane;  // of 2 D
    const bool in = c < 2 * a.dim;
    float v = 0.f;
    if (in) {
#pragma unroll 8
      for (int k = part; k < a.parts; k += kSumLanes)
        v += a.partial[2 * k * a.dim + c];
    }
    lds[part][lane] = v;
    __syncthreads();
    if (part == 0 && in) {
#pragma unroll
      for (int k = 1; k < kSumLanes; ++k) v += lds[k][lane];
      if (c < a.dim) {
        if (a.dw) ((W*)a.dw)[c] = (W)v;
      } else {
        if (a.db) ((W*)a.db)[c - a.dim] = (W)v;
      }
    }
    __syncthreads();  // the next turn writes what this one reads
  }
}

// Blocks of 1024 lanes at most, of which a launch has fewer than 2^32; more
// rows or columns are looped over.
constexpr int64_t kGrid = 1 << 21;

// How a row lies on lanes: G of them with N vectors each; G = 0: too long.
// Two vectors a lane, for twice the bytes in flight: with one, 131072 x 256
// bf16 took 29 us forward and 47 backward, 32768 x 1024 28 and 72. A row of
// more than 2048 vectors would not leave registers for its share of dw and db:
// it is walked and read again.
struct Shape {
  int G, N;
};

Shape shape_of(int64_t dim, int bytes) {
  const int64_t n = (dim * bytes + 15) / 16;  // vectors
  if (n <= 8) return {8, 1};
  for (int G = 8; G <= 1024; G *= 2)
    if (n <= 2 * G) return {G, 2};
  return {0, 0};
}

// Blocks of the backward pass, each with a share: 2048 to 4096 waves, which is
// what 128 registers a lane leave room for. Fewer wide ones for fewer shares
// gain nothing: 5003 x 1021 fp32 takes 22 us with 625 as with 1024 of them.
int parts_of(int64_t rows, int64_t dim, int bytes) {
  const Shape s = shape_of(dim, bytes);
  const int64_t at_once = s.G == 0 ? 32 : s.G <= kWave ? 512 / s.G : 1;
  const int64_t most = s.G == 0     ? 128
                       : s.G <= kWave ? 512
                       : s.G < 256    ? 1024
                       : s.G < 1024   ? 512
                                      : 256;
  const int64_t p = (rows + at_once - 1) / at_once;
  return (int)(p < 1 ? 1 : p < most ? p : most);
}

constexpr int64_t kFwdLanes = 256 * 2048;  // of the forward pass, at most

template <typename T, int G, int N>
hipError_t fwd_with(const NormFwd& p, hipStream_t s) {
  constexpr int64_t R = kBlock<G> / G;
  const int64_t want = (p.rows + R - 1) / R;
  const int64_t most = kFwdLanes / kBlock<G>;  // each walks rows from there on
  return launch(norm_fwd_kernel<T, G, N>, dim3(want < most ? want : most),
                dim3(kBlock<G>), 0, s, p);
}

template <typename T>
hipError_t fwd(const NormFwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  const Shape h = shape_of(p.dim, sizeof(T));
  switch (h.G * 8 + h.N) {
    case 8 * 8 + 1: return fwd_with<T, 8, 1>(p, s);
    case 8 * 8 + 2: return fwd_with<T, 8, 2>(p, s);
    case 16 * 8 + 2: return fwd_with<T, 16, 2>(p, s);
    case 32 * 8 + 2: return fwd_with<T, 32, 2>(p, s);
    case 64 * 8 + 2: return fwd_with<T, 64, 2>(p, s);
    case 128 * 8 + 2: return fwd_with<T, 128, 2>(p, s);
    case 256 * 8 + 2: return fwd_with<T, 256, 2>(p, s);
    case 512 * 8 + 2: return fwd_with<T, 512, 2>(p, s);
    case 1024 * 8 + 2: return fwd_with<T, 1024, 2>(p, s);
  }
  return launch(norm_long_fwd_kernel<T>,
                dim3(p.rows < kGrid ? p.rows : kGrid), dim3(1024), 0, s, p);
}

template <typename T, int G, int N>
hipError_t bwd_with(const NormBwd& p, hipStream_t s) {
  return launch(norm_bwd_kernel<T, G, N>, dim3(p.parts), dim3(kBlock<G>), 0,
                s, p);
}

template <typename T>
hipError_t bwd(const NormBwd& p, const NormSum& z, hipStream_t s) {
  const Shape h = shape_of(p.dim, sizeof(T));
  hipError_t e = hipSuccess;
  switch (h.G * 8 + h.N) {
    case 8 * 8 + 1: e = bwd_with<T, 8, 1>(p, s); break;
    case 8 * 8 + 2: e = bwd_with<T, 8, 2>(p, s); break;
    case 16 * 8 + 2: e = bwd_with<T, 16, 2>(p, s); break;
    case 32 * 8 + 2: e = bwd_with<T, 32, 2>(p, s); break;
    case 64 * 8 + 2: e = bwd_with<T, 64, 2>(p, s); break;
    case 128 * 8 + 2: e = bwd_with<T, 128, 2>(p, s); break;
    case 256 * 8 + 2: e = bwd_with<T, 256, 2>(p, s); break;
    case 512 * 8 + 2: e = bwd_with<T, 512, 2>(p, s); break;
    case 1024 * 8 + 2: e = bwd_with<T, 1024, 2>(p, s); break;
    default:
      if (p.dx && p.rows > 0)
        e = launch(norm_long_dx_kernel<T>,
                   dim3(p.rows < kGrid ? p.rows : kGrid), dim3(1024), 0, s, p);
      if (e == hipSuccess && p.partial)
        e = launch(norm_long_dw_kernel<T>,
                   dim3((p.dim + 255) / 256, p.parts), dim3(256), 0, s, p);
  }
  if (e != hipSuccess || !p.partial) return e;
  const int64_t sums = (2 * p.dim + 31) / 32;
  const dim3 grid(sums < kGrid ? sums : kGrid);
  if (p.w32) return launch(norm_sum_kernel<float>, grid, dim3(32 * kSumLanes), 0, s, z);
  return launch(norm_sum_kernel<T>, grid, dim3(32 * kSumLanes), 0, s, z);
}

}  // namespace

extern "C" int rlsched_norm_fwd(int device, void* stream, const void* x,
                                const void* w, const void* b, void* y,
                                float* mean, float* rstd, int64_t rows,
                                int64_t dim, int64_t x_stride, double eps,
                                int type, int wtype) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  if (wtype != F32 && wtype != type) return hipErrorInvalidValue;
  const NormFwd a = {x,    w,   b,        y,          mean,        rstd,
                     rows, dim, x_stride, (float)eps, wtype == F32};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return fwd<float>(a, s);
  if (type == BF16) return fwd<bf16>(a, s);
  if (type == F16) return fwd<f16>(a, s);
  return hipErrorInvalidValue;
}

// Row groups whose sums of dy n and dy the backward pass keeps apart: its
// scratch holds 2 * parts * dim floats.
extern "C" int64_t rlsched_norm_parts(int64_t rows, int64_t dim, int type) {
  return parts_of(rows, dim, type == F32 ? 4 : 2);
}

extern "C" int rlsched_norm_bwd(int device, void* stream, const void* dy,
                                const void* x, const void* w,
                                const float* mean, const float* rstd, void* dx,
                                void* dw, void* db, float* partial,
                                int64_t rows, int64_t dim, int64_t x_stride,
                                int64_t dy_stride, int type, int wtype) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  if (wtype != F32 && wtype != type) return hipErrorInvalidValue;
  const int parts = (int)rlsched_norm_parts(rows, dim, type);
  const NormBwd a = {dy,   x,   w,        mean,      rstd,  dx,         partial,
                     rows, dim, x_stride, dy_stride, parts, wtype == F32};
  const NormSum z = {partial, dw, db, dim, parts};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return bwd<float>(a, z, s);
  if (type == BF16) return bwd<bf16>(a, z, s);
  if (type == F16) return bwd<f16>(a, z, s);
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
