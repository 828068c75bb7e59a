// Log probabilities of taken actions over the allowed ones, with the
// distribution's entropy and its top alternatives, and their gradient.
//
//   m = max x, s = sum e^(x-m), u = sum e^(x-m) (x-m)   over allowed actions
//   logp_j = (x_j - m) - log s,  H = log s - u / s
//   dx_j = dlogp (1[j = action] - p_j) - dH p_j (logp_j + H)
//
// An action that the mask leaves out and one of logit -inf are the same:
// probability 0, no gradient, never an alternative. Sums are held in 32 bits;
// m and log s are kept apart: where every logit is the type's lowest value,
// their sum would lose log s.
#include "seq_api.h"
#include "seq_common.h"

namespace {
using namespace seq;

struct LogpFwd {
  const void* logits;
  const int64_t* actions;
  const uint8_t* mask;  // null: all allowed
  float* logp;
  float* entropy;
  float* stats;  // [rows, 3]: m, log s, H; or null
  float* top_logp;     // [rows, k]
  int64_t* top_index;  // [rows, k]
  int64_t rows, A, x_stride, mask_stride;
  int k;
};

struct LogpBwd {
  const float* dlogp;     // null: zeros
  const float* dentropy;  // null: zeros
  const void* logits;
  const int64_t* actions;
  const uint8_t* mask;
  const float* stats;
  void* dlogits;
  int64_t rows, A, x_stride, mask_stride;
};

// One vector is 16 bytes of logits and as many bytes of mask.
template <typename T>
constexpr int kVec = 16 / sizeof(T);

constexpr float kFloor = -1e4f;  // e^kFloor is 0, and so is kFloor e^kFloor

// Whole numbers in the order of (value, lowest index first); 0 is nothing.
__device__ __forceinline__ uint64_t key_of(float v, int64_t i) {
  uint32_t b = __float_as_uint(v + 0.f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)b << 32 | (0xffffffffu - (uint32_t)i);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  const uint32_t b = (uint32_t)(key >> 32);
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ int64_t index_of(uint64_t key) {
  return (int64_t)(0xffffffffu - (uint32_t)key);
}

// Vector j of a row as floats, -inf where nothing is or may be taken. The
// last vector of a row of no whole number of them begins early enough to end
// with the row; what it shares with the one before is left out unless
// `shared`, so no element is counted twice.
template <typename T, bool shared = false>
__device__ __forceinline__ int64_t load_row(const T* x, const uint8_t* ok,
                                            int64_t A, int64_t j,
                                            float (&f)[kVec<T>]) {
  constexpr int V = kVec<T>;
  const int64_t base = j * V;
  int64_t from = base;
  if (A >= V) {
    from = base < A - V ? base : A - V;
    load<T, V>(x + from, f);
    if (ok) {
      const Vec<uint8_t, V> m = load<uint8_t, V>(ok + from);
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (!m.v[e]) f[e] = -INFINITY;
    }
    if (!shared && from != base) {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (from + e < base) f[e] = -INFINITY;
    }
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      f[e] = -INFINITY;
      if (e < A && !(ok && !ok[e])) f[e] = (float)x[e];
    }
  }
  return from;
}

template <typename T>
__device__ __forceinline__ void store_row(T* y, int64_t A, int64_t from,
                                          const float (&g)[kVec<T>]) {
  constexpr int V = kVec<T>;
  if (A >= V) {
    store<T, V>(y + from, g);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < A) y[e] = (T)g[e];
  }
}

// What a row's forward pass writes. `q` is the taken action's logit, -inf
// where it may not be taken.
__device__ __forceinline__ void finish_row(const LogpFwd& p, int64_t row,
                                           int64_t act, float q, float m,
                                           float s, float u) {
  const bool broken = s != s, some = s > 0.f;
  const float ls = some || broken ? logf(s) : 0.f;
  const float H = some || broken ? ls - u / s : 0.f;
  const float lp = some || broken ? q - m - ls : -INFINITY;
  p.logp[row] = act < 0 ? 0.f : lp;
  p.entropy[row] = H;
  if (p.stats) {
    p.stats[3 * row] = some || broken ? m : 0.f;
    p.stats[3 * row + 1] = ls;
    p.stats[3 * row + 2] = H;
  }
}

__device__ __forceinline__ void finish_top(const LogpFwd& p, int64_t row,
                                           int j, uint64_t key, float m,
                                           float s) {
  const bool broken = s != s;
  float lp = -INFINITY;
  int64_t ix = -1;
  if (key && !broken) {
    lp = value_of(key) - m - logf(s);
    ix = index_of(key);
  }
  p.top_logp[row * p.k + j] = broken ? NAN : lp;
  p.top_index[row * p.k + j] = ix;
}

template <typename T>
__device__ __forceinline__ float taken(const T* x, const uint8_t* ok,
                                       int64_t A, int64_t act) {
  return act >= 0 && act < A && !(ok && !ok[act]) ? (float)x[act] : -INFINITY;
}

// What the gradient of one row's elements needs.
struct Row {
  float m, ls, H, dl, dh;
  int64_t act;
};

template <typename T>
__device__ __forceinline__ Row row_of(const LogpBwd& p, const T* x,
                                      const uint8_t* ok, int64_t row) {
  Row r;
  r.act = p.actions[row];
  r.m = p.stats[3 * row];
  r.ls = p.stats[3 * row + 1];
  r.H = p.stats[3 * row + 2];
  r.dl = p.dlogp ? p.dlogp[row] : 0.f;
  r.dh = p.dentropy ? p.dentropy[row] : 0.f;
  // a taken action of probability 0 is a constant -inf
  if (taken(x, ok, p.A, r.act) == -INFINITY) r.dl = 0.f;
  return r;
}

__device__ __forceinline__ float gradient(const Row& r, float v, int64_t i) {
  const float d = maximum(v - r.m, kFloor) - r.ls, pr = __expf(d);
  const float g = -pr * (r.dl + r.dh * (d + r.H));
  return v == -INFINITY ? 0.f : i == r.act ? g + r.dl : g;
}

// ---- rows of up to 64 * N vectors: G lanes a row, all of it in registers
template <typename T, int G, int N>
__global__ __launch_bounds__(256) void logp_group_kernel(LogpFwd p) {
  constexpr int V = kVec<T>, R = 256 / G;
  const int l = threadIdx.x % G;
  for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G; row < p.rows;
       row += (int64_t)gridDim.x * R) {
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    const int64_t act = p.actions[row];
    float f[N][V], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = -INFINITY;
      if ((l + G * i) * V < p.A) load_row<T>(x, ok, p.A, l + G * i, f[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) m = maximum(m, f[i][e]);
    }
    const float q = taken(x, ok, p.A, act);
    m = group_max<G>(m);
    if (m == -INFINITY) m = 0.f;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = maximum(f[i][e] - m, kFloor), w = __expf(d);
        s += w;
        u += w * d;
      }
    s = group_sum<G>(s);
    u = group_sum<G>(u);
    if (l == 0) finish_row(p, row, act, q, m, s, u);
    uint64_t last = ~0ull;
    for (int j = 0; j < p.k; ++j) {
      uint64_t best = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int64_t base = (int64_t)(l + G * i) * V;
        const int64_t from = p.A < V || base < p.A - V ? base : p.A - V;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const uint64_t key = key_of(f[i][e], from + e);
          if (f[i][e] > -INFINITY && key < last && key > best) best = key;
        }
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)best, o, kWave);
        best = other > best ? other : best;
      }
      last = best;
      if (l == 0) finish_top(p, row, j, best, m, s);
    }
  }
}

template <typename T, int G, int N>
__global__ __launch_bounds__(256) void logp_group_bwd_kernel(LogpBwd p) {
  constexpr int V = kVec<T>, R = 256 / G;
  const int l = threadIdx.x % G;
  for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G; row < p.rows;
       row += (int64_t)gridDim.x * R) {
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    const Row r = row_of(p, x, ok, row);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if ((l + G * i) * V >= p.A) break;
      float f[V];
      const int64_t from = load_row<T, true>(x, ok, p.A, l + G * i, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = gradient(r, f[e], from + e);
      store_row<T>((T*)p.dlogits + row * p.A, p.A, from, f);
    }
  }
}

// ---- longer rows, forward: W waves a row, one pass over it
// A lane's running maximum, sum and weighted sum. m starts at the lowest
// finite value, so differences of it are never -inf minus -inf.
struct Running {
  float m = -3.402823466e38f, s = 0.f, u = 0.f;

  template <int N>
  __device__ __forceinline__ void take(const float (&f)[N], float top) {
    const float n = maximum(m, top);
    const float d0 = maximum(m - n, kFloor), w0 = __expf(d0);
    u = w0 * (u + d0 * s);
    s = w0 * s;
    m = n;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = maximum(f[e] - m, kFloor), w = __expf(d);
      s += w;
      u += w * d;
    }
  }
  // as they would be below a larger maximum
  __device__ __forceinline__ void lower(float n) {
    const float d0 = maximum(m - n, kFloor), w0 = __expf(d0);
    u = w0 * (u + d0 * s);
    s = w0 * s;
    m = n;
  }
  __device__ __forceinline__ void join_wave() {
    lower(group_max(m));
    s = group_sum(s);
    u = group_sum(u);
  }
};

constexpr int kHeads = 128;   // groups of lanes whose best bound the top k
constexpr int kFound = 1024;  // alternatives that are sorted out at once

template <int NT>
struct RowLds {
  float m[NT / kWave], s[NT / kWave], u[NT / kWave];
  uint64_t heads[kHeads];
  uint64_t found[kFound];
  uint64_t bound;
  int count;
};

template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void logp_row_kernel(LogpFwd p) {
  constexpr int V = kVec<T>, W = NT / kWave, U = 4;
  __shared__ RowLds<NT> lds;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int64_t n = (p.A + V - 1) / V;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    const int64_t act = p.actions[row];
    const float q = taken(x, ok, p.A, act);
    Running r;
    int64_t best = -1;  // the first vector that holds the lane's maximum
    auto take = [&](const float(&f)[V], int64_t j) {
      float top = f[0];
#pragma unroll
      for (int e = 1; e < V; ++e) top = maximum(top, f[e]);
      if (TOP && (top > r.m || (best < 0 && top > -INFINITY))) best = j;
      r.take(f, top);
    };
    int64_t j = tid;
    for (; j + (U - 1) * NT < n; j += U * NT) {
      float f[U][V];
#pragma unroll
      for (int i = 0; i < U; ++i) load_row<T>(x, ok, p.A, j + i * NT, f[i]);
#pragma unroll
      for (int i = 0; i < U; ++i) take(f[i], j + i * NT);
    }
    for (; j < n; j += NT) {
      float f[V];
      load_row<T>(x, ok, p.A, j, f);
      take(f, j);
    }
    const float own = r.m;
    r.join_wave();
    if (lane == 0) {
      lds.m[wave] = r.m;
      lds.s[wave] = r.s;
      lds.u[wave] = r.u;
    }
    __syncthreads();
    float m = lds.m[0], s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 1; i < W; ++i) m = maximum(m, lds.m[i]);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Running part{lds.m[i], lds.s[i], lds.u[i]};
      part.lower(m);
      s += part.s;
      u += part.u;
    }
    if (tid == 0) finish_row(p, row, act, q, m, s, u);
    if (TOP) {
      // Each of kHeads groups of lanes has its best; the k-th of those is a
      // lower bound of the k-th of all, and only lanes whose own best
      // reaches it have more to give: about k elements, at most k groups'.
      uint64_t key = 0;
      if (best >= 0 && s == s) {
        float f[V];
        const int64_t from = load_row<T>(x, ok, p.A, best, f);
#pragma unroll
        for (int e = V - 1; e >= 0; --e)
          if (f[e] == own) key = key_of(f[e], from + e);
      }
      uint64_t head = key;
#pragma unroll
      for (int o = 1; o < NT / kHeads; o <<= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)head, o, kWave);
        head = other > head ? other : head;
      }
      if (tid % (NT / kHeads) == 0) lds.heads[tid / (NT / kHeads)] = head;
      if (tid == 0) {
        lds.bound = 1;
        lds.count = 0;
      }
      __syncthreads();
      if (tid < kHeads) {
        const uint64_t mine = lds.heads[tid];
        int rank = 0;
        for (int i = 0; i < kHeads; ++i) rank += lds.heads[i] > mine;
        if (mine && rank == p.k - 1) lds.bound = mine;
      }
      __syncthreads();
      const uint64_t bound = lds.bound;
      if (key >= bound) {
        for (int64_t i = tid; i < n; i += NT) {
          float f[V];
          const int64_t from = load_row<T>(x, ok, p.A, i, f);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const uint64_t k = key_of(f[e], from + e);
            if (f[e] > -INFINITY && k >= bound) {
              const int at = atomicAdd(&lds.count, 1);
              if (at < kFound) lds.found[at] = k;
            }
          }
        }
      }
      __syncthreads();
      const int count = lds.count;
      if (count <= kFound) {
        for (int i = tid; i < count; i += NT) {
          const uint64_t mine = lds.found[i];
          int rank = 0;
          for (int c = 0; c < count; ++c) rank += lds.found[c] > mine;
          if (rank < p.k) finish_top(p, row, rank, mine, m, s);
        }
        for (int i = count + tid; i < p.k; i += NT)
          finish_top(p, row, i, 0, m, s);
      } else {
        // More than fit: few lanes hold many of the largest. One round an
        // alternative, each a maximum below the one before.
        uint64_t last = ~0ull;
        for (int a = 0; a < p.k; ++a) {
          uint64_t top = 0;
          if (key >= bound) {
            for (int64_t i = tid; i < n; i += NT) {
              float f[V];
              const int64_t from = load_row<T>(x, ok, p.A, i, f);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const uint64_t k = key_of(f[e], from + e);
                if (f[e] > -INFINITY && k < last && k > top) top = k;
              }
            }
          }
#pragma unroll
          for (int o = kWave / 2; o > 0; o >>= 1) {
            const uint64_t other =
                __shfl_xor((unsigned long long)top, o, kWave);
            top = other > top ? other : top;
          }
          if (lane == 0) lds.heads[wave] = top;
          __syncthreads();
#pragma unroll
          for (int i = 0; i < W; ++i)
            top = lds.heads[i] > top ? lds.heads[i] : top;
          __syncthreads();
          last = top;
          if (tid == 0) finish_top(p, row, a, top, m, s);
        }
      }
    }
    __syncthreads();  // the next row writes what this one reads
  }
}

// ---- longer rows, backward: blocks of 256 lanes with U vectors each
constexpr int kBwdVecs = 4;

template <typename T>
__global__ __launch_bounds__(256) void logp_row_bwd_kernel(LogpBwd p,
                                                           int64_t pieces) {
  constexpr int V = kVec<T>, U = kBwdVecs;
  const int64_t n = (p.A + V - 1) / V;
  for (int64_t b = blockIdx.x; b < p.rows * pieces; b += gridDim.x) {
    const int64_t row = b / pieces;
    const int64_t j = b % pieces * (256 * U) + threadIdx.x;
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    float f[U][V];
    int64_t from[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j + 256 * i < n)
        from[i] = load_row<T, true>(x, ok, p.A, j + 256 * i, f[i]);
    const Row r = row_of(p, x, ok, row);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (j + 256 * i >= n) break;
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = gradient(r, f[i][e], from[i] + e);
      store_row<T>((T*)p.dlogits + row * p.A, p.A, from[i], f[i]);
    }
  }
}

constexpr int64_t kGrid = 1 << 22;  // blocks at most; more rows are looped over

template <typename T, int G, int N>
hipError_t group_fwd(const LogpFwd& p, hipStream_t s) {
  const int64_t grid = (p.rows + 256 / G - 1) / (256 / G);
  return launch(logp_group_kernel<T, G, N>, dim3(grid < kGrid ? grid : kGrid),
                dim3(256), 0, s, p);
}
template <typename T, int G, int N>
hipError_t group_bwd(const LogpBwd& p, hipStream_t s) {
  const int64_t grid = (p.rows + 256 / G - 1) / (256 / G);
  return launch(logp_group_bwd_kernel<T, G, N>,
                dim3(grid < kGrid ? grid : kGrid), dim3(256), 0, s, p);
}

template <typename T, int NT>
hipError_t row_fwd(const LogpFwd& p, hipStream_t s) {
  const dim3 grid(p.rows < kGrid ? p.rows : kGrid);
  if (p.k)
    return launch(logp_row_kernel<T, NT, true>, grid, dim3(NT), 0, s, p);
  return launch(logp_row_kernel<T, NT, false>, grid, dim3(NT), 0, s, p);
}

template <typename T>
hipError_t fwd(const LogpFwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  const int64_t n = (p.A + kVec<T> - 1) / kVec<T>;
  if (n <= 1) return group_fwd<T, 1, 1>(p, s);
  if (n <= 2) return group_fwd<T, 2, 1>(p, s);
  if (n <= 4) return group_fwd<T, 4, 1>(p, s);
  if (n <= 8) return group_fwd<T, 8, 1>(p, s);
  if (n <= 16) return group_fwd<T, 16, 1>(p, s);
  if (n <= 32) return group_fwd<T, 32, 1>(p, s);
  if (n <= 64) return group_fwd<T, 64, 1>(p, s);
  if (n <= 128) return group_fwd<T, 64, 2>(p, s);
  if (n <= 256) return group_fwd<T, 64, 4>(p, s);
  if (n >= 2048 && p.rows < 512) return row_fwd<T, 1024>(p, s);
  return row_fwd<T, 256>(p, s);
}

template <typename T>
hipError_t bwd(const LogpBwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  const int64_t n = (p.A + kVec<T> - 1) / kVec<T>;
  if (n <= 1) return group_bwd<T, 1, 1>(p, s);
  if (n <= 2) return group_bwd<T, 2, 1>(p, s);
  if (n <= 4) return group_bwd<T, 4, 1>(p, s);
  if (n <= 8) return group_bwd<T, 8, 1>(p, s);
  if (n <= 16) return group_bwd<T, 16, 1>(p, s);
  if (n <= 32) return group_bwd<T, 32, 1>(p, s);
  if (n <= 64) return group_bwd<T, 64, 1>(p, s);
  if (n <= 128) return group_bwd<T, 64, 2>(p, s);
  const int64_t pieces = (n + 256 * kBwdVecs - 1) / (256 * kBwdVecs);
  const int64_t grid = p.rows * pieces;
  return launch(logp_row_bwd_kernel<T>, dim3(grid < kGrid ? grid : kGrid),
                dim3(256), 0, s, p, pieces);
}

}  // namespace

extern "C" int rlsched_logp_fwd(int device, void* stream, const void* logits,
                                const int64_t* actions, const uint8_t* mask,
                                float* logp, float* entropy, float* stats,
                                float* top_logp, int64_t* top_index,
                                int64_t rows, int64_t A, int64_t x_stride,
                                int64_t mask_stride, int k, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const LogpFwd p = {logits, actions,  mask,      logp, entropy,  stats,
                     top_logp, top_index, rows, A, x_stride, mask_stride, k};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return fwd<float>(p, s);
  if (type == BF16) return fwd<bf16>(p, s);
  if (type == F16) return fwd<f16>(p, s);
  return hipErrorInvalidValue;
}

extern "C" int rlsched_logp_bwd(int device, void* stream, const float* dlogp,
                                const float* dentropy, const void* logits,
                                const int64_t* actions, const uint8_t* mask,
                                const float* stats, void* dlogits,
                                int64_t rows, int64_t A, int64_t x_stride,
                                int64_t mask_stride, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const LogpBwd p = {dlogp, dentropy, logits, actions,  mask,       stats,
                     dlogits, rows,   A,      x_stride, mask_stride};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return bwd<float>(p, s);
  if (type == BF16) return bwd<bf16>(p, s);
  if (type == F16) return bwd<f16>(p, s);
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
