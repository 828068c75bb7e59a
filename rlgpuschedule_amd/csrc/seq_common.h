// Shared pieces of the sequence operators (layer_norm.hip, gated_scan.hip,
// logprob.hip): element types, wide loads and stores, wave reductions, and
// launches that stay on the caller's device and stream.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

namespace seq {

constexpr int kWave = 64;

// element type codes, as ops/_seq.py passes them
enum Type { F32 = 0, BF16 = 1, F16 = 2 };

typedef __bf16 bf16;
typedef _Float16 f16;

// N elements as one load or store of N * sizeof(T) bytes, at any address:
// global accesses of this part need no alignment beyond the byte's, so rows
// of odd lengths go the same way as even ones.
template <typename T, int N>
struct Vec {
  T v[N];
};

template <typename T, int N>
__device__ __forceinline__ Vec<T, N> load(const T* p) {
  Vec<T, N> r;
  __builtin_memcpy(&r, p, sizeof(r));
  return r;
}

template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float (&f)[N]) {
  const Vec<T, N> r = load<T, N>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)r.v[i];
}

// One rounding to nearest even, of a value held in 32 bits.
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float (&f)[N]) {
  Vec<T, N> r;
#pragma unroll
  for (int i = 0; i < N; ++i) r.v[i] = (T)f[i];
  __builtin_memcpy(p, &r, sizeof(r));
}

// Of two values the larger, and NaN if either is (one instruction).
__device__ __forceinline__ float maximum(float a, float b) {
  return __builtin_elementwise_maximum(a, b);
}

template <int W = kWave>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, kWave);
  return v;
}

template <int W = kWave>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = maximum(v, __shfl_xor(v, o, kWave));
  return v;
}

// Runs the scope on one device and goes back to the caller's.
struct OnDevice {
  int before = -1;
  hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) {
      err = hipSetDevice(device);
    } else {
      before = -1;
    }
  }
  ~OnDevice() {
    if (before >= 0) (void)hipSetDevice(before);
  }
};

// The launch's own status: an error left by other code stays where it is.
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block,
                         size_t lds, hipStream_t stream, A... args) {
  void* list[] = {(void*)&args...};
  static_assert(sizeof...(P) == sizeof...(A), "one value for each parameter");
  return hipLaunchKernel((const void*)kernel, grid, block, list, lds, stream);
}

}  // namespace seq
