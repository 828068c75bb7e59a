// Shared pieces of the sequence operators (layer_norm.hip, gated_scan.hip,
// logprob.hip): element types, wide loads and stores, wave reductions, and
// launches that stay on the caller's device and stream.
#pragma once
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include <tuple>
#include <type_traits>

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

// A reduction over groups of W lanes, its result in every one of them, by
// moves between registers alone: quads, halves of a row of 16, the row, then
// swaps of rows and of halves of the wave. A step's two operands may lie in
// other lanes than an exclusive-or's would, but hold the same sums.
template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}

template <int W = kWave, typename Op>
__device__ __forceinline__ uint32_t group_reduce(uint32_t v, Op op) {
  if constexpr (W >= 2) v = op(v, dpp<0xb1>(v));   // quad 1 0 3 2
  if constexpr (W >= 4) v = op(v, dpp<0x4e>(v));   // quad 2 3 0 1
  if constexpr (W >= 8) v = op(v, dpp<0x141>(v));  // half mirror
  if constexpr (W >= 16) v = op(v, dpp<0x140>(v));  // mirror
  if constexpr (W >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  if constexpr (W >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    v = op(r[0], r[1]);
  }
  return v;
}

// Not contracted: fused with a product before it, an addition would see one
// lane's rounded and another's not, and the lanes' sums would differ.
__device__ __forceinline__ float add(float a, float b) {
#pragma clang fp contract(off)
  return a + b;
}

template <int W = kWave>
__device__ __forceinline__ float group_sum(float f) {
  return __uint_as_float(
      group_reduce<W>(__float_as_uint(f), [](uint32_t a, uint32_t b) {
        return __float_as_uint(add(__uint_as_float(a), __uint_as_float(b)));
      }));
}

template <int W = kWave>
__device__ __forceinline__ float group_max(float f) {
  return __uint_as_float(
      group_reduce<W>(__float_as_uint(f), [](uint32_t a, uint32_t b) {
        return __float_as_uint(
            maximum(__uint_as_float(a), __uint_as_float(b)));
      }));
}

// The largest of 64-bit keys.
template <int W = kWave>
__device__ __forceinline__ uint64_t group_larger(uint64_t k) {
  auto step = [&](uint32_t lo, uint32_t hi) {
    const uint64_t other = (uint64_t)hi << 32 | lo;
    k = other > k ? other : k;
  };
  auto lo = [&] { return (uint32_t)k; };
  auto hi = [&] { return (uint32_t)(k >> 32); };
  if constexpr (W >= 2) step(dpp<0xb1>(lo()), dpp<0xb1>(hi()));
  if constexpr (W >= 4) step(dpp<0x4e>(lo()), dpp<0x4e>(hi()));
  if constexpr (W >= 8) step(dpp<0x141>(lo()), dpp<0x141>(hi()));
  if constexpr (W >= 16) step(dpp<0x140>(lo()), dpp<0x140>(hi()));
  if constexpr (W >= 32) {
    const auto l = __builtin_amdgcn_permlane16_swap(lo(), lo(), false, false);
    const auto h = __builtin_amdgcn_permlane16_swap(hi(), hi(), false, false);
    step(l[0], h[0]);
    step(l[1], h[1]);
  }
  if constexpr (W >= 64) {
    const auto l = __builtin_amdgcn_permlane32_swap(lo(), lo(), false, false);
    const auto h = __builtin_amdgcn_permlane32_swap(hi(), hi(), false, false);
    step(l[0], h[0]);
    step(l[1], h[1]);
  }
  return k;
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
// 2^32 lanes or more along one axis are refused here: the runtime refuses
// 2^32 itself, but a launch of a few blocks more left most of its work undone
// without an error.
template <typename... P, typename... A>
inline hipError_t launch(void (*kernel)(P...), dim3 grid, dim3 block,
                         size_t lds, hipStream_t stream, A... args) {
  void* list[] = {(void*)&args...};
  static_assert(std::is_same_v<std::tuple<P...>, std::tuple<A...>>,
                "a value of its own type for each parameter");
  if (((uint64_t)grid.x * block.x | (uint64_t)grid.y * block.y) >> 32)
    return hipErrorInvalidConfiguration;
  return hipLaunchKernel((const void*)kernel, grid, block, list, lds, stream);
}

}  // namespace seq
