// Gated linear recurrence over time-major sequences, forward and backward.
//
//   z = sigmoid(gate), a = 1 - z
//   c_t = done_{t-1} ? 0 : h_{t-1}  (c_0 = h0),  h_t = a_t c_t + z_t x_t
//   h_last = done_{T-1} ? 0 : h_{T-1}
//   D_t = dh_t + (done_t ? 0 : a_{t+1} D_{t+1}),  the last with dh_last
//   dx = z D,  dgate = D (x - c) z a,  dh0 = a_0 D_0
//
// A reset is a selection, not a product: nothing before an episode's end,
// not even a NaN, is seen after it. The state is held in 32 bits throughout;
// the backward pass does not read the rounded hs but computes c again from
// the 32-bit states kept at every kKeep-th step.
#include "seq_api.h"
#include "seq_common.h"

namespace {
using namespace seq;

constexpr int kKeep = 64;  // steps from one kept state to the next

struct ScanFwd {
  const void* gate;
  const void* x;
  const float* h0;      // null: zeros
  const uint8_t* done;  // null: no episode ends
  void* hs;
  float* h_last;
  float* states;  // [ceil(T / kKeep), E, H]: c at t = 0, kKeep, ...; or null
  int64_t T, E, H;
  int64_t gate_t, gate_e, x_t, x_e;  // strides of time and environment
};

struct ScanBwd {
  const void* dhs;       // null: zeros
  const float* dh_last;  // null: zeros
  const void* gate;
  const void* x;
  const float* states;
  const uint8_t* done;
  void* dgate;
  void* dx;
  float* dh0;  // null: not asked for
  int64_t T, E, H;
  int64_t gate_t, gate_e, x_t, x_e, dhs_t, dhs_e;
};

// z and 1 - z, each to its own last bits: neither is taken as a difference.
__device__ __forceinline__ void gates(float g, float& z, float& a) {
  const float e = __expf(-fabsf(g));
  const float r = __frcp_rn(1.f + e);
  const float q = e * r;
  z = g >= 0.f ? r : q;
  a = g >= 0.f ? q : r;
  if (g != g) z = a = g;
}

template <typename T>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanFwd p) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.E * p.H) return;
  const int64_t e = col / p.H, i = col % p.H;
  float c = p.h0 ? p.h0[col] : 0.f;
  for (int64_t t = 0; t < p.T; ++t) {
    if (p.states && t % kKeep == 0) p.states[t / kKeep * p.E * p.H + col] = c;
    float z, a;
    gates((float)((const T*)p.gate)[t * p.gate_t + e * p.gate_e + i], z, a);
    const float x = (float)((const T*)p.x)[t * p.x_t + e * p.x_e + i];
    const float h = a * c + z * x;
    ((T*)p.hs)[t * p.E * p.H + col] = (T)h;
    c = p.done && p.done[t * p.E + e] ? 0.f : h;
  }
  p.h_last[col] = c;
}

template <typename T>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanBwd p) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.E * p.H) return;
  const int64_t e = col / p.H, i = col % p.H;
  float carry = p.dh_last ? p.dh_last[col] : 0.f;  // a_{t+1} D_{t+1}
  float before[kKeep];
  for (int64_t t0 = (p.T - 1) / kKeep * kKeep; t0 >= 0; t0 -= kKeep) {
    const int n = (int)(p.T - t0 < kKeep ? p.T - t0 : kKeep);
    float c = p.states[t0 / kKeep * p.E * p.H + col];
    for (int k = 0; k < n; ++k) {
      const int64_t t = t0 + k;
      before[k] = c;
      float z, a;
      gates((float)((const T*)p.gate)[t * p.gate_t + e * p.gate_e + i], z, a);
      const float x = (float)((const T*)p.x)[t * p.x_t + e * p.x_e + i];
      const float h = a * c + z * x;
      c = p.done && p.done[t * p.E + e] ? 0.f : h;
    }
    for (int k = n - 1; k >= 0; --k) {
      const int64_t t = t0 + k;
      float z, a;
      gates((float)((const T*)p.gate)[t * p.gate_t + e * p.gate_e + i], z, a);
      const float x = (float)((const T*)p.x)[t * p.x_t + e * p.x_e + i];
      float d = p.done && p.done[t * p.E + e] ? 0.f : carry;
      if (p.dhs) d += (float)((const T*)p.dhs)[t * p.dhs_t + e * p.dhs_e + i];
      ((T*)p.dx)[t * p.E * p.H + col] = (T)(z * d);
      ((T*)p.dgate)[t * p.E * p.H + col] = (T)(d * (x - before[k]) * z * a);
      carry = a * d;
    }
  }
  if (p.dh0) p.dh0[col] = carry;
}

struct ScanStep {
  const void* gate;
  const void* x;
  const uint8_t* done;  // environments that restart from zero; null: none
  float* h;             // in place
  void* hs;
  int64_t E, H, gate_e, x_e;
};

template <typename T>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanStep p) {
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= p.E * p.H) return;
  const int64_t e = col / p.H, i = col % p.H;
  const float c = p.done && p.done[e] ? 0.f : p.h[col];
  float z, a;
  gates((float)((const T*)p.gate)[e * p.gate_e + i], z, a);
  const float h = a * c + z * (float)((const T*)p.x)[e * p.x_e + i];
  p.h[col] = h;
  ((T*)p.hs)[col] = (T)h;
}

template <typename T>
hipError_t step(const ScanStep& p, hipStream_t s) {
  if (p.E * p.H == 0) return hipSuccess;
  const int64_t grid = (p.E * p.H + 255) / 256;
  return launch(scan_step_kernel<T>, dim3(grid), dim3(256), 0, s, p);
}

template <typename T>
hipError_t fwd(const ScanFwd& p, hipStream_t s) {
  if (p.E * p.H == 0) return hipSuccess;
  const int64_t grid = (p.E * p.H + 255) / 256;
  return launch(scan_fwd_kernel<T>, dim3(grid), dim3(256), 0, s, p);
}

template <typename T>
hipError_t bwd(const ScanBwd& p, hipStream_t s) {
  if (p.E * p.H == 0) return hipSuccess;
  const int64_t grid = (p.E * p.H + 255) / 256;
  return launch(scan_bwd_kernel<T>, dim3(grid), dim3(256), 0, s, p);
}

}  // namespace

extern "C" int rlsched_scan_fwd(int device, void* stream, const void* gate,
                                const void* x, const float* h0,
                                const uint8_t* done, void* hs, float* h_last,
                                float* states, int64_t T, int64_t E, int64_t H,
                                int64_t gate_t, int64_t gate_e, int64_t x_t,
                                int64_t x_e, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const ScanFwd p = {gate, x, h0, done,   hs,     h_last, states, T,
                     E,    H, gate_t, gate_e, x_t,    x_e};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return fwd<float>(p, s);
  if (type == BF16) return fwd<bf16>(p, s);
  if (type == F16) return fwd<f16>(p, s);
  return hipErrorInvalidValue;
}

extern "C" int rlsched_scan_bwd(int device, void* stream, const void* dhs,
                                const float* dh_last, const void* gate,
                                const void* x, const float* states,
                                const uint8_t* done, void* dgate, void* dx,
                                float* dh0, int64_t T, int64_t E, int64_t H,
                                int64_t gate_t, int64_t gate_e, int64_t x_t,
                                int64_t x_e, int64_t dhs_t, int64_t dhs_e,
                                int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const ScanBwd p = {dhs, dh_last, gate,   x,      states, done,  dgate,
                     dx,  dh0,     T,      E,      H,      gate_t, gate_e,
                     x_t, x_e,     dhs_t,  dhs_e};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return bwd<float>(p, s);
  if (type == BF16) return bwd<bf16>(p, s);
  if (type == F16) return bwd<f16>(p, s);
  return hipErrorInvalidValue;
}

extern "C" int rlsched_scan_step(int device, void* stream, const void* gate,
                                 const void* x, const uint8_t* done, float* h,
                                 void* hs, int64_t E, int64_t H,
                                 int64_t gate_e, int64_t x_e, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const ScanStep p = {gate, x, done, h, hs, E, H, gate_e, x_e};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return step<float>(p, s);
  if (type == BF16) return step<bf16>(p, s);
  if (type == F16) return step<f16>(p, s);
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
