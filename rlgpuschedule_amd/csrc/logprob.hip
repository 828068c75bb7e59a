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

// Running maximum, sum and weighted sum of a set of logits.
struct Part {
  float m, s, u;
};

__device__ __forceinline__ void join(Part& a, const Part& b) {
  if (b.m == -INFINITY) return;
  if (a.m == -INFINITY) {
    a = b;
    return;
  }
  const float m = fmaxf(a.m, b.m);
  const float da = a.m - m, db = b.m - m;
  const float ea = __expf(da), eb = __expf(db);
  a.u = (ea > 0.f ? ea * (a.u + da * a.s) : 0.f) +
        (eb > 0.f ? eb * (b.u + db * b.s) : 0.f);
  a.s = a.s * ea + b.s * eb;
  a.m = m;
}

// Whole numbers in the order of (value, lowest index first); 0 is nothing.
__device__ __forceinline__ uint64_t key_of(float v, int64_t i) {
  uint32_t b = __float_as_uint(v + 0.f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return (uint64_t)b << 32 | (0xffffffffu - (uint32_t)i);
}

template <typename T>
__global__ __launch_bounds__(256) void logp_fwd_kernel(LogpFwd p) {
  __shared__ Part parts[256];
  __shared__ uint64_t keys[256];
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.logits + row * p.x_stride;
  const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
  const int tid = threadIdx.x;
  Part q = {-INFINITY, 0.f, 0.f};
  float bad = 0.f;
  for (int64_t i = tid; i < p.A; i += 256) {
    if (ok && !ok[i]) continue;
    const float v = (float)x[i];
    if (v != v || v == INFINITY) bad = NAN;
    join(q, Part{v, 1.f, 0.f});
  }
  q.s += bad;
  q.u += bad;
  parts[tid] = q;
  for (int n = 128; n > 0; n >>= 1) {
    __syncthreads();
    if (tid < n) {
      const float s = parts[tid].s + parts[tid + n].s;
      join(parts[tid], parts[tid + n]);
      if (s != s) parts[tid].s = s;
    }
  }
  __syncthreads();
  q = parts[0];
  const bool broken = q.s != q.s;
  const bool some = q.m > -INFINITY && !broken;
  const float ls = logf(q.s);
  if (tid == 0) {
    const int64_t a = p.actions[row];
    float lp = broken ? NAN : -INFINITY;
    if (some && a < p.A && a >= 0 && !(ok && !ok[a]))
      lp = (float)x[a] - q.m - ls;
    p.logp[row] = a < 0 ? 0.f : lp;
    const float H = broken ? NAN : some ? ls - q.u / q.s : 0.f;
    p.entropy[row] = H;
    if (p.stats) {
      p.stats[3 * row] = broken ? NAN : some ? q.m : 0.f;
      p.stats[3 * row + 1] = broken ? NAN : some ? ls : 0.f;
      p.stats[3 * row + 2] = H;
    }
  }
  uint64_t last = ~0ull;
  for (int j = 0; j < p.k; ++j) {
    uint64_t best = 0;
    if (some) {
      for (int64_t i = tid; i < p.A; i += 256) {
        if (ok && !ok[i]) continue;
        const float v = (float)x[i];
        if (v == -INFINITY) continue;
        const uint64_t key = key_of(v, i);
        if (key < last && key > best) best = key;
      }
    }
    keys[tid] = best;
    for (int n = 128; n > 0; n >>= 1) {
      __syncthreads();
      if (tid < n && keys[tid + n] > keys[tid]) keys[tid] = keys[tid + n];
    }
    __syncthreads();
    last = keys[0];
    __syncthreads();
    if (tid == 0) {
      const int64_t i = last ? (int64_t)(0xffffffffu - (uint32_t)last) : -1;
      p.top_index[row * p.k + j] = i;
      p.top_logp[row * p.k + j] =
          broken ? NAN : i >= 0 ? (float)x[i] - q.m - ls : -INFINITY;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void logp_bwd_kernel(LogpBwd p) {
  const int64_t row = blockIdx.x;
  const T* x = (const T*)p.logits + row * p.x_stride;
  const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
  T* out = (T*)p.dlogits + row * p.A;
  const int64_t act = p.actions[row];
  const float m = p.stats[3 * row], ls = p.stats[3 * row + 1];
  const float H = p.stats[3 * row + 2];
  float dl = p.dlogp ? p.dlogp[row] : 0.f;
  const float dh = p.dentropy ? p.dentropy[row] : 0.f;
  // a taken action of probability 0 is a constant -inf
  if (act < 0 || act >= p.A || (ok && !ok[act]) ||
      (float)x[act] == -INFINITY)
    dl = 0.f;
  for (int64_t i = threadIdx.x; i < p.A; i += 256) {
    float g = 0.f;
    const float v = (float)x[i];
    if (!(ok && !ok[i]) && v != -INFINITY) {
      const float lp = v - m - ls, pr = __expf(lp);
      g = -dl * pr;
      if (pr != 0.f) g -= dh * pr * (lp + H);
      if (i == act) g += dl;
    }
    out[i] = (T)g;
  }
}

template <typename T>
hipError_t fwd(const LogpFwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  return launch(logp_fwd_kernel<T>, dim3(p.rows), dim3(256), 0, s, p);
}

template <typename T>
hipError_t bwd(const LogpBwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  return launch(logp_bwd_kernel<T>, dim3(p.rows), dim3(256), 0, s, p);
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
