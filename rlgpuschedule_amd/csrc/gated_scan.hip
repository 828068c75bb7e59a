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
// the 32-bit states kept at every kKeep-th step, which also reads less.
//
// A lane owns V neighbouring columns of one environment and walks time. With
// columns enough for the chip it walks all of it, in one pass. With fewer,
// time is cut into chunks: a first kernel finds each chunk's effect on the
// state, c_end = A c_start + B, those are joined from chunk to chunk, and a
// last kernel walks every chunk from its own start.
//
// Bound by memory where it is walked: 64 x 2048 x 256 bf16 with ends takes 44
// us forward (218 MB with the kept states, 5.0 TB/s) and 66 us backward (352
// MB, 5.3; part of both lies in the 256 MB cache), a large copy's rate being
// 4.9. In chunks gate and x are read twice: 32768 x 2 x 1000 takes 68 us for
// the effects (262 MB), 9 to join 512 chunks and 68 to walk. Small calls are
// bound by the latency of kKeep steps after another: 65 x 64 x 256 bf16 with
// ends takes 7.5 and 11 us.
//
// In chunks a state that has become infinite may go on as NaN: the product of
// a chunk's a may be 0 where none of them is, and 0 times an infinity is NaN.
#include "seq_api.h"
#include "seq_common.h"

namespace {
using namespace seq;

// Steps from one kept state to the next: what the backward pass holds at once.
// 16 of them took twice the registers for half as wide loads, and a training
// pass of 64 x 2048 x 256 bf16 a seventh longer.
constexpr int kKeep = 8;

// A sequence's columns as lanes: n lanes an environment, the last of which
// begins early enough to end with it and computes shared columns twice, to
// the same bits.
struct Cols {
  int64_t E, H, n;
};

// A lane's environment and columns, counted from the block's first
// environment e0: what is far is the same for the block, and a lane's own
// distance fits 32 bits (the host sees to it).
struct Lane {
  int64_t e0;
  uint32_t e, i;
};

template <int V>
__device__ __forceinline__ bool lane_of(const Cols& c, Lane& l) {
  const int64_t g0 = (int64_t)blockIdx.x * 256;
  l.e0 = g0 / c.n;
  const uint32_t n = (uint32_t)c.n, H = (uint32_t)c.H;
  const uint32_t r = (uint32_t)(g0 - l.e0 * c.n) + threadIdx.x;
  l.e = r / n;
  if (l.e0 + l.e >= c.E) return false;
  const uint32_t i = (r - l.e * n) * V;
  l.i = i < H - V ? i : H - V;
  return true;
}

// One step's values of a lane's environment and columns: `at` is the step's,
// stride_e from one environment to the next.
template <typename T>
__device__ __forceinline__ T* here(T* at, const Lane& l, int64_t stride_e) {
  const uint32_t own = (l.e * (uint32_t)stride_e + l.i) * sizeof(T);
  return (T*)((char*)(at + l.e0 * stride_e) + own);
}

struct ScanFwd {
  const void* gate;
  const void* x;
  const float* h0;      // null: zeros
  const uint8_t* done;  // null: no episode ends
  void* hs;
  float* h_last;
  float* states;  // [ceil(T / kKeep), E, H]: c at t = 0, kKeep, ...; or null
  const float* ways;  // [chunks, 2, E, H]: the chunks' effects, or null
  float* carry;       // [chunks, E, H]: c at the chunks' starts, or null
  Cols c;
  int64_t T, chunk;
  int64_t gate_t, gate_e, x_t, x_e;  // strides of time and environment
};

struct ScanBwd {
  const void* dhs;       // of which dhs_bits are taken
  const float* dh_last;  // null: zeros
  const void* gate;
  const void* x;
  const float* states;
  const uint8_t* done;
  void* dgate;
  void* dx;
  float* dh0;    // null: not asked for
  const float* ways;  // [chunks, 2, E, H]: the chunks' effects, or null
  float* carry;       // [chunks, E, H]: a D of the step behind each, or null
  Cols c;
  int64_t T, chunk;
  int64_t gate_t, gate_e, x_t, x_e, dhs_t, dhs_e;
  uint32_t dhs_bits;
};

// e^-|g|, to its own last bits: of m = |g|, e^-m = 2^p (1 + t), p the rounded
// product -m / ln 2 and t = -m - p ln 2 what its rounding left out. Without t
// it is off by up to m half steps, and with it the smaller of z and 1 - z.
// That is three instructions, of which a small call sees most: 512x32x256 bf16
// takes 14.4 us forward instead of 13.9, 65x64x256 6.8 instead of 6.6 (without
// ends).
__device__ __forceinline__ float decay(float g) {
  constexpr double kLn2 = 0.69314718055994530942;
  constexpr float kHigh = (float)kLn2, kLow = (float)(kLn2 - (double)kHigh);
  // 1 / ln 2 is taken a little large: so t is in [0, 2^-15], and a clamp that
  // costs nothing makes that of an infinite gate 0 instead of NaN.
  constexpr float kOver = (float)(-1.0 / kLn2) - 0x1p-22f;
  const float m = fabsf(g), p = m * kOver;
  const float t = fmaf(-p, kLow, fmaf(-p, kHigh, -m));
  const float w = __builtin_amdgcn_exp2f(p);
  return fmaf(w, fminf(fmaxf(t, 0.f), 1.f), w);
}

// The smaller of z and 1 - z, and the other: neither is taken as a difference
// of two near values.
struct Gates {
  float small, large;
  __device__ __forceinline__ explicit Gates(float g) {
    const float e = decay(g);
    large = __builtin_amdgcn_rcpf(1.f + e);
    small = e * large;
  }
};
__device__ __forceinline__ void gates(float g, float& z, float& a) {
  const Gates s(g);
  z = g >= 0.f ? s.large : s.small;
  a = g >= 0.f ? s.small : s.large;
}

// A state's way through some steps: c_end = A c_start + B, or B alone (A
// below zero) where an episode ended within them.
struct Way {
  float A = 1.f, B = 0.f;
  template <bool DONE>
  __device__ __forceinline__ void step(float a, float b) {
    A = DONE && A < 0.f ? A : A * a;
    B = a * B + b;
  }
  __device__ __forceinline__ void end() {
    A = -1.f;
    B = 0.f;
  }
  __device__ __forceinline__ void then(float a, float b) {
    B = a < 0.f ? b : a * B + b;
    A = a < 0.f || A < 0.f ? -1.f : A * a;
  }
};

// A state's way through `count` chunks, from the `first` on or back.
template <int V>
__device__ __forceinline__ void follow(const float* ways, const Cols& cols,
                                       const Lane& l, int64_t first, int count,
                                       bool reverse, float (&c)[V]) {
  const int64_t EH = cols.E * cols.H;
#pragma unroll 4
  for (int i = 0; i < count; ++i) {
    const int64_t k = reverse ? first - i : first + i;
    float A[V], B[V];
    load<float, V>(here(ways + 2 * k * EH, l, cols.H), A);
    load<float, V>(here(ways + (2 * k + 1) * EH, l, cols.H), B);
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = A[v] < 0.f ? B[v] : A[v] * c[v] + B[v];
  }
}

// ---- forward
// N steps of a lane's columns from t on. FULL: all of them are before `end`;
// else what is not is not read.
template <bool FULL, typename T, int V, int N>
__device__ __forceinline__ void read_steps(Vec<T, V> (&to)[N], const T* from,
                                           int64_t stride_t, int64_t stride_e,
                                           const Lane& l, int64_t t,
                                           int64_t end) {
  const T* at = here(from + t * stride_t, l, stride_e);
#pragma unroll
  for (int k = 0; k < N; ++k) {
    if (!FULL) to[k] = {};
    if (FULL || t + k < end) to[k] = load<T, V>(at + k * stride_t);
  }
}

// Which of kKeep steps end an episode: their flags as they are read, and before
// the rest, so that nothing waits for them alone: 256x1024x256 bf16 takes 83 us
// forward so, and 95 where they are made bits of one word behind it.
struct Ends {
  uint8_t flags[kKeep];

  template <bool FULL>
  __device__ __forceinline__ void read(const uint8_t* done, int64_t E,
                                       const Lane& l, int64_t t, int64_t end) {
    const uint8_t* at = done + t * E + l.e0 + l.e;
#pragma unroll
    for (int k = 0; k < kKeep; ++k)
      flags[k] = FULL || t + k < end ? at[k * E] : 0;
  }
  __device__ __forceinline__ bool operator[](int k) const {
    return flags[k] != 0;
  }
};

// kKeep steps of a lane's columns, and which of them end an episode.
template <typename T, int V>
struct Steps {
  Vec<T, V> gate[kKeep], x[kKeep];
  Ends ends;

  template <bool FULL, bool DONE>
  __device__ __forceinline__ void read(const ScanFwd& p, const Lane& l,
                                       int64_t t, int64_t end) {
    if constexpr (DONE) ends.template read<FULL>(p.done, p.c.E, l, t, end);
    read_steps<FULL>(gate, (const T*)p.gate, p.gate_t, p.gate_e, l, t, end);
    read_steps<FULL>(x, (const T*)p.x, p.x_t, p.x_e, l, t, end);
  }
};

template <bool FULL, bool DONE, typename T, int V>
__device__ __forceinline__ void walk(const ScanFwd& p, const Lane& l,
                                     const Steps<T, V>& s, int64_t t,
                                     int64_t end, float (&c)[V]) {
  const int64_t EH = p.c.E * p.c.H;
  if (p.states)
    store<float, V>(here(p.states + t / kKeep * EH, l, p.c.H), c);
  T* out = here((T*)p.hs + t * EH, l, p.c.H);
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    if (!FULL && t + k >= end) continue;
    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float z, a;
      gates((float)s.gate[k].v[v], z, a);
      h[v] = a * c[v] + z * (float)s.x[k].v[v];
      c[v] = DONE && s.ends[k] ? 0.f : h[v];
    }
    store<T, V>(out + k * EH, h);
  }
}

// A chunk is a multiple of kKeep, so states are kept where steps are read.
template <typename T, int V, bool DONE>
__global__ __launch_bounds__(256) void scan_fwd_kernel(ScanFwd p) {
  constexpr int L = kKeep;
  Lane l;
  if (!lane_of<V>(p.c, l)) return;
  const int64_t EH = p.c.E * p.c.H;
  int64_t t = blockIdx.y * p.chunk;
  const int64_t end = t + p.chunk < p.T ? t + p.chunk : p.T;
  float c[V] = {};
  if (p.carry) {
    load<float, V>(here(p.carry + blockIdx.y * EH, l, p.c.H), c);
  } else if (p.h0) {
    load<float, V>(here(p.h0, l, p.c.H), c);
  }
  if (p.ways) follow<V>(p.ways, p.c, l, 0, blockIdx.y, false, c);
  if (t + L <= end) {
    // the next steps are read while these are walked
    Steps<T, V> s, n;
    s.template read<true, DONE>(p, l, t, end);
    for (; t + 2 * L <= end; t += L) {
      n.template read<true, DONE>(p, l, t + L, end);
      walk<true, DONE>(p, l, s, t, end, c);
      s = n;
    }
    walk<true, DONE>(p, l, s, t, end, c);
    t += L;
  }
  if (t < end) {
    Steps<T, V> s;
    s.template read<false, DONE>(p, l, t, end);
    walk<false, DONE>(p, l, s, t, end, c);
  }
  if (end == p.T) store<float, V>(here(p.h_last, l, p.c.H), c);
}

template <bool FULL, bool DONE, typename T, int V>
__device__ __forceinline__ void way(const ScanFwd& p, const Lane& l, int64_t t,
                                    int64_t end, Way (&w)[V]) {
  Steps<T, V> s;
  s.template read<FULL, DONE>(p, l, t, end);
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    if (!FULL && t + k >= end) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float z, a;
      gates((float)s.gate[k].v[v], z, a);
      w[v].template step<DONE>(a, z * (float)s.x[k].v[v]);
      if (DONE && s.ends[k]) w[v].end();
    }
  }
}

// The chunks' effects are found from the last to the first, so that the
// kernel that walks them begins with what was read last and is still cached.
__device__ __forceinline__ int64_t from_last() {
  return gridDim.y - 1 - blockIdx.y;
}

template <int V>
__device__ __forceinline__ void keep_way(const Cols& c, const Lane& l,
                                         const Way (&w)[V], float* ways) {
  float A[V], B[V];
#pragma unroll
  for (int v = 0; v < V; ++v) A[v] = w[v].A, B[v] = w[v].B;
  const int64_t EH = c.E * c.H, k = from_last();
  store<float, V>(here(ways + 2 * k * EH, l, c.H), A);
  store<float, V>(here(ways + (2 * k + 1) * EH, l, c.H), B);
}

template <typename T, int V, bool DONE>
__global__ __launch_bounds__(256) void scan_fwd_way_kernel(ScanFwd p,
                                                           float* ways) {
  constexpr int L = kKeep;
  Lane l;
  if (!lane_of<V>(p.c, l)) return;
  int64_t t = from_last() * p.chunk;
  const int64_t end = t + p.chunk < p.T ? t + p.chunk : p.T;
  Way w[V];
  for (; t + L <= end; t += L) way<true, DONE, T, V>(p, l, t, end, w);
  if (t < end) way<false, DONE, T, V>(p, l, t, end, w);
  keep_way<V>(p.c, l, w, ways);
}

// ---- from chunk to chunk, in either direction: kCols columns a block, its
// kGroups groups of as many lanes one after the other in time, JOIN chunks
// each. With 64 columns a block few have work: 32768x1x256 fp32's 2048 chunks
// took 37 us to join, 22 so.
constexpr int kCols = 32, kGroups = 1024 / kCols;

struct Join {
  const float* ways;   // [chunks, 2, EH]
  const float* first;  // [EH] or null: zeros
  float* carry;        // [chunks, EH]
  int64_t EH, chunks;
  bool reverse;
};

template <int JOIN>
__global__ __launch_bounds__(1024) void scan_join_kernel(Join p) {
  __shared__ float lds[2][kGroups][2][kCols];
  const int group = threadIdx.x / kCols, lane = threadIdx.x % kCols;
  const int64_t col = (int64_t)blockIdx.x * kCols + lane;
  const bool mine = col < p.EH;
  float c = mine && p.first ? p.first[col] : 0.f;
  int turn = 0;
  for (int64_t k0 = 0; k0 < p.chunks; k0 += kGroups * JOIN, turn ^= 1) {
    const int64_t k = k0 + group * JOIN;
    float A[JOIN], B[JOIN];
    Way w;
#pragma unroll
    for (int i = 0; i < JOIN; ++i) {
      A[i] = 1.f;
      B[i] = 0.f;
      if (k + i < p.chunks && mine) {
        const int64_t at = p.reverse ? p.chunks - 1 - (k + i) : k + i;
        A[i] = p.ways[2 * at * p.EH + col];
        B[i] = p.ways[(2 * at + 1) * p.EH + col];
      }
    }
#pragma unroll
    for (int i = 0; i < JOIN; ++i) w.then(A[i], B[i]);
    lds[turn][group][0][lane] = w.A;
    lds[turn][group][1][lane] = w.B;
    // one barrier a turn: the next turn writes the other half
    __syncthreads();
    float start = c;
#pragma unroll
    for (int i = 0; i < kGroups; ++i) {
      if (i == group) start = c;
      const float a = lds[turn][i][0][lane], b = lds[turn][i][1][lane];
      c = a < 0.f ? b : a * c + b;
    }
#pragma unroll
    for (int i = 0; i < JOIN; ++i) {
      if (k + i < p.chunks && mine) {
        const int64_t at = p.reverse ? p.chunks - 1 - (k + i) : k + i;
        p.carry[at * p.EH + col] = start;
      }
      start = A[i] < 0.f ? B[i] : A[i] * start + B[i];
    }
  }
}

// ---- backward
// The bits of a vector that a mask of 32 bits leaves.
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> masked(Vec<T, V> x, uint32_t bits) {
  if constexpr (sizeof(x) == 2) {
    uint16_t w;
    __builtin_memcpy(&w, &x, 2);
    w &= (uint16_t)bits;
    __builtin_memcpy(&x, &w, 2);
  } else {
    uint32_t w[sizeof(x) / 4];
    __builtin_memcpy(w, &x, sizeof(x));
#pragma unroll
    for (int i = 0; i < (int)(sizeof(x) / 4); ++i) w[i] &= bits;
    __builtin_memcpy(&x, w, sizeof(x));
  }
  return x;
}

// kKeep steps of a lane's columns.
template <typename T, int V>
struct Back {
  Vec<T, V> gate[kKeep], dhs[kKeep];
  Ends ends;

  template <bool FULL, bool DONE>
  __device__ __forceinline__ void read(const ScanBwd& p, const Lane& l,
                                       int64_t t, int64_t end) {
    if constexpr (DONE) ends.template read<FULL>(p.done, p.c.E, l, t, end);
    read_steps<FULL>(gate, (const T*)p.gate, p.gate_t, p.gate_e, l, t, end);
    read_steps<FULL>(dhs, (const T*)p.dhs, p.dhs_t, p.dhs_e, l, t, end);
#pragma unroll
    for (int k = 0; k < kKeep; ++k) dhs[k] = masked(dhs[k], p.dhs_bits);
  }
};

template <bool FULL, bool DONE, typename T, int V>
__device__ __forceinline__ void way_back(const ScanBwd& p, const Lane& l,
                                         int64_t t, int64_t end, Way (&w)[V]) {
  Back<T, V> s;
  s.template read<FULL, DONE>(p, l, t, end);
#pragma unroll
  for (int k = kKeep - 1; k >= 0; --k) {
    if (!FULL && t + k >= end) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float z, a;
      gates((float)s.gate[k].v[v], z, a);
      if (DONE && s.ends[k]) w[v].end();
      w[v].template step<DONE>(a, a * (float)s.dhs[k].v[v]);
    }
  }
}

template <typename T, int V, bool DONE>
__global__ __launch_bounds__(256) void scan_bwd_way_kernel(ScanBwd p,
                                                           float* ways) {
  Lane l;
  if (!lane_of<V>(p.c, l)) return;
  const int64_t t0 = from_last() * p.chunk;
  const int64_t end = t0 + p.chunk < p.T ? t0 + p.chunk : p.T;
  int64_t t = t0 + (end - t0) / kKeep * kKeep;
  Way w[V];
  if (t < end) way_back<false, DONE, T, V>(p, l, t, end, w);
  for (t -= kKeep; t >= t0; t -= kKeep)
    way_back<true, DONE, T, V>(p, l, t, end, w);
  keep_way<V>(p.c, l, w, ways);
}

// What kKeep steps of a lane's columns are walked back with.
template <typename T, int V>
struct Sheet {
  Back<T, V> s;
  Vec<T, V> x[kKeep];
  float c[V];  // before the first

  template <bool FULL, bool DONE>
  __device__ __forceinline__ void read(const ScanBwd& p, const Lane& l,
                                       int64_t t, int64_t end) {
    s.template read<FULL, DONE>(p, l, t, end);
    load<float, V>(here(p.states + t / kKeep * p.c.E * p.c.H, l, p.c.H), c);
    read_steps<FULL>(x, (const T*)p.x, p.x_t, p.x_e, l, t, end);
  }
};

template <bool FULL, bool DONE, typename T, int V>
__device__ __forceinline__ void walk_back(const ScanBwd& p, const Lane& l,
                                          Sheet<T, V>& now, int64_t t,
                                          int64_t end, float (&carry)[V]) {
  const int64_t EH = p.c.E * p.c.H;
  Back<T, V>& s = now.s;
  // x - c, and the smaller gates with their gates' signs: the other one is 1
  // less them, so a pair takes one register.
  float diff[kKeep][V], small[kKeep][V];
#pragma unroll
  for (int k = 0; k < kKeep; ++k) {
    if (!FULL && t + k >= end) continue;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float g = (float)s.gate[k].v[v];
      const Gates both(g);
      small[k][v] = copysignf(both.small, g);
      const float z = g >= 0.f ? both.large : both.small;
      const float a = g >= 0.f ? both.small : both.large;
      const float xv = (float)now.x[k].v[v];
      diff[k][v] = xv - now.c[v];
      now.c[v] = DONE && s.ends[k] ? 0.f : a * now.c[v] + z * xv;
    }
  }
  T* out_x = here((T*)p.dx + t * EH, l, p.c.H);
  T* out_g = here((T*)p.dgate + t * EH, l, p.c.H);
#pragma unroll
  for (int k = kKeep - 1; k >= 0; --k) {
    if (!FULL && t + k >= end) continue;
    float dg[V], dx[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float less = fabsf(small[k][v]), more = 1.f - less;
      const bool open = __float_as_int(small[k][v]) >= 0;
      const float z = open ? more : less, a = open ? less : more;
      const bool ends = DONE && s.ends[k];
      const float D = (ends ? 0.f : carry[v]) + (float)s.dhs[k].v[v];
      dx[v] = z * D;
      dg[v] = D * diff[k][v] * (z * a);
      carry[v] = a * D;
    }
    store<T, V>(out_x + k * EH, dx);
    store<T, V>(out_g + k * EH, dg);
  }
}

template <typename T, int V, bool DONE>
__global__ __launch_bounds__(256) void scan_bwd_kernel(ScanBwd p) {
  Lane l;
  if (!lane_of<V>(p.c, l)) return;
  const int64_t EH = p.c.E * p.c.H;
  const int64_t t0 = blockIdx.y * p.chunk;
  const int64_t end = t0 + p.chunk < p.T ? t0 + p.chunk : p.T;
  float carry[V] = {};  // a_{t+1} D_{t+1}
  if (p.carry) {
    load<float, V>(here(p.carry + blockIdx.y * EH, l, p.c.H), carry);
  } else if (p.dh_last) {
    load<float, V>(here(p.dh_last, l, p.c.H), carry);
  }
  if (p.ways)
    follow<V>(p.ways, p.c, l, gridDim.y - 1, gridDim.y - 1 - blockIdx.y, true,
              carry);
  int64_t t = t0 + (end - t0) / kKeep * kKeep;
  Sheet<T, V> now;
  if (t < end) {
    now.template read<false, DONE>(p, l, t, end);
    walk_back<false, DONE>(p, l, now, t, end, carry);
  }
  t -= kKeep;
  if constexpr (sizeof(T) * V < 8) {
    // few waves: the steps before are read while these are walked
    Sheet<T, V> next;
    if (t >= t0) now.template read<true, DONE>(p, l, t, end);
    for (; t >= t0; t -= kKeep) {
      if (t > t0) next.template read<true, DONE>(p, l, t - kKeep, end);
      walk_back<true, DONE>(p, l, now, t, end, carry);
      now = next;
    }
  } else {
    for (; t >= t0; t -= kKeep) {
      now.template read<true, DONE>(p, l, t, end);
      // No read is put off until a register is free: 64x2048x256 bf16 takes 74
      // us so and 78 otherwise. With ends, or in 32 bits, none is.
      if constexpr (sizeof(T) == 2 && !DONE) __builtin_amdgcn_sched_barrier(0);
      walk_back<true, DONE>(p, l, now, t, end, carry);
    }
  }
  if (t0 == 0 && p.dh0) store<float, V>(here(p.dh0, l, p.c.H), carry);
}

// ---- one step
struct ScanStep {
  const void* gate;
  const void* x;
  const uint8_t* done;  // environments that restart from zero; null: none
  float* h;             // in place
  void* hs;
  Cols c;
  int64_t gate_e, x_e;
};

template <typename T, int V>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanStep p) {
  Lane l;
  if (!lane_of<V>(p.c, l)) return;
  const bool end = p.done && p.done[l.e0 + l.e];
  const Vec<T, V> gate = load<T, V>(here((const T*)p.gate, l, p.gate_e));
  const Vec<T, V> x = load<T, V>(here((const T*)p.x, l, p.x_e));
  float h[V];
  load<float, V>(here(p.h, l, p.c.H), h);
#pragma unroll
  for (int v = 0; v < V; ++v) {
    float z, a;
    gates((float)gate.v[v], z, a);
    h[v] = a * (end ? 0.f : h[v]) + z * (float)x.v[v];
  }
  store<float, V>(here(p.h, l, p.c.H), h);
  store<T, V>(here((T*)p.hs, l, p.c.H), h);
}

// In place, so no column may be computed twice: V divides H.
template <typename T, int V>
hipError_t step_with(ScanStep p, hipStream_t s) {
  p.c.n = p.c.H / V;
  const int64_t grid = (p.c.E * p.c.n + 255) / 256;
  return launch(scan_step_kernel<T, V>, dim3(grid), dim3(256), 0, s, p);
}

template <typename T>
hipError_t step(const ScanStep& p, hipStream_t s) {
  if (p.c.E * p.c.H == 0) return hipSuccess;
  if (p.c.H % 4 == 0) return step_with<T, 4>(p, s);
  if (p.c.H % 2 == 0) return step_with<T, 2>(p, s);
  return step_with<T, 1>(p, s);
}

// How the columns of a call lie on lanes, and its time in chunks.
struct Plan {
  int V;
  int64_t n, chunk, chunks;
};

constexpr int64_t kWaves = 4096;  // as many keep the memory busy
constexpr int64_t kShort = 64;    // steps that one lane walks in any case

// Lanes take 8 bytes of columns, as few load instructions as the memory's
// rate allows, or fewer where that leaves too few waves: 64x256x256 bf16 runs
// in 10.2 us forward and 19 us backward with 2 bytes, in 19 and 26 us with 8;
// 64x1024x256 in 24 and 38 us with 8. (Here and below with ends.)
//
// Time is cut where a lane would walk more than kShort steps among few waves:
// 512x32x256 bf16 runs in 16 and 22 us in chunks, in 48 and 113 us walked;
// 65x64x256 in 7.5 and 11 us instead of 9 and 19; 32x64x64 fp32 would take 6.7
// and 8.9 instead of 5.0 and 8.7. With 1024 waves it is walked (256x1024x256
// bf16: 83 and 135 us, in chunks 142 and 191, which read more), but backward
// not by lanes of 2 bytes (512x256x256 bf16: 64 us walked forward, 80 in
// chunks; 141 us walked backward, 106 in chunks).
Plan plan(int64_t T, int64_t E, int64_t H, int bytes, bool back) {
  Plan p;
  int64_t waves = 0;
  auto lay = [&](int64_t cuts) {
    for (p.V = 8 / bytes; p.V >= 1; p.V /= 2) {
      if (p.V > H) continue;
      p.n = (H + p.V - 1) / p.V;
      waves = (E * p.n + kWave - 1) / kWave;
      if (p.V == 1 || waves * cuts >= kWaves / 4) break;
    }
  };
  lay(1);
  p.chunk = T;
  p.chunks = 1;
  if (T > kShort && (waves < kWaves / 4 || (back && p.V * bytes < 4))) {
    lay(T / 64);
    int64_t want = kWaves / waves;  // chunks
    const int64_t most = (T + 15) / 16;
    want = want < most ? want : most;
    want = want < 32768 ? want : 32768;
    if (want > 1) {
      p.chunk = (T + want - 1) / want;
      p.chunk = (p.chunk + kKeep - 1) / kKeep * kKeep;
      p.chunks = (T + p.chunk - 1) / p.chunk;
    }
  }
  return p;
}

// A chunk follows the ways of up to kFollow others itself, without a kernel
// between: 509x37x263 fp16's 22 chunks are walked 4.5 us sooner each way,
// 663x36x64 bf16's 42 0.8 and 1.4 us, and a launch is saved. More would read
// too much (2063x3x64 fp32's 129: 19 us instead of 12.3): scratch then holds
// the chunks' starts as well.
constexpr int64_t kFollow = 64;
static_assert(kFollow >= 1, "a call that is not cut has no scratch");

template <typename P>
void give_ways(P& p, const Plan& q, float* scratch) {
  const int64_t EH = p.c.E * p.c.H;
  p.c.n = q.n;
  p.chunk = q.chunk;
  p.ways = q.chunks > 1 && q.chunks <= kFollow ? scratch : nullptr;
  p.carry = q.chunks > kFollow ? scratch + 2 * q.chunks * EH : nullptr;
}

hipError_t join(const float* ways, const float* first, float* carry,
                const Plan& q, int64_t EH, bool reverse, hipStream_t s) {
  const Join j = {ways, first, carry, EH, q.chunks, reverse};
  const dim3 grid((EH + kCols - 1) / kCols), block(1024);
  // fewer chunks a group where one turn is enough: 1473x1x181 bf16 runs in
  // 10.6 us so and in 11.4 with 16; 7065x11x64's 295 in 24.2 and 23.1
  if (q.chunks <= 8 * kGroups)
    return launch(scan_join_kernel<8>, grid, block, 0, s, j);
  return launch(scan_join_kernel<16>, grid, block, 0, s, j);
}

template <typename T, int V, bool DONE>
hipError_t fwd_with(const ScanFwd& p, const Plan& q, float* ways,
                    hipStream_t s) {
  const int64_t EH = p.c.E * p.c.H;
  const dim3 grid((p.c.E * p.c.n + 255) / 256, q.chunks);
  if (q.chunks > 1) {
    hipError_t e = launch(scan_fwd_way_kernel<T, V, DONE>, grid, dim3(256), 0, s,
                          p, ways);
    if (e == hipSuccess && p.carry)
      e = join(ways, p.h0, p.carry, q, EH, false, s);
    if (e != hipSuccess) return e;
  }
  return launch(scan_fwd_kernel<T, V, DONE>, grid, dim3(256), 0, s, p);
}

template <typename T>
hipError_t fwd(ScanFwd p, float* scratch, hipStream_t s) {
  if (p.c.E * p.c.H == 0) return hipSuccess;
  const Plan q = plan(p.T, p.c.E, p.c.H, sizeof(T), false);
  give_ways(p, q, scratch);
  switch (q.V * 2 + (p.done != nullptr)) {
    case 2: return fwd_with<T, 1, false>(p, q, scratch, s);
    case 3: return fwd_with<T, 1, true>(p, q, scratch, s);
    case 4: return fwd_with<T, 2, false>(p, q, scratch, s);
    case 5: return fwd_with<T, 2, true>(p, q, scratch, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (p.done) return fwd_with<T, 4, true>(p, q, scratch, s);
    return fwd_with<T, 4, false>(p, q, scratch, s);
  }
  return hipErrorInvalidValue;
}

template <typename T, int V, bool DONE>
hipError_t bwd_with(const ScanBwd& p, const Plan& q, float* ways,
                    hipStream_t s) {
  const int64_t EH = p.c.E * p.c.H;
  const dim3 grid((p.c.E * p.c.n + 255) / 256, q.chunks);
  if (q.chunks > 1) {
    hipError_t e =
        launch(scan_bwd_way_kernel<T, V, DONE>, grid, dim3(256), 0, s, p, ways);
    if (e == hipSuccess && p.carry)
      e = join(ways, p.dh_last, p.carry, q, EH, true, s);
    if (e != hipSuccess) return e;
  }
  return launch(scan_bwd_kernel<T, V, DONE>, grid, dim3(256), 0, s, p);
}

template <typename T>
hipError_t bwd(ScanBwd p, float* scratch, hipStream_t s) {
  if (p.c.E * p.c.H == 0) return hipSuccess;
  const Plan q = plan(p.T, p.c.E, p.c.H, sizeof(T), true);
  give_ways(p, q, scratch);
  switch (q.V * 2 + (p.done != nullptr)) {
    case 2: return bwd_with<T, 1, false>(p, q, scratch, s);
    case 3: return bwd_with<T, 1, true>(p, q, scratch, s);
    case 4: return bwd_with<T, 2, false>(p, q, scratch, s);
    case 5: return bwd_with<T, 2, true>(p, q, scratch, s);
  }
  if constexpr (sizeof(T) == 2) {
    if (p.done) return bwd_with<T, 4, true>(p, q, scratch, s);
    return bwd_with<T, 4, false>(p, q, scratch, s);
  }
  return hipErrorInvalidValue;
}

}  // namespace

// Floats of scratch that the forward or the backward call needs.
extern "C" int64_t rlsched_scan_scratch(int64_t T, int64_t E, int64_t H,
                                        int type, int back) {
  if (E * H == 0) return 0;
  const Plan q = plan(T, E, H, type == F32 ? 4 : 2, back);
  if (q.chunks == 1) return 0;
  return (q.chunks > kFollow ? 3 : 2) * q.chunks * E * H;
}

// Elements from one environment to the next that a lane's 32-bit distance
// covers for any number of them in a block; beyond it the caller copies.
extern "C" int64_t rlsched_scan_reach(int64_t H) {
  const int64_t envs = 256 * 4 / (H < 1 ? 1 : H) + 2;
  return ((1ll << 31) / 4 - H) / (envs < 256 ? envs : 256);
}

extern "C" int64_t rlsched_scan_states(int64_t T) {
  return (T + kKeep - 1) / kKeep;
}

extern "C" int rlsched_scan_fwd(int device, void* stream, const void* gate,
                                const void* x, const float* h0,
                                const uint8_t* done, void* hs, float* h_last,
                                float* states, float* scratch, int64_t T,
                                int64_t E, int64_t H, int64_t gate_t,
                                int64_t gate_e, int64_t x_t, int64_t x_e,
                                int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const ScanFwd p = {gate,    x,       h0,     done, hs, h_last, states,
                     nullptr, nullptr, {E, H}, T,    0,  gate_t, gate_e,
                     x_t,     x_e};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return fwd<float>(p, scratch, s);
  if (type == BF16) return fwd<bf16>(p, scratch, s);
  if (type == F16) return fwd<f16>(p, scratch, s);
  return hipErrorInvalidValue;
}

extern "C" int rlsched_scan_bwd(int device, void* stream, const void* dhs,
                                const float* dh_last, const void* gate,
                                const void* x, const float* states,
                                const uint8_t* done, void* dgate, void* dx,
                                float* dh0, float* scratch, int64_t T,
                                int64_t E, int64_t H, int64_t gate_t,
                                int64_t gate_e, int64_t x_t, int64_t x_e,
                                int64_t dhs_t, int64_t dhs_e, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  ScanBwd p = {dhs, dh_last, gate,    x,       states, done,  dgate,
               dx,  dh0,     nullptr, nullptr, {E, H}, T,     0,
               gate_t, gate_e, x_t,   x_e,     dhs_t,  dhs_e, ~0u};
  if (!dhs) {
    // zeros: no bit of what is there anyway, so the kernels need no branch
    p.dhs = gate;
    p.dhs_t = gate_t;
    p.dhs_e = gate_e;
    p.dhs_bits = 0;
  }
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return bwd<float>(p, scratch, s);
  if (type == BF16) return bwd<bf16>(p, scratch, s);
  if (type == F16) return bwd<f16>(p, scratch, s);
  return hipErrorInvalidValue;
}

extern "C" int rlsched_scan_step(int device, void* stream, const void* gate,
                                 const void* x, const uint8_t* done, float* h,
                                 void* hs, int64_t E, int64_t H,
                                 int64_t gate_e, int64_t x_e, int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const ScanStep p = {gate, x, done, h, hs, {E, H}, gate_e, x_e};
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
