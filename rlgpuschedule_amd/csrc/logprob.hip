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
//
// A probability below 2^-126 counts as 0.
//
// Bound by memory: one pass over the logits each way. On an MI355X 4096 x
// 32768 bf16 takes 75 us forward (268 MB, 3.6 TB/s; a large sum of torch's
// reads at 4.0 there) and 114 us backward (537 MB, 4.7 TB/s; a large copy's
// rate is 4.9); 524288 x 17 fp32 with a mask 16 and 25 us. One row of 131072
// with 20 alternatives takes 7 us in 32 parts and 5 to join them, its latency.
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
__device__ __forceinline__ uint64_t key_of(float v, int i) {
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

__device__ __forceinline__ uint64_t larger(uint64_t a, uint64_t b) {
  return a > b ? a : b;
}

// Vector j of a row. The last vector of a row of no whole number of them
// begins early enough to end with the row; what it shares with the one
// before is left out unless SHARED, so no element is counted twice.
template <typename T>
struct Piece {
  Vec<T, kVec<T>> x;
  Vec<uint8_t, kVec<T>> ok;
  int from, skip;

  __device__ __forceinline__ void read(const T* row, const uint8_t* mask,
                                       int A, int j) {
    constexpr int V = kVec<T>;
    const int base = j * V;
    from = A < V || base < A - V ? base : A - V;
    skip = base - from;
    if (A >= V) {
      x = load<T, V>(row + from);
      if (mask) ok = load<uint8_t, V>(mask + from);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        x.v[e] = e < A ? row[e] : (T)-INFINITY;
        if (mask) ok.v[e] = e < A ? mask[e] : 0;
      }
    }
  }
  // its logits, -inf where nothing may be taken
  template <bool SHARED = false>
  __device__ __forceinline__ void values(bool masked,
                                         float (&f)[kVec<T>]) const {
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) f[e] = (float)x.v[e];
    if (masked) {
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e)
        if (!ok.v[e]) f[e] = -INFINITY;
    }
    if (!SHARED && skip) {
#pragma unroll
      for (int e = 0; e < kVec<T>; ++e)
        if (e < skip) f[e] = -INFINITY;
    }
  }
};

template <typename T>
__device__ __forceinline__ void store_row(T* y, int A, int from,
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
  const bool any = !(s <= 0.f);  // NaN: a broken row
  const float ls = any ? logf(s) : 0.f;
  const float H = any ? ls - u / s : 0.f;
  const float lp = any ? q - m - ls : -INFINITY;
  p.logp[row] = act < 0 ? 0.f : lp;
  p.entropy[row] = H;
  if (p.stats) {
    p.stats[3 * row] = any ? m : 0.f;
    p.stats[3 * row + 1] = ls;
    p.stats[3 * row + 2] = H;
  }
}

// Where a row's alternatives go.
struct Top {
  float* logp;
  int64_t* index;
  float m, ls;
  bool broken;

  __device__ __forceinline__ Top(const LogpFwd& p, int64_t row, float m_,
                                 float s)
      : logp(p.top_logp + row * p.k),
        index(p.top_index + row * p.k),
        m(m_),
        ls(logf(s)),
        broken(s != s) {}
  __device__ __forceinline__ void put(int rank, uint64_t key) const {
    const bool some = key && !broken;
    logp[rank] = broken ? NAN : some ? value_of(key) - m - ls : -INFINITY;
    index[rank] = some ? index_of(key) : -1;
  }
};

template <typename T>
__device__ __forceinline__ float taken(const T* x, const uint8_t* ok,
                                       int64_t A, int64_t act) {
  return act >= 0 && act < A && !(ok && !ok[act]) ? (float)x[act] : -INFINITY;
}

// What the gradient of one row's elements needs.
struct Row {
  float m, ls, H, dl, dh;
  int act;
};

template <typename T>
__device__ __forceinline__ Row row_of(const LogpBwd& p, const T* x,
                                      const uint8_t* ok, int64_t row) {
  Row r;
  const int64_t act = p.actions[row];
  r.act = (int)act;
  r.m = p.stats[3 * row];
  r.ls = p.stats[3 * row + 1];
  r.H = p.stats[3 * row + 2];
  r.dl = p.dlogp ? p.dlogp[row] : 0.f;
  r.dh = p.dentropy ? p.dentropy[row] : 0.f;
  // a taken action of probability 0 is a constant -inf
  if (taken(x, ok, p.A, act) == -INFINITY) r.dl = 0.f;
  return r;
}

__device__ __forceinline__ float gradient(const Row& r, float v, int i) {
  const float d = maximum(v - r.m, kFloor) - r.ls, pr = __expf(d);
  const float g = -pr * (r.dl + r.dh * (d + r.H));
  return v == -INFINITY ? 0.f : i == r.act ? g + r.dl : g;
}

// How many of n keys are larger; reads of several in flight, up to kAhead
// keys behind the last, which are not counted.
constexpr int kAhead = 7;

__device__ __forceinline__ int rank_of(uint64_t mine, const uint64_t* keys,
                                       int n) {
  int rank = 0;
  for (int i = 0; i < n; i += 8) {
    uint64_t k[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = keys[i + j];
#pragma unroll
    for (int j = 0; j < 8; ++j) rank += (k[j] > mine) & (i + j < n);
  }
  return rank;
}

// The largest of a lane's logits, and where it is first.
template <int N, int V>
__device__ __forceinline__ float first_best(const float (&f)[N][V],
                                            int& slot) {
  float top = -INFINITY;
  slot = 0;
#pragma unroll
  for (int i = 0; i < N * V; ++i)
    if (f[i / V][i % V] > top) top = f[i / V][i % V], slot = i;
  return top;
}

template <int N, int V>
__device__ __forceinline__ void take_out(float (&f)[N][V], int slot) {
#pragma unroll
  for (int i = 0; i < N * V; ++i)
    f[i / V][i % V] = i == slot ? -INFINITY : f[i / V][i % V];
}

// Where in its row the at-th logit of lane l is, of lanes with every G-th
// vector.
template <typename T, int G>
__device__ __forceinline__ int place_of(int l, int at, int A) {
  constexpr int V = kVec<T>;
  const int base = (l + G * (at / V)) * V;
  return (A < V || base < A - V ? base : A - V) + at % V;
}

// A lower bound of the k-th largest element that few more than k reach: a
// bisection between the least and the largest of G lanes' H bests each, no
// element the best of two, by how many of them reach the middle. First the
// middle of the values is taken; where that does not come near, as with one
// value far above the others, that of their exponents. Wherever it ends, its
// lower end holds.
template <int G, int H>
__device__ __forceinline__ float bound_of(const float (&heads)[H], float most,
                                          int k) {
  const int enough = k + k / 4 + 2;
  float lo = INFINITY, hi = most;
#pragma unroll
  for (int h = 0; h < H; ++h)
    lo = fminf(lo, heads[h] == -INFINITY ? INFINITY : heads[h]);
  lo = -group_max<G>(-lo);
  auto reach = [&](float v) {
    uint32_t n = 0;
    if constexpr (G == kWave) {
#pragma unroll
      for (int h = 0; h < H; ++h) n += __popcll(__ballot(heads[h] >= v));
      return (int)n;
    }
#pragma unroll
    for (int h = 0; h < H; ++h) n += heads[h] >= v;
    return (int)group_reduce<G>(n,
                                [](uint32_t a, uint32_t b) { return a + b; });
  };
  int n = reach(lo);
  if (n < k) return -3.402823466e38f;
  for (int i = 0; i < 24 && n > enough && lo < hi; ++i) {
    float mid = 0.5f * lo + 0.5f * hi;
    if (i >= 6) {
      // whole numbers in the order of the values
      const int a = __float_as_int(lo), b = __float_as_int(hi);
      const int from = a ^ (a >> 31 & 0x7fffffff);
      const int to = b ^ (b >> 31 & 0x7fffffff);
      const int at = from + (int)(((uint32_t)to - (uint32_t)from + 1) / 2);
      mid = __int_as_float(at ^ (at >> 31 & 0x7fffffff));
    }
    const int some = reach(mid);
    if (some < k) {
      hi = mid;
    } else {
      lo = mid;
      n = some;
    }
  }
  return lo;
}

// A wave's writes to LDS are there for its reads behind this.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Keys of short rows: 19 bits hold a 16-bit type's values in 32 bits, the
// other 13 an index below 2^13. 0 is nothing, as for the wide ones.
template <typename T>
using Key = std::conditional_t<sizeof(T) == 2, uint32_t, uint64_t>;

template <typename K>
__device__ __forceinline__ K short_key(float v, int i) {
  const uint64_t key = key_of(v, i);
  if constexpr (sizeof(K) == 8) return key;
  return ((uint32_t)(key >> 32) & ~0x1fffu) | (0x1fffu - (uint32_t)i);
}
__device__ __forceinline__ uint64_t wide_key(uint64_t key) { return key; }
__device__ __forceinline__ uint64_t wide_key(uint32_t key) {
  const uint32_t low = key & 0x80000000u ? 0 : 0x1fffu;
  return (uint64_t)((key & ~0x1fffu) | low) << 32 |
         (0xffffffffu - (0x1fffu - (key & 0x1fffu)));
}

// ---- rows of up to G * N vectors: G lanes a row, all of it in registers
// Few lanes with up to four vectors each share a row's bookkeeping among few:
// 524288 x 17 fp32 takes two thirds of the time with 2 lanes of 3 vectors (16
// us) that it takes with 8 of one.

// So many lanes or more find a row's alternatives by a bound: 64199 x 886 bf16
// with 14 takes 57 us so, in rounds 164. Fewer take a round an alternative:
// 1582 x 51 fp32 with 20 takes 11.4 us so, by a bound 17.8.
template <int G>
constexpr bool kRanked = G >= 8;
// Bests of a row that its bound is found from: of 64, 8192 x 2048 bf16 with 64
// alternatives takes 119 us instead of 29, and 17 with 20 alternatives as well.
constexpr int kBests = 128;
// Keys that a row's lanes rank among themselves: what reaches the bound, of
// 128 bests' 82 about 130.
template <int G>
constexpr int kCap = G >= 32 ? 256 : G == 16 ? 192 : 128;

template <typename T, int G, int N, bool TOP>
__global__ __launch_bounds__(256, TOP && kRanked<G> && N <= 4 ? 4 : 1)
void logp_group_kernel(LogpFwd p) {
  constexpr int V = kVec<T>, R = 256 / G;
  // a row's bests, each of C of a lane's elements
  constexpr int C = (N * V + kBests / G - 1) / (kBests / G);
  constexpr int H = (N * V + C - 1) / C;
  constexpr bool kFind = TOP && kRanked<G>;
  using K = Key<T>;
  // zeros behind the last, and no two rows at one bank
  constexpr int kRow = kFind ? kCap<G> + 80 / sizeof(K) : 1;
  static_assert(!kFind || kRow >= kCap<G> + kAhead);
  __shared__ alignas(16) K found[kFind ? R : 1][kRow];
  __shared__ int counts[kFind ? R : 1];
  const int l = threadIdx.x % G, A = (int)p.A;
  for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G; row < p.rows;
       row += (int64_t)gridDim.x * R) {
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    const int64_t act = p.actions[row];
    Piece<T> piece[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((l + G * i) * V < A) piece[i].read(x, ok, A, l + G * i);
    const float q = taken(x, ok, A, act);
    float f[N][V], m = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = -INFINITY;
      if ((l + G * i) * V < A) piece[i].values(ok, f[i]);
#pragma unroll
      for (int e = 0; e < V; ++e) m = maximum(m, f[i][e]);
    }
    m = group_max<G>(m);
    const float most = m;
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
    if constexpr (!TOP) continue;
    const Top to_row(p, row, m, s);
    int count = kCap<G> + 1;
    if constexpr (kRanked<G>) {
      K* keys = found[threadIdx.x / G];
      int* at = &counts[threadIdx.x / G];
      float heads[H];
#pragma unroll
      for (int h = 0; h < H; ++h) {
        heads[h] = -INFINITY;
#pragma unroll
        for (int i = h * C; i < (h + 1) * C && i < N * V; ++i)
          heads[h] = fmaxf(heads[h], f[i / V][i % V]);
      }
      const float least =
          bound_of<G, H>(heads, to_row.broken ? -INFINITY : most, p.k);
      // a bit for each element that reaches it
      std::conditional_t<(N * V > 32), uint64_t, uint32_t> mine = 0;
#pragma unroll
      for (int i = N * V - 1; i >= 0; --i)
        mine = mine + mine + (f[i / V][i % V] >= least);
      if (to_row.broken) mine = 0;
      if (l == 0) *at = 0;
      wave_sync();
      int to = mine ? atomicAdd(at, __popcll(mine)) : 0;
      for (; mine; mine &= mine - 1, ++to) {
        const int j = place_of<T, G>(l, __builtin_ctzll(mine), A);
        if (to < kCap<G>) keys[to] = short_key<K>((float)x[j], j);
      }
      wave_sync();
      count = *at;
      if (count <= kCap<G>) {
        for (int i = l; i < kAhead; i += G) keys[count + i] = 0;
        wave_sync();
        for (int i = l; i < count; i += G) {
          const K own = keys[i];
          int rank = 0;
          for (int j = 0; j < count; j += 8) {
            K other[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) other[e] = keys[j + e];
#pragma unroll
            for (int e = 0; e < 8; ++e) rank += other[e] > own;
          }
          if (rank < p.k) to_row.put(rank, wide_key(own));
        }
        for (int i = count + l; i < p.k; i += G) to_row.put(i, 0);
        wave_sync();
      }
    }
    if (count <= kCap<G>) continue;
    // a round an alternative
    if constexpr (sizeof(K) == 4 && !kRanked<G>) {
      K keys[N * V], last = ~(K)0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int from = place_of<T, G>(l, i * V, A);
        asm volatile("" : "+v"(from));  // its sums are not kept for later rows
#pragma unroll
        for (int e = 0; e < V; ++e)
          keys[i * V + e] =
              f[i][e] > -INFINITY ? short_key<K>(f[i][e], from + e) : 0;
      }
      for (int j = 0; j < p.k; ++j) {
        // Below the last one, differences to it wrap: the largest of all is
        // the nearest below it.
        if (last) {
          K best = 0;
#pragma unroll
          for (int i = 0; i < N * V; ++i) best = max(best, keys[i] - last);
          last += group_reduce<G>(best,
                                  [](K a, K b) { return a > b ? a : b; });
        }
        if (l == 0) to_row.put(j, last ? wide_key(last) : 0);
      }
    } else {
      // the one found is taken out
      for (int j = 0; j < p.k; ++j) {
        int slot;
        const float top = first_best(f, slot);
        const uint64_t own =
            top > -INFINITY ? key_of(top, place_of<T, G>(l, slot, A)) : 0;
        const uint64_t best = group_larger<G>(own);
        if (own == best) take_out(f, slot);
        if (l == 0) to_row.put(j, best);
      }
    }
  }
}

template <typename T, int G, int N>
__global__ __launch_bounds__(256) void logp_group_bwd_kernel(LogpBwd p) {
  constexpr int V = kVec<T>, R = 256 / G;
  const int l = threadIdx.x % G, A = (int)p.A;
  for (int64_t row = (int64_t)blockIdx.x * R + threadIdx.x / G; row < p.rows;
       row += (int64_t)gridDim.x * R) {
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    T* out = (T*)p.dlogits + row * p.A;
    Piece<T> piece[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if ((l + G * i) * V < A) piece[i].read(x, ok, A, l + G * i);
    const Row r = row_of(p, x, ok, row);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if ((l + G * i) * V >= A) continue;
      float f[V];
      piece[i].template values<true>(ok, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = gradient(r, f[e], piece[i].from + e);
      store_row<T>(out, A, piece[i].from, f);
    }
  }
}

// ---- longer rows, forward: a block of 256 lanes a row, or a part of one
// A lane's running maximum, sum and weighted sum. m starts at the lowest
// finite value, so differences of it are never -inf minus -inf.
struct Running {
  float m = -3.402823466e38f, s = 0.f, u = 0.f;

  // as they would be below a larger maximum
  __device__ __forceinline__ void lower(float n) {
    const float d0 = maximum(m - n, kFloor), w0 = __expf(d0);
    u = w0 * (u + d0 * s);
    s = w0 * s;
    m = n;
  }
  template <int N>
  __device__ __forceinline__ void take(const float (&f)[N], float top) {
    lower(maximum(m, top));
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float d = maximum(f[e] - m, kFloor), w = __expf(d);
      s += w;
      u += w * d;
    }
  }
  __device__ __forceinline__ void join_wave() {
    lower(group_max(m));
    s = group_sum(s);
    u = group_sum(u);
  }
};

constexpr int kLanes = 256;
// Elements that are ranked at once.
constexpr int kFound = 512;

// bound_of a block's lanes. `count` is cleared.
__device__ __forceinline__ float block_bound(float own, int k, float* heads,
                                             float* at, int* count) {
  heads[threadIdx.x] = own;
  __syncthreads();
  if (threadIdx.x < kWave) {
    constexpr int H = kLanes / kWave;
    float mine[H], most = -INFINITY;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      mine[h] = heads[threadIdx.x + h * kWave];
      most = maximum(most, mine[h]);
    }
    const float bound = bound_of<kWave, H>(mine, group_max(most), k);
    if (threadIdx.x == 0) *at = bound, *count = 0;
  }
  __syncthreads();
  return *at;
}

// The largest of a block's keys; `keys` has one for each wave.
__device__ __forceinline__ uint64_t block_larger(uint64_t k, uint64_t* keys) {
  k = group_larger(k);
  if (threadIdx.x % kWave == 0) keys[threadIdx.x / kWave] = k;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kLanes / kWave; ++i) k = larger(k, keys[i]);
  __syncthreads();
  return k;
}

// The parts of a row that blocks of their own have seen: (m, s, u) of each,
// and its k best keys in their order, zeros behind the last.
struct Parts {
  float* sums;     // [rows, parts, 3]
  uint64_t* keys;  // [rows, parts, k]
  int parts;       // of each row; 1: the block writes the row's results
};

template <typename T, bool TOP>
__global__ __launch_bounds__(kLanes) void logp_row_kernel(LogpFwd p,
                                                          Parts parts) {
  constexpr int V = kVec<T>, W = kLanes / kWave, U = 4;
  __shared__ float sums[3][W], heads[kLanes], least_at;
  __shared__ uint64_t found[kFound + kAhead], waves[W];
  __shared__ int count_at, hot_at, hot[kLanes];
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int A = (int)p.A, all = (A + V - 1) / V, P = parts.parts;
  for (int64_t b = blockIdx.x; b < p.rows * P; b += gridDim.x) {
    const int64_t row = P == 1 ? b : b / P;
    const int part = P == 1 ? 0 : (int)(b - row * P);
    const int first = (int)((int64_t)all * part / P);
    const int n = (int)((int64_t)all * (part + 1) / P);
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    Running r;
    float own = -INFINITY;
    auto take = [&](const Piece<T>& v) {
      float f[V];
      v.values(ok, f);
      float top = f[0];
#pragma unroll
      for (int e = 1; e < V; ++e) top = maximum(top, f[e]);
      if (TOP) own = maximum(own, top);
      r.take(f, top);
    };
    int j = first + tid;
    for (; j + (U - 1) * kLanes < n; j += U * kLanes) {
      Piece<T> v[U];
#pragma unroll
      for (int i = 0; i < U; ++i) v[i].read(x, ok, A, j + i * kLanes);
#pragma unroll
      for (int i = 0; i < U; ++i) take(v[i]);
    }
    for (; j < n; j += kLanes) {
      Piece<T> v;
      v.read(x, ok, A, j);
      take(v);
    }
    r.join_wave();
    if (lane == 0) {
      sums[0][wave] = r.m;
      sums[1][wave] = r.s;
      sums[2][wave] = r.u;
    }
    __syncthreads();
    float m = sums[0][0], s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 1; i < W; ++i) m = maximum(m, sums[0][i]);
#pragma unroll
    for (int i = 0; i < W; ++i) {
      Running one{sums[0][i], sums[1][i], sums[2][i]};
      one.lower(m);
      s += one.s;
      u += one.u;
    }
    if (tid == 0) {
      if (P == 1) {
        const int64_t act = p.actions[row];
        finish_row(p, row, act, taken(x, ok, A, act), m, s, u);
      } else {
        parts.sums[3 * b] = m;
        parts.sums[3 * b + 1] = s;
        parts.sums[3 * b + 2] = u;
      }
    }
    if (TOP) {
      const Top to_row(p, row, m, s);
      auto put = [&](int i, uint64_t key) {
        if (P == 1) {
          to_row.put(i, key);
        } else {
          parts.keys[b * p.k + i] = key;
        }
      };
      if (tid == 0) hot_at = 0;
      const float least =
          block_bound(own, p.k, heads, &least_at, &count_at);
      // Only the vectors of lanes whose own best reaches the bound have more to
      // give: they are read again, by all lanes.
      if (own >= least) hot[atomicAdd(&hot_at, 1)] = tid;
      __syncthreads();
      const int each = (n - first + kLanes - 1) / kLanes, some = hot_at * each;
      for (int i = tid; i < some; i += 2 * kLanes) {
        Piece<T> v[2];
        bool in[2];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int at = i + c * kLanes, h = at / each;
          const int j = at < some ? first + hot[h] + (at - h * each) * kLanes : n;
          in[c] = j < n;
          if (in[c]) v[c].read(x, ok, A, j);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if (!in[c]) continue;
          float f[V];
          v[c].values(ok, f);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            if (!(f[e] >= least)) continue;
            const int at = atomicAdd(&count_at, 1);
            if (at < kFound) found[at] = key_of(f[e], v[c].from + e);
          }
        }
      }
      __syncthreads();
      const int count = count_at;
      if (count <= kFound) {
        // whatever order they were found in, each goes to its rank
        for (int i = tid; i < count; i += kLanes) {
          const uint64_t mine = found[i];
          const int rank = rank_of(mine, found, count);
          if (rank < p.k) put(rank, mine);
        }
        for (int i = count + tid; i < p.k; i += kLanes) put(i, 0);
      } else {
        // More than fit, such as many equal ones: one round an alternative,
        // each a maximum below the one before.
        uint64_t last = ~0ull;
        for (int a = 0; a < p.k; ++a) {
          uint64_t top = 0;
          if (own >= least) {
            for (int i = first + tid; i < n; i += kLanes) {
              Piece<T> v;
              v.read(x, ok, A, i);
              float f[V];
              v.values(ok, f);
#pragma unroll
              for (int e = 0; e < V; ++e) {
                const uint64_t k = key_of(f[e], v.from + e);
                if (f[e] > -INFINITY && k < last && k > top) top = k;
              }
            }
          }
          last = block_larger(top, waves);
          if (tid == 0) put(a, last);
        }
      }
    }
    __syncthreads();  // the next turn writes what this one reads
  }
}

// The same for parts of up to N * kLanes vectors with alternatives, N of them
// in a lane's registers: nothing is read twice, 30000 x 4500 bf16 with 20 takes
// 168 us so and 212 walked, 8192 x 4096 38 and 70.
template <typename T, int N>
__global__ __launch_bounds__(kLanes) void logp_part_kernel(LogpFwd p,
                                                           Parts parts) {
  constexpr int V = kVec<T>, W = kLanes / kWave;
  __shared__ float sums[3][W], heads[kLanes], least_at;
  __shared__ uint64_t found[kFound + kAhead], waves[W];
  __shared__ int count_at;
  const int tid = threadIdx.x, wave = tid / kWave, lane = tid % kWave;
  const int A = (int)p.A, all = (A + V - 1) / V, P = parts.parts;
  for (int64_t b = blockIdx.x; b < p.rows * P; b += gridDim.x) {
    const int64_t row = P == 1 ? b : b / P;
    const int part = P == 1 ? 0 : (int)(b - row * P);
    const int first = (int)((int64_t)all * part / P);
    const int n = (int)((int64_t)all * (part + 1) / P);
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    Piece<T> v[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first + tid + i * kLanes < n)
        v[i].read(x, ok, A, first + tid + i * kLanes);
    float f[N][V], tops[N], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int e = 0; e < V; ++e) f[i][e] = -INFINITY;
      if (first + tid + i * kLanes < n) v[i].values(ok, f[i]);
      tops[i] = f[i][0];
#pragma unroll
      for (int e = 1; e < V; ++e) tops[i] = maximum(tops[i], f[i][e]);
      top = maximum(top, tops[i]);
    }
    float m = group_max(top);
    if (lane == 0) sums[0][wave] = m;
    const float least =
        block_bound(top, p.k, heads, &least_at, &count_at);
#pragma unroll
    for (int i = 0; i < W; ++i) m = maximum(m, sums[0][i]);
    if (m == -INFINITY) m = -3.402823466e38f;
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float d = maximum(f[i][e] - m, kFloor), w = __expf(d);
        s += w;
        u += w * d;
      }
    s = group_sum(s);
    u = group_sum(u);
    if (lane == 0) sums[1][wave] = s, sums[2][wave] = u;
    auto index = [&](int at) {
      const int base = (first + tid + at / V * kLanes) * V;
      return (base < A - V ? base : A - V) + at % V;
    };
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!(tops[i] >= least)) continue;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (!(f[i][e] >= least)) continue;
        const int at = atomicAdd(&count_at, 1);
        if (at < kFound) found[at] = key_of(f[i][e], index(i * V + e));
      }
    }
    __syncthreads();
    s = u = 0.f;
#pragma unroll
    for (int i = 0; i < W; ++i) s += sums[1][i], u += sums[2][i];
    if (tid == 0) {
      if (P == 1) {
        const int64_t act = p.actions[row];
        finish_row(p, row, act, taken(x, ok, A, act), m, s, u);
      } else {
        parts.sums[3 * b] = m;
        parts.sums[3 * b + 1] = s;
        parts.sums[3 * b + 2] = u;
      }
    }
    const Top to_row(p, row, m, s);
    auto put = [&](int i, uint64_t key) {
      if (P == 1) {
        to_row.put(i, key);
      } else {
        parts.keys[b * p.k + i] = key;
      }
    };
    const int count = count_at;
    if (count <= kFound) {
      // whatever order they were found in, each goes to its rank
      for (int i = tid; i < count || i < p.k; i += kLanes) {
        const uint64_t mine = i < count ? found[i] : 0;
        const int at = i < count ? rank_of(mine, found, count) : i;
        if (at < p.k) put(at, mine);
      }
    } else {
      // many equal ones: a round an alternative, and it is taken out
      for (int j = 0; j < p.k; ++j) {
        int slot;
        const float best = first_best(f, slot);
        const uint64_t own =
            best > -INFINITY ? key_of(best, index(slot)) : 0;
        const uint64_t key = block_larger(own, waves);
        if (own == key) take_out(f, slot);
        if (tid == 0) put(j, key);
      }
    }
    __syncthreads();  // the next turn writes what this one reads
  }
}

// The k-th largest of n keys, none of them twice but 0; 1 if there are fewer
// than k. Whole blocks, n <= kLanes; `keys` is in LDS and complete.
__device__ __forceinline__ uint64_t kth(const uint64_t* keys, int n, int k,
                                        uint64_t* out) {
  const int tid = threadIdx.x;
  if (tid == 0) *out = 1;
  __syncthreads();
  if (tid < n) {
    const uint64_t mine = keys[tid];
    if (rank_of(mine, keys, n) == k - 1 && mine) *out = mine;
  }
  __syncthreads();
  return *out;
}

// One row's results from its parts'. Of each part's sorted keys the first
// few bound the k-th of all, and what reaches the bound goes to its rank.
constexpr int kMostParts = 64;

__global__ __launch_bounds__(kLanes) void logp_join_kernel(LogpFwd p,
                                                           Parts parts,
                                                           int type) {
  __shared__ uint64_t heads[kLanes], found[kMostParts * 64 + kAhead];
  __shared__ uint64_t bound_at;
  __shared__ int count_at;
  const int tid = threadIdx.x, P = parts.parts, k = p.k;
  for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float* sums = parts.sums + 3 * row * P;
    const int i0 = tid % kWave < P ? tid % kWave : 0;
    Running r{sums[3 * i0], sums[3 * i0 + 1], sums[3 * i0 + 2]};
    if (tid % kWave >= P) r.s = r.u = 0.f;
    r.join_wave();
    if (tid == 0) {
      const int64_t act = p.actions[row];
      const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
      float q;
      if (type == F32) {
        q = taken((const float*)p.logits + row * p.x_stride, ok, p.A, act);
      } else if (type == BF16) {
        q = taken((const bf16*)p.logits + row * p.x_stride, ok, p.A, act);
      } else {
        q = taken((const f16*)p.logits + row * p.x_stride, ok, p.A, act);
      }
      finish_row(p, row, act, q, r.m, r.s, r.u);
      count_at = 0;
    }
    if (k == 0) continue;
    const uint64_t* keys = parts.keys + row * P * k;
    const Top to_row(p, row, r.m, r.s);
    const int each = (k + P - 1) / P, n = P * each;  // < k + P
    if (tid < n) heads[tid] = keys[tid / each * k + tid % each];
    __syncthreads();
    const uint64_t bound = kth(heads, n, k, &bound_at);
    for (int i = tid; i < P * k; i += kLanes) {
      const uint64_t key = keys[i];
      if (key >= bound) found[atomicAdd(&count_at, 1)] = key;
    }
    __syncthreads();
    const int count = count_at;
    for (int i = tid; i < count; i += kLanes) {
      const uint64_t mine = found[i];
      const int rank = rank_of(mine, found, count);
      if (rank < k) to_row.put(rank, mine);
    }
    for (int i = count + tid; i < k; i += kLanes) to_row.put(i, 0);
    __syncthreads();
  }
}

// ---- longer rows, backward: blocks of 256 lanes with U vectors each
constexpr int kBwdVecs = 4;

template <typename T>
__global__ __launch_bounds__(256) void logp_row_bwd_kernel(LogpBwd p,
                                                           int64_t pieces) {
  constexpr int V = kVec<T>, U = kBwdVecs;
  const int A = (int)p.A, n = (A + V - 1) / V;
  for (int64_t b = blockIdx.x; b < p.rows * pieces; b += gridDim.x) {
    const int64_t row = b / pieces;
    const int j = (int)(b - row * pieces) * (256 * U) + threadIdx.x;
    const T* x = (const T*)p.logits + row * p.x_stride;
    const uint8_t* ok = p.mask ? p.mask + row * p.mask_stride : nullptr;
    T* out = (T*)p.dlogits + row * p.A;
    Piece<T> v[U];
#pragma unroll
    for (int i = 0; i < U; ++i)
      if (j + 256 * i < n) v[i].read(x, ok, A, j + 256 * i);
    const Row r = row_of(p, x, ok, row);
#pragma unroll
    for (int i = 0; i < U; ++i) {
      if (j + 256 * i >= n) break;
      float f[V];
      v[i].template values<true>(ok, f);
#pragma unroll
      for (int e = 0; e < V; ++e) f[e] = gradient(r, f[e], v[i].from + e);
      store_row<T>(out, A, v[i].from, f);
    }
  }
}

constexpr int64_t kGrid = 1 << 22;  // blocks at most; more are looped over

// Rows that G lanes hold in registers: G as few as four vectors a lane allow,
// and a wave with 6 or 8.
struct Group {
  int G, N;
};

Group group_of(int64_t A, int V) {
  const int64_t n = (A + V - 1) / V;
  int G = 1;
  while (4 * G < n && G < kWave) G *= 2;
  const int N = (int)((n + G - 1) / G);
  return {G, N <= 4 ? N : (N + 1) / 2 * 2};
}

// Vectors of the longest row that a wave's lanes hold, as many a lane as
// leave registers for three waves or more; longer ones take blocks. 4 forward
// and backward: 8192 x 1000 bf16 takes 6.3 us so, 12.6 in blocks, 8192 x 2048
// 10.4 and 15.2. Forward, 32 bits go to 6: 8192 x 1400 12.4 and 15.5 us (to 8:
// 8192 x 2048 18.3 and 16.3). With alternatives, which a block finds between
// barriers, 16 bits go to 6 and 32 to 8: 13938 x 2780 fp16 with 6 takes 37 and
// 51 us, 8192 x 2048 fp32 with 20 25 and 33 (16 bits to 8: 8192 x 4096 with 20
// 38 and 37).
constexpr int64_t kGroupVecs = 4 * kWave;
constexpr int64_t group_vecs(bool top, int V) {
  return (V == 4 ? top ? 8 : 6 : top ? 6 : 4) * kWave;
}

template <typename T, bool BWD, int G, int N, typename P>
hipError_t group_with(const P& p, hipStream_t s) {
  constexpr int B = 256;
  const int64_t want = (p.rows + B / G - 1) / (B / G);
  const dim3 grid(want < kGrid ? want : kGrid);
  // only what rows of so many vectors come to is built
  if constexpr (BWD) {
    static_assert(G * N <= kGroupVecs);
    return launch(logp_group_bwd_kernel<T, G, N>, grid, dim3(B), 0, s, p);
  } else {
    static_assert(G * N <= group_vecs(true, kVec<T>));
    if (p.k)
      return launch(logp_group_kernel<T, G, N, true>, grid, dim3(B), 0, s, p);
    if constexpr (G * N <= group_vecs(false, kVec<T>))
      return launch(logp_group_kernel<T, G, N, false>, grid, dim3(B), 0, s, p);
    return hipErrorInvalidValue;
  }
}

template <typename T, bool BWD, typename P>
hipError_t group(const P& p, hipStream_t s) {
  const Group g = group_of(p.A, kVec<T>);
  if constexpr (!BWD) {
    if (g.N == 6) return group_with<T, false, 64, 6>(p, s);
    if constexpr (64 * 8 <= group_vecs(true, kVec<T>))
      if (g.N == 8) return group_with<T, false, 64, 8>(p, s);
  }
  switch (g.G * 8 + g.N) {
    case 1 * 8 + 1: return group_with<T, BWD, 1, 1>(p, s);
    case 1 * 8 + 2: return group_with<T, BWD, 1, 2>(p, s);
    case 1 * 8 + 3: return group_with<T, BWD, 1, 3>(p, s);
    case 1 * 8 + 4: return group_with<T, BWD, 1, 4>(p, s);
    case 2 * 8 + 3: return group_with<T, BWD, 2, 3>(p, s);
    case 2 * 8 + 4: return group_with<T, BWD, 2, 4>(p, s);
    case 4 * 8 + 3: return group_with<T, BWD, 4, 3>(p, s);
    case 4 * 8 + 4: return group_with<T, BWD, 4, 4>(p, s);
    case 8 * 8 + 3: return group_with<T, BWD, 8, 3>(p, s);
    case 8 * 8 + 4: return group_with<T, BWD, 8, 4>(p, s);
    case 16 * 8 + 3: return group_with<T, BWD, 16, 3>(p, s);
    case 16 * 8 + 4: return group_with<T, BWD, 16, 4>(p, s);
    case 32 * 8 + 3: return group_with<T, BWD, 32, 3>(p, s);
    case 32 * 8 + 4: return group_with<T, BWD, 32, 4>(p, s);
    case 64 * 8 + 3: return group_with<T, BWD, 64, 3>(p, s);
    case 64 * 8 + 4: return group_with<T, BWD, 64, 4>(p, s);
  }
  return hipErrorInvalidValue;
}

// Parts of a row: of 512 vectors at least, while there are fewer blocks than
// keep the chip busy (97 x 100000 bf16: 10 us in parts, 20 whole; 512 x 32768:
// 13 and 10). With alternatives too: cut into as many parts as registers hold,
// 4096 x 32768 bf16 with 8 took 131 us, walked whole 71. Rows of up to kWhole
// vectors are not cut, which would take a second launch: 16 x 16384 bf16 with
// 10 takes 8.3 us whole and 9.8 in parts, 16 x 24000 10.8 and 10.6.
constexpr int64_t kWhole = 2048;
constexpr int64_t kBlocks = 512;

int parts_of(int64_t rows, int64_t A, int V) {
  const int64_t n = (A + V - 1) / V;
  if (n <= kWhole || rows <= 0) return 1;
  int64_t p = (kBlocks + rows - 1) / rows;
  p = p < n / 512 ? p : n / 512;
  p = p < kMostParts ? p : kMostParts;
  return p < 1 ? 1 : (int)p;
}

template <typename T>
hipError_t fwd(const LogpFwd& p, void* scratch, int type, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  const int64_t n = (p.A + kVec<T> - 1) / kVec<T>;
  if (n <= group_vecs(p.k, kVec<T>)) return group<T, false>(p, s);
  const int P = parts_of(p.rows, p.A, kVec<T>);
  const int64_t blocks = p.rows * P;
  const Parts parts = {(float*)((uint64_t*)scratch + blocks * p.k),
                       (uint64_t*)scratch, P};
  const dim3 grid(blocks < kGrid ? blocks : kGrid);
  const dim3 lanes(kLanes);
  hipError_t e;
  if (p.k == 0) {
    e = launch(logp_row_kernel<T, false>, grid, lanes, 0, s, p, parts);
  } else if (n <= 2 * (int64_t)kLanes * P) {
    e = launch(logp_part_kernel<T, 2>, grid, lanes, 0, s, p, parts);
  } else if (n <= 3 * (int64_t)kLanes * P) {
    e = launch(logp_part_kernel<T, 3>, grid, lanes, 0, s, p, parts);
  } else if (n <= 4 * (int64_t)kLanes * P) {
    e = launch(logp_part_kernel<T, 4>, grid, lanes, 0, s, p, parts);
  } else {
    e = launch(logp_row_kernel<T, true>, grid, lanes, 0, s, p, parts);
  }
  if (e != hipSuccess || P == 1) return e;
  return launch(logp_join_kernel, dim3(p.rows < kGrid ? p.rows : kGrid),
                dim3(kLanes), 0, s, p, parts, type);
}

template <typename T>
hipError_t bwd(const LogpBwd& p, hipStream_t s) {
  if (p.rows == 0) return hipSuccess;
  const int64_t n = (p.A + kVec<T> - 1) / kVec<T>;
  if (n <= kGroupVecs) return group<T, true>(p, s);
  const int64_t pieces = (n + 256 * kBwdVecs - 1) / (256 * kBwdVecs);
  const int64_t grid = p.rows * pieces;
  return launch(logp_row_bwd_kernel<T>, dim3(grid < kGrid ? grid : kGrid),
                dim3(256), 0, s, p, pieces);
}

}  // namespace

// Bytes of scratch that the forward call needs.
extern "C" int64_t rlsched_logp_scratch(int64_t rows, int64_t A, int k,
                                        int type) {
  const int P = parts_of(rows, A, type == F32 ? 4 : 8);
  return P == 1 ? 0 : rows * P * (8 * (int64_t)k + 12);
}

extern "C" int rlsched_logp_fwd(int device, void* stream, const void* logits,
                                const int64_t* actions, const uint8_t* mask,
                                float* logp, float* entropy, float* stats,
                                float* top_logp, int64_t* top_index,
                                void* scratch, int64_t rows, int64_t A,
                                int64_t x_stride, int64_t mask_stride, int k,
                                int type) {
  OnDevice on(device);
  if (on.err != hipSuccess) return on.err;
  const LogpFwd p = {logits, actions,  mask,      logp, entropy,  stats,
                     top_logp, top_index, rows, A, x_stride, mask_stride, k};
  const hipStream_t s = (hipStream_t)stream;
  if (type == F32) return fwd<float>(p, scratch, type, s);
  if (type == BF16) return fwd<bf16>(p, scratch, type, s);
  if (type == F16) return fwd<f16>(p, scratch, type, s);
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
