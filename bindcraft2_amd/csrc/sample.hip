// Drawing a class from each row of logits x[V] by a given uniform number u.
// With m = max x and the classes ranked by x, ties to the lowest index:
//
//   e_j   = exp((x_j - m) / temperature)
//   top-k  keeps the first k; top-p those whose forerunners hold less than
//   top_p of what top-k kept; min-p those with e_j >= min_p; the first stays
//   index = the first class, by index, at which the running sum of the kept
//           e_j exceeds u times their whole sum
//   logp  = log of its share of that sum
//
// The class hangs on which side of a border a sum lies, so nothing here may
// depend on the order of a sum: e_j is held as a whole number of 2^-S (its
// exponential in 64 bits), 2^S as large as a row's sum in 64 bits allows (2^44
// for 131 k classes), and sums of those are exact in any order.  An e_j below
// half of that counts as zero and can be left out of everything.
//
// Rows of up to 64 classes take a lane a class, up to 1024 a wave a row, with the
// row in registers; longer ones a workgroup a row.  Read once they are bound by
// memory (1021 rows of 50 k f32: 40 us at the rate of a copy, 62 taken), so their one pass leaves the
// maxima of short runs: what a cut can keep lies in the runs whose maxima reach
// it, and those alone are read again.  The few classes of them (1024 at most) are put
// in buckets by value and by index, compared with their own buckets, and drawn
// from by sums in both orders.
//
// Where more stay, a rank or a share of the mass becomes a threshold on (x, index)
// in one pass that counts the classes by their distance to the maximum, in 2048
// steps, and an exact ranking of the few in the step that the border falls into;
// where ties or odd distributions leave many there, further passes divide that
// step.  Exponentials in 64 bits cost twenty instructions and are made only of
// classes still in play; the passes that need them of all classes are bound by
// them (64 rows of 131 k bfloat16: nothing cut 86 us, top-p of 0.9 191, top-k of
// 50 19).
#include "sample.h"

#include "common.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace bc2n {

namespace {

typedef unsigned long long u64;

constexpr int BINS = 2048;
constexpr int LIST = 256;  // classes ranked one against all
constexpr float NEG_INF = -__builtin_inff();
constexpr float MAX_F32 = 3.402823466e38f;

// bits of a mass: V of them fit 62 bits
__host__ __device__ constexpr int mass_bits(int V) {
  int b = 0;
  while ((int64_t(1) << b) < V) ++b;
  return 61 - b < 48 ? 61 - b : 48;
}

// 2^t for t <= 0 in units of 2^-S, in whole ones.  The series of e^(f log 2) for
// |f| <= 1/2 ends at 4e-16.
__device__ __forceinline__ u64 mass_of(double t, int S) {
  if (!(t > -(double)(S + 2))) return 0;
  const double n = rint(t), f = (t - n) * 0.69314718055994530942;
  double p = 1.0 / 479001600.0;
  p = fma(p, f, 1.0 / 39916800.0);
  p = fma(p, f, 1.0 / 3628800.0);
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return (u64)(ldexp(p, (int)n + S) + 0.5);
}

// Larger for larger x; -0 as 0.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
// Larger for a better rank; no two classes have the same.
__device__ __forceinline__ u64 rank_key(float x, int j) {
  return (u64)key_of(x) << 32 | (uint32_t)(~j);
}

struct Settings {
  double inv;    // log2(e) / temperature
  int64_t k;     // 0: all
  double p;
  double floor;  // log2 of min-p, at most 0
  float u;
  bool greedy, bad;
};
__device__ __forceinline__ Settings settings_of(const Sample& a, int64_t r) {
  Settings s;
  const double t = a.temperature.row ? (double)a.temperature.row[r] : a.temperature.v;
  s.k = a.top_k_row ? (int64_t)a.top_k_row[r] : a.top_k;
  if (s.k < 1 || s.k >= a.V) s.k = 0;
  s.p = a.top_p.row ? (double)a.top_p.row[r] : a.top_p.v;
  const double floor = a.min_p.row ? (double)a.min_p.row[r] : a.min_p.v;
  s.floor = floor > 0 ? log2(fmin(floor, 1.0)) : (double)NEG_INF;
  s.u = a.u[r];
  s.bad = !(s.u == s.u) || !(fabs(t) < (double)-NEG_INF);
  s.greedy = !(t > 0) || s.k == 1;
  s.inv = fmin(1.4426950408889634 / t, 1e300);
  return s;
}
// A value a little below the last with a mass beside a maximum of m: in 64 bits, so
// that at temperatures about 1e37 the distance may pass f32's numbers, and no
// lower than the lowest of those.
__device__ __forceinline__ float last_with_mass(float m, double inv, int S) {
  return (float)fmax((double)m - (S + 2) / inv * 1.0001, -(double)MAX_F32);
}
// the least sum of forerunners that ends top-p: p of the mass, at least 1
__device__ __forceinline__ u64 share_of(double p, u64 mass) {
  const double x = ceil(fmax(p, 0.0) * (double)mass);
  return x < 1.0 ? 1 : x >= (double)mass ? mass : (u64)x;
}
__device__ __forceinline__ u64 target_of(float u, u64 mass) {
  const double x = fmax((double)u, 0.0) * (double)mass;
  return x >= (double)mass ? mass - 1 : min((u64)x, mass - 1);
}
__device__ __forceinline__ void write(const Sample& a, int64_t r, int j, float logp) {
  a.index[r] = j;
  if (a.logp) a.logp[r] = logp;
}
// log of e^((x - m) / t) 2^S / mass; d = (x - m) inv in log 2
__device__ __forceinline__ float log_share(double d, u64 mass, int S) {
  return (float)((d - (log2((double)mass) - (double)S)) * 0.69314718055994530942);
}

// DPP moves: what a fold or a scan waits for is its latency, a tenth of a shuffle's.
constexpr int ROW_SHR = 0x110, ROW_BCAST15 = 0x142, ROW_BCAST31 = 0x143;
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 dpp64(u64 v, u64 none) {
  const uint32_t lo = __builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp((int)(none >> 32), (int)(v >> 32), CTRL, ROWS, 0xF, false);
  return (u64)hi << 32 | lo;
}
struct Sum {
  static constexpr u64 NONE = 0;
  __device__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
  static constexpr u64 NONE = 0;
  __device__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};
struct Min {
  static constexpr u64 NONE = ~u64(0);
  __device__ u64 operator()(u64 a, u64 b) const { return a < b ? a : b; }
};
// of the lanes up to this one
template <class F>
__device__ __forceinline__ u64 wave_scan(u64 v, F f) {
  v = f(v, dpp64<ROW_SHR + 1, 0xF>(v, F::NONE));
  v = f(v, dpp64<ROW_SHR + 2, 0xF>(v, F::NONE));
  v = f(v, dpp64<ROW_SHR + 4, 0xF>(v, F::NONE));
  v = f(v, dpp64<ROW_SHR + 8, 0xF>(v, F::NONE));
  v = f(v, dpp64<ROW_BCAST15, 0xA>(v, F::NONE));
  return f(v, dpp64<ROW_BCAST31, 0xC>(v, F::NONE));
}
__device__ __forceinline__ u64 lane_value(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
template <class F>
__device__ __forceinline__ u64 wave_fold(u64 v, F f) {
  return lane_value(wave_scan(v, f), 63);
}
// ---------------------------------------------------------------------------
// Rows of at most W classes: a class a lane, W lanes a row.  Ranks and sums of
// forerunners by comparing each class with all.
template <class T, int W>
__global__ __launch_bounds__(256) void sample_few_kernel(Sample a) {
  const int lane = threadIdx.x & (W - 1);
  const int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
  if (r >= a.rows) return;  // whole groups
  const int S = mass_bits(a.V);
  const Settings s = settings_of(a, r);
  const float x = lane < a.V ? (float)reinterpret_cast<const T*>(a.x)[r * a.ld + lane] : NEG_INF;
  const u64 c = rank_key(x, lane);
  const float m = group_max<W>(x);
  const float nan = group_max<W>(x != x || x == -NEG_INF ? 1.f : 0.f);
  if (nan != 0.f || m == NEG_INF || s.bad) {
    if (lane == 0) write(a, r, -1, __builtin_nanf(""));
    return;
  }
  const double d = ((double)x - (double)m) * s.inv;
  u64 w = s.greedy ? 0 : mass_of(d, S);
  auto sum = [&](u64 v) {
#pragma unroll
    for (int i = 1; i < W; i *= 2) v += __shfl_xor(v, i, W);
    return v;
  };
  int rank = 0;
  if (s.k || s.greedy) {
    for (int j = 0; j < a.V; ++j) rank += __shfl(c, j, W) > c;
    if (s.greedy) {
      if (rank == 0) write(a, r, lane, 0.f);
      return;
    }
    if (rank >= s.k) w = 0;
  }
  if (s.p < 1.0) {
    const u64 end = share_of(s.p, sum(w));
    u64 before = 0;
    for (int j = 0; j < a.V; ++j) {
      const u64 cj = __shfl(c, j, W), wj = __shfl(w, j, W);
      before += cj > c ? wj : 0;
    }
    if (before >= end) w = 0;
  }
  if (d < s.floor) w = 0;
  u64 run = w;
#pragma unroll
  for (int i = 1; i < W; i *= 2) {
    const u64 v = __shfl_up(run, i, W);
    if (lane >= i) run += v;
  }
  const u64 mass = __shfl(run, W - 1, W), t = target_of(s.u, mass);
  if (w && run > t && run - w <= t) write(a, r, lane, log_share(d, mass, S));
}

// ---------------------------------------------------------------------------
// Rows of at most 64 R classes: a wave a row, R consecutive classes a lane in its
// registers.  A cut is a threshold on x found by halving: the sum of what is above
// a value, all lanes', against the cut's end, until one class is left between.
template <class T, int R>
struct WaveRow {
  float x[R];
  uint32_t key[R];  // 0: not in play
  u64 w[R];
  int lane, j0;

  template <bool MASS>
  __device__ __forceinline__ u64 above(uint32_t v) const {
    if constexpr (MASS) {
      u64 sum = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) sum += key[i] > v ? w[i] : 0;
      return wave_fold(sum, Sum());
    } else {
      int n = 0;
#pragma unroll
      for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] > v));
      return (u64)n;
    }
  }
  __device__ __forceinline__ int between(uint32_t lo, uint32_t hi) const {  // in (lo, hi]
    int n = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) n += __popcll(__ballot(key[i] > lo && key[i] <= hi));
    return n;
  }
  // Takes out of play the classes whose forerunners weigh `end` or more, by number
  // or (MASS) by mass; low: a value below all that count.
  template <bool MASS>
  __device__ __forceinline__ void cut(u64 end, float m, float low) {
    // above hi all stay, up to lo none
    uint32_t hi = key_of(m), lo = key_of(low) - 1;
    if (above<MASS>(lo) <= (MASS ? end - 1 : end)) lo = 0;  // all stay, the last in any case
    float a = low, b = m;
    for (int turn = 0; lo && hi - lo > 1; ++turn) {
      // halves of the values first, which logits are spread over, then of the keys
      uint32_t mid = lo + (hi - lo) / 2;
      if (turn < 16) {
        const uint32_t v = key_of(0.5f * a + 0.5f * b);
        if (v > lo && v < hi) mid = v;
      }
      const bool stays = above<MASS>(mid) < end;
      if (stays) hi = mid;
      else lo = mid;
      const uint32_t bits = mid & 0x80000000u ? mid & 0x7fffffffu : ~mid;
      (stays ? b : a) = __builtin_bit_cast(float, bits);
      if (between(lo, hi) <= 1) {
        hi = lo;  // one class, whose forerunners are those above: it stays
        break;
      }
    }
    if (!lo) return;
    if (hi == lo) {
#pragma unroll
      for (int i = 0; i < R; ++i)
        if (key[i] <= lo) key[i] = 0;
      return;
    }
    // classes of one value, hi: the first of them by index
    const u64 before = above<MASS>(hi);
    int mine = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) mine += key[i] == hi;
    u64 rank = wave_scan((u64)mine, Sum()) - mine;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const bool tie = key[i] == hi;
      if (key[i] < hi || (tie && before + rank * (MASS ? w[i] : 1) >= end)) key[i] = 0;
      rank += tie;
    }
  }
};

template <class T, int R>
__global__ __launch_bounds__(256) void sample_wave_kernel(Sample a) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const int S = mass_bits(a.V);
  WaveRow<T, R> row;
  row.lane = threadIdx.x & 63;
  row.j0 = row.lane * R;
  const T* x = reinterpret_cast<const T*>(a.x) + r * a.ld;
#pragma unroll
  for (int i = 0; i < R; ++i) row.x[i] = NEG_INF;
  if (row.j0 + R <= a.V) {
    constexpr int N = R < 16 / (int)sizeof(T) ? R : 16 / (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < R; i += N) Few<T, N>::template load<false>(x + row.j0 + i, row.x + i);
  } else {
#pragma unroll
    for (int i = 0; i < R; ++i)
      if (row.j0 + i < a.V) row.x[i] = (float)x[row.j0 + i];
  }
  const Settings s = settings_of(a, r);
  float m = NEG_INF;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    nan |= row.x[i] != row.x[i];
    m = fmaxf(m, row.x[i]);
  }
  m = group_max<64>(m);
  if (__any(nan) || m == -NEG_INF || m == NEG_INF || s.bad) {
    if (row.lane == 0) write(a, r, -1, __builtin_nanf(""));
    return;
  }
  if (s.greedy) {
    int first = 0x7fffffff;
#pragma unroll
    for (int i = R - 1; i >= 0; --i)
      if (row.x[i] == m) first = row.j0 + i;
    first = (int)wave_fold((u64)first, Min());
    if (row.lane == 0) write(a, r, first, 0.f);
    return;
  }
  const float low = last_with_mass(m, s.inv, S);
  u64 mine = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const bool counts = row.x[i] >= low;
    const double t = ((double)row.x[i] - (double)m) * s.inv;
    row.key[i] = counts ? key_of(row.x[i]) : 0;
    row.w[i] = counts ? mass_of(t, S) : 0;
  }
  if (s.k) row.template cut<false>((u64)s.k, m, low);
  if (s.p < 1.0) {
    mine = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) mine += row.key[i] ? row.w[i] : 0;
    row.template cut<true>(share_of(s.p, wave_fold(mine, Sum())), m, low);
  }
  mine = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const double t = ((double)row.x[i] - (double)m) * s.inv;
    if (!row.key[i] || t < s.floor) row.w[i] = 0;
    mine += row.w[i];
  }
  const u64 run = wave_scan(mine, Sum()), mass = lane_value(run, 63), target = target_of(s.u, mass);
  u64 before = run - mine;
  if (before > target || run <= target) return;
#pragma unroll
  for (int i = 0; i < R; ++i) {  // one lane's
    if (before <= target && before + row.w[i] > target)
      write(a, r, row.j0 + i, log_share(((double)row.x[i] - (double)m) * s.inv, mass, S));
    before += row.w[i];
  }
}

// ---------------------------------------------------------------------------
// A workgroup a row.
constexpr int CANDIDATES = 1024;
constexpr int RUNS = 2048;  // runs of a row's vectors whose maxima are kept
template <int NT>
struct Shared {
  u64 mass[BINS];
  uint32_t count[BINS];
  union {
    struct {
      u64 list_key[LIST];
      u64 list_mass[LIST];
    };
    uint32_t live_runs[CANDIDATES];  // beside the steps' counts, which a cut of the row takes up
  };
  union {
    struct {
      float x[CANDIDATES];
      int j[CANDIDATES];
    };
    float run_max[RUNS];  // until the candidates are collected
  };
  u64 wave_a[NT / 64], wave_b[NT / 64];
  u64 out[4];
  uint32_t n, found;
};

// The larger of two (of a NaN and a number either), in one instruction: fmaxf takes
// one more an operand, which signalling NaNs need.
__device__ __forceinline__ float larger(float a, float b) {
  return __builtin_amdgcn_fmed3f(a, b, __builtin_inff());
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float row_below(float v) {
  const int b = __builtin_bit_cast(int, v);
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(b, b, CTRL, ROWS, 0xF, false));
}

// over the workgroup, the result in every thread
template <int NT, class F>
__device__ __forceinline__ u64 block_fold(u64 v, u64* waves, F f) {
  v = wave_fold(v, f);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = v;
  __syncthreads();
  v = waves[0];
#pragma unroll 4
  for (int i = 1; i < NT / 64; ++i) v = f(v, waves[i]);
  return lane_value(v, 0);  // in scalar registers
}
template <int NT>
__device__ __forceinline__ u64 block_scan(u64 v, u64* waves) {  // exclusive
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const u64 run = wave_scan(v, Sum());
  __syncthreads();
  if (lane == 63) waves[wave] = run;
  __syncthreads();
  u64 before = 0;
#pragma unroll 4
  for (int i = 0; i < NT / 64; ++i) before += i < wave ? waves[i] : 0;
  return before + run - v;
}

// A row, read at each pass: out of the caches after the first.  (Held in registers
// it needs so many for the vectors' places that they spill: 64 rows of 131 k
// bfloat16 67 us against 25.)  Passes of a few instructions a class take vectors;
// those with exponentials take a class at a time, their loads are the least of it.
template <class T, int NT>
struct RowOf {
  static constexpr int E = Vec<T>::N;
  typedef T Type;
  const T* x;
  int V;

  // f(x, index) of a thread's classes
  template <class F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int j = threadIdx.x; j < V; j += NT) f((float)x[j], j);
  }
  __device__ __forceinline__ int count() const { return (V + E - 1) / E; }
  // Vector q's place.  One that would pass the row's end is read ending there, and
  // its classes that the one before has are -infinity.
  __device__ __forceinline__ int first(int q) const { return min(q * E, V - E); }
  __device__ __forceinline__ void values(u32x4 raw, int q, float (&v)[E]) const {
    Vec<T>::unpack(raw, v);
    const int twice = q * E - first(q);
    if (twice) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = e < twice ? NEG_INF : v[e];
    }
  }
  // f(classes' values, number, whether it may be past the last) of a thread's vectors,
  // lanes next to each other having vectors next to each other; past the last all
  // of them are -infinity.
  template <class F>
  __device__ __forceinline__ void vectors(F f) const {
    constexpr int AT_ONCE = NT == 1024 ? 8 : 4;
    const int n = (count() + NT - 1) / NT;
    auto one = [&](u32x4 raw, int q, auto end) __attribute__((always_inline)) {
      float v[E];
      if (decltype(end)::value) values(raw, q, v);
      else Vec<T>::unpack(raw, v);
      f(v, q, end);
    };
    int i = 0;
    for (; i + AT_ONCE < n; i += AT_ONCE) {
      u32x4 raw[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) raw[u] = Vec<T>::load(x + (int64_t)((i + u) * NT + (int)threadIdx.x) * E);
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) one(raw[u], (i + u) * NT + (int)threadIdx.x, std::false_type());
    }
    u32x4 raw[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (i + u < n) raw[u] = Vec<T>::load(x + first((i + u) * NT + (int)threadIdx.x));
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u)
      if (i + u < n) one(raw[u], (i + u) * NT + (int)threadIdx.x, std::true_type());
  }
};
template <int NT>
struct Drawer {
  Shared<NT>& sh;
  float m, last, range, steps;  // maximum, lowest value with a mass, their distance, steps a distance
  double inv;
  int S;

  __device__ __forceinline__ double distance(float x) const { return ((double)x - (double)m) * inv; }
  __device__ __forceinline__ u64 mass(float x) const { return mass_of(distance(x), S); }
  // a class that can have a mass
  __device__ __forceinline__ bool counts(float x) const { return x >= last; }
  __device__ __forceinline__ int step_of(float x) const {
    return (int)fminf((m - x) * steps, (float)(BINS - 1));
  }
  __device__ __forceinline__ void clear(bool masses) {
    for (int i = threadIdx.x; i < BINS; i += NT) {
      sh.count[i] = 0;
      if (masses) sh.mass[i] = 0;
    }
    if (threadIdx.x == 0) sh.n = 0;
    __syncthreads();
  }
  // The last filled step whose forerunners, `before` and the steps before it,
  // weigh less than the end; `before` becomes what those weigh.
  template <bool MASS>
  __device__ __forceinline__ int last_step(u64 end, u64& before) {
    constexpr int PER = BINS / NT;
    u64 w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = threadIdx.x * PER + i;
      w += MASS ? sh.mass[b] : sh.count[b];
    }
    u64 run = before + block_scan<NT>(w, sh.wave_a);
    u64 best = 0, best_run = 0;  // step + 1
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int b = threadIdx.x * PER + i;
      if (sh.count[b] && run < end) {
        best = b + 1;
        best_run = run;
      }
      run += MASS ? sh.mass[b] : sh.count[b];
    }
    const u64 top = block_fold<NT>(best, sh.wave_b, Max());
    if (best == top && best) sh.out[0] = best_run;
    __syncthreads();
    before = sh.out[0];
    return (int)top - 1;
  }

  // Counts and (masses) masses of the classes of `from` in steps of distance, those
  // of rank keys >= least.
  template <class S_>
  __device__ __forceinline__ void fill(const S_& from, bool masses, u64 least) {
    clear(masses);
    from.each([&](float x, int j) {
      if (!counts(x) || rank_key(x, j) < least) return;
      const int b = step_of(x);
      atomicAdd(&sh.count[b], 1u);
      if (masses) atomicAdd(&sh.mass[b], mass(x));
    });
    __syncthreads();
  }
  // The weight of all steps.
  __device__ __forceinline__ u64 filled_mass(int steps_) {
    u64 w = 0;
    for (int b = threadIdx.x; b < steps_; b += NT) w += sh.mass[b];
    return block_fold<NT>(w, sh.wave_b, Sum());
  }

  // The rank key of the last class of `from` whose forerunners, among those of
  // rank keys >= least, weigh less than `end`: by number, or (MASS) by mass.  The
  // steps have to be filled, with those at least.  False is left in `intact` where
  // they were filled anew; else, with `tell` and the steps' masses filled, `kept`
  // gets the mass of the classes up to that one.
  template <bool MASS, class S_>
  __device__ __forceinline__ u64 last_before(const S_& from, u64 end, u64 least, bool& intact, bool tell, u64& kept) {
    u64 lo = 0, hi = ~u64(0), before = 0;
    int shift = -1;  // -1: steps of distance
    for (;;) {
      auto bin_of = [&](float x, u64 c) { return shift < 0 ? step_of(x) : (int)((hi - c) >> shift); };
      const int bin = last_step<MASS>(end, before);
      if (threadIdx.x == 0) sh.n = 0;
      const uint32_t in_bin = sh.count[bin];
      __syncthreads();
      if (in_bin <= LIST) {
        from.each([&](float x, int j) {
          if (!counts(x)) return;
          const u64 c = rank_key(x, j);
          if (c < least || c < lo || c > hi || bin_of(x, c) != bin) return;
          const uint32_t at = atomicAdd(&sh.n, 1u);
          sh.list_key[at] = c;
          sh.list_mass[at] = MASS || tell ? mass(x) : 1;
        });
        __syncthreads();
        const int n = (int)sh.n;
        u64 key = ~u64(0);
        for (int i = threadIdx.x; i < n; i += NT) {
          const u64 c = sh.list_key[i];
          u64 f = before;
          for (int k = 0; k < n; ++k) f += sh.list_key[k] > c ? (MASS ? sh.list_mass[k] : 1) : 0;
          if (f < end) key = min(key, c);
        }
        key = block_fold<NT>(key, sh.wave_a, Min());
        if (tell && intact) {
          u64 w = 0;
          for (int i = threadIdx.x; i < n; i += NT) w += sh.list_key[i] >= key ? sh.list_mass[i] : 0;
          kept = filled_mass(bin) + block_fold<NT>(w, sh.wave_a, Sum());
        }
        return key;
      }
      // too many: their range of rank keys in 2048 parts
      u64 a = ~u64(0), b = 0;
      from.each([&](float x, int j) {
        if (!counts(x)) return;
        const u64 c = rank_key(x, j);
        if (c < least || c < lo || c > hi || bin_of(x, c) != bin) return;
        a = min(a, c);
        b = max(b, c);
      });
      a = block_fold<NT>(a, sh.wave_a, Min());
      b = block_fold<NT>(b, sh.wave_b, Max());
      lo = a;
      hi = b;
      shift = 0;
      while (((hi - lo) >> shift) >= BINS) ++shift;
      intact = false;
      clear(MASS);
      from.each([&](float x, int j) {
        if (!counts(x)) return;
        const u64 c = rank_key(x, j);
        if (c < least || c < lo || c > hi) return;
        const int b_ = bin_of(x, c);
        atomicAdd(&sh.count[b_], 1u);
        if (MASS) atomicAdd(&sh.mass[b_], mass(x));
      });
      __syncthreads();
    }
  }

  // The classes that are at least `low` to LDS, from the runs of 2^shift vectors
  // that have one; how many there are, more than CANDIDATES where not all fit.
  template <class R>
  __device__ __forceinline__ int collect(const R& row, float low, int runs, int shift) {
    if (threadIdx.x == 0) sh.n = sh.found = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < runs; i += NT) {
      if (sh.run_max[i] >= low) {
        const uint32_t at = atomicAdd(&sh.n, 1u);
        if (at < CANDIDATES) sh.live_runs[at] = i;
      }
    }
    __syncthreads();
    const int live = (int)sh.n, n = min(live, CANDIDATES) << shift;
    __syncthreads();  // what follows may clear it
    if (live > CANDIDATES) return live;
    constexpr int AT_ONCE = 4;
    for (int i0 = threadIdx.x; i0 < n; i0 += AT_ONCE * NT) {
      u32x4 raw[AT_ONCE];
      int q[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = min(i0 + u * NT, n - 1);
        q[u] = ((int)sh.live_runs[i >> shift] << shift) + (i & ((1 << shift) - 1));
        raw[u] = Vec<typename R::Type>::load(row.x + row.first(q[u]));
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        if (i0 + u * NT >= n || q[u] >= row.count()) continue;
        float v[R::E];
        row.values(raw[u], q[u], v);
#pragma unroll
        for (int e = 0; e < R::E; ++e) {
          if (v[e] >= low) {
            const uint32_t at = atomicAdd(&sh.found, 1u);
            if (at < CANDIDATES) {
              sh.x[at] = v[e];
              sh.j[at] = row.first(q[u]) + e;
            }
          }
        }
      }
    }
    __syncthreads();
    return (int)sh.found;
  }
  // a value that no class of the steps up to `step` is below
  __device__ __forceinline__ float lowest(int step) const {
    if (step >= BINS - 1) return last;
    const float d = (float)(step + 1) / steps;  // of the next step's first, but for rounding
    return fmaxf(m - d * 1.0001f - 1e-6f * fabsf(m), last);
  }

  // The same as cut and draw, of at most 64 candidates by one wave: ranks by value and
  // by index from comparing each with all, sums of forerunners by scans in
  // their orders.
  template <class ST>
  __device__ __forceinline__ void draw_few(const Sample& a, int64_t r, int n, const ST& s, u64 whole) {
    const int lane = threadIdx.x;
    const float x = lane < n ? sh.x[lane] : NEG_INF;
    const int j = lane < n ? sh.j[lane] : 0x7fffffff;
    const uint32_t key = lane < n ? key_of(x) : 0;
    const double t = distance(x);
    u64 w = lane < n && counts(x) ? mass_of(t, S) : 0;
    int rank = 0, place = 0;
#pragma unroll 4
    for (int i = 0; i < n; ++i) {
      const uint32_t k = (uint32_t)__builtin_amdgcn_readlane((int)key, i);
      const int before = __builtin_amdgcn_readlane(j, i) < j;
      place += before;
      rank += k > key || (k == key && before);
    }
    if (s.k && rank >= s.k) w = 0;
    auto forerunners = [&](u64 v, int at) {  // by the order that `at` numbers
      if (lane < n) sh.list_mass[at] = v;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      const u64 mine = lane < n ? sh.list_mass[lane] : 0, run = wave_scan(mine, Sum()) - mine;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (lane < n) sh.list_key[lane] = run;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      return lane < n ? sh.list_key[at] : 0;
    };
    if (s.p < 1.0) {
      if (s.k) whole = wave_fold(w, Sum());
      if (forerunners(w, rank) >= share_of(s.p, whole)) w = 0;
    }
    if (t < s.floor) w = 0;
    const u64 mass = wave_fold(w, Sum()), target = target_of(s.u, mass), before = forerunners(w, place);
    if (w && before <= target && before + w > target) write(a, r, j, log_share(t, mass, S));
  }

  // The same of up to CANDIDATES by the workgroup: in buckets by distance (least: the
  // candidates' least value) and in buckets by index, and only those of its own are
  // compared with a class.
  template <class ST>
  __device__ __forceinline__ void draw_some(const Sample& a, int64_t r, int n, float least, const ST& s, u64 whole) {
    constexpr int U = CANDIDATES / NT, BUCKETS = 256, PER = BUCKETS / 64;
    const int t = threadIdx.x, lane = t & 63;
    int shift = 0;
    while ((a.V - 1) >> shift >= BUCKETS) ++shift;
    const float f = fminf((BUCKETS - 1) / fminf(m - least, range), 3e38f);
    auto bucket = [&](float x) { return (int)fminf((m - x) * f, (float)(BUCKETS - 1)); };
    uint32_t *count = sh.count, *start = sh.count + 2 * BUCKETS;  // by value, then by index
    for (int i = t; i < 2 * BUCKETS; i += NT) count[i] = 0;
    __syncthreads();
    float x[U];
    int j[U], slot[U], rank[U], place[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = t + u * NT;
      x[u] = c < n ? sh.x[c] : NEG_INF;
      j[u] = c < n ? sh.j[c] : 0;
      if (c < n)
        slot[u] = (int)(atomicAdd(&count[bucket(x[u])], 1u) |
                        atomicAdd(&count[BUCKETS + (j[u] >> shift)], 1u) << 16);
    }
    __syncthreads();
    if (t < 128) {  // a wave for each
      const uint32_t* from = count + (t >> 6) * BUCKETS + lane * PER;
      uint32_t own = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) own += from[i];
      uint32_t run = (uint32_t)wave_scan((u64)own, Sum()) - own;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        start[(t >> 6) * BUCKETS + lane * PER + i] = run;
        run += from[i];
      }
    }
    __syncthreads();
    float* by_value = reinterpret_cast<float*>(sh.mass);  // values, and their indexes
    int* index_of = reinterpret_cast<int*>(by_value + CANDIDATES);
    int* by_index = index_of + CANDIDATES;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u * NT >= n) continue;
      const int at = (int)start[bucket(x[u])] + (slot[u] & 0xffff);
      by_value[at] = x[u];
      index_of[at] = j[u];
      by_index[start[BUCKETS + (j[u] >> shift)] + (slot[u] >> 16)] = j[u];
    }
    __syncthreads();
    u64 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      w[u] = 0;
      rank[u] = place[u] = 0;
      if (t + u * NT >= n) continue;
      int b = bucket(x[u]), i = (int)start[b], end = i + (int)count[b];
      rank[u] = i;
      for (; i < end; ++i) {
        const float y = by_value[i];
        rank[u] += y > x[u] || (y == x[u] && index_of[i] < j[u]);
      }
      b = BUCKETS + (j[u] >> shift);
      i = (int)start[b];
      end = i + (int)count[b];
      place[u] = i;
      for (; i < end; ++i) place[u] += by_index[i] < j[u];
      if (counts(x[u]) && !(s.k && rank[u] >= s.k)) w[u] = mass(x[u]);
    }
    // what the forerunners weigh, in the order that `at` numbers
    auto forerunners = [&](const int (&at)[U], u64 (&v)[U]) {
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (t + u * NT < n) sh.mass[at[u]] = w[u];
      __syncthreads();
      u64 own = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) own += t * U + u < n ? sh.mass[t * U + u] : 0;
      u64 run = block_scan<NT>(own, sh.wave_a);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (t * U + u >= n) continue;
        sh.mass[CANDIDATES + t * U + u] = run;
        run += sh.mass[t * U + u];
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = t + u * NT < n ? sh.mass[CANDIDATES + at[u]] : 0;
    };
    auto all = [&] {
      u64 sum = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) sum += w[u];
      return block_fold<NT>(sum, sh.wave_b, Sum());
    };
    u64 before[U];
    if (s.p < 1.0) {
      if (s.k) whole = all();
      const u64 end = share_of(s.p, whole);
      forerunners(rank, before);
#pragma unroll
      for (int u = 0; u < U; ++u) w[u] = before[u] >= end ? 0 : w[u];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = distance(x[u]) < s.floor ? 0 : w[u];
    const u64 sum = all(), target = target_of(s.u, sum);
    forerunners(place, before);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (w[u] && before[u] <= target && before[u] + w[u] > target)
        write(a, r, j[u], log_share(distance(x[u]), sum, S));
  }
};

template <class T, int NT>
__global__ __launch_bounds__(NT) void sample_row_kernel(Sample a) {
  __shared__ Shared<NT> sh;
  constexpr int WAVES = NT / 64;
  const int64_t r = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  typedef RowOf<T, NT> R;
  const R row{reinterpret_cast<const T*>(a.x) + r * a.ld, a.V};
  const Settings s = settings_of(a, r);
  // Maxima of runs of 2^shift vectors, as short as there is room for (up to 8, and
  // from 64 on): later passes over few classes read their runs alone.
  int shift = 0;
  while (((row.count() - 1) >> shift) >= RUNS) shift += shift == 3 ? 3 : 1;
  const int runs = ((row.count() - 1) >> shift) + 1;
  float hi = NEG_INF;
  bool nan = false;
  auto maxima = [&](auto lanes) __attribute__((always_inline)) {
    constexpr int L = decltype(lanes)::value;
    const bool last = (lane & (L - 1)) == L - 1;  // has its run's maximum
    row.vectors([&](const float (&v)[R::E], int q, auto end) __attribute__((always_inline)) {
      float g = v[0];
#pragma unroll
      for (int e = 0; e < R::E; e += 2) {
        nan |= __builtin_isunordered(v[e], v[e + 1]);
        if (e) g = larger(g, v[e]);
        g = larger(g, v[e + 1]);
      }
      hi = larger(hi, g);
      if (L >= 2) g = larger(g, dpp_mov<DPP_QUAD_1032>(g));
      if (L >= 4) g = larger(g, dpp_mov<DPP_QUAD_2301>(g));
      if (L >= 8) g = larger(g, dpp_mov<DPP_ROW_HALF_MIRROR>(g));
      if (L == 64) {
        g = larger(g, dpp_mov<DPP_ROW_MIRROR>(g));
        g = larger(g, row_below<ROW_BCAST15, 0xA>(g));
        g = larger(g, row_below<ROW_BCAST31, 0xC>(g));
      }
      const int run = q >> shift;
      if (last && (!decltype(end)::value || run < runs)) {
        if (L < 64 || shift == 6) sh.run_max[run] = g;
        else __hip_atomic_fetch_max(&sh.run_max[run], g, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      }
    });
  };
  if (shift == 0) {
    maxima(std::integral_constant<int, 1>());
  } else if (shift == 1) {
    maxima(std::integral_constant<int, 2>());
  } else if (shift == 2) {
    maxima(std::integral_constant<int, 4>());
  } else if (shift == 3) {
    maxima(std::integral_constant<int, 8>());
  } else {
    for (int i = threadIdx.x; i < runs; i += NT) sh.run_max[i] = NEG_INF;
    __syncthreads();
    maxima(std::integral_constant<int, 64>());
  }
  const u64 top = block_fold<NT>(nan ? ~u64(0) : (u64)key_of(hi), sh.wave_a, Max());
  const uint32_t bits = (uint32_t)top;
  const float m = __builtin_bit_cast(float, bits & 0x80000000u ? bits & 0x7fffffffu : ~bits);
  if (top == ~u64(0) || m == -NEG_INF || m == NEG_INF || s.bad) {
    if (threadIdx.x == 0) write(a, r, -1, __builtin_nanf(""));
    return;
  }
  if (s.greedy) {
    u64 first = ~u64(0);
    for (int i = threadIdx.x; i < runs; i += NT)
      if (sh.run_max[i] == m) first = min(first, (u64)i);
    first = block_fold<NT>(first, sh.wave_b, Min());
    u64 at = ~u64(0);
    for (int i = threadIdx.x; i < 1 << shift; i += NT) {
      const int q = ((int)first << shift) + i;
      if (q >= row.count()) break;
      float v[R::E];
      row.values(Vec<T>::load(row.x + row.first(q)), q, v);
#pragma unroll
      for (int e = 0; e < R::E; ++e)
        if (v[e] == m) at = min(at, (u64)(row.first(q) + e));
    }
    at = block_fold<NT>(at, sh.wave_a, Min());
    if (threadIdx.x == 0) write(a, r, (int)at, 0.f);
    return;
  }
  Drawer<NT> d{sh, m, 0.f, 0.f, 0.f, s.inv, mass_bits(a.V)};
  d.last = last_with_mass(m, s.inv, d.S);
  // one that passes the numbers, as an infinite distance does, is in the last step
  d.range = fminf(m - d.last, MAX_F32);
  d.steps = fminf((float)(BINS - 1) / d.range, 3e38f);

  u64 least = 0, whole = 0;
  // The candidates: with top-k, what is at least the k-th of the runs' maxima,
  // but for a coarse step, which the k-th class is, or where that is too many (1.9 k
  // of random rows with 4/3 k runs, more with fewer) what is within the k-th
  // class's step; with top-p alone, what is within the step in which the mass
  // passes it; with min-p alone, what is that large.
  int n = CANDIDATES + 1;
  float low = NEG_INF;
  if (s.k && 4 * s.k <= 3 * runs && s.k <= CANDIDATES / 2) {
    constexpr int COARSE = 4, BINS_K = BINS / COARSE, PER = BINS_K / 64;
    for (int i = threadIdx.x; i < BINS_K; i += NT) sh.count[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < runs; i += NT) {
      const float x = sh.run_max[i];
      if (d.counts(x)) atomicAdd(&sh.count[d.step_of(x) / COARSE], 1u);
    }
    __syncthreads();
    // each wave for itself
    uint32_t own = 0, c[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) own += c[i] = sh.count[lane * PER + i];
    u64 run = wave_scan((u64)own, Sum()) - own;
    int step = BINS_K;  // fewer than k runs that count: all classes that do
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (run < (u64)s.k && run + c[i] >= (u64)s.k) step = lane * PER + i;
      run += c[i];
    }
    step = (int)wave_fold((u64)step, Min());
    low = d.lowest(min(step * COARSE + COARSE - 1, BINS - 1));
  } else if (s.k && s.k < CANDIDATES) {
    d.clear(false);
    row.vectors([&](const float (&v)[R::E], int, auto) {
#pragma unroll
      for (int e = 0; e < R::E; ++e)
        if (d.counts(v[e])) atomicAdd(&sh.count[d.step_of(v[e])], 1u);
    });
    __syncthreads();
    u64 before = 0;
    low = d.lowest(d.template last_step<false>((u64)s.k, before));
  } else if (!s.k && s.p < 1.0) {
    d.fill(row, true, 0);
    whole = d.filled_mass(BINS);
    u64 before = 0;
    low = d.lowest(d.template last_step<true>(share_of(s.p, whole), before));
  } else if (!s.k && s.floor > (double)NEG_INF) {
    low = (float)((double)m + s.floor / s.inv);
    low = fmaxf(low - 1e-6f * (fabsf(low) + fabsf(m)) - 1e-37f, d.last);
  }
  if (low > NEG_INF) n = d.collect(row, low, runs, shift);
  auto kept_mass = [&](float x, int j) -> u64 {
    if (!d.counts(x) || rank_key(x, j) < least) return 0;
    const double t = d.distance(x);
    return t < s.floor ? 0 : mass_of(t, d.S);
  };
  if (n <= 64) {
    if (wave == 0) d.draw_few(a, r, n, s, whole);
    return;
  }
  if (n <= CANDIDATES) {
    d.draw_some(a, r, n, low, s, whole);
    return;
  }
  // The cuts, each by the steps that the one before has left where they tell it.
  const bool by_mass = s.p < 1.0;
  bool intact = true;
  if (s.k) {
    d.fill(row, by_mass, 0);
    least = d.template last_before<false>(row, (u64)s.k, 0, intact, by_mass, whole);
    if (by_mass && !intact) {
      d.fill(row, true, least);
      whole = d.filled_mass(BINS);
      intact = true;
    }
  }
  // steps beyond the k-th class weigh nothing here: what is before them is the whole
  if (by_mass) least = d.template last_before<true>(row, share_of(s.p, whole), least, intact, false, whole);

  // the running sum over the whole row in tiles of OWN classes a thread: groups of
  // tiles, then the tiles of one group, then the waves of one tile
  constexpr int OWN = 8, TILE = OWN * NT;
  int t0 = 0, t1 = (a.V + TILE - 1) / TILE;
  u64 before = 0, mass = 0, target = 0;
  bool first = true;
  for (;;) {
    const int per = (t1 - t0 + BINS / WAVES - 1) / (BINS / WAVES);
    __syncthreads();
    for (int i = threadIdx.x; i < BINS; i += NT) sh.mass[i] = 0;
    __syncthreads();
    for (int i = t0; i < t1; ++i) {
      const int j0 = i * TILE + (int)threadIdx.x * OWN;
      u64 sum = 0;
#pragma unroll 2
      for (int j = j0; j < min(j0 + OWN, a.V); ++j) sum += kept_mass((float)row.x[j], j);
      sum = wave_fold(sum, Sum());
      if (lane == 0) sh.mass[(i - t0) / per * WAVES + wave] += sum;
    }
    __syncthreads();
    // entries within a group are in the classes' order where it is one tile
    const int entries = ((t1 - t0 + per - 1) / per) * WAVES;
    constexpr int PER = BINS / NT;
    u64 w = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) w += sh.mass[threadIdx.x * PER + i];
    u64 run = before + block_scan<NT>(w, sh.wave_a);
    if (first) {
      mass = block_fold<NT>(w, sh.wave_b, Sum());
      target = target_of(s.u, mass);
      first = false;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = threadIdx.x * PER + i;
      const u64 v = sh.mass[e];
      if (e < entries && run <= target && run + v > target) {
        sh.out[0] = e;
        sh.out[1] = run;
      }
      run += v;
    }
    __syncthreads();
    const int e = (int)sh.out[0], group = e / WAVES;
    before = sh.out[1];
    if (per == 1) {
      t0 += group;
      if (wave != e % WAVES) return;
      break;
    }
    for (int i = group * WAVES; i < e; ++i) before -= sh.mass[i];
    t0 += group * per;
    t1 = min(t0 + per, t1);
  }
  // one wave's classes of tile t0
  const int j0 = t0 * TILE + (int)threadIdx.x * OWN;
  u64 own = 0;
  for (int j = j0; j < min(j0 + OWN, a.V); ++j) own += kept_mass((float)row.x[j], j);
  u64 run = before + wave_scan(own, Sum()) - own;
  if (run > target || run + own <= target) return;
  for (int j = j0; j < min(j0 + OWN, a.V); ++j) {  // one thread's
    const float x = (float)row.x[j];
    const u64 w = kept_mass(x, j);
    if (run <= target && run + w > target) write(a, r, j, log_share(d.distance(x), mass, d.S));
    run += w;
  }
}

template <class T, int NT>
void row_go(hipStream_t st, const Sample& a) {
  sample_row_kernel<T, NT><<<(unsigned)a.rows, NT, 0, st>>>(a);
}
template <class T>
void go(hipStream_t st, const Sample& a) {
  constexpr int E = Vec<T>::N;
  if (a.V <= 64) {
    const int W = a.V <= 16 ? 16 : a.V <= 32 ? 32 : 64;
    const unsigned grid = (unsigned)((a.rows * W + 255) / 256);
    if (W == 16) sample_few_kernel<T, 16><<<grid, 256, 0, st>>>(a);
    else if (W == 32) sample_few_kernel<T, 32><<<grid, 256, 0, st>>>(a);
    else sample_few_kernel<T, 64><<<grid, 256, 0, st>>>(a);
  } else if (a.V <= 1024) {
    const unsigned grid = (unsigned)((a.rows + 3) / 4);
    if (a.V <= 128) sample_wave_kernel<T, 2><<<grid, 256, 0, st>>>(a);
    else if (a.V <= 256) sample_wave_kernel<T, 4><<<grid, 256, 0, st>>>(a);
    else if (a.V <= 512) sample_wave_kernel<T, 8><<<grid, 256, 0, st>>>(a);
    else sample_wave_kernel<T, 16><<<grid, 256, 0, st>>>(a);
  } else if (a.V <= 16 * 256 * E) {
    row_go<T, 256>(st, a);  // 16 vectors a thread at most: more workgroups a unit
  } else if (a.rows > device_cus()) {
    row_go<T, 512>(st, a);  // two a unit
  } else {
    row_go<T, 1024>(st, a);  // one: 64 rows of 131 k 99 us of 512 threads, 82 so
  }
}

}  // namespace

void sample(hipStream_t st, const Sample& a) {
  // a grid holds fewer than 2^32 threads
  constexpr int64_t SLICE = int64_t(1) << 21;
  for (int64_t r = 0; r < a.rows; r += SLICE) {
    Sample b = a;
    b.rows = std::min(SLICE, a.rows - r);
    const int64_t w = a.dtype == BC2N_F32 ? 4 : 2;
    b.x = (const char*)a.x + r * a.ld * w;
    b.u += r;
    b.index += r;
    if (b.logp) b.logp += r;
    if (b.top_k_row) b.top_k_row += r;
    for (Setting* s : {&b.temperature, &b.top_p, &b.min_p})
      if (s->row) s->row += r;
    KTimed kt("sample", st);
    if (a.dtype == BC2N_F32) go<float>(st, b);
    else if (a.dtype == BC2N_F16) go<h16>(st, b);
    else go<bf16>(st, b);
    hip_check(hipGetLastError(), "sample launch");
  }
}

}  // namespace bc2n
