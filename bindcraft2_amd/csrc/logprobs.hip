// Log-probabilities of given classes, entropies and top alternatives of rows
// of logits x[V], and their gradient.  Per row, with m = max_j x_j,
// s = sum_j e^(x_j - m) and u = sum_j e^(x_j - m) (x_j - m):
//
//   logp     = (x_t - m) - log s
//   H        = log s - u / s                      (entropy)
//   top k    : the K largest x, ties to the lowest index; (x_i - m) - log s
//   d x_j    = g [j = t] + sum_k h_k [j = i_k] - p_j (g + sum_k h_k)
//              - e p_j (log p_j + H),             log p_j = x_j - m - log s
//
// (g, e, h the cotangents of logp, H and top k).  A row with t < 0 is left
// out (zeros, indices -1); a row of -inf alone has log-probabilities -inf,
// entropy and gradient 0; a NaN or +inf makes its row NaN and its indices -1;
// a target at or past V makes its row's log-probability and gradient NaN,
// whichever cotangents are given.
//
// Rows are independent and every element is read once and (gradient) written
// once, a few operations a byte, so memory bounds most of it: the kernels have
// to keep enough 16-byte loads in flight and the row on chip.  A read-only pass
// reaches 6.2 to 6.9 TB/s on this card, a copy 5.0 to 6.5.  16-bit logits come
// near the vector units' rate too (ten operations an element, one of them a
// quarter-rate exp2), and alternatives cost instructions by their number, for
// longer rows also by the logits' order: where they rise along the classes,
// every element enters a wave's list (one that falls, or random ones, leave it
// to the first chunk's bound).  Five alternatives of 2047 rows of 50 k binary16:
// random 47 us, falling 40, rising 706; eight of 4 rows of 131 k bfloat16: 12,
// 39, 36.
// Measured on random logits (bytes read and written once over the time):
//   forward, f32:  262 k rows of 64 4.9 TB/s, 50 k of 1000 5.1, 4084 of 33 k 5.9
//   forward, binary16: 2047 rows of 50 k 4.8 TB/s, with five alternatives 4.1
//   with gradient: 262 k of 64 f32 4.6 TB/s, 50 k of 1000 f32 5.7, 5000 of 20 k
//   bfloat16 4.4, 2048 of 131 k bfloat16 4.9
#include "logprobs.h"

#include "common.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

#include <algorithm>
#include <type_traits>

namespace bc2n {

namespace {

// e^(x - m) is 0 in f32 long before this difference, which stands in for
// -inf so that 0 * (x - m) stays 0.
constexpr float FAR = -200.f;
constexpr float LOWEST = -3.4028234663852886e38f;
constexpr float NEG_INF = -__builtin_inff();

__device__ __forceinline__ float exp_f(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

__device__ __forceinline__ int64_t target_of(const LogProbs& a, int64_t r) {
  if (!a.target) return 0;
  return a.target64 ? reinterpret_cast<const int64_t*>(a.target)[r]
                    : (int64_t) reinterpret_cast<const int32_t*>(a.target)[r];
}
// A target past the classes makes its row's gradient NaN, whatever the
// cotangents and the logits.  (Without targets t is 0.)
__device__ __forceinline__ bool past_classes(const LogProbs& a, int64_t t) { return t >= a.V; }

// m, s, u of a part of a row
struct Stat {
  float m = LOWEST, s = 0.f, u = 0.f;
  // the sums taken relative to a maximum m2 >= m
  __device__ __forceinline__ void raise(float m2) {
    const float d = fmaxf(m - m2, FAR), k = exp_f(d);
    u = k * fmaf(s, d, u);
    s *= k;
    m = m2;
  }
  // x <= m.  e is NaN where x is, and where x and m are +inf: the sum of such
  // a row is NaN.
  __device__ __forceinline__ void add(float x) {
    const float d = x - m, e = exp_f(d);
    s += e;
    u = fmaf(e, fmaxf(d, FAR), u);
  }
};

// What the outputs and the gradient of a row are made of.
struct RowStat {
  float m, logs, h;
  float live;  // 1; 0 for a row left out or without a logit above -inf
};
__device__ __forceinline__ RowStat finish(Stat t, bool counts) {
  RowStat r;
  const bool some = counts && !(t.s == 0.f);
  r.m = some ? t.m : 0.f;
  r.logs = some ? logf(t.s) : 0.f;
  r.h = some ? r.logs - t.u / t.s : 0.f;
  r.live = some ? 1.f : 0.f;
  return r;
}
__device__ __forceinline__ float log_prob(const RowStat& r, float x) {
  return r.live != 0.f ? (x - r.m) - r.logs : NEG_INF;
}
__device__ __forceinline__ bool is_nan(float x) { return x != x; }

// logp, entropy and save of row r, by one lane
template <class T>
__device__ __forceinline__ void write_row(const LogProbs& a, int64_t r, const RowStat& st,
                                          int64_t t) {
  if (a.logp) {
    float v = 0.f;
    if (t >= a.V) v = __builtin_nanf("");
    else if (t >= 0) v = log_prob(st, (float)reinterpret_cast<const T*>(a.x)[r * a.ld + t]);
    a.logp[r] = v;
  }
  if (a.entropy) a.entropy[r] = st.h;
  if (a.save) reinterpret_cast<float4*>(a.save)[r] = make_float4(st.m, st.logs, st.h, st.live);
}

// The gradient at one element without the terms of single classes:
// -p (g + e (log p + H)), in units of log 2.
struct Cotangent {
  float m, l2;    // log2 of the sum
  float gh, e2;   // g + e H, e log 2; g with those of the alternatives
  __device__ __forceinline__ Cotangent(const RowStat& st, float g, float e)
      : m(st.m), l2(st.logs * LOG2E), gh(fmaf(e, st.h, g)), e2(e * LN2) {}
  __device__ __forceinline__ float at(float x) const {
    const float lp2 = fmaf(x - m, LOG2E, -l2), p = __builtin_amdgcn_exp2f(lp2);
    return -p * fmaf(e2, fmaxf(lp2, FAR), gh);
  }
  template <int N>
  __device__ __forceinline__ void all(float (&x)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = at(x[i]);
  }
};

// ---------------------------------------------------------------------------
// Rows of at most W * NV vectors: a group of W lanes holds one row in
// registers, lane l the elements [l * E, l * E + E).  A vector that would run
// past the row's end is read ending there instead, and its first elements,
// which are the vector's before it, do not count (`skip` of them), so that
// every lane reads whole vectors whatever V.  VN = 1: rows shorter than one
// vector.  MODE 1 forward, 2 backward, 3 both.
// ---------------------------------------------------------------------------
__device__ __forceinline__ uint32_t order_key(float x) {
  // larger floats, larger keys; -0 and 0 alike; 0 for no element
  const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
  return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of_key(uint32_t k) {
  return __builtin_bit_cast(float, k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// with the other 16-lane row of its pair, with the other half of the wave
__device__ __forceinline__ uint32_t swap16_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return umax(a[0], a[1]);
}
__device__ __forceinline__ uint32_t swap32_max(uint32_t v) {
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return umax(a[0], a[1]);
}
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
  if constexpr (W >= 2) v = umax(v, dpp_u32<DPP_QUAD_1032>(v));
  if constexpr (W >= 4) v = umax(v, dpp_u32<DPP_QUAD_2301>(v));
  if constexpr (W >= 8) v = umax(v, dpp_u32<DPP_ROW_HALF_MIRROR>(v));
  if constexpr (W >= 16) v = umax(v, dpp_u32<DPP_ROW_MIRROR>(v));
  if constexpr (W >= 32) v = swap16_max(v);
  if constexpr (W >= 64) v = swap32_max(v);
  return v;
}

template <class Op>
__device__ __forceinline__ float wave_reduce(float v, Op op) {
  v = group_reduce<16>(v, op);
  auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, v),
                                            __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t a0 = a[0], a1 = a[1];
  v = op(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
  auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, v),
                                            __builtin_bit_cast(uint32_t, v), false, false);
  const uint32_t b0 = b[0], b1 = b[1];
  return op(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}
__device__ __forceinline__ float wave_max(float v) {
  return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_sum(float v) {
  return wave_reduce(v, [](float a, float b) { return a + b; });
}

template <int N>
__device__ __forceinline__ float max_of(const float (&x)[N]) {
  float m = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, x[i]);
  return m;
}
__device__ __forceinline__ float read_lane(float v, int lane) {
  return __builtin_bit_cast(float,
                            __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
// key of the float just below the one of this key; there is none below -inf
__device__ __forceinline__ uint32_t key_below(uint32_t k) {
  return k == 0x80000000u ? k - 2 : k - 1;  // below 0 lies the smallest negative, not -0
}

// Candidates in LDS are one word each: the value's order key over the index's
// complement, so that the larger word is the better candidate; 0: none.
__device__ __forceinline__ uint64_t candidate(float v, int i) {
  return i < 0 ? 0 : (uint64_t)order_key(v) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ int index_of(uint64_t c) { return (int)~(uint32_t)c; }
__device__ __forceinline__ float value_of(uint64_t c) { return value_of_key((uint32_t)(c >> 32)); }
// how many of the n candidates (n a multiple of 8) are better than c
__device__ __forceinline__ int rank_of(const uint64_t* cand, int n, uint64_t c) {
  int rank = 0;
  for (int o = 0; o < n; o += 8) {
#pragma unroll
    for (int k = 0; k < 8; ++k) rank += cand[o + k] > c;
  }
  return rank;
}
constexpr int up8(int n) { return (n + 7) / 8 * 8; }

// A wave's largest elements, the k-th in lane k (index -1: none yet).  An
// element not above `floor` is not among the row's: the wave has K as large
// that come before it.  Waves of one row tell each other, through LDS, values
// that K elements reach (*shared, as a key), so that a wave does not collect
// what another has better; when they learn it changes only what is collected
// beside the answer.
struct TopList {
  float v = NEG_INF;
  int i = -1;
  float floor = NEG_INF;

  __device__ __forceinline__ void insert(float cv, int ci, int K) {
    const int lane = threadIdx.x & 63;
    const int before = __popcll(__ballot(v > cv) | (__ballot(v == cv) & __ballot(i < ci)));
    const float pv = dpp_mov<0x138>(v);  // the lane before
    const int pi = (int)dpp_u32<0x138>((uint32_t)i);
    v = lane > before ? pv : lane == before ? cv : v;
    i = lane > before ? pi : lane == before ? ci : i;
    floor = fmaxf(floor, read_lane(v, K - 1));
  }

  // K lanes hold an element as large as the K-th largest of the lanes' maxima
  // mx, so nothing below it can stay: without this bound the first elements
  // would enter the list one by one.  Returns its key (0: none).
  __device__ __forceinline__ uint32_t bound(float mx, int K) {
    const int lane = threadIdx.x & 63;
    float t = NEG_INF;
    if (K <= 6) {  // the largest, K times
      for (int k = 0; k < K; ++k) {
        t = wave_max(mx);
        const uint64_t b = __ballot(mx == t);
        if (b == 0) break;
        if (lane == __ffsll((unsigned long long)b) - 1) mx = NEG_INF;
      }
    } else {  // the smallest of those that fewer than K are above
      int above = 0;
#pragma unroll
      for (int j = 0; j < 64; ++j) above += read_lane(mx, j) > mx;
      t = -wave_max(above < K ? -mx : NEG_INF);
    }
    if (!(t > NEG_INF)) return 0;
    const uint32_t reached = order_key(t);
    floor = fmaxf(floor, value_of_key(key_below(reached)));
    return reached;
  }
  // element x of each lane; index(lane) its index
  template <class F>
  __device__ __forceinline__ void offer(float x, int K, F index) {
    // out of order among the lanes' elements, so an equal one may be better
    for (uint64_t b = __ballot(x >= floor); b; b &= b - 1) {
      const int from = __ffsll((unsigned long long)b) - 1;
      const float cv = read_lane(x, from);
      if (cv > NEG_INF && cv >= floor) insert(cv, index(from), K);  // else the list rose since
    }
  }

  // x: this lane's elements of one chunk, vector u from index i0 + u * step;
  // mx: their maximum
  template <int VN, bool SHARE, int N>
  __device__ __forceinline__ void take(const float (&x)[N], float mx, int i0, int step, int K,
                                       bool first, uint32_t* shared) {
    if (!__any(mx > floor)) return;
    if (SHARE) {
      const uint32_t k = __hip_atomic_load(shared, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
      if (k) floor = fmaxf(floor, value_of_key(key_below(k)));
      if (!__any(mx > floor)) return;
    }
    uint32_t reached = first ? bound(mx, K) : 0;
    const float before = floor;
#pragma unroll
    for (int n = 0; n < N; ++n)
      offer(x[n], K, [&](int from) {
        return __builtin_amdgcn_readlane(i0, from) + n / VN * step + n % VN;
      });
    if (SHARE) {
      if (floor > before) reached = order_key(floor);
      if (reached && (threadIdx.x & 63) == 0)
        __hip_atomic_fetch_max(shared, reached, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    }
  }
};

// A row's alternative k, by one lane
__device__ __forceinline__ void write_top(const LogProbs& a, int64_t r, int k, const RowStat& st,
                                          bool counts, float v, int i) {
  const bool bad = is_nan(st.logs);
  a.top_logp[r * a.K + k] = bad ? st.logs : counts ? log_prob(st, v) : 0.f;
  a.top_index[r * a.K + k] = bad || !counts ? -1 : i;
}

// Where a row has only `have` < K alternatives above -inf, its first -inf
// elements follow; by one wave.
template <class T>
__device__ __forceinline__ void fill_tops(const LogProbs& a, int64_t r, int have) {
  const int lane = threadIdx.x & 63;
  const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
  for (int b = 0; have < a.K && b < a.V; b += 64) {
    const bool gone = b + lane < a.V && (float)p[b + lane] == NEG_INF;
    const uint64_t m = __ballot(gone);
    const int k = have + __popcll(m & ((1ull << lane) - 1));
    if (gone && k < a.K) {
      a.top_logp[r * a.K + k] = NEG_INF;
      a.top_index[r * a.K + k] = b + lane;
    }
    have += __popcll(m);
  }
}

// 16-bit logits: a key holds an element's order and its index's complement
// (rows here have at most 1024), so the largest of a group is the next
// alternative, index and all, and is taken out by comparing keys.
template <class T, int W, int E>
__device__ __forceinline__ void tops_by_key(const LogProbs& a, int64_t r, bool mine,
                                            const RowStat& st, bool counts, uint32_t (&key)[E]) {
  const int l = threadIdx.x & (W - 1);
  uint32_t kept = 0;
  for (int k = 0; k < a.K; ++k) {
    uint32_t best = 0;
#pragma unroll
    for (int i = 0; i < E; ++i) best = umax(best, key[i]);
    best = group_umax<W>(best);
#pragma unroll
    for (int i = 0; i < E; ++i) key[i] = key[i] == best ? 0u : key[i];
    if (l == (k & (W - 1))) kept = best;
    if ((k & (W - 1)) == W - 1 || k == a.K - 1) {  // W of them together
      const int at = (k & ~(W - 1)) + l;
      const uint32_t o = kept >> 16, bits = o & 0x8000u ? o ^ 0x8000u : o ^ 0xffffu;
      if (mine && at <= k)
        write_top(a, r, at, st, counts, (float)__builtin_bit_cast(T, (uint16_t)bits),
                  0xffff - (int)(kept & 0xffffu));
    }
  }
}
template <class T>
__device__ __forceinline__ uint32_t key16(float x, int i) {
  const uint32_t b = __builtin_bit_cast(uint16_t, (T)(x + 0.f));
  return (b & 0x8000u ? b ^ 0xffffu : b ^ 0x8000u) << 16 | (0xffffu - (uint32_t)i);
}

// f32 logits: each lane's elements in descending order, equal ones as they
// were (neighbours change places); the largest first element of the group is
// the next alternative, and the lowest lane that has it holds the lowest index.
template <int W, int E>
__device__ __forceinline__ void tops_by_lane(const LogProbs& a, int64_t r, bool mine,
                                             const RowStat& st, bool counts, uint32_t (&key)[E],
                                             int (&at)[E]) {
  const int l = threadIdx.x & (W - 1), lane0 = (threadIdx.x & 63) - l;
  if (a.K == 1) {  // the first of the largest is enough
#pragma unroll
    for (int i = 1; i < E; ++i) {
      const bool more = key[i] > key[0];
      key[0] = more ? key[i] : key[0];
      at[0] = more ? at[i] : at[0];
    }
  } else {
#pragma unroll
    for (int p = 0; p < E; ++p)
#pragma unroll
      for (int i = p & 1; i + 1 < E; i += 2) {
        const bool swap = key[i] < key[i + 1];
        const uint32_t x = key[i], y = key[i + 1];
        const int u = at[i], v = at[i + 1];
        key[i] = swap ? y : x;
        key[i + 1] = swap ? x : y;
        at[i] = swap ? v : u;
        at[i + 1] = swap ? u : v;
      }
  }
  for (int k = 0; k < a.K; ++k) {
    const uint32_t top = group_umax<W>(key[0]);
    const uint64_t b = __ballot(key[0] == top) >> lane0;
    const int first = W <= 32 ? __ffs((int)b) : __ffsll((unsigned long long)b);
    if (l == first - 1) {
      if (mine) write_top(a, r, k, st, counts, value_of_key(top), at[0]);
#pragma unroll
      for (int i = 0; i + 1 < E; ++i) {
        key[i] = key[i + 1];
        at[i] = at[i + 1];
      }
      key[E - 1] = 0;
    }
  }
}

// f32 logits of a row that is a wave's, more than four a lane: a sort of them
// would cost more than the list (K = 3 of 100 k rows of 500: 79 us).
template <class T, int VN, int W, int NV>
__device__ __forceinline__ void tops_by_list(const LogProbs& a, int64_t r, bool mine,
                                             const RowStat& st, bool counts,
                                             const float (&x)[VN * NV], const int (&pos)[NV],
                                             const int (&skip)[NV]) {
  static_assert(W == 64, "the list is a whole wave's, of one row");
  const int lane = threadIdx.x & 63;
  TopList top;
  if (counts && !is_nan(st.logs)) {
    float y[VN * NV];
#pragma unroll
    for (int i = 0; i < VN * NV; ++i) y[i] = i % VN >= skip[i / VN] ? x[i] : NEG_INF;
    top.bound(max_of(y), a.K);
#pragma unroll
    for (int i = 0; i < VN * NV; ++i)
      top.offer(y[i], a.K, [&](int from) {
        return __builtin_amdgcn_readlane(pos[i / VN], from) + i % VN;
      });
  }
  if (!mine) return;
  const bool some = counts && !is_nan(st.logs);
  if (lane < a.K && (top.i >= 0 || !some)) write_top(a, r, lane, st, counts, top.v, top.i);
  if (some) fill_tops<T>(a, r, __popcll(__ballot(lane < a.K && top.i >= 0)));
}

template <class T, int VN, int W, int NV, int MODE>
__global__ __launch_bounds__(256) void lp_rows_kernel(LogProbs a) {
  constexpr int E = VN * NV;
  const int l = threadIdx.x & (W - 1);
  const int64_t r0 = (int64_t)blockIdx.x * (256 / W) + threadIdx.x / W;
  const bool mine = r0 < a.rows;
  const int64_t r = mine ? r0 : a.rows - 1;  // whole groups stay active
  const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
  float x[E];
  int pos[NV], skip[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = l * E + i * VN;
    pos[i] = min(at, a.V - VN);
    skip[i] = at - pos[i];
    if constexpr (VN == 1) {
      x[i] = (float)p[pos[i]];
    } else {
      Vec<T>::unpack(Vec<T>::load(p + pos[i]), x + i * VN);
    }
  }
  const int64_t t = target_of(a, r);
  const bool counts = t >= 0;

  RowStat st;
  if constexpr (MODE & 1) {
    Stat q;
    float m = LOWEST;
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (i % VN >= skip[i / VN]) m = fmaxf(m, x[i]);
    q.m = group_max<W>(m);
#pragma unroll
    for (int i = 0; i < E; ++i) q.add(i % VN >= skip[i / VN] ? x[i] : NEG_INF);
    q.s = group_sum<W>(q.s);
    q.u = group_sum<W>(q.u);
    st = finish(q, counts);
    if (mine && l == 0) write_row<T>(a, r, st, a.target ? t : -1);

    // two vectors a lane by fewer than 64 lanes: without alternatives alone
    if constexpr (MODE == 1 && (NV == 1 || W == 64)) {
      if (a.K > 0) {
        if constexpr (sizeof(T) == 4 && E > 4) {
          tops_by_list<T, VN, W, NV>(a, r, mine, st, counts, x, pos, skip);
        } else {
          uint32_t key[E];
          int at[E];
#pragma unroll
          for (int i = 0; i < E; ++i) {
            at[i] = pos[i / VN] + i % VN;
            const bool real = i % VN >= skip[i / VN];
            if constexpr (sizeof(T) == 2) key[i] = real ? key16<T>(x[i], at[i]) : 0u;
            else key[i] = real ? order_key(x[i]) : 0u;
          }
          if constexpr (sizeof(T) == 2) tops_by_key<T, W>(a, r, mine, st, counts, key);
          else tops_by_lane<W>(a, r, mine, st, counts, key, at);
        }
      }
    }
  } else {
    const float4 s = reinterpret_cast<const float4*>(a.save)[r];
    st = RowStat{s.x, s.y, s.z, s.w};
  }

  if constexpr (MODE & 2) {
    const float g = a.d_logp ? a.d_logp[r] : 0.f;
    float all = g;
    if (MODE == 2 && a.d_top)
      for (int k = 0; k < a.K; ++k) all += a.d_top[r * a.K + k];
    const Cotangent c(st, all, a.d_entropy ? a.d_entropy[r] : 0.f);
    float d[E];
#pragma unroll
    for (int i = 0; i < E; ++i) d[i] = c.at(x[i]);
    if (a.d_logp) {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (pos[i / VN] + i % VN == t) d[i] += g;
    }
    if (MODE == 2 && a.d_top) {
      for (int k = 0; k < a.K; ++k) {
        const int at = a.top_index[r * a.K + k];
        const float h = a.d_top[r * a.K + k];
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (pos[i / VN] + i % VN == at) d[i] += h;
      }
    }
    T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
    const bool past = past_classes(a, t), one = past || st.live == 0.f || !counts;
    const float all_of = past ? __builtin_nanf("") : 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VN; ++j)
        if (one) d[i * VN + j] = all_of;
      if (mine && skip[i] < VN) {
        if constexpr (VN == 1) o[pos[i]] = (T)d[i];
        else Vec<T>::store(o + pos[i], Vec<T>::pack(d + i * VN));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Longer rows: whole workgroups.  A row is the elements before the first
// 16-byte boundary (`head`), aligned vectors, and what is left behind them;
// head and rest together are fewer than 16 elements, the `edge`, one a lane of
// the first wave.  (Aligned vectors: 50 against 56 us for 2047 rows of 50 k
// binary16 logits that start anywhere.)
// ---------------------------------------------------------------------------
template <class T>
struct Row {
  static constexpr int VN = Vec<T>::N;
  const T* p;
  int head, nv, edges;  // vector g holds the elements from head + g * VN
  __device__ __forceinline__ Row(const T* row, int V) : p(row) {
    const int past = (int)(reinterpret_cast<uintptr_t>(row) & 15);
    head = min(V, ((16 - past) & 15) / (int)sizeof(T));
    nv = (V - head) / VN;
    edges = V - nv * VN;
  }
  // index of edge element t < edges
  __device__ __forceinline__ int edge(int t) const { return t < head ? t : t + nv * VN; }
  __device__ __forceinline__ u32x4 load(int g) const { return Vec<T>::load(p + head + g * VN); }
  static __device__ __forceinline__ u32x4 none() {  // -inf
    constexpr uint32_t w = sizeof(T) == 4 ? 0xff800000u
                           : std::is_same<T, h16>::value ? 0xfc00fc00u : 0xff80ff80u;
    return u32x4{w, w, w, w};
  }
};

// A chunk: E elements a lane, U vectors apart by the workgroup's width
constexpr int E = 16;

// f(chunk, base) for the chunks of U vectors a lane of [v0, v1): chunk[u] is
// vector base + u * NT + lane, -inf past v1.  While one is worked on the next
// is on its way: two buffers that take turns, so that no copy waits for it.
template <class T, int NT, int U, class F>
__device__ __forceinline__ void each_chunk(const Row<T>& r, int v0, int v1, F f) {
  constexpr int STEP = U * NT;
  const int t = threadIdx.x;
  u32x4 a[U], b[U];
  auto fetch = [&](int base, u32x4(&c)[U]) {
#pragma unroll
    for (int u = 0; u < U; ++u) c[u] = r.load(base + u * NT + t);
  };
  const int full = (v1 - v0) / STEP, end = v0 + full * STEP;
  int base = v0;
  if (full > 0) {
    fetch(base, a);
    for (; base + 2 * STEP < end; base += 2 * STEP) {
      fetch(base + STEP, b);
      f(a, base);
      fetch(base + 2 * STEP, a);
      f(b, base + STEP);
    }
    if (base + STEP < end) {
      fetch(base + STEP, b);
      f(a, base);
      f(b, base + STEP);
    } else {
      f(a, base);
    }
  }
  if (end < v1) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      a[u] = Row<T>::none();
      if (end + u * NT + t < v1) a[u] = r.load(end + u * NT + t);
    }
    f(a, end);
  }
}
// Keeps the compiler from holding a vector's f32 values from one use to the
// next, in twice the registers.
__device__ __forceinline__ void as_stored(u32x4& v) { asm volatile("" : "+v"(v)); }
// a lane's running sums over one more chunk of maximum mx
template <int N>
__device__ __forceinline__ void add_chunk(Stat& q, const float (&x)[N], float mx) {
  if (__any(mx > q.m)) q.raise(fmaxf(q.m, mx));
#pragma unroll
  for (int i = 0; i < N; ++i) q.add(x[i]);
}

// Sum of a row over a wave's lanes, and over the workgroup's waves, in every lane
__device__ __forceinline__ Stat join_wave(Stat q) {
  q.raise(wave_max(q.m));
  q.s = wave_sum(q.s);
  q.u = wave_sum(q.u);
  return q;
}
__device__ __forceinline__ Stat join(Stat q, float (*buf)[4], int waves) {
  q = join_wave(q);
  if (waves == 1) return q;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  if (lane == 0) {
    buf[w][0] = q.m;
    buf[w][1] = q.s;
    buf[w][2] = q.u;
  }
  __syncthreads();
  Stat o;
  if (lane < waves) {
    o.m = buf[lane][0];
    o.s = buf[lane][1];
    o.u = buf[lane][2];
  }
  return join_wave(o);
}

// Writes the K best of n candidates (LDS, zeros behind up to a multiple of 8)
// as row r's alternatives; where there are fewer than K above -inf, the first
// -inf elements of the row follow.
template <class T, int NT>
__device__ __forceinline__ void write_tops(const LogProbs& a, int64_t r, const RowStat& st,
                                           const uint64_t* cand, int n) {
  float* ov = a.top_logp + r * a.K;
  int32_t* oi = a.top_index + r * a.K;
  if (is_nan(st.logs)) {
    for (int k = threadIdx.x; k < a.K; k += NT) {
      ov[k] = st.logs;
      oi[k] = -1;
    }
    return;
  }
  for (int c = threadIdx.x; c < n; c += NT) {
    const uint64_t mine = cand[c];
    const int k = mine ? rank_of(cand, n, mine) : a.K;
    if (k < a.K) {
      ov[k] = log_prob(st, value_of(mine));
      oi[k] = index_of(mine);
    }
  }
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int have = 0;
    for (int c = 0; c < n; c += 64) have += __popcll(__ballot(c + lane < n && cand[c + lane] != 0));
    fill_tops<T>(a, r, have);
  }
}
__device__ __forceinline__ void no_tops(const LogProbs& a, int64_t r, int nt) {
  for (int k = threadIdx.x; k < a.K; k += nt) {
    a.top_logp[r * a.K + k] = 0.f;
    a.top_index[r * a.K + k] = -1;
  }
}

// Parts of rows: their sums and their largest elements
struct Parts {
  float4* stat = nullptr;    // [rows][splits]
  uint64_t* top = nullptr;   // [rows][splits][K] candidates
};
template <class A>
Parts parts_of(A& c, int64_t rows, int splits, int K) {
  Parts p;
  const size_t n = (size_t)rows * splits;
  p.stat = c.template take<float4>(n);
  p.top = c.template take<uint64_t>(n * K);
  return p;
}

// A workgroup reads a row, or one of `splits` parts of `part` vectors of it
// (the first with the edge), a chunk ahead of the one it works on, with a
// running maximum a lane.
template <class T, bool TOP, int NT>
__global__ __launch_bounds__(NT, 8) void lp_stream_kernel(LogProbs a, int splits, int part,
                                                          Parts parts) {
  constexpr int VN = Vec<T>::N, NW = NT / 64, U = E / VN;
  __shared__ float buf[NW][4];
  __shared__ uint64_t cand[TOP ? NW * LP_MAX_TOP : 1];
  __shared__ uint32_t shared;
  constexpr bool SHARE = TOP && NT > 64;
  const int64_t r = blockIdx.x / splits;
  const int sp = blockIdx.x % splits;
  const int64_t t = target_of(a, r);
  // left out: not read.  (A part's rows are few, and waiting for the target
  // first costs each a load's latency: the join leaves them out.)
  if (splits == 1 && t < 0) {
    if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
    if (TOP) no_tops(a, r, NT);
    return;
  }
  const Row<T> row(reinterpret_cast<const T*>(a.x) + r * a.ld, a.V);
  const int v0 = sp * part, v1 = min(row.nv, v0 + part);
  const bool edge = sp == 0 && (int)threadIdx.x < row.edges;
  const int edge_at = edge ? row.edge(threadIdx.x) : -1;
  const float ex = edge ? (float)row.p[edge_at] : NEG_INF;
  Stat q;
  TopList top;
  if (SHARE) {
    if (threadIdx.x == 0) shared = 0;
    __syncthreads();
  }
  each_chunk<T, NT, U>(row, v0, v1, [&](const u32x4(&raw)[U], int base) {
    float x[E];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(raw[u], x + u * VN);
    const float mx = max_of(x);
    add_chunk(q, x, mx);
    if (TOP)
      top.take<VN, SHARE>(x, mx, row.head + (base + (int)threadIdx.x) * VN, NT * VN, a.K,
                          base == v0, &shared);
  });
  if (threadIdx.x < 64 && sp == 0) {
    const float one[1] = {ex};
    add_chunk(q, one, ex);
    if (TOP)
      top.offer(ex, a.K, [&](int from) { return __builtin_amdgcn_readlane(edge_at, from); });
  }
  if (TOP) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = NW * a.K;
    if (lane < a.K) cand[w * a.K + lane] = candidate(top.v, top.i);
    if ((int)threadIdx.x < up8(n) - n) cand[n + threadIdx.x] = 0;
  }
  const Stat all = join(q, buf, NT / 64);
  if (TOP && NT == 64) __syncthreads();  // else join's
  if (splits == 1) {
    const RowStat st = finish(all, true);
    if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
    if (TOP) write_tops<T, NT>(a, r, st, cand, NW * a.K);
    return;
  }
  const int64_t o = r * splits + sp;
  if (threadIdx.x == 0) parts.stat[o] = make_float4(all.m, all.s, all.u, 0.f);
  if (TOP) {
    // in any order; places that no candidate ranks for are none
    const int n = NW * a.K;
    uint64_t mine = 0;
    int have = 0;
    for (int c = 0; c < n; c += 64) {
      const int lane = threadIdx.x & 63;
      have += __popcll(__ballot(c + lane < n && cand[c + lane] != 0));
    }
    for (int c = threadIdx.x; c < n; c += NT) {
      mine = cand[c];
      const int k = mine ? rank_of(cand, n, mine) : a.K;
      if (k < a.K) parts.top[o * a.K + k] = mine;
    }
    for (int k = have + threadIdx.x; k < a.K; k += NT) parts.top[o * a.K + k] = 0;
  }
}

// Joins the parts of a row.
constexpr int MAX_SPLITS = 32;
template <class T>
__global__ __launch_bounds__(256) void lp_join_kernel(LogProbs a, int splits, Parts parts) {
  __shared__ uint64_t cand[MAX_SPLITS * LP_MAX_TOP];
  const int64_t r = blockIdx.x;
  const int n = splits * a.K;
  for (int c = threadIdx.x; c < up8(n); c += 256) cand[c] = c < n ? parts.top[r * n + c] : 0;
  const int lane = threadIdx.x & 63;
  Stat q;
  if (lane < splits) {  // each wave by itself
    const float4 s = parts.stat[r * splits + lane];
    q.m = s.x;
    q.s = s.y;
    q.u = s.z;
  }
  const int64_t t = target_of(a, r);
  if (t < 0) {
    if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
    no_tops(a, r, 256);
    return;
  }
  const RowStat st = finish(join_wave(q), true);
  if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
  __syncthreads();
  if (a.K > 0) write_tops<T, 256>(a, r, st, cand, n);
}

// One value over [lo, hi) of row r's gradient: NaN for a target past the
// classes, else zero.
template <class T>
__device__ __forceinline__ void write_one(const LogProbs& a, int64_t r, int64_t t, int64_t lo,
                                          int64_t hi) {
  constexpr int VN = Vec<T>::N;
  const int NT = blockDim.x;
  T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
  float x[VN];
#pragma unroll
  for (int i = 0; i < VN; ++i) x[i] = past_classes(a, t) ? __builtin_nanf("") : 0.f;
  const u32x4 v = Vec<T>::pack(x);
  for (int64_t at = lo + threadIdx.x * VN; at < hi; at += NT * VN) {
    if (at + VN <= hi) Vec<T>::store(o + at, v);
    else
      for (int64_t j = at; j < hi; ++j) o[j] = (T)x[0];
  }
}

// The classes of a row with terms of their own, one a lane of each wave:
// lane k < K alternative k, lane K the target.  g: the sum of those terms.
struct Special {
  int64_t at = -1;  // class, or none
  float own = 0.f;  // its own terms
};
__device__ __forceinline__ Special special_of(const LogProbs& a, int64_t r, int64_t t, int K,
                                              float& g) {
  const int lane = threadIdx.x & 63;
  Special s;
  if (a.d_top && lane < K) {
    s.at = a.top_index[r * K + lane];
    s.own = a.d_top[r * K + lane];
  }
  g = a.d_top ? wave_sum(s.own) : 0.f;
  if (a.d_logp) {
    const float gt = a.d_logp[r];
    const uint64_t same = __ballot(lane < K && s.at == t);  // the target among the alternatives
    if (lane < K && s.at == t) s.own += gt;
    if (lane == K && !same) {
      s.at = t;
      s.own = gt;
    }
    g += gt;
  }
  if (past_classes(a, t)) g = __builtin_nanf("");
  return s;
}
__device__ __forceinline__ Cotangent cotangent_of(const LogProbs& a, int64_t r, const RowStat& st,
                                                  float g) {
  return Cotangent(st, g, a.d_entropy ? a.d_entropy[r] : 0.f);
}

// The gradient of vectors [v0, v1) and, where `edge`, the edge of row r from
// its statistics.  The special classes are computed first, by one wave, and
// stored last: a row may be written in place.
template <class T, int NT, bool ONCE>
__device__ __forceinline__ void write_gradient(const LogProbs& a, int64_t r, int64_t t,
                                               const RowStat& st, int K, const Row<T>& row, int v0,
                                               int v1, bool edge) {
  constexpr int VN = Vec<T>::N, U = E / VN;
  T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
  float g;
  const Special sp = special_of(a, r, t, K, g);
  const Cotangent c = cotangent_of(a, r, st, g);
  const int lo = row.head + v0 * VN, hi = row.head + v1 * VN;
  const bool inside = sp.at >= lo && sp.at < hi;
  const bool outside = edge && sp.at >= 0 && sp.at < a.V &&
                       (sp.at < row.head || sp.at >= row.head + row.nv * VN);
  const bool mine = threadIdx.x < 64 && (inside || outside);
  T sv = (T)0.f;
  if (mine) sv = (T)(c.at((float)row.p[sp.at]) + sp.own);
  __syncthreads();
  if (edge && (int)threadIdx.x < row.edges) {
    const int at = row.edge(threadIdx.x);
    o[at] = (T)c.at((float)row.p[at]);
  }
  each_chunk<T, NT, U>(row, v0, v1, [&](const u32x4(&raw)[U], int base) {
    float x[E];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(raw[u], x + u * VN);
    c.all(x);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = base + u * NT + (int)threadIdx.x;
      if (g < v1) Vec<T>::template store<ONCE>(o + row.head + g * VN, Vec<T>::pack(x + u * VN));
    }
  });
  __syncthreads();
  if (mine) o[sp.at] = sv;
}

constexpr int BWD_NT = 256;
template <class T, bool ONCE>
__global__ __launch_bounds__(BWD_NT) void lp_gradient_kernel(LogProbs a, int splits, int part) {
  const int64_t r = blockIdx.x / splits;
  const int sp = blockIdx.x % splits;
  const int64_t t = target_of(a, r);
  const float4 s = reinterpret_cast<const float4*>(a.save)[r];
  const RowStat st{s.x, s.y, s.z, s.w};
  const Row<T> row(reinterpret_cast<const T*>(a.x) + r * a.ld, a.V);
  const int v0 = min(row.nv, sp * part), v1 = min(row.nv, v0 + part);
  if (st.live == 0.f || t < 0) {
    constexpr int VN = Vec<T>::N;
    write_one<T>(a, r, t, sp == 0 ? 0 : row.head + v0 * VN,
                 sp == splits - 1 ? a.V : row.head + v1 * VN);
    return;
  }
  write_gradient<T, BWD_NT, ONCE>(a, r, t, st, a.K, row, v0, v1, sp == 0);
}

// Forward and backward of a row held in the registers of one workgroup, as wide
// as the row takes at NV vectors a lane.
template <class T, int NV, bool ONCE>
__global__ __launch_bounds__(1024) void lp_block_kernel(LogProbs a) {
  constexpr int VN = Vec<T>::N;
  const int NT = blockDim.x;
  __shared__ float buf[16][4];
  const int64_t r = blockIdx.x;
  const int64_t t = target_of(a, r);
  if (t < 0) {
    if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
    write_one<T>(a, r, t, 0, a.V);
    return;
  }
  const Row<T> row(reinterpret_cast<const T*>(a.x) + r * a.ld, a.V);
  u32x4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int g = i * NT + (int)threadIdx.x;
    raw[i] = Row<T>::none();
    if (g < row.nv) raw[i] = row.load(g);
  }
  const bool edge = (int)threadIdx.x < row.edges;
  const int edge_at = edge ? row.edge(threadIdx.x) : -1;
  const float ex = edge ? (float)row.p[edge_at] : NEG_INF;
  Stat q;
  q.m = fmaxf(LOWEST, ex);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float x[VN];
    Vec<T>::unpack(raw[i], x);
    q.m = fmaxf(q.m, max_of(x));
    as_stored(raw[i]);
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    float x[VN];
    Vec<T>::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < VN; ++j) q.add(x[j]);
    as_stored(raw[i]);
  }
  q.add(ex);
  const RowStat st = finish(join(q, buf, NT / 64), true);
  if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
  if (st.live == 0.f) {
    __syncthreads();  // the target's logit is read before its place is written
    write_one<T>(a, r, t, 0, a.V);
    return;
  }
  float g;
  const Special sp = special_of(a, r, t, 0, g);
  const Cotangent c = cotangent_of(a, r, st, g);
  const bool mine = threadIdx.x < 64 && sp.at >= 0 && sp.at < a.V;
  T sv = (T)0.f;
  if (mine) sv = (T)(c.at((float)row.p[sp.at]) + sp.own);
  __syncthreads();
  T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
  if (edge) o[edge_at] = (T)c.at(ex);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int g = i * NT + (int)threadIdx.x;
    float x[VN];
    Vec<T>::unpack(raw[i], x);
    c.all(x);
    if (g < row.nv) Vec<T>::template store<ONCE>(o + row.head + g * VN, Vec<T>::pack(x));
  }
  __syncthreads();
  if (mine) o[sp.at] = sv;
}

// Rows longer than that: what a workgroup can hold of one (half of the CU's
// registers and LDS, at two workgroups a CU) it reads once, the rest twice,
// the second time out of the caches.
// 2048 rows of 131 k bfloat16: nothing held 228 us, registers alone 217, LDS
// too 210; six vectors a lane in registers 217, a workgroup of 512 250.
constexpr int BOTH_NT = 1024, BOTH_KEEP = 4, BOTH_LDS = 4;  // vectors a lane
template <class T, bool ONCE>
__global__ __launch_bounds__(BOTH_NT, 8) void lp_both_kernel(LogProbs a) {
  constexpr int VN = Vec<T>::N, NT = BOTH_NT, U = 2, KEEP = BOTH_KEEP, LDS = BOTH_LDS;
  __shared__ float buf[NT / 64][4];
  __shared__ u32x4 held[LDS * NT];
  const int64_t r = blockIdx.x;
  const int64_t t = target_of(a, r);
  if (t < 0) {
    if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
    write_one<T>(a, r, t, 0, a.V);
    return;
  }
  const Row<T> row(reinterpret_cast<const T*>(a.x) + r * a.ld, a.V);
  const int lane = threadIdx.x, rest = min(row.nv, (KEEP + LDS) * NT);
  const bool edge = lane < row.edges;
  const int edge_at = edge ? row.edge(lane) : -1;
  const float ex = edge ? (float)row.p[edge_at] : NEG_INF;
  Stat q;
  auto add = [&](const u32x4(&raw)[U]) {
    float x[U * VN];
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(raw[u], x + u * VN);
    add_chunk(q, x, max_of(x));
  };
  u32x4 keep[KEEP / U][U];  // vectors [0, KEEP * NT): all there
#pragma unroll
  for (int i = 0; i < KEEP; ++i) keep[i / U][i % U] = row.load(i * NT + lane);
#pragma unroll
  for (int i = 0; i < LDS / U; ++i) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int g = (KEEP + i * U + u) * NT + lane;
      raw[u] = Row<T>::none();
      if (g < row.nv) raw[u] = row.load(g);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) held[(i * U + u) * NT + lane] = raw[u];
    add(raw);
  }
#pragma unroll
  for (int i = 0; i < KEEP / U; ++i) {
    add(keep[i]);
#pragma unroll
    for (int u = 0; u < U; ++u) as_stored(keep[i][u]);
  }
  each_chunk<T, NT, U>(row, rest, row.nv, [&](const u32x4(&raw)[U], int) { add(raw); });
  const float one[1] = {ex};
  add_chunk(q, one, ex);
  const RowStat st = finish(join(q, buf, NT / 64), true);
  if (lane == 0) write_row<T>(a, r, st, a.target ? t : -1);
  if (st.live == 0.f) {
    __syncthreads();  // the target's logit is read before its place is written
    return write_one<T>(a, r, t, 0, a.V);
  }
  float g;
  const Special sp = special_of(a, r, t, 0, g);
  const Cotangent c = cotangent_of(a, r, st, g);
  const bool mine = lane < 64 && sp.at >= 0 && sp.at < a.V;
  T sv = (T)0.f;
  if (mine) sv = (T)(c.at((float)row.p[sp.at]) + sp.own);
  __syncthreads();
  T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
  if (edge) o[edge_at] = (T)c.at(ex);
  auto put = [&](u32x4 raw, int v) {
    float x[VN];
    Vec<T>::unpack(raw, x);
    c.all(x);
    if (v < row.nv) Vec<T>::template store<ONCE>(o + row.head + v * VN, Vec<T>::pack(x));
  };
  each_chunk<T, NT, U>(row, rest, row.nv, [&](const u32x4(&raw)[U], int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) put(raw[u], base + u * NT + lane);
  });
#pragma unroll
  for (int i = 0; i < LDS; ++i) put(held[i * NT + lane], (KEEP + i) * NT + lane);
#pragma unroll
  for (int i = 0; i < KEEP; ++i) put(keep[i / U][i % U], i * NT + lane);
  __syncthreads();
  if (mine) o[sp.at] = sv;
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
constexpr int ROW_VECS = 128;      // vectors that a group of lanes holds
constexpr int PART_MIN = 8192;     // longest row that is always read whole
constexpr int BLOCK_VECS = 8192;   // vectors that one workgroup holds in registers

template <class T>
bool short_row(int V) {
  return V <= ROW_VECS * Vec<T>::N;
}

// How a long row is divided among workgroups of 256: into as many parts as
// fill the card, each at least one chunk.
struct Split {
  int splits = 1, part = 0;  // part in vectors
};
Split split_of(int dtype, int64_t rows, int V, int K) {
  const int vn = dtype == BC2N_F32 ? 4 : 8, nv = (V + vn - 1) / vn;
  const int64_t chunk = (int64_t)E / vn * 256;
  const int64_t fill = (4 * (int64_t)device_cus() + rows / 2) / rows;
  // the join ranks splits * K candidates against each other: at most 256 (K =
  // 20 of 32 rows of 150 k: 32 parts 39 us, 8 parts 24)
  const int64_t most = K > 0 ? std::min(MAX_SPLITS, std::max(4, 256 / K)) : MAX_SPLITS;
  int64_t s = std::min<int64_t>({(nv + chunk - 1) / chunk, fill, most});
  if (s < 1 || V <= PART_MIN) s = 1;
  return Split{(int)s, (int)((nv + s - 1) / s)};
}

void launched() { hip_check(hipGetLastError(), "logprobs launch"); }

template <class T, int VN, int W, int NV, int MODE>
void rows_go(hipStream_t st, const LogProbs& a) {
  const int64_t per = 256 / W;
  lp_rows_kernel<T, VN, W, NV, MODE><<<(unsigned)((a.rows + per - 1) / per), 256, 0, st>>>(a);
}

template <class T, int MODE>
void rows_launch(hipStream_t st, const LogProbs& a) {
  constexpr int N = Vec<T>::N;
  const int vecs = (a.V + N - 1) / N;
  if (a.V < N) return rows_go<T, 1, 8, 1, MODE>(st, a);
  // Two vectors a lane keep more loads in flight and halve the lanes that a sum
  // joins: V = 64 f32 with gradient 32.8 -> 29.3 us, forward 17.2 -> 14.1 (262 k
  // rows); four (64 bytes between a lane's stores and the next's) 38.  With
  // alternatives one, for the least time of few rows with two or three (50 k of
  // 64 f32: two 6.8 against 7.3 us, eight 10.0 against 9.5).  Many rows would
  // gain from two there as well (262 k of 64 f32: one alternative 21.8 against
  // 19.7 us, eight 37.4 against 32.7; 100 k of 500 bfloat16: 45 against 37, 77
  // against 62), which this rule does not take.
  if constexpr (MODE == 1) {
    if (a.K > 0) {
      if (vecs <= 4) return rows_go<T, N, 4, 1, MODE>(st, a);
      if (vecs <= 8) return rows_go<T, N, 8, 1, MODE>(st, a);
      if (vecs <= 16) return rows_go<T, N, 16, 1, MODE>(st, a);
      if (vecs <= 32) return rows_go<T, N, 32, 1, MODE>(st, a);
      if (vecs <= 64) return rows_go<T, N, 64, 1, MODE>(st, a);
    }
  }
  if (vecs <= 8) rows_go<T, N, 4, 2, MODE>(st, a);
  else if (vecs <= 16) rows_go<T, N, 8, 2, MODE>(st, a);
  else if (vecs <= 32) rows_go<T, N, 16, 2, MODE>(st, a);
  else if (vecs <= 64) rows_go<T, N, 32, 2, MODE>(st, a);
  else rows_go<T, N, 64, 2, MODE>(st, a);
}

template <class T, int NT>
void stream_go(hipStream_t st, const LogProbs& a, const Split& s, const Parts& parts) {
  const unsigned grid = (unsigned)(a.rows * s.splits);
  if (a.K > 0) lp_stream_kernel<T, true, NT><<<grid, NT, 0, st>>>(a, s.splits, s.part, parts);
  else lp_stream_kernel<T, false, NT><<<grid, NT, 0, st>>>(a, s.splits, s.part, parts);
}

template <class T>
void fwd(hipStream_t st, const LogProbs& a, void* work) {
  if (short_row<T>(a.V)) return rows_launch<T, 1>(st, a);
  const Split s = split_of(a.dtype, a.total, a.V, a.K);
  Parts parts;
  if (s.splits > 1) {
    Carver c(work);
    parts = parts_of(c, a.rows, s.splits, a.K);
  }
  // A wave by itself collects its row's alternatives once, and joins nothing,
  // where rows enough fill the card with waves: five alternatives of 2048 rows
  // of 8000 bfloat16 15.5 us against 17.5, 8000 rows of 5003 28 against 47; of
  // 256 rows of 8000 11.5 against 8.3.
  const bool waves = a.V <= 2048 || (a.V <= PART_MIN && a.total >= 6 * (int64_t)device_cus());
  if (waves) stream_go<T, 64>(st, a, s, parts);
  else stream_go<T, 256>(st, a, s, parts);
  if (s.splits > 1) lp_join_kernel<T><<<(unsigned)a.rows, 256, 0, st>>>(a, s.splits, parts);
}

// Logits and gradient of more than half of the Infinity Cache's 256 MiB: the
// gradient is stored past the caches, which leaves them to the logits (1021
// rows of 33 k f32, forward and backward: 95 -> 82 us; 30 k of 1.5 k: 113 ->
// 102).  Smaller ones stay for whoever reads them next.
template <class F>
void with_once(const LogProbs& a, F f) {
  const int64_t bytes = 2 * a.total * a.V * (a.dtype == BC2N_F32 ? 4 : 2);
  if (bytes > int64_t(128) << 20) f(std::true_type());
  else f(std::false_type());
}

template <class T>
void bwd(hipStream_t st, const LogProbs& a) {
  if (short_row<T>(a.V)) return rows_launch<T, 2>(st, a);
  const Split s = split_of(a.dtype, a.total, a.V, a.K);
  const unsigned grid = (unsigned)(a.rows * s.splits);
  with_once(a, [&](auto once) {
    lp_gradient_kernel<T, once><<<grid, BWD_NT, 0, st>>>(a, s.splits, s.part);
  });
}

// Few rows that no workgroup holds: forward in parts, then backward
bool in_parts(int dtype, int64_t rows, int V) {
  return V / (dtype == BC2N_F32 ? 4 : 8) > BLOCK_VECS && rows < device_cus();
}

template <class T, int NV>
void block_go(hipStream_t st, const LogProbs& a) {
  const int vecs = a.V / Vec<T>::N, nt = (vecs + 64 * NV - 1) / (64 * NV) * 64;
  with_once(a, [&](auto once) {
    lp_block_kernel<T, NV, once><<<(unsigned)a.rows, nt, 0, st>>>(a);
  });
}

template <class T>
void both(hipStream_t st, const LogProbs& a, void* work) {
  if (short_row<T>(a.V)) return rows_launch<T, 3>(st, a);
  const int vecs = a.V / Vec<T>::N;
  if (vecs <= BLOCK_VECS / 2) block_go<T, 4>(st, a);
  else if (vecs <= BLOCK_VECS) block_go<T, 8>(st, a);
  else if (!in_parts(a.dtype, a.total, a.V)) {
    with_once(a, [&](auto once) {
      lp_both_kernel<T, once><<<(unsigned)a.rows, BOTH_NT, 0, st>>>(a);
    });
  } else {
    LogProbs b = a;
    Carver c(work);
    b.save = c.take<float>(4 * (size_t)a.rows);
    fwd<T>(st, b, c.p + c.off);
    bwd<T>(st, b);
  }
}

template <class F>
void by_type(int dtype, F f) {
  if (dtype == BC2N_F32) f(float());
  else if (dtype == BC2N_F16) f(h16());
  else f(bf16());
  launched();
}

}  // namespace

size_t logprobs_work_bytes(int dtype, int64_t rows, int V, int K) {
  if (rows <= 0 || V <= PART_MIN) return 0;
  const Split s = split_of(dtype, rows, V, K);
  Sizer z;
  if (s.splits > 1 || in_parts(dtype, rows, V)) z.take<float>(4 * (size_t)rows);
  if (s.splits > 1) parts_of(z, rows, s.splits, K);
  return z.off;
}

namespace {

// rows [r0, r0 + n) of a call
LogProbs slice(const LogProbs& a, int64_t r0, int64_t n) {
  const int64_t w = a.dtype == BC2N_F32 ? 4 : 2;
  auto bytes = [](auto*& p, int64_t by) {
    typedef std::remove_reference_t<decltype(p)> P;
    if (p) p = (P)((uintptr_t)p + (uintptr_t)by);
  };
  LogProbs b = a;
  b.rows = n;
  bytes(b.x, r0 * a.ld * w);
  bytes(b.d, r0 * a.d_ld * w);
  bytes(b.target, r0 * (a.target64 ? 8 : 4));
  for (auto** p : {&b.logp, &b.entropy}) bytes(*p, r0 * 4);
  for (auto** p : {&b.d_logp, &b.d_entropy}) bytes(*p, r0 * 4);
  bytes(b.top_logp, r0 * a.K * 4);
  bytes(b.top_index, r0 * a.K * 4);
  bytes(b.d_top, r0 * a.K * 4);
  bytes(b.save, r0 * 16);
  return b;
}

// A grid holds fewer than 2^32 threads, at most 1024 of them a row here.
constexpr int64_t SLICE = int64_t(1) << 21;
template <class F>
void by_slices(const LogProbs& a, F f) {
  for (int64_t r = 0; r < a.rows; r += SLICE)
    f(a.rows <= SLICE ? a : slice(a, r, std::min(SLICE, a.rows - r)));
}

}  // namespace

void logprobs_fwd(hipStream_t st, const LogProbs& a, void* work) {
  by_slices(a, [&](const LogProbs& b) {
    KTimed t("logprobs.fwd", st);
    by_type(a.dtype, [&](auto v) { fwd<decltype(v)>(st, b, work); });
  });
}

void logprobs_bwd(hipStream_t st, const LogProbs& a) {
  by_slices(a, [&](const LogProbs& b) {
    KTimed t("logprobs.bwd", st);
    by_type(a.dtype, [&](auto v) { bwd<decltype(v)>(st, b); });
  });
}

void logprobs_grad(hipStream_t st, const LogProbs& a, void* work) {
  by_slices(a, [&](const LogProbs& b) {
    KTimed t("logprobs.grad", st);
    by_type(a.dtype, [&](auto v) { both<decltype(v)>(st, b, work); });
  });
}

}  // namespace bc2n
