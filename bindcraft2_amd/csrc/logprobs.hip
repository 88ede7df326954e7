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
// a target at or past V makes its row's log-probability and gradient NaN.
//
// Rows are independent and every element is read once and (gradient) written
// once, a few operations a byte, so memory bounds all of it: the kernels only
// have to keep enough 16-byte loads in flight and the row on chip.
#include "logprobs.h"

#include "common.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

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

// The gradient at one element without the terms of single classes.
struct Cotangent {
  float m, logs, h, g, e;  // g: those of logp and the alternatives together
  __device__ __forceinline__ float at(float x) const {
    const float lp = (x - m) - logs;
    return -exp_f(lp) * fmaf(e, fmaxf(lp, FAR) + h, g);
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
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
}
__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int W>
__device__ __forceinline__ uint32_t group_umax(uint32_t v) {
  if constexpr (W >= 2) v = umax(v, dpp_u32<DPP_QUAD_1032>(v));
  if constexpr (W >= 4) v = umax(v, dpp_u32<DPP_QUAD_2301>(v));
  if constexpr (W >= 8) v = umax(v, dpp_u32<DPP_ROW_HALF_MIRROR>(v));
  if constexpr (W >= 16) v = umax(v, dpp_u32<DPP_ROW_MIRROR>(v));
  if constexpr (W >= 32) v = umax(v, (uint32_t)__shfl_xor((int)v, 16, 64));
  if constexpr (W >= 64) v = umax(v, (uint32_t)__shfl_xor((int)v, 32, 64));
  return v;
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

    if (MODE == 1 && a.K > 0) {
      uint32_t key[E];
#pragma unroll
      for (int i = 0; i < E; ++i) key[i] = i % VN >= skip[i / VN] ? order_key(x[i]) : 0u;
      const int lane0 = (threadIdx.x & 63) - l;
      for (int k = 0; k < a.K; ++k) {
        uint32_t best = 0;
#pragma unroll
        for (int i = 0; i < E; ++i) best = umax(best, key[i]);
        const uint32_t top = group_umax<W>(best);
        const uint64_t at = __ballot(best == top) >> lane0;
        if (l == __ffsll((unsigned long long)at) - 1) {
          // the first of this lane's elements that holds it
          int idx = 0;
          float v = 0.f;
#pragma unroll
          for (int i = E - 1; i >= 0; --i)
            if (key[i] == top) {
              idx = i;
              v = x[i];
            }
          int where = 0;
#pragma unroll
          for (int i = 0; i < E; ++i)
            if (i == idx) {
              key[i] = 0u;
              where = pos[i / VN] + i % VN;
            }
          if (mine) {
            const bool bad = is_nan(st.logs);
            a.top_logp[r * a.K + k] = bad ? st.logs : counts ? log_prob(st, v) : 0.f;
            a.top_index[r * a.K + k] = bad || !counts ? -1 : where;
          }
        }
      }
    }
  } else {
    const float4 s = reinterpret_cast<const float4*>(a.save)[r];
    st = RowStat{s.x, s.y, s.z, s.w};
  }

  if constexpr (MODE & 2) {
    const float g = a.d_logp ? a.d_logp[r] : 0.f;
    Cotangent c{st.m, st.logs, st.h, g, a.d_entropy ? a.d_entropy[r] : 0.f};
    if (MODE == 2 && a.d_top)
      for (int k = 0; k < a.K; ++k) c.g += a.d_top[r * a.K + k];
    if (a.d_logp && t >= a.V) c.g = __builtin_nanf("");
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
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VN; ++j)
        if (st.live == 0.f || !counts) d[i * VN + j] = 0.f;
      if (mine && skip[i] < VN) {
        if constexpr (VN == 1) o[pos[i]] = (T)d[i];
        else Vec<T>::store(o + pos[i], Vec<T>::pack(d + i * VN));
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Longer rows: a workgroup reads a row, or one of `splits` parts of it, 16
// bytes a lane and U vectors at a time, with a running maximum a lane (the
// sums are rescaled once a chunk of U * VN elements).
// ---------------------------------------------------------------------------
constexpr int U = 4;

// A wave's largest elements, the k-th in lane k (index -1: none yet); above
// `floor` an element belongs to them.  A wave takes its elements in ascending
// order of index, so a later one equal to the last kept is never better.
struct TopList {
  float v = NEG_INF;
  int i = -1;
  float floor = NEG_INF;

  // x: this lane's elements of one chunk, vector u starting at index i0 + u *
  // step; mx: their maximum
  template <int VN>
  __device__ __forceinline__ void take(const float (&x)[U * VN], float mx, int i0, int step, int K,
                                       bool first) {
    if (!__ballot(mx > floor)) return;
    const int lane = threadIdx.x & 63;
    if (first) {
      // K lanes hold an element as large as the K-th largest of the lanes'
      // maxima, so nothing below it can stay: without this bound the first
      // chunk would enter the list one by one
      float w = mx, t = NEG_INF;
      for (int k = 0; k < K; ++k) {
        t = group_max<64>(w);
        const uint64_t b = __ballot(w == t);
        if (b == 0) break;
        if (lane == __ffsll((unsigned long long)b) - 1) w = NEG_INF;
      }
      if (t > NEG_INF) {  // the float just below
        const int b = __builtin_bit_cast(int, t);
        floor = __builtin_bit_cast(float, t > 0.f ? b - 1 : t < 0.f ? b + 1 : (int)0x80000001);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      unsigned want = 0;
#pragma unroll
      for (int j = 0; j < VN; ++j) want |= x[u * VN + j] > floor ? 1u << j : 0u;
      for (uint64_t b = __ballot(want != 0); b; b = __ballot(want != 0)) {
        const int from = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)b) - 1);
        const int j = __ffs(want) - 1;
        float xv = x[u * VN];
#pragma unroll
        for (int q = 1; q < VN; ++q)
          if (j == q) xv = x[u * VN + q];
        const float cv = __builtin_bit_cast(
            float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, xv), from));
        const int ci = __builtin_amdgcn_readlane(i0 + u * step + j, from);
        if (lane == from) want &= want - 1;
        if (!(cv > floor)) continue;  // the list rose since
        const int before = __popcll(__ballot(i >= 0 && v >= cv));
        const float pv = __shfl_up(v, 1, 64);
        const int pi = __shfl_up(i, 1, 64);
        if (lane > before) {
          v = pv;
          i = pi;
        } else if (lane == before) {
          v = cv;
          i = ci;
        }
        floor = fmaxf(floor, __builtin_bit_cast(float, __builtin_amdgcn_readlane(
                                                           __builtin_bit_cast(int, v), K - 1)));
      }
    }
  }
};

// The chunk of U vectors a lane at `pos` (VN elements a lane a vector, NT
// lanes), elements at or past `hi` as -inf
template <class T, int NT>
__device__ __forceinline__ void read_chunk(const T* p, int64_t pos, int64_t hi,
                                           float (&x)[U * Vec<T>::N]) {
  constexpr int VN = Vec<T>::N;
  if (pos + (int64_t)U * NT * VN <= hi) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = Vec<T>::load(p + pos + (u * NT + (int)threadIdx.x) * VN);
#pragma unroll
    for (int u = 0; u < U; ++u) Vec<T>::unpack(raw[u], x + u * VN);
    return;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t at = pos + (u * NT + (int)threadIdx.x) * VN;
    if (at + VN <= hi) {
      Vec<T>::unpack(Vec<T>::load(p + at), x + u * VN);
    } else {
#pragma unroll
      for (int j = 0; j < VN; ++j) x[u * VN + j] = at + j < hi ? (float)p[at + j] : NEG_INF;
    }
  }
}

// Sum of a part of a row over the workgroup's NT lanes, in every lane
template <int NT>
__device__ __forceinline__ Stat join(Stat q, float (*buf)[4]) {
  q.raise(group_max<64>(q.m));
  q.s = group_sum<64>(q.s);
  q.u = group_sum<64>(q.u);
  const int w = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) {
    buf[w][0] = q.m;
    buf[w][1] = q.s;
    buf[w][2] = q.u;
  }
  __syncthreads();
  float m = buf[0][0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, buf[i][0]);
  Stat all;
  all.m = m;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) {
    Stat o;
    o.m = buf[i][0];
    o.s = buf[i][1];
    o.u = buf[i][2];
    o.raise(m);
    all.s += o.s;
    all.u += o.u;
  }
  return all;
}

// Of n candidates (cv, ci; ci < 0: none) in LDS the rank of candidate c among
// all, by value and then by index
__device__ __forceinline__ int rank_of(const float* cv, const int* ci, int n, int c) {
  const float v = cv[c];
  const int i = ci[c];
  int rank = 0;
  for (int o = 0; o < n; ++o)
    rank += ci[o] >= 0 && (cv[o] > v || (cv[o] == v && ci[o] < i));
  return rank;
}

// Writes the K best of n candidates in LDS as row r's alternatives; where
// there are fewer than K above -inf, the first -inf elements of the row follow.
template <class T, int NT>
__device__ __forceinline__ void write_tops(const LogProbs& a, int64_t r, const RowStat& st,
                                           const float* cv, const int* ci, int n) {
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
    if (ci[c] < 0) continue;
    const int k = rank_of(cv, ci, n, c);
    if (k < a.K) {
      ov[k] = log_prob(st, cv[c]);
      oi[k] = ci[c];
    }
  }
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int have = 0;
    for (int c = lane; c < n; c += 64) have += ci[c] >= 0;
    have = (int)group_sum<64>((float)have);  // at most 1024: exact
    const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
    for (int64_t b = 0; have < a.K && b < a.V; b += 64) {
      const bool gone = b + lane < a.V && (float)p[b + lane] == NEG_INF;
      const uint64_t m = __ballot(gone);
      const int k = have + __popcll(m & ((1ull << lane) - 1));
      if (gone && k < a.K) {
        ov[k] = NEG_INF;
        oi[k] = (int)(b + lane);
      }
      have += __popcll(m);
    }
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
  float4* stat = nullptr;  // [rows][splits]
  float* v = nullptr;      // [rows][splits][K]
  int* i = nullptr;
};
template <class A>
Parts parts_of(A& c, int64_t rows, int splits, int K) {
  Parts p;
  const size_t n = (size_t)rows * splits;
  p.stat = c.template take<float4>(n);
  p.v = c.template take<float>(n * (K > 0 ? K : 1));
  p.i = c.template take<int>(n * (K > 0 ? K : 1));
  return p;
}

constexpr int FWD_NT = 256;

template <class T, bool TOP>
__global__ __launch_bounds__(FWD_NT) void lp_stream_kernel(LogProbs a, int splits, int64_t part,
                                                           Parts parts) {
  constexpr int VN = Vec<T>::N, NT = FWD_NT, NW = NT / 64;
  __shared__ float buf[NW][4];
  __shared__ float cv[TOP ? NW * LP_MAX_TOP : 1];
  __shared__ int ci[TOP ? NW * LP_MAX_TOP : 1];
  const int64_t r = blockIdx.x / splits;
  const int sp = blockIdx.x % splits;
  const int64_t t = target_of(a, r);
  if (t < 0) {  // left out: not read
    if (splits == 1) {
      if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
      if (TOP) no_tops(a, r, NT);
    }
    return;
  }
  const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
  const int64_t lo = sp * part, hi = min((int64_t)a.V, lo + part);
  Stat q;
  TopList top;
  for (int64_t pos = lo; pos < hi; pos += (int64_t)U * NT * VN) {
    float x[U * VN];
    read_chunk<T, NT>(p, pos, hi, x);
    float mx = x[0];
#pragma unroll
    for (int i = 1; i < U * VN; ++i) mx = fmaxf(mx, x[i]);
    q.raise(fmaxf(q.m, mx));
#pragma unroll
    for (int i = 0; i < U * VN; ++i) q.add(x[i]);
    if (TOP) top.take<VN>(x, mx, (int)pos + threadIdx.x * VN, NT * VN, a.K, pos == lo);
  }
  if (TOP) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (lane < a.K) {
      cv[w * a.K + lane] = top.v;
      ci[w * a.K + lane] = top.i;
    }
  }
  const Stat all = join<NT>(q, buf);  // its barrier also covers cv, ci
  if (splits == 1) {
    const RowStat st = finish(all, true);
    if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
    if (TOP) write_tops<T, NT>(a, r, st, cv, ci, NW * a.K);
    return;
  }
  const int64_t o = r * splits + sp;
  if (threadIdx.x == 0) parts.stat[o] = make_float4(all.m, all.s, all.u, 0.f);
  if (TOP) {
    const int n = NW * a.K;
    int have = 0;
    for (int c = 0; c < n; ++c) have += ci[c] >= 0;
    for (int c = threadIdx.x; c < n; c += NT) {
      if (ci[c] < 0) continue;
      const int k = rank_of(cv, ci, n, c);
      if (k < a.K) {
        parts.v[o * a.K + k] = cv[c];
        parts.i[o * a.K + k] = ci[c];
      }
    }
    for (int k = have + threadIdx.x; k < a.K; k += NT) parts.i[o * a.K + k] = -1;
  }
}

// Joins the parts of a row.
constexpr int MAX_SPLITS = 32;
template <class T>
__global__ __launch_bounds__(FWD_NT) void lp_join_kernel(LogProbs a, int splits, Parts parts) {
  __shared__ float cv[MAX_SPLITS * LP_MAX_TOP];
  __shared__ int ci[MAX_SPLITS * LP_MAX_TOP];
  const int64_t r = blockIdx.x;
  const int64_t t = target_of(a, r);
  if (t < 0) {
    if (threadIdx.x == 0) write_row<T>(a, r, finish(Stat(), false), -1);
    no_tops(a, r, FWD_NT);
    return;
  }
  const int lane = threadIdx.x & 63;
  Stat q;
  if (lane < splits) {  // each wave by itself
    const float4 s = parts.stat[r * splits + lane];
    q.m = s.x;
    q.s = s.y;
    q.u = s.z;
  }
  q.raise(group_max<64>(q.m));
  q.s = group_sum<64>(q.s);
  q.u = group_sum<64>(q.u);
  const RowStat st = finish(q, true);
  if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
  if (a.K > 0) {
    const int n = splits * a.K;
    for (int c = threadIdx.x; c < n; c += FWD_NT) {
      cv[c] = parts.v[r * n + c];
      ci[c] = parts.i[r * n + c];
    }
    __syncthreads();
    write_tops<T, FWD_NT>(a, r, st, cv, ci, n);
  }
}

// The gradient of [lo, hi) of row r from its statistics.  The classes with
// terms of their own (the target and the alternatives) are computed first, by
// one wave, and stored last: a row may be written in place.
template <class T, int NT>
__device__ __forceinline__ void write_gradient(const LogProbs& a, int64_t r, int64_t t,
                                               const RowStat& st, int K, int64_t lo, int64_t hi) {
  constexpr int VN = Vec<T>::N;
  T* o = reinterpret_cast<T*>(a.d) + r * a.d_ld;
  if (st.live == 0.f || t < 0) {
    const float zero[VN] = {};
    for (int64_t at = lo + threadIdx.x * VN; at < hi; at += NT * VN) {
      if (at + VN <= hi) Vec<T>::store(o + at, Vec<T>::pack(zero));
      else
        for (int64_t j = at; j < hi; ++j) o[j] = (T)0.f;
    }
    return;
  }
  const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
  const int lane = threadIdx.x & 63;
  const float g = a.d_logp ? a.d_logp[r] : 0.f;
  Cotangent c{st.m, st.logs, st.h, g, a.d_entropy ? a.d_entropy[r] : 0.f};
  // lane k < K: alternative k; lane K: the target
  int64_t at = -1;
  float own = 0.f;
  if (a.d_top && lane < K) {
    at = a.top_index[r * K + lane];
    own = a.d_top[r * K + lane];
  }
  c.g += group_sum<64>(own);
  if (lane == K && a.d_logp) {
    at = t;
    own = g;
  }
  if (a.d_logp && t >= a.V) c.g = __builtin_nanf("");
  if (a.d_top && a.d_logp) {  // a target among the alternatives has both terms
    const uint64_t same = __ballot(lane < K && at == t);
    if (lane < K && at == t) own += g;
    if (lane == K && same) at = -1;
  }
  const bool special = threadIdx.x < 64 && at >= lo && at < hi;
  T sv = (T)0.f;
  if (special) sv = (T)(c.at((float)p[at]) + own);
  __syncthreads();
  for (int64_t pos = lo; pos < hi; pos += (int64_t)U * NT * VN) {
    float x[U * VN];
    read_chunk<T, NT>(p, pos, hi, x);
#pragma unroll
    for (int i = 0; i < U * VN; ++i) x[i] = c.at(x[i]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t b = pos + (u * NT + (int)threadIdx.x) * VN;
      if (b + VN <= hi) {
        Vec<T>::store(o + b, Vec<T>::pack(x + u * VN));
      } else {
#pragma unroll
        for (int j = 0; j < VN; ++j)
          if (b + j < hi) o[b + j] = (T)x[u * VN + j];
      }
    }
  }
  __syncthreads();
  if (special) o[at] = sv;
}

template <class T>
__global__ __launch_bounds__(FWD_NT) void lp_gradient_kernel(LogProbs a, int splits, int64_t part) {
  const int64_t r = blockIdx.x / splits, lo = (blockIdx.x % splits) * part;
  const float4 s = reinterpret_cast<const float4*>(a.save)[r];
  write_gradient<T, FWD_NT>(a, r, target_of(a, r), RowStat{s.x, s.y, s.z, s.w}, a.K, lo,
                            min((int64_t)a.V, lo + part));
}

// A workgroup takes a whole row twice, the second time out of the caches.
constexpr int BOTH_NT = 1024;
template <class T>
__global__ __launch_bounds__(BOTH_NT) void lp_both_kernel(LogProbs a) {
  constexpr int VN = Vec<T>::N, NT = BOTH_NT;
  __shared__ float buf[NT / 64][4];
  const int64_t r = blockIdx.x;
  const int64_t t = target_of(a, r);
  Stat q;
  if (t >= 0) {
    const T* p = reinterpret_cast<const T*>(a.x) + r * a.ld;
    for (int64_t pos = 0; pos < a.V; pos += (int64_t)U * NT * VN) {
      float x[U * VN];
      read_chunk<T, NT>(p, pos, a.V, x);
      float mx = x[0];
#pragma unroll
      for (int i = 1; i < U * VN; ++i) mx = fmaxf(mx, x[i]);
      q.raise(fmaxf(q.m, mx));
#pragma unroll
      for (int i = 0; i < U * VN; ++i) q.add(x[i]);
    }
  }
  const RowStat st = finish(join<NT>(q, buf), t >= 0);
  if (threadIdx.x == 0) write_row<T>(a, r, st, a.target ? t : -1);
  __syncthreads();  // the target's logit is read before its place is written
  write_gradient<T, NT>(a, r, t, st, 0, 0, a.V);
}

// ---------------------------------------------------------------------------
// Which kernel
// ---------------------------------------------------------------------------
constexpr int ROW_MAX = 1024;  // longest row held by a group of lanes

// Parts a row is read in: as many as fill the card, each at least one chunk
// of a workgroup.
int splits_of(int dtype, int64_t rows, int V) {
  if (V <= ROW_MAX) return 1;
  const int64_t chunk = (int64_t)U * FWD_NT * (dtype == BC2N_F32 ? 4 : 8);
  const int64_t fill = (2 * (int64_t)device_cus() + rows - 1) / rows;
  int64_t s = (V + chunk - 1) / chunk;
  if (s > fill) s = fill;
  if (s > MAX_SPLITS) s = MAX_SPLITS;
  return s < 1 ? 1 : (int)s;
}
int64_t part_of(int V, int splits) {
  // a multiple of 64 elements, so that parts begin like the row
  const int64_t p = (V + splits - 1) / splits;
  return (p + 63) / 64 * 64;
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
  if (a.V < N) rows_go<T, 1, 8, 1, MODE>(st, a);
  else if (vecs <= 4) rows_go<T, N, 4, 1, MODE>(st, a);
  else if (vecs <= 8) rows_go<T, N, 8, 1, MODE>(st, a);
  else if (vecs <= 16) rows_go<T, N, 16, 1, MODE>(st, a);
  else if (vecs <= 32) rows_go<T, N, 32, 1, MODE>(st, a);
  else if (vecs <= 64) rows_go<T, N, 64, 1, MODE>(st, a);
  else if (N == 8 || vecs <= 128) rows_go<T, N, 64, 2, MODE>(st, a);
  else if constexpr (N == 4) rows_go<T, N, 64, 4, MODE>(st, a);
}

template <class T>
void fwd(hipStream_t st, const LogProbs& a, void* work) {
  if (a.V <= ROW_MAX) return rows_launch<T, 1>(st, a);
  const int s = splits_of(a.dtype, a.rows, a.V);
  Parts parts;
  if (s > 1) {
    Carver c(work);
    parts = parts_of(c, a.rows, s, a.K);
  }
  const unsigned grid = (unsigned)(a.rows * s);
  if (a.K > 0) lp_stream_kernel<T, true><<<grid, FWD_NT, 0, st>>>(a, s, part_of(a.V, s), parts);
  else lp_stream_kernel<T, false><<<grid, FWD_NT, 0, st>>>(a, s, part_of(a.V, s), parts);
  if (s > 1) lp_join_kernel<T><<<(unsigned)a.rows, FWD_NT, 0, st>>>(a, s, parts);
}

template <class T>
void bwd(hipStream_t st, const LogProbs& a) {
  if (a.V <= ROW_MAX) return rows_launch<T, 2>(st, a);
  const int s = splits_of(a.dtype, a.rows, a.V);
  lp_gradient_kernel<T><<<(unsigned)(a.rows * s), FWD_NT, 0, st>>>(a, s, part_of(a.V, s));
}

template <class T>
void both(hipStream_t st, const LogProbs& a, void* work) {
  if (a.V <= ROW_MAX) return rows_launch<T, 3>(st, a);
  if (splits_of(a.dtype, a.rows, a.V) == 1) {
    lp_both_kernel<T><<<(unsigned)a.rows, BOTH_NT, 0, st>>>(a);
    return;
  }
  LogProbs b = a;
  Carver c(work);
  b.save = c.take<float>(4 * (size_t)a.rows);
  fwd<T>(st, b, c.p + c.off);
  bwd<T>(st, b);
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
  if (rows <= 0) return 0;
  const int s = splits_of(dtype, rows, V);
  if (s == 1) return 0;
  Sizer z;
  z.take<float>(4 * (size_t)rows);
  parts_of(z, rows, s, K);
  return z.off;
}

void logprobs_fwd(hipStream_t st, const LogProbs& a, void* work) {
  if (a.rows == 0) return;
  KTimed t("logprobs.fwd", st);
  by_type(a.dtype, [&](auto v) { fwd<decltype(v)>(st, a, work); });
}

void logprobs_bwd(hipStream_t st, const LogProbs& a) {
  if (a.rows == 0) return;
  KTimed t("logprobs.bwd", st);
  by_type(a.dtype, [&](auto v) { bwd<decltype(v)>(st, a); });
}

void logprobs_grad(hipStream_t st, const LogProbs& a, void* work) {
  if (a.rows == 0) return;
  KTimed t("logprobs.grad", st);
  by_type(a.dtype, [&](auto v) { both<decltype(v)>(st, a, work); });
}

}  // namespace bc2n
