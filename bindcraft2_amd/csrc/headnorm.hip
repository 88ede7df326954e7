// Norms of queries and keys for each head with the position rotation in the
// same pass.  Per head x[D] with weight w[D] and pairs (i, j) of its first R
// elements -- (i, i + R/2), or interleaved (2 i, 2 i + 1) -- at angle
// t = position * freq[i]:
//
//   y = x r w,  r = (mean x^2 + eps)^-1/2
//   (y_i, y_j) -> (y_i cos t - y_j sin t, y_j cos t + y_i sin t)
//
// and, with g the cotangent turned back by -t and n = x r:
//
//   dw = sum over tokens and heads of g n,   dx = r (g w - n mean(g w n))
//
// Every element is read once and written once (the gradient reads two), some
// ten operations each, so memory bounds it: 16-byte loads, a head in the
// registers of a few lanes, and the angles, which all heads of a token share,
// made once for all of them.  16384 tokens of 40 heads of 128 bfloat16: 76 us, 4.4
// TB/s (when it took 98: vectors of 8 bytes 114, stores past the caches 111); the
// gradient of 8191 tokens of 20 heads of 64 f32 25 us, 5.0 TB/s, and 4 of its join.
//
// A lane holds units of two vectors of N elements that rotate into each other
// (or, past R, two vectors side by side; interleaved, one run of 2 N), N the
// widest of 16 bytes and less that R/2 and D - R are made of; W lanes hold a
// head, 64 / W heads at a time in a wave, and a wave walks a token's heads
// with its lanes' units, and so their cosines and weights, unchanged.
#include "headnorm.h"

#include "common.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

#include <algorithm>

namespace bc2n {

namespace {

constexpr int NT = 256;      // threads of a workgroup
constexpr int WAVES = NT / 64;

template <class T>
__device__ __forceinline__ T* at(const HeadView& v, int64_t t, int h) {
  return (T*)v.p + t * v.st + h * v.sh;
}

// sums over the aligned groups of W lanes, W known at run time
__device__ __forceinline__ float sum_lanes(float v, int W) {
  if (W >= 2) v += dpp_mov<DPP_QUAD_1032>(v);
  if (W >= 4) v += dpp_mov<DPP_QUAD_2301>(v);
  if (W >= 8) v += dpp_mov<DPP_ROW_HALF_MIRROR>(v);
  if (W >= 16) v += dpp_mov<DPP_ROW_MIRROR>(v);
  if (W >= 32) v += __shfl_xor(v, 16, 64);
  if (W >= 64) v += __shfl_xor(v, 32, 64);
  return v;
}

// Where a lane's unit lies in its head.
struct Unit {
  int a, b;     // first elements of its two vectors
  int pair;     // its first pair's frequency
  int turned;   // pairs of it that rotate (the first ones)
  bool live;
};
template <int N>
__device__ __forceinline__ Unit unit_of(const HeadNorm& p, int u) {
  Unit r;
  r.live = 2 * N * u < p.width;
  const int half = p.rotated / 2;
  if (p.interleaved) {
    r.a = 2 * N * u;
    r.b = r.a + N;
    r.pair = N * u;
    r.turned = min(max(half - r.pair, 0), N);
  } else if (N * u < half) {
    r.a = N * u;
    r.b = r.a + half;
    r.pair = N * u;
    r.turned = N;
  } else {
    r.a = 2 * N * u;  // past the rotated ones: 2 N u = R + 2 N (u - half / N)
    r.b = r.a + N;
    r.pair = 0;
    r.turned = 0;
  }
  return r;
}

// cos and sin of position * freq.  The product is taken in 64 bits (at a position of
// 10^6 one of 32 would lose a tenth of a radian), in turns: the frequency in turns and
// its product with the position round to 53 bits each, 2^-52 of the turns with the
// constant's own rounding.  Whole turns leave there; the rest, in f32, is good to 2^-26
// of one.  Then
// quarters of a turn, and the series of both for an eighth at most, which end
// below 2^-29 (a library call for both, with its own reductions, takes twice the
// instructions).
template <int N>
struct Turn {
  double f[N];  // a lane's frequencies in turns; 0 where it does not rotate
  float c[N], s[N];
  __device__ __forceinline__ void init(const HeadNorm& p, const Unit& u) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      f[i] = i < u.turned ? (double)p.freq[u.pair + i] * 0.15915494309189535 : 0.0;
  }
  __device__ __forceinline__ double position(const HeadNorm& p, int64_t t) const {
    if (!p.pos) return 0.0;
    return p.pos64 ? (double)reinterpret_cast<const int64_t*>(p.pos)[t]
                   : (double)reinterpret_cast<const int32_t*>(p.pos)[t];
  }
  __device__ __forceinline__ void make(double pos) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const double turns = pos * f[i];
      const float t = (float)(turns - rint(turns)), q = rintf(4.f * t), r = fmaf(4.f, t, -q), z = r * r;
      // of r quarters: powers of pi / 2 over factorials
      float sn = fmaf(z, 1.6044118e-4f, -4.6817541e-3f);
      sn = fmaf(z, sn, 7.9692626e-2f);
      sn = fmaf(z, sn, -6.4596410e-1f);
      sn = r * fmaf(z, sn, 1.5707963e0f);
      float cs = fmaf(z, -2.5202042e-5f, 9.1926028e-4f);
      cs = fmaf(z, cs, -2.0863481e-2f);
      cs = fmaf(z, cs, 2.5366951e-1f);
      cs = fmaf(z, cs, -1.2337005e0f);
      cs = fmaf(z, cs, 1.f);
      const int k = (int)q;
      const float a = k & 1 ? cs : sn, b = k & 1 ? sn : cs;
      s[i] = k & 2 ? -a : a;
      c[i] = (k + 1) & 2 ? -b : b;
    }
  }
};

// (a, b) turned by t, or by -t (BACK); interleaved pairs lie side by side.
template <int N, bool BACK>
__device__ __forceinline__ void rotate(const Turn<N>& t, bool interleaved, float* a, float* b) {
  auto turn = [&](float& x, float& y, int i) {
    const float c = t.c[i], s = BACK ? -t.s[i] : t.s[i], u = x, v = y;
    x = fmaf(u, c, -(v * s));
    y = fmaf(v, c, u * s);
  };
  if (interleaved) {
    if constexpr (N == 1) {
      turn(a[0], b[0], 0);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        turn(a[2 * i], a[2 * i + 1], i);
        turn(b[2 * i], b[2 * i + 1], N / 2 + i);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) turn(a[i], b[i], i);
  }
}

template <int N>
__device__ __forceinline__ void load_weight(const HeadNorm& p, int which, const Unit& u, float (&a)[N],
                                            float (&b)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = b[i] = 0.f;
  if (!u.live || !p.heads[which]) return;
  auto load = [&](auto type) {
    typedef decltype(type) T;
    Few<T, N>::template load<false>(reinterpret_cast<const T*>(p.weight[which]) + u.a, a);
    Few<T, N>::template load<false>(reinterpret_cast<const T*>(p.weight[which]) + u.b, b);
  };
  if (p.weight_dtype == BC2N_F32) load(float());
  else if (p.weight_dtype == BC2N_F16) load(h16());
  else load(bf16());
}

// Waves walk the tokens; each takes `per` rounds of 64 / W heads of a token, the
// blockIdx.y-th share of them, first the queries' `q_rounds`, then the keys'.  The
// first round's loads are issued ahead of the angles, each other's ahead of the
// work before it.
template <class T, int N>
__global__ __launch_bounds__(NT) void headnorm_fwd_kernel(HeadNorm p, int W, int q_rounds, int rounds, int per) {
  const int lane = threadIdx.x & 63;
  const Unit u = unit_of<N>(p, lane & (W - 1));
  const int step = 64 / W, mine = lane / W;
  const int r0 = blockIdx.y * per, r1 = min(rounds, r0 + per);
  Turn<N> turn;
  turn.init(p, u);
  const float inv = 1.f / (float)p.width;
  float wa[2][N], wb[2][N];
#pragma unroll
  for (int k = 0; k < 2; ++k) load_weight<N>(p, k, u, wa[k], wb[k]);
  for (int64_t t = (int64_t)blockIdx.x * WAVES + (threadIdx.x >> 6); t < p.tokens;
       t += (int64_t)gridDim.x * WAVES) {
    float na[N] = {}, nb[N] = {};
    // the head of a lane in round r, the same tensor for all lanes
    auto fetch = [&](int r) __attribute__((always_inline)) {
      if (r >= r1) return;
      auto from = [&](const HeadView& v, int h, int heads) __attribute__((always_inline)) {
        if (h >= heads || !u.live) return;
        const T* x = at<const T>(v, t, h);
        Few<T, N>::template load<false>(x + u.a, na);
        Few<T, N>::template load<false>(x + u.b, nb);
      };
      if (r < q_rounds) from(p.x[0], r * step + mine, p.heads[0]);
      else from(p.x[1], (r - q_rounds) * step + mine, p.heads[1]);
    };
    auto round = [&](int r, const HeadView& v, int h, int heads, const float (&wa)[N], const float (&wb)[N])
                     __attribute__((always_inline)) {
      float a[N], b[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] = na[i];
        b[i] = nb[i];
      }
      fetch(r + 1);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(a[i], a[i], fmaf(b[i], b[i], s));
      const float scale = rsqrtf(fmaf(sum_lanes(s, W), inv, p.eps));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        a[i] = a[i] * scale * wa[i];
        b[i] = b[i] * scale * wb[i];
      }
      rotate<N, false>(turn, p.interleaved, a, b);
      if (h < heads && u.live) {
        T* y = at<T>(v, t, h);
        Few<T, N>::template store<false>(y + u.a, a);
        Few<T, N>::template store<false>(y + u.b, b);
      }
    };
    fetch(r0);
    turn.make(turn.position(p, t));
    for (int r = r0; r < r1; ++r) {
      if (r < q_rounds) round(r, p.out[0], r * step + mine, p.heads[0], wa[0], wb[0]);
      else round(r, p.out[1], (r - q_rounds) * step + mine, p.heads[1], wa[1], wb[1]);
    }
  }
}

// Waves walk the tokens; each keeps its lanes' sums of g n for both weights,
// which a workgroup adds in LDS and leaves in partial [workgroup][2][D].
template <class T, int N>
__global__ __launch_bounds__(NT) void headnorm_bwd_kernel(HeadNorm p, int W, float* partial) {
  extern __shared__ float sums[];  // [waves][64 / W][2][D]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Unit u = unit_of<N>(p, lane & (W - 1));
  const int step = 64 / W;
  const float inv = 1.f / (float)p.width;
  float da[2][N] = {}, db[2][N] = {};
  float wa[2][N], wb[2][N];
#pragma unroll
  for (int k = 0; k < 2; ++k) load_weight<N>(p, k, u, wa[k], wb[k]);
  Turn<N> turn;
  turn.init(p, u);
  for (int64_t t = (int64_t)blockIdx.x * WAVES + wave; t < p.tokens; t += (int64_t)gridDim.x * WAVES) {
    turn.make(turn.position(p, t));
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      for (int h = lane / W; h < p.heads[k]; h += step) {
        float a[N] = {}, b[N] = {}, ga[N] = {}, gb[N] = {};
        if (u.live) {
          const T* x = at<const T>(p.x[k], t, h);
          const T* d = at<const T>(p.d[k], t, h);
          Few<T, N>::template load<false>(x + u.a, a);
          Few<T, N>::template load<false>(x + u.b, b);
          Few<T, N>::template load<false>(d + u.a, ga);
          Few<T, N>::template load<false>(d + u.b, gb);
        }
        rotate<N, true>(turn, p.interleaved, ga, gb);
        float s = 0.f, m = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s = fmaf(a[i], a[i], fmaf(b[i], b[i], s));
        const float r = rsqrtf(fmaf(sum_lanes(s, W), inv, p.eps));
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a[i] *= r;
          b[i] *= r;
          da[k][i] = fmaf(ga[i], a[i], da[k][i]);
          db[k][i] = fmaf(gb[i], b[i], db[k][i]);
          ga[i] *= wa[k][i];
          gb[i] *= wb[k][i];
          m = fmaf(ga[i], a[i], fmaf(gb[i], b[i], m));
        }
        m = sum_lanes(m, W) * inv;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          a[i] = r * fmaf(-a[i], m, ga[i]);
          b[i] = r * fmaf(-b[i], m, gb[i]);
        }
        if (u.live) {
          T* y = at<T>(p.out[k], t, h);
          Few<T, N>::template store<false>(y + u.a, a);
          Few<T, N>::template store<false>(y + u.b, b);
        }
      }
    }
  }
  const int D = p.width;
  if (u.live) {
    float* mine = sums + (wave * step + lane / W) * 2 * D;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        mine[k * D + u.a + i] = da[k][i];
        mine[k * D + u.b + i] = db[k][i];
      }
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < 2 * D; e += NT) {
    double s = 0;
    for (int i = 0; i < WAVES * step; ++i) s += sums[i * 2 * D + e];
    partial[(int64_t)blockIdx.x * 2 * D + e] = (float)s;
  }
}

// d_weight from the workgroups' partial sums, in a fixed order: 4 columns a
// workgroup, 64 threads a column.
__global__ __launch_bounds__(NT) void headnorm_join_kernel(HeadNorm p, const float* partial, int parts) {
  __shared__ double sums[4][65];
  const int c = threadIdx.x & 3, r = threadIdx.x >> 2;
  const int e = blockIdx.x * 4 + c, D = p.width;
  double s = 0;
  if (e < 2 * D) {
#pragma unroll 8
    for (int i = r; i < parts; i += 64) s += partial[(int64_t)i * 2 * D + e];
  }
  sums[c][r] = s;
  __syncthreads();
  if (threadIdx.x < 4 && blockIdx.x * 4 + threadIdx.x < 2 * D) {
    const int col = blockIdx.x * 4 + threadIdx.x;
    s = 0;
    for (int i = 0; i < 64; ++i) s += sums[threadIdx.x][i];
    const int k = col >= D;
    if (p.d_weight[k]) p.d_weight[k][col - k * D] = (float)s;
  }
}

int bwd_blocks(int64_t tokens) {
  // two workgroups a CU of the largest grids: more leave the join more rows
  return (int)std::min<int64_t>((tokens + WAVES - 1) / WAVES, 512);
}

// lanes a head
int lanes(const HeadNorm& a, int N) {
  int W = 1;
  while (W * 2 * N < a.width) W *= 2;
  return W;
}

template <class F, class T>
void by_vector(int N, T, F f) {
  if constexpr (sizeof(T) == 2) {
    if (N == 8) return f(T(), std::integral_constant<int, 8>());
  }
  if (N == 4) f(T(), std::integral_constant<int, 4>());
  else if (N == 2) f(T(), std::integral_constant<int, 2>());
  else f(T(), std::integral_constant<int, 1>());
}
template <class F>
void by_type(const HeadNorm& a, F f) {
  const int N = headnorm_vector(a.dtype, a.width, a.rotated, a.interleaved);
  if (a.dtype == BC2N_F32) by_vector(N, float(), f);
  else if (a.dtype == BC2N_F16) by_vector(N, h16(), f);
  else by_vector(N, bf16(), f);
  hip_check(hipGetLastError(), "headnorm launch");
}

}  // namespace

int headnorm_vector(int dtype, int width, int rotated, int interleaved) {
  for (int n = dtype == BC2N_F32 ? 4 : 8; n; n /= 2) {
    const bool fits = width % (2 * n) == 0 && (interleaved || (rotated / 2) % n == 0);
    if (fits) return width / (2 * n) <= 64 ? n : 0;
  }
  return 0;
}

size_t headnorm_work_bytes(int64_t tokens, int width) {
  return tokens > 0 ? (size_t)bwd_blocks(tokens) * 2 * width * 4 : 0;
}

void headnorm_fwd(hipStream_t st, const HeadNorm& a) {
  if (a.tokens == 0) return;
  KTimed kt("headnorm.fwd", st);
  by_type(a, [&](auto v, auto n) {
    const int W = lanes(a, n), step = 64 / W;
    const int q_rounds = (a.heads[0] + step - 1) / step, rounds = q_rounds + (a.heads[1] + step - 1) / step;
    // All heads by one wave make the angles once; few tokens spread their heads.
    int per = rounds;
    while (per > 1 && a.tokens * ((rounds + per - 1) / per) < 8 * (int64_t)device_cus()) per = (per + 1) / 2;
    // eight workgroups a CU, what its registers hold twice over
    const int64_t blocks = std::min<int64_t>((a.tokens + WAVES - 1) / WAVES, 8 * (int64_t)device_cus());
    const dim3 grid((unsigned)blocks, (rounds + per - 1) / per);
    headnorm_fwd_kernel<decltype(v), n><<<grid, NT, 0, st>>>(a, W, q_rounds, rounds, per);
  });
}

void headnorm_bwd(hipStream_t st, const HeadNorm& a, void* work) {
  KTimed kt("headnorm.bwd", st);
  const int blocks = bwd_blocks(a.tokens), D = a.width;
  float* partial = reinterpret_cast<float*>(work);
  if (a.tokens) by_type(a, [&](auto v, auto n) {
    const int W = lanes(a, n);
    const size_t lds = (size_t)WAVES * (64 / W) * 2 * D * 4;
    headnorm_bwd_kernel<decltype(v), n><<<blocks, NT, lds, st>>>(a, W, partial);
  });
  headnorm_join_kernel<<<(2 * D + 3) / 4, NT, 0, st>>>(a, partial, a.tokens ? blocks : 0);
  hip_check(hipGetLastError(), "headnorm launch");
}

}  // namespace bc2n
