// Lists of gradients g: norm = sqrt(sum over all tensors of g^2), the clipped
// gradients c g with c = 1 where norm < max_norm and max_norm / norm
// elsewhere, and Adam with decoupled weight decay on the clipped gradients:
//
//   m <- b1 m + (1 - b1) c g,  v <- b2 v + (1 - b2) (c g)^2
//   p <- p - lr ((m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + decay p)
//
// All of it streams: a few operations an element, so memory bounds it.  A
// list is cut into chunks of one tensor, a workgroup each, whatever the
// tensors' sizes, so a list of thousands costs the launches of one tensor.
// The squares are summed in f64: an f32 gradient's square can pass f32's
// range, and the chunks' sums are added in one fixed order, so a norm is the
// same every time.  (Its cost is hidden: a read-only pass with f32 squares is
// as long.)  Measured on 4080 tensors of 88 M f32 elements: the squares' pass
// 60 us (5.9 TB/s), the clipping's 108 (6.5, part of it read from the Infinity
// Cache), Adam's 437 (5.6); a copy reaches 5.0 to 6.5 TB/s on this card.
#include "optim.h"

#include "common.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace bc2n {

namespace {

constexpr int NT = 256;          // threads of a chunk's workgroup
constexpr int64_t CHUNK = 8192;  // elements of a chunk, at least
constexpr uint32_t MANY = 16384; // chunks of a list beyond which they grow
constexpr int ONE_NT = 1024;     // threads of a small list's one workgroup
// elements of a small list.  One workgroup against three launches, in a graph,
// one tensor of f32: clip of 4480 elements 3.6 against 7.0 us, of 32 k 5.6
// against 7.6, of 61 k 9.2 against 8.0; clipped Adam of 4480 4.6 against 9.2, of
// 16 k 8.3 against 11.9.  Three tensors: clip of 12 k 5.3 against 8.0, of 33 k
// 7.3 against 7.9; clipped Adam of 12 k 7.6 against 9.2.  The workgroup takes a
// list's tensors one after another, so it falls behind from six to eight of them
// (six of 1000: clip 6.3 against 6.7 us, clipped Adam 8.6 against 7.1; eight 7.7
// against 6.8 and 10.7 against 7.2; 32 of 100 22.5 against 6.8 and 36 against
// 7.2): this rule, by elements alone, is for lists of a few states.
constexpr int64_t SMALL_CLIP = 32768, SMALL_ADAM = 12288;
// The Infinity Cache holds 256 MiB.  A list whose operands pass it goes by it
// once (nontemporal loads and stores) and, after the norm, from its end: what
// the norm's pass read last is still in the cache.  88 M f32 gradients: clip
// 218 -> 175 us a call, Adam 575 -> 507; a list of 2 M, which stays in the
// cache, is faster with ordinary accesses (clip 12.5 against 13.5 us, Adam
// 18.5 against 20.8).
constexpr int64_t CACHE = int64_t(256) << 20;

// What the later kernels of a call need of the norm, at the front of its
// scratch; the chunks' sums follow.
struct Scales {
  float c, pre;   // clipping factor c * pre: pre = 2^-64 keeps a small c normal
  float lr;       // learning rate / (1 - b1^t)
  float inv2;     // 1 / sqrt(1 - b2^t)
  float decay;    // learning rate * weight decay
};
constexpr size_t SCALES = 256;

// The entries with the launch (a short list) or in a device table; of(b) is
// that of workgroup b's chunk, the same for every lane.
struct InlineList {
  ListEntry e[LIST_INLINE];
  int count;
  int64_t chunk;
  __device__ __forceinline__ ListEntry of(uint32_t b) const {
    const int lane = threadIdx.x & 63;
    const bool begun = lane < count && e[lane < LIST_INLINE ? lane : 0].chunk0 <= b;
    return e[__popcll(__ballot(begun)) - 1];
  }
};
struct TableList {
  const ListEntry* table;
  const int32_t* owner;
  int64_t chunk;
  __device__ __forceinline__ ListEntry of(uint32_t b) const {
    return table[__builtin_amdgcn_readfirstlane(owner[b])];
  }
};

template <class F>
__device__ __forceinline__ void by_type(int type, F f) {
  if (type == BC2N_F32) f(float());
  else if (type == BC2N_F16) f(h16());
  else f(bf16());
}

// sum of a value over the workgroup's N threads, in every thread, in one order
template <int N>
__device__ __forceinline__ double block_sum(double v, double* buf) {
#pragma unroll
  for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o, 64);
  if ((threadIdx.x & 63) == 0) buf[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0;
#pragma unroll
  for (int i = 0; i < N / 64; ++i) s += buf[i];
  __syncthreads();
  return s;
}

// sum of squares of [lo, hi) by N threads
template <class T, int N>
__device__ __forceinline__ double squares(const T* p, int64_t lo, int64_t hi) {
  constexpr int VN = Vec<T>::N, U = sizeof(T) == 4 ? 8 : 4;
  double s[2] = {0, 0};
  int64_t at = lo + (int64_t)threadIdx.x * VN;
  for (; at + (int64_t)(U - 1) * N * VN + VN <= hi; at += (int64_t)U * N * VN) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = Vec<T>::load(p + at + (int64_t)u * N * VN);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VN];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < VN; ++i) s[i & 1] = fma((double)x[i], (double)x[i], s[i & 1]);
    }
  }
  for (; at < hi; at += (int64_t)N * VN) {
    if (at + VN <= hi) {
      float x[VN];
      Vec<T>::unpack(Vec<T>::load(p + at), x);
#pragma unroll
      for (int i = 0; i < VN; ++i) s[i & 1] = fma((double)x[i], (double)x[i], s[i & 1]);
    } else {
      for (int64_t j = at; j < hi; ++j) s[0] = fma((double)(float)p[j], (double)(float)p[j], s[0]);
    }
  }
  return s[0] + s[1];
}

template <class L>
__global__ __launch_bounds__(NT) void list_squares_kernel(L l, double* part) {
  __shared__ double buf[NT / 64];
  const ListEntry e = l.of(blockIdx.x);
  const int64_t lo = (int64_t)(blockIdx.x - e.chunk0) * l.chunk, hi = min(e.n, lo + l.chunk);
  double s = 0;
  by_type(e.g_type, [&](auto t) {
    typedef decltype(t) T;
    s = squares<T, NT>(reinterpret_cast<const T*>(e.g), lo, hi);
  });
  s = block_sum<NT>(s, buf);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// A step's scalars.  lr, inv2, decay: Scales's of the host's learning rate and
// step; device: {learning rate, step} to compute them from instead.
struct StepArgs {
  double max_norm = 0;
  Scales host{1.f, 1.f, 0.f, 0.f, 0.f};
  const float* device = nullptr;
  double beta1 = 0, beta2 = 0, decay = 0;
};

// 1 - b^t, exact where b^t is near 1
__host__ __device__ __forceinline__ double one_less_power(double b, double t) {
  return b > 0 ? -expm1(t * log(b)) : 1.0;
}
__host__ __device__ __forceinline__ void schedule(Scales& s, double lr, double t, double beta1,
                                                  double beta2, double decay) {
  s.lr = (float)(lr / one_less_power(beta1, t));
  s.inv2 = (float)(1.0 / sqrt(one_less_power(beta2, t)));
  s.decay = (float)(lr * decay);
}
__device__ __forceinline__ Scales scales(const StepArgs& a, double norm) {
  Scales s = a.host;
  if (a.device) schedule(s, a.device[0], a.device[1], a.beta1, a.beta2, a.decay);
  // not below: also where the norm is NaN, which makes every gradient NaN
  const double c = a.max_norm > 0 && !(norm < a.max_norm) ? a.max_norm / norm : 1.0;
  s.pre = c < 0x1p-100 ? 0x1p-64f : 1.f;
  s.c = (float)(c < 0x1p-100 ? c * 0x1p64 : c);
  return s;
}

// the chunks' sums (none: no norm was asked for) -> norm and scales
__global__ __launch_bounds__(ONE_NT) void list_scales_kernel(const double* part, uint32_t n,
                                                             StepArgs a, float* norm, Scales* out) {
  __shared__ double buf[ONE_NT / 64];
  double s = 0;
  constexpr uint32_t U = 8;  // loads in flight
  uint32_t i = threadIdx.x;
  for (; i + (U - 1) * ONE_NT < n; i += U * ONE_NT) {
    double x[U];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) x[u] = part[i + u * ONE_NT];
#pragma unroll
    for (uint32_t u = 0; u < U; ++u) s += x[u];
  }
  for (; i < n; i += ONE_NT) s += part[i];
  s = sqrt(block_sum<ONE_NT>(s, buf));
  if (threadIdx.x == 0) {
    if (norm) *norm = (float)s;
    if (out) *out = scales(a, s);
  }
}

template <class T, int N, bool ONCE>
__device__ __forceinline__ void scale_range(const T* p, T* o, const Scales& s, int64_t lo,
                                            int64_t hi) {
  constexpr int VN = Vec<T>::N, U = 4;
  int64_t at = lo + (int64_t)threadIdx.x * VN;
  for (; at + (int64_t)(U - 1) * N * VN + VN <= hi; at += (int64_t)U * N * VN) {
    u32x4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = Vec<T>::template load<ONCE>(p + at + (int64_t)u * N * VN);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[VN];
      Vec<T>::unpack(raw[u], x);
#pragma unroll
      for (int i = 0; i < VN; ++i) x[i] = x[i] * s.pre * s.c;
      Vec<T>::template store<ONCE>(o + at + (int64_t)u * N * VN, Vec<T>::pack(x));
    }
  }
  for (; at < hi; at += (int64_t)N * VN) {
    if (at + VN <= hi) {
      float x[VN];
      Vec<T>::unpack(Vec<T>::load(p + at), x);
#pragma unroll
      for (int i = 0; i < VN; ++i) x[i] = x[i] * s.pre * s.c;
      Vec<T>::store(o + at, Vec<T>::pack(x));
    } else {
      for (int64_t j = at; j < hi; ++j) o[j] = (T)((float)p[j] * s.pre * s.c);
    }
  }
}

template <int N, bool ONCE>
__device__ __forceinline__ void clip_range(const ListEntry& e, const Scales& s, int64_t lo,
                                           int64_t hi) {
  by_type(e.g_type, [&](auto t) {
    typedef decltype(t) T;
    scale_range<T, N, ONCE>(reinterpret_cast<const T*>(e.g), reinterpret_cast<T*>(e.g_out), s, lo, hi);
  });
}

template <class L, bool ONCE>
__global__ __launch_bounds__(NT) void list_clip_kernel(L l, const Scales* s) {
  const uint32_t b = ONCE ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const ListEntry e = l.of(b);
  const int64_t lo = (int64_t)(b - e.chunk0) * l.chunk;
  clip_range<NT, ONCE>(e, *s, lo, min(e.n, lo + l.chunk));
}

struct AdamArgs {
  float b1, b1c, b2, b2c, eps;  // b1c = 1 - b1
};

__device__ __forceinline__ void adam_one(const AdamArgs& a, const Scales& s, float& p, float g,
                                         float& m, float& v) {
  g = g * s.pre * s.c;
  m = fmaf(a.b1, m, a.b1c * g);
  v = fmaf(a.b2, v, a.b2c * g * g);
  const float move = m / fmaf(sqrtf(v), s.inv2, a.eps);
  p = p - fmaf(s.lr, move, s.decay * p);
}

template <class P, class G, int N, bool ONCE>
__device__ __forceinline__ void adam_typed(const ListEntry& e, const AdamArgs& a, const Scales& s,
                                           int64_t lo, int64_t hi) {
  const P* p = reinterpret_cast<const P*>(e.p);
  const G* g = reinterpret_cast<const G*>(e.g);
  P* po = reinterpret_cast<P*>(e.p_out);
  for (int64_t at = lo + (int64_t)threadIdx.x * 4; at < hi; at += (int64_t)N * 4) {
    if (at + 4 <= hi) {
      float x[4], y[4], m[4], v[4];
      Few<P, 4>::template load<ONCE>(p + at, x);
      Few<G, 4>::template load<ONCE>(g + at, y);
      Few<float, 4>::template load<ONCE>(e.m + at, m);
      Few<float, 4>::template load<ONCE>(e.v + at, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) adam_one(a, s, x[i], y[i], m[i], v[i]);
      Few<P, 4>::template store<ONCE>(po + at, x);
      Few<float, 4>::template store<ONCE>(e.m_out + at, m);
      Few<float, 4>::template store<ONCE>(e.v_out + at, v);
    } else {
      for (int64_t j = at; j < hi; ++j) {
        float x = (float)p[j], m = e.m[j], v = e.v[j];
        adam_one(a, s, x, (float)g[j], m, v);
        po[j] = (P)x;
        e.m_out[j] = m;
        e.v_out[j] = v;
      }
    }
  }
}

template <int N, bool ONCE>
__device__ __forceinline__ void adam_range(const ListEntry& e, const AdamArgs& a, const Scales& s,
                                           int64_t lo, int64_t hi) {
  by_type(e.p_type, [&](auto p) {
    by_type(e.g_type,
            [&](auto g) { adam_typed<decltype(p), decltype(g), N, ONCE>(e, a, s, lo, hi); });
  });
}

template <class L, bool ONCE>
__global__ __launch_bounds__(NT) void list_adam_kernel(L l, AdamArgs a, const Scales* sp) {
  const uint32_t b = ONCE ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const ListEntry e = l.of(b);
  const int64_t lo = (int64_t)(b - e.chunk0) * l.chunk;
  adam_range<NT, ONCE>(e, a, *sp, lo, min(e.n, lo + l.chunk));
}

// A small list in one workgroup: norm, scales and the writes in one launch.
// CLIP, ADAM: which of them follows the norm.
template <bool CLIP, bool ADAM>
__global__ __launch_bounds__(ONE_NT) void list_small_kernel(InlineList in, StepArgs sa, AdamArgs a,
                                                            float* norm) {
  __shared__ double buf[ONE_NT / 64];
  double s = 0;
  if (norm || sa.max_norm > 0)
    for (int i = 0; i < in.count; ++i)
      by_type(in.e[i].g_type, [&](auto t) {
        typedef decltype(t) T;
        s += squares<T, ONE_NT>(reinterpret_cast<const T*>(in.e[i].g), 0, in.e[i].n);
      });
  s = sqrt(block_sum<ONE_NT>(s, buf));
  if (norm && threadIdx.x == 0) *norm = (float)s;
  if (!CLIP && !ADAM) return;
  const Scales sc = scales(sa, s);
  for (int i = 0; i < in.count; ++i) {
    if (CLIP) clip_range<ONE_NT, false>(in.e[i], sc, 0, in.e[i].n);
    if (ADAM) adam_range<ONE_NT, false>(in.e[i], a, sc, 0, in.e[i].n);
  }
}

void launched() { hip_check(hipGetLastError(), "list launch"); }

// Device memory of lists that are gone, for the next ones: freeing a list
// makes no HIP call, so it may happen at any time (by a garbage collector
// while a stream is captured, say).
struct Tables {
  std::mutex mu;
  std::vector<DeviceBlock> free;
  DeviceBlock take(size_t n) {
    std::lock_guard<std::mutex> lk(mu);
    int dev = 0;
    BC2N_HIP(hipGetDevice(&dev));
    for (size_t i = 0; i < free.size(); ++i)
      if (free[i].n >= n && free[i].device == dev) {
        // a launch that reads the old table may still be queued
        BC2N_HIP(hipDeviceSynchronize());
        const DeviceBlock b = free[i];
        free.erase(free.begin() + i);
        return b;
      }
    DeviceBlock b;
    BC2N_HIP(hipMalloc(reinterpret_cast<void**>(&b.p), n));
    b.n = n;
    b.device = dev;
    return b;
  }
  void give(DeviceBlock b) {
    std::lock_guard<std::mutex> lk(mu);
    free.push_back(b);
  }
};
Tables& tables() {
  static Tables* t = new Tables;  // outlives every list
  return *t;
}

int width(int type) { return type == BC2N_F32 ? 4 : 2; }

// One operand's memory
struct Range {
  uintptr_t a, b;
  int of;     // tensor
  bool out;
};

InlineList inline_of(const TensorList& l) {
  InlineList a;
  a.count = (int)l.entries.size();
  a.chunk = l.chunk;
  std::copy(l.entries.begin(), l.entries.end(), a.e);
  return a;
}
// f with the list as the kernels of more than one workgroup take it
template <class F>
void with_list(const TensorList& l, F f) {
  if (l.dev) f(TableList{l.dev, l.dev_owner, l.chunk});
  else f(inline_of(l));
}
// and with whether its operands are more than the caches hold
template <class F>
void with_list_once(const TensorList& l, F f) {
  with_list(l, [&](const auto& a) {
    if (l.bytes > CACHE) f(a, std::true_type());
    else f(a, std::false_type());
  });
}
bool small(const TensorList& l) { return !l.dev && l.total <= (l.adam ? SMALL_ADAM : SMALL_CLIP); }

StepArgs clip_args(double max_norm) {
  StepArgs a;
  a.max_norm = max_norm;
  return a;
}

double* sums(void* work) {
  return reinterpret_cast<double*>(reinterpret_cast<char*>(work) + SCALES);
}

// norm (where `want`) and, where `out`, the scales
void reduce(hipStream_t st, const TensorList& l, bool want, const StepArgs& sa, float* norm,
            Scales* out, void* work) {
  if (want) {
    KTimed t("list.squares", st);
    with_list(l, [&](const auto& a) {
      list_squares_kernel<<<l.chunks, NT, 0, st>>>(a, sums(work));
    });
    launched();
  }
  KTimed t("list.scales", st);
  list_scales_kernel<<<1, ONE_NT, 0, st>>>(sums(work), want ? l.chunks : 0, sa, norm, out);
  launched();
}

}  // namespace

TensorList::TensorList(std::vector<ListEntry> all, bool clips_, bool adam_)
    : clips(clips_), adam(adam_) {
  std::vector<Range> r;
  for (size_t i = 0; i < all.size(); ++i) {
    ListEntry& e = all[i];
    const std::string at = "tensor " + std::to_string(i);
    if (all.size() > (size_t(1) << 22)) throw std::invalid_argument("list: too many tensors");
    if (e.n < 0) throw std::invalid_argument("list: " + at + " has a negative size");
    if (e.n > (int64_t(1) << 40)) throw std::invalid_argument("list: " + at + " is too large");
    if (e.n == 0) continue;
    auto put = [&](const void* p, int w, bool out, const char* what) {
      if (!p) throw std::invalid_argument("list: " + at + " has a null " + what);
      const uintptr_t u = reinterpret_cast<uintptr_t>(p);
      if (u % (uintptr_t)w) throw std::invalid_argument("list: " + at + ": unaligned " + what);
      r.push_back({u, u + (uintptr_t)e.n * w, (int)i, out});
    };
    // an operand and its output, which may be the operand itself
    auto pair = [&](const void* p, const void* o, int w, const char* what) {
      if (p != o) put(p, w, false, what);
      put(o, w, true, (std::string(what) + " output").c_str());
    };
    const int gw = width(e.g_type), pw = width(e.p_type);
    if (clips) pair(e.g, e.g_out, gw, "gradient");
    else put(e.g, gw, false, "gradient");
    if (adam) {
      pair(e.p, e.p_out, pw, "parameter");
      pair(e.m, e.m_out, 4, "first moment");
      pair(e.v, e.v_out, 4, "second moment");
    }
    entries.push_back(e);
    total += e.n;
    bytes += e.n * (adam ? gw + 2 * pw + 16 : clips ? 2 * gw : gw);
  }
  // An output shares memory with nothing else: workgroups run in any order.
  // (Inputs may share memory.)
  std::sort(r.begin(), r.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
  uintptr_t end = 0, out_end = 0;  // of the ranges before, and of the outputs among them
  for (const Range& x : r) {
    if (x.a < out_end || (x.out && x.a < end))
      throw std::invalid_argument("list: an operand of tensor " + std::to_string(x.of) +
                                  " shares memory with an output");
    end = std::max(end, x.b);
    if (x.out) out_end = std::max(out_end, x.b);
  }

  chunk = CHUNK;
  for (;;) {
    uint64_t c = 0;
    for (const ListEntry& e : entries) c += (uint64_t)((e.n + chunk - 1) / chunk);
    if (c <= MANY + entries.size()) break;
    chunk *= 2;
  }
  std::vector<int32_t> owner;
  for (size_t i = 0; i < entries.size(); ++i) {
    entries[i].chunk0 = chunks;
    const uint32_t c = (uint32_t)((entries[i].n + chunk - 1) / chunk);
    chunks += c;
    if (entries.size() > (size_t)LIST_INLINE) owner.insert(owner.end(), c, (int32_t)i);
  }
  if (entries.size() > (size_t)LIST_INLINE) {
    const size_t eb = (entries.size() * sizeof(ListEntry) + 255) & ~size_t(255);
    block_ = tables().take(eb + owner.size() * sizeof(int32_t));
    dev = reinterpret_cast<ListEntry*>(block_.p);
    dev_owner = reinterpret_cast<int32_t*>(block_.p + eb);
    try {
      BC2N_HIP(hipMemcpy(dev, entries.data(), entries.size() * sizeof(ListEntry),
                         hipMemcpyHostToDevice));
      BC2N_HIP(hipMemcpy(dev_owner, owner.data(), owner.size() * sizeof(int32_t),
                         hipMemcpyHostToDevice));
    } catch (...) {
      tables().give(block_);
      throw;
    }
  }
}

TensorList::~TensorList() {
  magic = 0;
  if (block_.p && !kept_) tables().give(block_);
}

size_t TensorList::work_bytes() const {
  return small(*this) ? 0 : SCALES + (size_t)chunks * sizeof(double);
}

void grad_norm(hipStream_t st, const TensorList& l, float* norm, void* work) {
  const StepArgs sa = clip_args(0);
  if (small(l)) {
    KTimed t("list.small", st);
    list_small_kernel<false, false><<<1, ONE_NT, 0, st>>>(inline_of(l), sa, AdamArgs{}, norm);
    return launched();
  }
  reduce(st, l, true, sa, norm, nullptr, work);
}

void grad_clip(hipStream_t st, const TensorList& l, float max_norm, float* norm, void* work) {
  const StepArgs sa = clip_args(max_norm);
  if (small(l)) {
    KTimed t("list.small", st);
    list_small_kernel<true, false><<<1, ONE_NT, 0, st>>>(inline_of(l), sa, AdamArgs{}, norm);
    return launched();
  }
  Scales* sc = reinterpret_cast<Scales*>(work);
  reduce(st, l, true, sa, norm, sc, work);
  KTimed t("list.clip", st);
  with_list_once(l, [&](const auto& a, auto once) {
    list_clip_kernel<std::decay_t<decltype(a)>, once><<<l.chunks, NT, 0, st>>>(a, sc);
  });
  launched();
}

void adam_step(hipStream_t st, const TensorList& l, const AdamScalars& s, float* norm,
               void* work) {
  StepArgs sa = clip_args(s.max_norm);
  if (s.device) {
    sa.device = s.device;
    sa.beta1 = s.beta1;
    sa.beta2 = s.beta2;
    sa.decay = s.decay;
  } else {
    schedule(sa.host, s.lr, (double)s.step, s.beta1, s.beta2, s.decay);
    if (!std::isfinite(sa.host.lr) || !std::isfinite(sa.host.decay))
      throw std::invalid_argument(
          "adam_step: the learning rate over 1 - beta1^step, or by weight_decay, is past f32");
  }
  const AdamArgs aa{(float)s.beta1, (float)(1 - s.beta1), (float)s.beta2, (float)(1 - s.beta2),
                    (float)s.eps};
  if (small(l)) {
    KTimed t("list.small", st);
    list_small_kernel<false, true><<<1, ONE_NT, 0, st>>>(inline_of(l), sa, aa, norm);
    return launched();
  }
  Scales* sc = reinterpret_cast<Scales*>(work);
  reduce(st, l, norm || s.max_norm > 0, sa, norm, sc, work);
  KTimed t("list.adam", st);
  with_list_once(l, [&](const auto& a, auto once) {
    list_adam_kernel<std::decay_t<decltype(a)>, once><<<l.chunks, NT, 0, st>>>(a, aa, sc);
  });
  launched();
}

}  // namespace bc2n
