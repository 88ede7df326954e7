// Attention of packed sequences: sequence b has queries q_off[b] ..
// q_off[b+1] - 1 and keys k_off[b] .. of two buffers of tokens, G = heads /
// kv_heads query heads share a head of keys and values, and
//
//   S = scale q k^T over the keys that a query sees, P = softmax(S), o = P v,
//   lse = log sum e^S;  D = sum_d (do o),  dS = P (do v^T - D),
//   dv = P^T do,  dq = scale dS k,  dk = scale dS^T q  (summed over the group).
//
// A causal query i of m sees keys j <= i + n - m.  A row that sees none has
// o = 0, lse = -inf and no gradient.
//
// The G heads of a group are rows of one problem, row r = i G + g, so that
// they share every key tile that is staged and a few queries still fill a
// tile.  All products are v_mfma_f32_32x32x16, arranged so that a result is
// the next product's operand as it lies in the registers:
//
//   forward, dq:  S^T[key][row] = K Q^T, a lane owns one row: row maxima and
//                 sums are a lane's own but for its other half's (lane ^ 32),
//                 and rescaling o^T[d][row] += V^T P^T is one factor a lane
//   dk, dv:       S[row][key] = Q K^T, a lane owns one key:
//                 dv^T[d][key] += do^T P,  dk^T[d][key] += Q^T dS
//
// The result of a product holds rows 8 (r/4) + 4 (l/32) + r%4 in register r of
// lane l; as the operand of the next one those are its contraction's slots, and
// the other operand, a column of the row-major tile in LDS, is read in the same
// order with two ds_read_b64_tr_b16.
//
// P and dS are rounded to the operands' type, which the second products' instructions
// take: half a step of a term, as the result's own rounding is of the sum.  Outputs of
// prompts are 2.1e-3 off 64 bits with it, 1.6e-3 with their own rounding alone, gradients
// 2.4e-3 and 1.7e-3 (bfloat16; binary16 an eighth); P and dS as two halves each would
// double those products.  Scores, maxima, sums, lse, D and all sums of products are f32.
//
// Tiles are copied global -> LDS directly through buffer descriptors whose
// bounds turn what lies past a sequence or past the width into zeros.  A copy
// fills LDS in lane order, so the source address carries the swizzle (fswz)
// that keeps both the 16-byte row reads and the transposed reads off each
// other's banks.
#include "packattn.h"

#include "common.h"
#include "packrows.h"
#include "runtime.h"
#include "vec.h"

#include "../../include/bc2n.h"

#include <algorithm>
#include <type_traits>

namespace bc2n {

namespace {

typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef const __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef const __attribute__((address_space(3))) f32x4 lds_f32x4;

constexpr int NT = 256, WAVES = 4;
constexpr int BN = 64;  // keys of a staged tile (rows of one in the dk, dv kernel)
constexpr float NEG_INF = -__builtin_inff();

template <class T>
struct Half;
template <>
struct Half<h16> {
  typedef h16 V2 __attribute__((ext_vector_type(2)));
  // Probabilities are kept 2^SHIFT times as large, within binary16's range
  // beside a reference that lags the maximum by at most LAG: small ones stay
  // normal numbers.
  static constexpr float SHIFT = 7.f;
  static constexpr bool SCALED = true;  // dS needs a scale (below)
  static constexpr uint32_t EXPONENT = 0x7c00;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a),
                                                  __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
  }
};
template <>
struct Half<bf16> {
  typedef bf16 V2 __attribute__((ext_vector_type(2)));
  static constexpr float SHIFT = 0.f;
  static constexpr bool SCALED = false;
  static constexpr uint32_t EXPONENT = 0x7f80;
  static __device__ __forceinline__ f32x16 mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};
// The running reference of a row's exponents is raised only where the maximum
// has passed it by this much (log2): the products hold what lies between.
constexpr float LAG = 8.f;

// two f32 rounded to nearest even, in one register
template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const f32x2 v = {a, b};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename Half<T>::V2));
}
// registers 8 s .. 8 s + 7 of a product as the operand of the next one
template <class T>
__device__ __forceinline__ u32x4 pack8(const f32x16& v, int s) {
  u32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = pack2<T>(v[8 * s + 2 * i], v[8 * s + 2 * i + 1]);
  return r;
}

__device__ __forceinline__ float exp2_f(float x) { return __builtin_amdgcn_exp2f(x); }

// v of lane l ^ 32
__device__ __forceinline__ float other_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v),
                                                  __builtin_bit_cast(int, v), false, false);
  return fmaxf(__builtin_bit_cast(float, (int)r[0]), __builtin_bit_cast(float, (int)r[1]));
}
__device__ __forceinline__ float other_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(int, v),
                                                  __builtin_bit_cast(int, v), false, false);
  return __builtin_bit_cast(float, (int)r[0]) + __builtin_bit_cast(float, (int)r[1]);
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform64(int64_t v) {
  return (int64_t)((uint64_t)(uint32_t)uniform((int)v) |
                   (uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32);
}

// ---------------------------------------------------------------- sequences
struct Seq {
  int64_t q0, k0;  // first tokens
  int lq, lk;      // its queries and keys
  int have;        // tokens of the searched side that are its own, in it or not
};

// First token of entry s of `off`: 0, off[0], ..., off[B], n -- the tokens before the
// first sequence and behind the last are sequences without queries or keys.
// Offsets past the tokens are cut to them.
__device__ __forceinline__ int start_of(const int32_t* off, int s, int B, int64_t n) {
  return s == 0 ? 0 : (int)min((int64_t)max(off[min(s, B + 1) - 1], 0), n);
}

// Tile x of the rows of all sequences, `unit` rows a token and `tile` rows a
// tile: sequence s's tiles take the numbers from floor(start * unit / tile) + s
// on, which leaves each of them enough.  Sets s, returns the tile's index in it
// (past its last one, and with offsets that fall below 0, for no tile).
__device__ __forceinline__ int64_t find_tile(const int32_t* off, int B, int64_t n, int unit, int tile,
                                             int64_t x, int& s) {
  const int lane = threadIdx.x & 63;
  int lo = 0, count = B + 2;
  auto first = [&](int e) { return (int64_t)start_of(off, e, B, n) * unit / tile + e; };
  while (count > 1) {  // 64 entries at a time
    const int step = (count + 63) / 64, e = lo + lane * step;
    const bool below = lane * step < count && first(min(e, B + 1)) <= x;
    const int passed = max(__popcll(__ballot(below)) - 1, 0) * step;
    lo += passed;
    count = min(step, count - passed);
  }
  s = uniform(lo);
  return uniform64(x - first(s));
}

// entry s: a sequence, or the tokens outside all
__device__ __forceinline__ Seq sequence(const PackedAttn& a, int s, bool keys) {
  const int B = a.sequences;
  Seq r = {};
  const int32_t* off = keys ? a.k_off : a.q_off;
  const int64_t n = keys ? a.k_tokens : a.q_tokens;
  const int from = start_of(off, s, B, n);
  const int to = s == B + 1 ? (int)n : start_of(off, s + 1, B, n);
  r.have = max(to - from, 0);
  (keys ? r.k0 : r.q0) = from;
  if (s == 0 || s == B + 1) return r;
  const int other = start_of(keys ? a.q_off : a.k_off, s, B, keys ? a.q_tokens : a.k_tokens);
  const int end = start_of(keys ? a.q_off : a.k_off, s + 1, B, keys ? a.q_tokens : a.k_tokens);
  (keys ? r.q0 : r.k0) = other;
  int lq = keys ? max(end - other, 0) : r.have, lk = keys ? r.have : max(end - other, 0);
  if (a.q_len) lq = min(lq, max(a.q_len[s - 1], 0));
  if (a.k_len) lk = min(lk, max(a.k_len[s - 1], 0));
  r.lq = lq;
  r.lk = lk;
  return r;
}

__device__ __forceinline__ int64_t lane64(int64_t v, int lane) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)v, lane) |
                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32);
}
__device__ __forceinline__ Seq lane_seq(const Seq& s, int lane) {
  Seq r;
  r.q0 = lane64(s.q0, lane);
  r.k0 = lane64(s.k0, lane);
  r.lq = __builtin_amdgcn_readlane(s.lq, lane);
  r.lk = __builtin_amdgcn_readlane(s.lk, lane);
  r.have = __builtin_amdgcn_readlane(s.have, lane);
  return r;
}

// Workgroups of `tiles` tiles for each head of keys: XCD b % 8 takes heads of
// one class mod gcd(kv_heads, 8), so that the tiles which read one head's keys
// and values share an L2.
struct Place {
  int head;
  int64_t tile;  // < 0: none
};
__host__ __device__ inline int head_classes(int kv_heads) {
  return kv_heads % 8 == 0 ? 8 : kv_heads % 4 == 0 ? 4 : kv_heads % 2 == 0 ? 2 : 1;
}
__device__ __forceinline__ Place place(int kv_heads, int64_t tiles) {
  const int g = head_classes(kv_heads), share = NUM_XCD / g;
  const int64_t per = (tiles + share - 1) / share;
  const int64_t b = blockIdx.x, x = b % NUM_XCD, j = b / NUM_XCD;
  Place r;
  r.head = (int)(x % g + g * (j / per));
  r.tile = (j % per) * share + x / g;
  if (r.tile >= tiles) r.tile = -1;
  return r;
}
unsigned place_grid(int kv_heads, int64_t tiles) {
  const int g = head_classes(kv_heads), share = NUM_XCD / g;
  const int64_t grid = NUM_XCD * (int64_t)(kv_heads / g) * ((tiles + share - 1) / share);
  // 512 threads each: a launch has fewer than 2^32
  if (grid >= int64_t(1) << 23) throw std::invalid_argument("attention: too many tiles for one call");
  return (unsigned)grid;
}

// over a wave, by DPP within 16 lanes: what a search waits for is its latency
template <class F>
__device__ __forceinline__ int wave_fold(int v, F f) {
  auto step = [&](auto ctrl) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, decltype(ctrl)::value, 0xF, 0xF, false));
  };
  step(std::integral_constant<int, DPP_QUAD_1032>());
  step(std::integral_constant<int, DPP_QUAD_2301>());
  step(std::integral_constant<int, DPP_ROW_HALF_MIRROR>());
  step(std::integral_constant<int, DPP_ROW_MIRROR>());
  return f(f(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
           f(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
}
__device__ __forceinline__ int wave_add(int v) {
  return wave_fold(v, [](int a, int b) { return a + b; });
}

// Tile x of 128 keys of all sequences, those with the most rows to see them first:
// a launch's workgroups are a few times what runs at once, and a long causal
// sequence's first tiles begun late would run alone at its end (packed prompts of
// 140 .. 3435 tokens: dk and dv 672 -> 579 us; the rows' tiles, whose sequences
// share an L2's keys in their own order, lost 2% by it).  A tile's weight falls
// by the same step in all sequences, so the x-th heaviest of all is found by
// bisecting the weight, every lane counting its sequence's tiles above it.
// Whole sequences, and more than 64 entries, are taken in their order.
__device__ __forceinline__ bool find_work(const PackedAttn& a, int64_t x, int& s, int64_t& t) {
  const int lane = threadIdx.x & 63, entries = a.sequences + 2;
  if (!a.causal || entries > 64) {
    t = find_tile(a.k_off, a.sequences, a.k_tokens, 1, 128, x, s);
    return t >= 0;
  }
  int n = 0, top = 0;  // a lane's sequence: tiles, weight of the heaviest
  if (lane < entries) {
    const Seq q = sequence(a, lane, true);
    n = ((a.fill ? q.have : q.lk) + 127) / 128;
    top = q.lk;
  }
  auto above = [&](int v) -> int {
    const int64_t d = (int64_t)top - v;
    return d <= 0 ? 0 : (int)min((int64_t)n, (d + 127) >> 7);
  };
  if (x >= wave_add(n)) return false;
  int hi = wave_fold(top, [](int a, int b) { return max(a, b); });
  // all tiles weigh more than lo; none more than hi
  int lo = wave_fold(top - n * 128, [](int a, int b) { return min(a, b); }) - 1;
  while (hi - lo > 1) {
    const int v = (int)(((int64_t)hi + lo) >> 1);
    if (wave_add(above(v)) > x) lo = v;
    else hi = v;
  }
  // tile x weighs hi: the x - (those above) -th of that weight
  int k = above(hi), rest = (int)x;
  const int same = above(hi - 1) - k;
  int before = same;
#pragma unroll
  for (int i = 1; i < 64; i *= 2) {
    const int o = __shfl_up(before, i, 64);
    if (lane >= i) before += o;
  }
  before -= same;
  rest -= wave_add(k);
  const unsigned long long at = __ballot(before <= rest && rest < before + same);
  if (!at) return false;
  s = uniform(__ffsll(at) - 1);
  t = __builtin_amdgcn_readlane(k, s) + rest - __builtin_amdgcn_readlane(before, s);
  return true;
}

// The order of the instructions around the products: left to itself the compiler
// reads an operand, waits for it and multiplies, which leaves the matrix cores
// idle for each read's latency.  order<M, N>: N instructions of kind M come next.
enum Kind { VALU = 0x2, MFMA = 0x8, LDS_READ = 0x100 };
template <int M, int N>
__device__ __forceinline__ void order() {
  if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(M, N, 0);
}

// ------------------------------------------------------------- tiles in LDS
// 16-byte chunk c of row r of a [rows][DP] tile lies at chunk c ^ fswz(r).
// A row read takes one chunk of 16 rows at a time and a transposed read 64
// bytes of 4 rows: over all 64 banks in both, whatever DP.
template <int DP>
__device__ __forceinline__ int fswz(int r) {
  if (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  if (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
  return (r >> 2) & 3;
}

__device__ __forceinline__ unsigned lds_addr(const void* p) {
  return (unsigned)(size_t)((const __attribute__((address_space(3))) unsigned char*)p);
}

// 1 KB global -> LDS, 16 bytes a lane; zeros where the offset is past the
// descriptor's bounds.
__device__ __forceinline__ void copy16(unsigned voff, u32x4 rsrc, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff),
               "s"(rsrc), "s"(lds)
               : "memory", "m0");
}
__device__ __forceinline__ u32x4 descriptor(uint64_t p) {
  return u32x4{(uint32_t)uniform((int)p), (uint32_t)uniform((int)(p >> 32)) & 0xffffu, 0x7fffffffu, 0x00027000u};
}
constexpr unsigned NOWHERE = 0x80000000u;  // past every descriptor's bounds

// a wave's copies done but the last N
template <int N>
__device__ __forceinline__ void wait_copies() {
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// all of a wave's LDS reads done: what they read may be written again
__device__ __forceinline__ void wait_reads() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// all of a wave's copies and LDS reads done, and every wave here
__device__ __forceinline__ void wait_all_and_sync() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// A wave's copies of a [ROWS][DP] tile by W waves: piece w + W i.
template <int DP, int ROWS, int W>
struct TileCopy {
  static constexpr int PIECES = ROWS * DP * 2 / 1024, PER = (PIECES + W - 1) / W;
  // waves past the pieces have none
  static __device__ __forceinline__ bool any(int i, int wave) { return PIECES % W == 0 || wave + W * i < PIECES; }
  static constexpr int CPR = DP / 8;  // chunks a row
  // row and element of lane's chunk of piece i
  static __device__ __forceinline__ int row(int i, int wave, int lane) {
    return ((wave + W * i) * 64 + lane) / CPR;
  }
  static __device__ __forceinline__ int elem(int i, int wave, int lane) {
    return (lane % CPR ^ fswz<DP>(row(i, wave, lane))) * 8;
  }
  static __device__ __forceinline__ unsigned dst(int i, int wave) { return (wave + W * i) * 1024; }
};

// A lane's LDS addresses of the operands in a [rows][DP] tile at address 0; a tile
// and the rows in it are constants beside them, which the reads take as offsets.
template <int DP>
struct Operands {
  unsigned row_[DP / 16], column_[DP / 32][2];
  __device__ __forceinline__ void init(unsigned base, int lane) {
    const int r = lane & 31, m = lane & 15;
#pragma unroll
    for (int ks = 0; ks < DP / 16; ++ks) {
      row_[ks] = base + r * (DP * 2) + (((2 * ks + (lane >> 5)) ^ fswz<DP>(r)) * 16);
      asm volatile("" : "+v"(row_[ks]));  // made once, not at each use
    }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int q = 8 * x + 4 * (lane >> 5) + (m >> 2);
        const int c = 4 * db + 2 * ((lane >> 4) & 1) + ((m & 3) >> 1);
        column_[db][x] = base + q * (DP * 2) + ((c ^ fswz<DP>(q)) * 16) + (m & 1) * 8;
        asm volatile("" : "+v"(column_[db][x]));
      }
  }
  // rows r0 + l%32, elements 16 ks + 8 (l/32) ..: of a contraction over the width;
  // at: r0 times the row's bytes, and the tile
  __device__ __forceinline__ u32x4 row(unsigned at, int ks) const { return *(lds_u32x4*)(row_[ks] + at); }
  // column 32 db + l%32, rows r0 + {4 h .. 4 h + 3, 8 + 4 h ..}, h = l/32: of a
  // contraction over the rows
  __device__ __forceinline__ u32x4 column(unsigned at, int db) const {
    u32x4 v;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const u32x2 t = __builtin_bit_cast(
          u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(column_[db][x] + at)));
      v[2 * x] = t[0];
      v[2 * x + 1] = t[1];
    }
    return v;
  }
};

// Infinities and NaN ("others") in masked places.  A tile's products multiply what a row
// does not see by a weight of 0, which makes 0 of a number but NaN of others.  So
// where some rows see less than a tile others in it are wiped, 0 in their place in
// LDS, and what they make of the rows that see them is made apart.  The forward and dq
// of 128 rows, whose sums tell whether there were any, look at those and go over
// their tiles once more if so; a few rows' blocks, of which one or two are cut, are
// wiped at once; dk and dv wipe rows whose lse or D tells of others.  Without any, on
// packed prompts, that costs the forward 1% (371 -> 375 us), dq 1%, dk and dv what a
// third division a tile did (below).  (Cut tiles wiped at once in the forward of 128
// rows: 4%.)
//
// The finite ones of two 16-bit numbers, 0 in the place of others
template <class T>
__device__ __forceinline__ uint32_t finite2(uint32_t v) {
  constexpr uint32_t E = Half<T>::EXPONENT;
  return ((v & E) == E ? 0 : v & 0xffff) | ((v >> 16 & E) == E ? 0 : v & 0xffff0000u);
}
// Wipes chunk `chunk` (16 bytes) of a tile at `lds`; whether there was something to wipe
template <class T>
__device__ __forceinline__ bool wipe(unsigned lds, int chunk) {
  typedef __attribute__((address_space(3))) u32x4 lds_chunk;
  const u32x4 v = *(lds_u32x4*)(lds + chunk * 16);
  u32x4 w;
  bool other = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    w[i] = finite2<T>(v[i]);
    other |= w[i] != v[i];
  }
  if (other) *(lds_chunk*)(lds + chunk * 16) = w;
  return other;
}
template <int DB>
__device__ __forceinline__ bool has_others(const f32x16 (&o)[DB]) {
  float t[4] = {};
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) t[i % 4] = fmaf(o[db][i], 0.f, t[i % 4]);
  return !(t[0] + t[1] + t[2] + t[3] == 0.f);
}
// Whether a wave of the workgroup says so; `word`: 4 bytes of LDS a wave, for this alone
constexpr int WORDS = 32;  // bytes of them
template <int W>
__device__ __forceinline__ bool any_wave(bool mine, int* word, int wave) {
  if ((threadIdx.x & 63) == 0) word[wave] = mine;
  __syncthreads();
  int r = 0;
#pragma unroll
  for (int i = 0; i < W; ++i) r |= word[i];
  return uniform(r) != 0;
}

// 8 elements from element e of a head's row, zeros past the width
template <class T>
__device__ __forceinline__ u32x4 load8(const T* row, int e, int width) {
  return e < width ? *global_ptr<const u32x4>(row + e) : u32x4{0, 0, 0, 0};
}

// Writes v[d][column] of a lane's column to `row` (16-bit, factor f): the halves
// of the wave swap so that a lane holds 8 elements side by side.
template <class T, int DB>
__device__ __forceinline__ void store_columns(const f32x16 (&v)[DB], float f, T* row, int width,
                                              int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db) {
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      u32x4 w;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const uint32_t x = pack2<T>(v[db][8 * p + 2 * j] * f, v[db][8 * p + 2 * j + 1] * f);
        const uint32_t y = pack2<T>(v[db][8 * p + 4 + 2 * j] * f, v[db][8 * p + 4 + 2 * j + 1] * f);
        const auto s = __builtin_amdgcn_permlane32_swap((int)x, (int)y, false, false);
        w[j] = s[0];
        w[2 + j] = s[1];
      }
      const int e = 32 * db + 16 * p + 8 * (lane >> 5);
      if (row && e < width) *global_ptr<u32x4>(row + e) = w;
    }
  }
}

// The same unrounded, to `row` of f32 of DP elements.
template <int DB>
__device__ __forceinline__ void store_sums(const f32x16 (&v)[DB], float f, float* row, int lane) {
  if (!row) return;
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4*>(row + 32 * db + 8 * i + 4 * (lane >> 5)) =
          make_float4(v[db][4 * i] * f, v[db][4 * i + 1] * f, v[db][4 * i + 2] * f, v[db][4 * i + 3] * f);
}

// A wave's 32 rows of a problem's G heads: a lane's own.
struct Row {
  int i, g;     // token in the sequence, head in the group
  int last;     // last key it sees, -1: none
  bool stored;  // in or (fill) behind its sequence
};
__device__ __forceinline__ Row row_of(const PackedAttn& a, const Seq& s, int r, int G) {
  const int have = a.fill ? s.have : s.lq;
  Row o;
  const int i = r / G;
  o.stored = i < have;
  o.i = o.stored ? i : max(have - 1, 0);
  o.g = r - i * G;
  o.last = -1;
  if (o.i < s.lq && o.stored) o.last = a.causal ? min(o.i + s.lk - s.lq, s.lk - 1) : s.lk - 1;
  return o;
}

template <class T>
__device__ __forceinline__ T* row_ptr(const HeadView& v, int64_t token, int head) {
  return (T*)v.p + token * v.st + (int64_t)head * v.sh;
}

__device__ __forceinline__ float finite_or_zero(float v) { return v < __builtin_inff() ? v : 0.f; }

// Largest (or smallest) over the lanes of a wave
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int m = 1; m < 64; m *= 2) v = max(v, __shfl_xor(v, m, 64));
  return uniform(v);
}
__device__ __forceinline__ int wave_min(int v) { return -wave_max(-v); }

// Copies of ROWS keys and of their values (zeros past the sequence), by W waves, from
// key k0 on and every `step` keys.
template <class T, int DP, int ROWS, int W>
struct KeyTiles {
  typedef TileCopy<DP, ROWS, W> C;
  static_assert(C::PIECES % W == 0, "every wave has as many pieces");
  unsigned ko[C::PER], vo[C::PER];  // a lane's offsets
  // the next ones' address, what is left of the sequence from there, and a step, in bytes
  uint64_t k, v;
  int64_t k_left, v_left, k_step, v_step;
  int wave;
  __device__ __forceinline__ void init(const PackedAttn& a, const Seq& s, int head, int k0, int step, int wave_,
                                       int lane) {
    wave = wave_;
    const int64_t kst = a.k.st, vst = a.v.st;
    k = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.k, s.k0 + k0, head));
    v = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.v, s.k0 + k0, head));
    k_left = uniform64(((int64_t)(s.lk - k0 - 1) * kst + a.width) * 2);
    v_left = uniform64(((int64_t)(s.lk - k0 - 1) * vst + a.width) * 2);
    k_step = uniform64(step * kst * 2);
    v_step = uniform64(step * vst * 2);
#pragma unroll
    for (int i = 0; i < C::PER; ++i) {
      const int r = C::row(i, wave, lane), e = C::elem(i, wave, lane);
      ko[i] = e < a.width ? (unsigned)(r * kst + e) * 2 : NOWHERE;
      vo[i] = e < a.width ? (unsigned)(r * vst + e) * 2 : NOWHERE;
    }
  }
  // a descriptor's bounds have 32 bits, and a tile's offsets 30
  static __device__ __forceinline__ u32x4 here(uint64_t p, int64_t left) {
    const uint32_t bytes = (uint64_t)left >> 31 ? 0x7fffffffu : (uint32_t)left;
    return u32x4{(uint32_t)p, (uint32_t)(p >> 32) & 0xffffu, bytes, 0x00027000u};
  }
  __device__ __forceinline__ void keys(unsigned lds) {
    const u32x4 d = here(k, k_left);
#pragma unroll
    for (int i = 0; i < C::PER; ++i) copy16(ko[i], d, lds + C::dst(i, wave));
    k += k_step;
    k_left -= k_step;
  }
  __device__ __forceinline__ void values(unsigned lds) {
    const u32x4 d = here(v, v_left);
#pragma unroll
    for (int i = 0; i < C::PER; ++i) copy16(vo[i], d, lds + C::dst(i, wave));
    v += v_step;
    v_left -= v_step;
  }
  __device__ __forceinline__ void both(unsigned lds) {
    keys(lds);
    values(lds + ROWS * DP * 2);
  }
};

// What the values of keys from .. to - 1 that are infinities or NaN make of the outputs
// of a lane's row, whose last key is `last`: its weights are positive.
template <class T, int DB>
__device__ __forceinline__ void add_others(const PackedAttn& a, const Seq& s, int head, int from, int to, int last,
                                           f32x16 (&o)[DB], int lane) {
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll 1
  for (int key = from; key < to; ++key) {
    const T* v = row_ptr<const T>(a.v, s.k0 + key, head) + 4 * (lane >> 5);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (32 * db + 8 * i >= a.width) continue;
        const t4 x = *global_ptr<const t4>(v + 32 * db + 8 * i);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y = (float)x[k];
          if (!(fabsf(y) < __builtin_inff()) && key <= last) o[db][4 * i + k] += y;
        }
        __builtin_amdgcn_sched_barrier(0);  // in few registers
      }
  }
}

// ------------------------------------------------------------------ forward
// A wave's 32 rows over tiles of 32 NB keys: outputs, sums and exponents'
// references of a lane's row.
template <class T, int DP, int NB>
struct Online {
  static constexpr int KS = DP / 16, DB = DP / 32;
  f32x16 o[DB];
  float ref, mc, sum;  // mc: ref times c; sum: of a lane's own keys

  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  }
  __device__ __forceinline__ void init() {
    clear();
    ref = NEG_INF;
    mc = sum = 0.f;
  }
  // S^T of a tile whose keys lie at `at`
  static __device__ __forceinline__ void scores(f32x16 (&p)[NB], const Operands<DP>& x, unsigned at,
                                                const u32x4 (&q)[KS]) {
    constexpr int N = NB * KS, AHEAD = N < 8 ? N : 8;  // reads ahead of their products
    u32x4 f[N];
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = x.row(at + 32 * (i % NB) * DP * 2, i / NB);
#pragma unroll
    for (int b = 0; b < NB; ++b) p[b] = f32x16{};
#pragma unroll
    for (int i = 0; i < N; ++i) p[i % NB] = Half<T>::mma(f[i], q[i / NB], p[i % NB]);
    order<LDS_READ, AHEAD>();
#pragma unroll
    for (int i = 0; i < N - AHEAD; ++i) {
      order<MFMA, 1>();
      order<LDS_READ, 1>();
    }
    order<MFMA, AHEAD>();
  }
  // the reference of their exponents.  last: the last key that the lane's row sees, from
  // the tile's first and its lane half's; cut: whether some row sees less than
  // the tile
  __device__ __forceinline__ void weights(f32x16 (&p)[NB], float c, int last, bool cut) {
    if (cut) {
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i / 4) + i % 4 > last) p[b][i] = NEG_INF;
    }
    float m = p[0][0];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, p[b][i]);
    m = other_half_max(m);
    // NaN scores leave m and end in the sum
    if (__any(m * c > ref * c + LAG || (ref == NEG_INF && m > NEG_INF))) {
      const float to = fmaxf(ref, m), f = ref == NEG_INF ? 0.f : exp2_f((ref - to) * c);
      ref = to;
      mc = ref == NEG_INF ? 0.f : ref * c;
      sum *= f;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= f;
    }
  }
  // exponents, and o^T += V^T P^T, the values at `at`: 16 keys' exponents beside the
  // products of the 16 before
  __device__ __forceinline__ void values(f32x16 (&p)[NB], float c, const Operands<DP>& x, unsigned at) {
    constexpr int N = 2 * NB;
    u32x4 v[N][DB];
#pragma unroll
    for (int g = 0; g < N; ++g)
#pragma unroll
      for (int db = 0; db < DB; ++db) v[g][db] = x.column(at + 16 * g * DP * 2, db);
    const float shift = Half<T>::SHIFT - mc;
#pragma unroll
    for (int g = 0; g < N; ++g) {
      f32x16& e = p[g / 2];
#pragma unroll
      for (int i = 8 * (g & 1); i < 8 * (g & 1) + 8; ++i) {
        e[i] = exp2_f(fmaf(e[i], c, shift));
        sum += e[i];
      }
      const u32x4 w = pack8<T>(e, g & 1);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = Half<T>::mma(v[g][db], w, o[db]);
    }
    order<LDS_READ, 2 * DB>();
    order<VALU, 28>();
#pragma unroll
    for (int g = 1; g < N; ++g) {
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        order<MFMA, 1>();
        order<LDS_READ, 2>();
        order<VALU, 28 / DB>();
      }
    }
    order<MFMA, DB>();
  }
};

// Workgroup = 128 rows of one sequence and head of keys, 4 waves x 32 rows;
// keys in tiles of 64, two buffers, one barrier a tile.
//
// Products and exponentials bound it: two workgroups a unit, one's products beside
// the other's exponentials.  11 causal sequences of 16384 tokens, 32 heads over 8
// of 128, bfloat16: 373 us, 828 TFLOP/s of what is seen, two thirds of what a
// large library product reaches; with the operands read as they are needed
// instead of up to eight ahead (the order below) 6% more.
template <class T, int DP>
__global__ __launch_bounds__(NT, 2) void packattn_fwd_kernel(PackedAttn a, int64_t tiles) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  constexpr int BM = 32 * WAVES, KS = DP / 16, DB = DP / 32, TILE = BN * DP * 2;
  const Place at = place(a.kv_heads, tiles);
  if (at.tile < 0) return;
  const int G = a.heads / a.kv_heads;
  int s;
  // from the last tile: a causal sequence's last rows see the most keys
  const int64_t t = find_tile(a.q_off, a.sequences, a.q_tokens, G, BM, tiles - 1 - at.tile, s);
  const Seq seq = lane_seq(sequence(a, s, false), 0);
  const int rows = (a.fill ? seq.have : seq.lq) * G;
  if (t < 0 || t * BM >= rows) return;
  const int r0 = (int)t * BM;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const Row row = row_of(a, seq, r0 + 32 * wave + (lane & 31), G);
  const int head = at.head * G + row.g;
  const int64_t token = seq.q0 + row.i;
  const int most = wave_max(row.last), least = wave_min(row.last);
  // the last row of the workgroup sees the most keys
  const Row end = row_of(a, seq, min(r0 + BM, rows) - 1, G);
  int far = uniform(end.last);
  if (a.fill && seq.lq < seq.have) far = seq.lk - 1;  // rows behind the queries see none
  const int nk = far < 0 ? 0 : far / BN + 1;

  u32x4 q[KS];
  const T* qrow = row_ptr<const T>(a.q, token, head);
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) q[ks] = load8(qrow, 16 * ks + 8 * h, a.width);
  const float c = a.scale * LOG2E;
  Online<T, DP, 2> st;
  const unsigned lds0 = lds_addr(smem);
  KeyTiles<T, DP, BN, WAVES> tile;
  Operands<DP> x;
  x.init(lds0, lane);
  // the first key that not all rows see, once others have to be wiped from there on
  int wiped = 0x7fffffff;
  auto step = [&](int kt, unsigned here, unsigned next) __attribute__((always_inline)) {
    const int k0 = kt * BN;
    wait_all_and_sync();
    if (k0 + BN > wiped) {
#pragma unroll 1
      for (int i = threadIdx.x; i < TILE / 16; i += NT) wipe<T>(lds0 + here + TILE, i);
      __syncthreads();
    }
    if (kt + 1 < nk) tile.both(lds0 + next);
    if (k0 > most) return;
    f32x16 p[2];
    st.scores(p, x, here, q);
    st.weights(p, c, row.last - k0 - 4 * h, k0 + BN - 1 > least);
    st.values(p, c, x, here + TILE);
  };
  for (;;) {
    st.init();
    tile.init(a, seq, at.head, 0, BN, wave, lane);
    if (nk > 0) tile.both(lds0);
    for (int kt = 0; kt < nk; kt += 2) {  // the two buffers at constant places
      step(kt, 0, 2 * TILE);
      if (kt + 1 < nk) step(kt + 1, 2 * TILE, 0);
    }
    if (!a.causal) break;
    if (wiped < 0x7fffffff) {
      add_others<T>(a, seq, at.head, wiped / BN * BN, most + 1, row.last, st.o, lane);
      break;
    }
    // others in a row that does not see all of its wave's last tile
    const bool others = row.last >= 0 && row.last < min(most / BN * BN + BN, seq.lk) - 1 && has_others(st.o);
    if (!any_wave<WAVES>(__any(others), reinterpret_cast<int*>(smem + 4 * TILE), wave)) break;
    wiped = uniform(row_of(a, seq, r0, G).last) + 1;
  }
  const float sum = other_half_sum(st.sum);
  // A row that sees keys has a sum of 0 where all its scores are -infinity: its
  // softmax is NaN, as 0 / 0 here, and its lse log 0.
  const bool none = row.last < 0;
  if (none) st.clear();
  store_columns<T, DB>(st.o, none ? 0.f : 1.f / sum,
                       row.stored ? row_ptr<T>(a.o, token, head) : nullptr, a.width, lane);
  if (row.stored && h == 0)
    a.lse[(int64_t)head * a.q_tokens + token] =
        none ? NEG_INF : (st.mc - Half<T>::SHIFT + log2f(sum)) * LN2;
}

// Few rows (single tokens against caches, short chains): a workgroup takes 32
// rows of one sequence and head of keys with a stretch of the sequence's keys, in
// blocks of 32 or 64.
//
// W = 1, long caches: a wave by itself is a workgroup.  What bounds it is the
// keys and values read once, so every stretch has to be as long as the others,
// whatever the sequences' lengths, and the card full of copies in flight: each
// wave adds up all sequences' blocks, which gives the length of a stretch for
// `goal` equal ones a head, and finds its own among them.  A wave has one
// buffer of keys and one of values, and refills each as soon as it is read, so
// that nearly all of the LDS is in flight nearly all of the time (64 sequences of
// 11 .. 8192 keys, 8 heads of 128: 240 MB in 56 us, 4.3 TB/s; one of 131 k, 4 heads
// of 64: 134 MB in 30).  Rows of more than one stretch go to packattn_join_kernel
// through memory.
// W = 4, few keys: all of a sequence's by one workgroup, every fourth block a
// wave, joined in LDS: no second launch.
// Calls of more entries than a wave holds: sums over the entries before each, and
// over all, made once a call and searched 64 at a time.  (Each wave adding up all
// entries for each of its items: 5000 sequences of one query and four keys, 32 heads
// over 8 of 128, 1408 us, 20 000 of 64 keys 16.8 ms.)
struct Table {
  int64_t *per, *items, *splits, *slots;  // [1], [entries + 1] each
};
struct Split {
  float* o;    // [slot][32 rows][DP], sums of exponents times values
  float2* ml;  // [slot][32]: reference in log 2, sum of exponents
  Table table;  // of more entries than a wave holds, else null
};
// keys of a block: 16 KB of keys and values at the widths 64 and 128
__host__ __device__ constexpr int block_keys(int DP) { return DP == 128 ? 32 : 64; }
constexpr int SHORTEST = 256;  // keys of a stretch at least

struct Item {
  Seq seq;
  int tile;         // of 32 rows
  int part, parts;  // stretch, of how many
  int64_t slot;     // of the tile's first stretch (parts > 1)
  int per;          // blocks of a stretch
};
// An entry (sequence, or the tokens outside) as one lane sees it.
struct Entry {
  int tiles, blocks;
};
template <int KN>
__device__ __forceinline__ Entry entry_of(const PackedAttn& a, int e, int G) {
  Entry r = {0, 0};
  if (e >= a.sequences + 2) return r;
  const Seq seq = sequence(a, e, false);
  r.tiles = (int)(((int64_t)(a.fill ? seq.have : seq.lq) * G + 31) / 32);
  r.blocks = seq.lq > 0 ? (seq.lk + KN - 1) / KN : 0;
  return r;
}
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) v += __shfl_xor(v, i, 64);
  return v;
}
// what the lanes before this one have
__device__ __forceinline__ int64_t wave_before(int64_t v, int lane) {
  int64_t run = v;
#pragma unroll
  for (int i = 1; i < 64; i *= 2) {
    const int64_t o = __shfl_up(run, i, 64);
    if (lane >= i) run += o;
  }
  return run - v;
}
// Blocks of a stretch.  work: of all tiles; all: how many tiles there are.
template <int KN>
__device__ __forceinline__ int stretch_of(int64_t work, int64_t all, int64_t goal) {
  // every tile may end in a short stretch: with those too one round of waves
  // (64 sequences of 11 .. 8192 keys, 8 heads of 128: 70.5 -> 62 us)
  if (all < goal / 2) goal -= all;
  return (int)max((int64_t)(SHORTEST / KN), (work + goal - 1) / goal);
}
// Of an entry: items, tiles of more than one stretch, and those tiles' stretches.
struct Counts {
  int64_t items, splits, slots;
};
__device__ __forceinline__ Counts counts_of(int tiles, int parts) {
  Counts c;
  c.items = (int64_t)tiles * parts;
  c.splits = parts > 1 ? tiles : 0;
  c.slots = parts > 1 ? c.items : 0;
  return c;
}
template <int KN>
__global__ __launch_bounds__(1024) void packattn_table_kernel(PackedAttn a, int64_t goal, Table table) {
  __shared__ int64_t sums[3][16];
  const int G = a.heads / a.kv_heads, entries = a.sequences + 2;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // v of the threads before this one, and of all
  auto scan = [&](int64_t v, int64_t* waves, int64_t& total) __attribute__((always_inline)) {
    const int64_t before = wave_before(v, lane);
    if (lane == 63) waves[wave] = before + v;
    __syncthreads();
    int64_t own = before;
    total = 0;
#pragma unroll 4
    for (int i = 0; i < 16; ++i) {
      if (i < wave) own += waves[i];
      total += waves[i];
    }
    return own;
  };
  int64_t work = 0, all = 0, of_items, of_splits, of_slots;
  for (int e = threadIdx.x; e < entries; e += 1024) {
    const Entry x = entry_of<KN>(a, e, G);
    work += (int64_t)x.tiles * x.blocks;
    all += x.tiles;
  }
  scan(work, sums[0], of_items);
  scan(all, sums[1], of_splits);
  const int per = stretch_of<KN>(of_items, of_splits, goal);
  if (threadIdx.x == 0) *table.per = per;
  Counts run = {};
  for (int e0 = 0; e0 < entries; e0 += 1024) {
    const int e = e0 + threadIdx.x;
    const Entry x = entry_of<KN>(a, e, G);
    const Counts c = counts_of(x.tiles, max(1, (x.blocks + per - 1) / per));
    __syncthreads();  // the sums before have been read
    const int64_t items = run.items + scan(c.items, sums[0], of_items);
    const int64_t splits = run.splits + scan(c.splits, sums[1], of_splits);
    const int64_t slots = run.slots + scan(c.slots, sums[2], of_slots);
    if (e <= entries) {
      table.items[e] = items;
      table.splits[e] = splits;
      table.slots[e] = slots;
    }
    run.items += of_items;
    run.splits += of_splits;
    run.slots += of_slots;
  }
  if (threadIdx.x == 0) {
    table.items[entries] = run.items;
    table.splits[entries] = run.splits;
    table.slots[entries] = run.slots;
  }
}

// The wave's view of all sequences: what up to 64 HELD entries come to lies in its
// lanes, more (TABLE) in the call's table.
constexpr int HELD = 4;
template <int KN, bool TABLE>
struct Stretches {
  int tiles[HELD], blocks[HELD];  // of entry 64 i + lane
  int per, G, lane, entries;
  Table table;

  __device__ __forceinline__ void init(const PackedAttn& a, int G_, int64_t goal, const Table& t) {
    G = G_;
    lane = threadIdx.x & 63;
    entries = a.sequences + 2;
    if constexpr (TABLE) {
      table = t;
      per = uniform((int)*table.per);
      return;
    }
    int64_t work = 0, all = 0;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
      const Entry x = entry_of<KN>(a, 64 * i + lane, G);
      tiles[i] = x.tiles;
      blocks[i] = x.blocks;
      work += (int64_t)x.tiles * x.blocks;
      all += x.tiles;
    }
    per = uniform(stretch_of<KN>(wave_sum64(work), wave_sum64(all), goal));
  }
  __device__ __forceinline__ int parts_of(int blocks_) const { return max(1, (blocks_ + per - 1) / per); }
  // tile or stretch y of entry e, whose stretches' slots begin at `slots`
  template <bool SPLIT>
  __device__ __forceinline__ void item(const PackedAttn& a, int e, int parts, int64_t y, int64_t slots, Item& r) const {
    r.seq = lane_seq(sequence(a, e, false), 0);
    r.parts = parts;
    r.tile = uniform((int)(SPLIT ? y : y / parts));
    r.part = SPLIT ? 0 : uniform((int)(y % parts));
    r.slot = slots + (int64_t)r.tile * parts;
    r.per = per;
  }
  // Item x of all (SPLIT: tile x of those with more stretches than one);
  // false past the last.
  template <bool SPLIT>
  __device__ __forceinline__ bool find(const PackedAttn& a, int64_t x, Item& r) const {
    if constexpr (TABLE) {
      const int64_t* from = SPLIT ? table.splits : table.items;
      if (x >= from[entries]) return false;
      int lo = 0, count = entries;  // the last entry that begins at x or before it
      while (count > 1) {
        const int step = (count + 63) / 64, i = lane * step;
        const bool below = i < count && from[lo + min(i, count - 1)] <= x;
        const int passed = max(__popcll(__ballot(below)) - 1, 0) * step;
        lo += passed;
        count = min(step, count - passed);
      }
      lo = uniform(lo);
      const Entry m = entry_of<KN>(a, lo, G);
      item<SPLIT>(a, lo, uniform(parts_of(m.blocks)), uniform64(x - from[lo]), uniform64(table.slots[lo]), r);
      return true;
    }
    int64_t slots = 0;
    auto look = [&](int i) {
      const int parts = parts_of(blocks[i]);
      const Counts c = counts_of(tiles[i], parts);
      const int64_t n = SPLIT ? c.splits : c.items, before = wave_before(n, lane);
      const unsigned long long at = __ballot(before <= x && x < before + n);
      if (at) {
        const int l = uniform(__ffsll(at) - 1);
        item<SPLIT>(a, 64 * i + l, __builtin_amdgcn_readlane(parts, l), x - lane64(before, l),
                    slots + lane64(wave_before(c.slots, lane), l), r);
        return true;
      }
      x -= wave_sum64(n);
      slots += wave_sum64(c.slots);
      return false;
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
      if (64 * i < entries && look(i)) return true;
    return false;
  }
};

template <class T, int DP, int W, bool TABLE>
__global__ __launch_bounds__(64 * W, 2) void packattn_keys_kernel(PackedAttn a, int64_t goal, Split split) {
  // goal: of equal stretches a head of keys; W = 4: tiles of 32 rows
  constexpr int KN = block_keys(DP), KS = DP / 16, DB = DP / 32, TILE = KN * DP * 2, LD = DP + 4;
  constexpr int JOIN = W > 1 ? W * 32 * (LD * 4 + 8) : 0;
  constexpr int LDS = W * 2 * TILE > JOIN ? W * 2 * TILE : JOIN;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[LDS];
  const int G = a.heads / a.kv_heads, lane = threadIdx.x & 63, h = lane >> 5;
  const int wave = W > 1 ? uniform(threadIdx.x >> 6) : 0;
  Stretches<KN, TABLE> all;
  if (W == 1) all.init(a, G, goal, split.table);
  // W = 4: every entry's keys whole, its tiles by their numbers
  auto tile_of = [&](int64_t x, Item& r) __attribute__((always_inline)) {
    int s;
    const int64_t t = find_tile(a.q_off, a.sequences, a.q_tokens, G, 32, x, s);
    r.seq = lane_seq(sequence(a, s, false), 0);
    r.tile = (int)t;
    r.part = 0;
    r.parts = 1;
    r.per = (r.seq.lk + KN - 1) / KN;
    return t >= 0 && t * 32 < (int64_t)(a.fill ? r.seq.have : r.seq.lq) * G;
  };
  const unsigned kb = lds_addr(smem) + wave * 2 * TILE, vb = kb + TILE;
  Operands<DP> ops;
  ops.init(kb, lane);
  const float c = a.scale * LOG2E;
  typedef KeyTiles<T, DP, KN, 1> Tiles;
  Item it;
  for (int64_t x = blockIdx.x;; x += gridDim.x) {
    if constexpr (W > 1) {
      if (x >= goal * a.kv_heads) break;
      if (!tile_of(x / a.kv_heads, it)) continue;
    } else {
      if (!all.template find<false>(a, x / a.kv_heads, it)) break;
    }
    const int kv = uniform((int)(x % a.kv_heads));
    const Seq& seq = it.seq;
    const Row row = row_of(a, seq, it.tile * 32 + (lane & 31), G);
    const int head = kv * G + row.g;
    const int64_t token = seq.q0 + row.i;
    const int most = wave_max(row.last), least = wave_min(row.last);
    const int b0 = it.part * it.per, b1 = min(b0 + it.per, (most + KN) / KN);
    u32x4 q[KS];
    const T* qrow = row_ptr<const T>(a.q, token, head);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = load8(qrow, 16 * ks + 8 * h, a.width);
    // The first key that not all rows see.  Few blocks have one (those of single tokens
    // none), and are wiped at once.
    const int sure = a.causal ? uniform(row_of(a, seq, it.tile * 32, G).last) + 1 : seq.lk;
    bool dirty = false;
    Online<T, DP, KN / 32> st;
    st.init();
    Tiles tile;
    wait_reads();
    wait_copies<0>();  // q: what follows counts copies alone
    int b = b0 + wave;
    tile.init(a, seq, kv, b * KN, W * KN, 0, lane);
    if (b < b1) tile.both(kb);
    for (; b < b1; b += W) {
      const bool more = b + W < b1;
      wait_copies<Tiles::C::PER>();  // the keys are here, the values on their way
      f32x16 p[KN / 32];
      st.scores(p, ops, 0, q);
      wait_reads();
      if (more) tile.keys(kb);
      st.weights(p, c, row.last - b * KN - 4 * h, b * KN + KN - 1 > least);
      if (more) wait_copies<Tiles::C::PER>();
      else wait_copies<0>();
      if (min(b * KN + KN, seq.lk) > sure) {
#pragma unroll 1
        for (int i = lane; i < TILE / 16; i += 64) dirty |= wipe<T>(vb, i);
        wait_reads();
      }
      st.values(p, c, ops, TILE);
      wait_reads();
      if (more) tile.values(vb);
    }
    if (__any(dirty))
      for (b = b0 + wave; b < b1; b += W)
        if (min(b * KN + KN, seq.lk) > sure)
          add_others<T>(a, seq, kv, b * KN, min(b * KN + KN, most + 1), row.last, st.o, lane);
    const float sum = other_half_sum(st.sum);
    if constexpr (W > 1) {
      // the waves' sums of a row, relative to the largest reference
      __syncthreads();
      float* so = reinterpret_cast<float*>(smem);                 // [wave][32 rows][LD]
      float2* sml = reinterpret_cast<float2*>(so + W * 32 * LD);  // [wave][32]
      if (h == 0) sml[wave * 32 + lane] = make_float2(st.mc, sum);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(so + (wave * 32 + (lane & 31)) * LD + 32 * db + 8 * i + 4 * h) =
              make_float4(st.o[db][4 * i], st.o[db][4 * i + 1], st.o[db][4 * i + 2], st.o[db][4 * i + 3]);
      __syncthreads();
      constexpr int PER_ROW = 2 * W;  // threads a row
      const int r = threadIdx.x / PER_ROW, part = threadIdx.x % PER_ROW;
      const Row mine = row_of(a, seq, it.tile * 32 + r, G);
      const int my_head = kv * G + mine.g;
      const int64_t my_token = seq.q0 + mine.i;
      float top = NEG_INF, l = 0.f, f[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 v = sml[w * 32 + r];
        if (!(v.y == 0.f)) top = fmaxf(top, v.x);
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float2 v = sml[w * 32 + r];
        f[w] = v.y == 0.f ? 0.f : exp2_f(v.x - top);
        l += v.y * f[w];
      }
      const bool none = mine.last < 0;
      const float inv = 1.f / l;
      if (mine.stored) {
        for (int e = part * 8; e < a.width; e += PER_ROW * 8) {
          float v[8] = {};
#pragma unroll
          for (int w = 0; w < W; ++w)
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = fmaf(so[(w * 32 + r) * LD + e + i], f[w], v[i]);
#pragma unroll
          for (int i = 0; i < 8; ++i) v[i] = none ? 0.f : v[i] * inv;
          Vec<T>::store(row_ptr<T>(a.o, my_token, my_head) + e, Vec<T>::pack(v));
        }
        if (part == 0)
          a.lse[(int64_t)my_head * a.q_tokens + my_token] =
              none ? NEG_INF : (top - Half<T>::SHIFT + log2f(l)) * LN2;
      }
      __syncthreads();
    } else if (it.parts == 1) {
      const bool none = row.last < 0;
      if (none) st.clear();
      store_columns<T, DB>(st.o, none ? 0.f : 1.f / sum,
                           row.stored ? row_ptr<T>(a.o, token, head) : nullptr, a.width, lane);
      if (row.stored && h == 0)
        a.lse[(int64_t)head * a.q_tokens + token] =
            none ? NEG_INF : (st.mc - Half<T>::SHIFT + log2f(sum)) * LN2;
    } else if (row.stored) {
      const int64_t at = ((it.slot + it.part) * a.kv_heads + kv) * 32 + (lane & 31);
      // of a row that sees no key, -0: the join need not find its sequence's keys again
      // (12.9 us for 12.3)
      if (h == 0) split.ml[at] = make_float2(st.mc, row.last < 0 ? -0.f : sum);
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4*>(split.o + at * DP + 32 * db + 8 * i + 4 * h) =
              make_float4(st.o[db][4 * i], st.o[db][4 * i + 1], st.o[db][4 * i + 2], st.o[db][4 * i + 3]);
    }
  }
}

// The stretches of rows, RW waves a row: DP / 4 lanes a stretch, each lane group
// with a reference of its own.  Bound by its launch and one round of loads: 10 us
// beside 56 of the stretches (64 sequences of 11 .. 8192 keys), 12 beside 30 (one of
// 131 k).
template <class T, int DP, int RW, bool TABLE>
__global__ __launch_bounds__(RW > 1 ? 64 * RW : NT) void packattn_join_kernel(PackedAttn a, int64_t goal, Split split) {
  constexpr int KN = block_keys(DP), LP = DP / 4, ROWS = RW > 1 ? 1 : WAVES, GROUPS = 64 * RW / LP;
  __shared__ float so[ROWS][RW][DP];
  __shared__ float2 sml[ROWS][RW];
  const int G = a.heads / a.kv_heads;
  Stretches<KN, TABLE> all;
  all.init(a, G, goal, split.table);
  const int mine = threadIdx.x / (64 * RW), t = threadIdx.x % (64 * RW);
  const int group = t / LP, e = t % LP * 4;
  Item it;
  for (int64_t x = blockIdx.x; all.template find<true>(a, x / a.kv_heads, it); x += gridDim.x) {
    const int kv = uniform((int)(x % a.kv_heads));
    for (int r0 = blockIdx.y * ROWS; r0 < 32; r0 += gridDim.y * ROWS) {
      if (!row_of(a, it.seq, it.tile * 32 + r0, G).stored) break;
      const int r = r0 + mine;
      const Row row = row_of(a, it.seq, it.tile * 32 + r, G);
      const int64_t stride = (int64_t)a.kv_heads * 32, at = (it.slot * a.kv_heads + kv) * 32 + r;
      float top = NEG_INF, sum = 0.f;
      bool blind = false;  // in the lanes that write the row, which read its first stretch
      f32x4 v = {};
      auto add = [&](float2 m, f32x4 o) __attribute__((always_inline)) {
        const float to = fmaxf(top, m.x), f = top == NEG_INF ? 0.f : exp2_f(top - to);
        const float g = exp2_f(m.x - to);
        top = to;
        sum = fmaf(sum, f, m.y * g);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf(v[k], f, o[k] * g);
      };
      for (int p = group; p < it.parts && row.stored; p += 4 * GROUPS) {
        float2 m[4];
        f32x4 o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // in flight together
          const int64_t s = at + min(p + i * GROUPS, it.parts - 1) * stride;
          m[i] = split.ml[s];
          o[i] = *reinterpret_cast<const f32x4*>(split.o + s * DP + e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (p + i * GROUPS >= it.parts) continue;
          blind |= __builtin_signbit(m[i].y);
          if (m[i].y == 0.f) continue;
          add(m[i], o[i]);
        }
      }
      // the lane groups of a wave, then the waves
#pragma unroll
      for (int i = LP; i < 64; i *= 2) {
        f32x4 o;
        const float2 m = make_float2(__shfl_xor(top, i, 64), __shfl_xor(sum, i, 64));
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = __shfl_xor(v[k], i, 64);
        if (!(m.y == 0.f)) add(m, o);
      }
      if constexpr (RW > 1) {
        __syncthreads();
        if (t % 64 < LP) *reinterpret_cast<float4*>(&so[mine][t / 64][e]) = make_float4(v[0], v[1], v[2], v[3]);
        if (t % 64 == 0) sml[mine][t / 64] = make_float2(top, sum);
        __syncthreads();
        top = NEG_INF;
        sum = 0.f;
        v = f32x4{};
        if (t < LP) {
#pragma unroll 4
          for (int i = 0; i < RW; ++i) {
            const float2 m = sml[mine][i];
            const float4 o = *reinterpret_cast<const float4*>(&so[mine][i][e]);
            if (!(m.y == 0.f)) add(m, f32x4{o.x, o.y, o.z, o.w});
          }
        }
      }
      if (t < LP && row.stored) {
        const bool none = blind && sum == 0.f;
        const float inv = 1.f / sum;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = none ? 0.f : v[k] * inv;
        const float w[4] = {v[0], v[1], v[2], v[3]};
        if (e < a.width) Few<T, 4>::template store<false>(row_ptr<T>(a.o, it.seq.q0 + row.i, kv * G + row.g) + e, w);
        if (t == 0)
          a.lse[(int64_t)(kv * G + row.g) * a.q_tokens + it.seq.q0 + row.i] =
              none ? NEG_INF : (top - Half<T>::SHIFT + log2f(sum)) * LN2;
      }
    }
  }
}

// ----------------------------------------------------------------- backward
// In binary16 a dS of many keys falls below the normal numbers, so it is made
// 2^e times as large, e from norms that bound it: |dS| <= 2 |do| max |v|.  dq has a
// scale for every row, from its own |do| and the values that its workgroup goes over;
// dk and dv one for a workgroup's keys, from the rows and values of their sequence
// and group of heads.  So no sequence's, group's or row's accuracy hangs on what
// others of the call hold; infinities and NaN are left out of the norms, and so are
// rows that see no key.
//
// The values' part: largest squares of 64 keys, a workgroup a tile and head, 16
// bytes a lane.
constexpr int NORM_KEYS = 64;
static_assert(NORM_KEYS == BN, "dq counts them by its tiles");
template <class T, int DP>
__global__ __launch_bounds__(NT) void packattn_norms_kernel(PackedAttn a, int64_t tiles, float* vmax) {
  __shared__ float best[WAVES];
  constexpr int LR = DP / 8;  // lanes a row
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, e = threadIdx.x % LR * 8;
  for (int64_t y = blockIdx.x; y < tiles * a.kv_heads; y += gridDim.x) {
    const int64_t x = y / a.kv_heads;
    const int head = (int)(y % a.kv_heads);
    int s;
    const int64_t t = find_tile(a.k_off, a.sequences, a.k_tokens, 1, NORM_KEYS, x, s);
    const Seq seq = sequence(a, s, true);
    const int n = t < 0 ? 0 : (int)min((int64_t)NORM_KEYS, seq.lk - t * NORM_KEYS);
    float m = 0.f;
    for (int r = threadIdx.x / LR; r < n; r += NT / LR) {
      float v[8], sq = 0.f;
      Vec<T>::unpack(load8(row_ptr<const T>(a.v, seq.k0 + t * NORM_KEYS + r, head), e, a.width), v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sq = fmaf(v[i], v[i], sq);
      sq = group_sum<LR>(sq);
      m = fmaxf(m, finite_or_zero(sq));
    }
    m = group_max<64>(m);
    __syncthreads();  // the tile before has been read
    if (lane == 0) best[wave] = m;
    __syncthreads();
    if (threadIdx.x == 0)
      vmax[head * tiles + x] = fmaxf(fmaxf(best[0], best[1]), fmaxf(best[2], best[3]));
  }
}
constexpr int NORM_BLOCKS = 2048;

// the largest of n squares, over a wave
__device__ __forceinline__ float largest(const float* squares, int n) {
  float m = 0.f;
#pragma unroll 4
  for (int i = threadIdx.x & 63; i < n; i += 64) m = fmaxf(m, squares[i]);
  return group_max<64>(m);
}
// the scale of dS from the largest squares of a row of do and of v: a power of two,
// dS below 2^14
__device__ __forceinline__ float ds_scale(float g, float v) {
  const float b = sqrtf(g) * sqrtf(v);  // |dS| <= 2 b
  if (!(b > 0.f)) return 1.f;
  return ldexpf(1.f, max(-100, min(100, 12 - (int)ceilf(log2f(b)))));
}

// What the gradient's two kernels share.  Where one has fewer workgroups than the
// card takes, each sequence's keys (of dq) or rows (of dk, dv) are cut into
// parts, whose sums packattn_sum_kernel adds in their order.
struct Back {
  float* delta;         // [heads][q_tokens]
  // binary16: the largest squares of a row, over 64 keys of v and 32 rows of do
  float *vmax, *gmax;  // [kv_heads][v_tiles], [kv_heads][4 * tiles of dq]
  int64_t v_tiles, g_tiles;
  int q_parts, k_parts;
  float* dq;            // [part][q_tokens][heads][DP]
  float *dk, *dv;       // [part][k_tokens][kv_heads][DP]
};

constexpr int FEW_KEYS = 1024;
// dq, and D = sum (do o) of every row for the other kernel.  The forward's layout
// with a product more, and as it bound by products and exponentials.  The scores
// are made in both kernels, so that neither adds to memory in an order of
// chance: nine products for seven, and for rows of up to 1024 keys eleven (below).
// 6 causal sequences of 10007 tokens, 32 heads over 8 of 128, bfloat16: this 371 us
// (the order of reads saved 6%), the other 469.
template <class T, int DP>
__global__ __launch_bounds__(NT, 2) void packattn_dq_kernel(PackedAttn a, int64_t tiles, Back back) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  constexpr int BM = 32 * WAVES, KS = DP / 16, DB = DP / 32, TILE = BN * DP * 2;
  const Place at = place(a.kv_heads, tiles);
  if (at.tile < 0) return;
  const int G = a.heads / a.kv_heads;
  int s;
  // from the last tile: a causal sequence's last rows see the most keys
  const int64_t number = tiles - 1 - at.tile, t = find_tile(a.q_off, a.sequences, a.q_tokens, G, BM, number, s);
  const Seq seq = lane_seq(sequence(a, s, false), 0);
  const int rows = (a.fill ? seq.have : seq.lq) * G;
  if (t < 0 || t * BM >= rows) return;
  const int r0 = (int)t * BM;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), h = lane >> 5;
  const Row row = row_of(a, seq, r0 + 32 * wave + (lane & 31), G);
  const int head = at.head * G + row.g;
  const int64_t token = seq.q0 + row.i, at_row = (int64_t)head * a.q_tokens + token;
  const int most = wave_max(row.last), least = wave_min(row.last);
  const Row end = row_of(a, seq, min(r0 + BM, rows) - 1, G);
  int far = uniform(end.last);
  if (a.fill && seq.lq < seq.have) far = seq.lk - 1;
  const int every = far < 0 ? 0 : far / BN + 1, per = (every + back.q_parts - 1) / back.q_parts;
  const int part = blockIdx.y, kt0 = part * per, nk = min(every, kt0 + per);
  float vmax = 0.f;
  if (Half<T>::SCALED) vmax = largest(back.vmax + at.head * back.v_tiles + seq.k0 / NORM_KEYS + s, every);

  u32x4 q[KS], g[KS];
  const T* qrow = row_ptr<const T>(a.q, token, head);
  const T* grow = row_ptr<const T>(a.d_o, token, head);
  const T* orow = row_ptr<const T>(a.o, token, head);
  float D = 0.f, gg = 0.f;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    q[ks] = load8(qrow, 16 * ks + 8 * h, a.width);
    g[ks] = load8(grow, 16 * ks + 8 * h, a.width);
    float x[8], y[8];
    Vec<T>::unpack(g[ks], x);
    Vec<T>::unpack(load8(orow, 16 * ks + 8 * h, a.width), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      D = fmaf(x[i], y[i], D);
      if (Half<T>::SCALED) gg = fmaf(x[i], x[i], gg);
    }
  }
  D = other_half_sum(D);
  float ds = 1.f;
  if (Half<T>::SCALED) {
    gg = other_half_sum(gg);
    gg = row.last < 0 ? 0.f : finite_or_zero(gg);
    ds = ds_scale(gg, vmax);
    const float m = group_max<64>(gg);
    if (part == 0 && lane == 0) back.gmax[at.head * back.g_tiles + number * WAVES + wave] = m;
  }
  float lse = a.lse[at_row] * LOG2E;
  if (row.last < 0) lse = -NEG_INF;  // a row without a key: P = 0
  const float c = a.scale * LOG2E;
  f32x16 o[DB];
  const unsigned lds0 = lds_addr(smem);
  // what was loaded above is here before the first copy is issued
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  KeyTiles<T, DP, BN, WAVES> tile;
  Operands<DP> x;
  x.init(lds0, lane);
  // Rows of few keys: out, an average of few values, is as large as each of them,
  // and its rounding would weigh as much in dS as that of dS itself.  Their D is
  // taken from the keys, sum P dP, by every part for itself (224 keys, binary16: dq
  // 1.56 times as far off as its own rounding with the rounded out, 1.46 so; up to
  // 1040 keys, bfloat16: 1.54 and 1.48).  It costs the packed prompts' gradient 3%.
  if (every <= FEW_KEYS / BN && (part == 0 || kt0 < nk)) {
    tile.init(a, seq, at.head, 0, BN, wave, lane);
    float sum = 0.f;
    for (int kt = 0; kt < every; ++kt) {
      if (kt == 0) tile.both(lds0);
      const unsigned here = (kt & 1) * 2 * TILE;
      wait_all_and_sync();
      if (kt + 1 < every) tile.both(lds0 + (~kt & 1) * 2 * TILE);
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        f32x16 p = {}, d = {};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          p = Half<T>::mma(x.row(here + 32 * b * DP * 2, ks), q[ks], p);
          d = Half<T>::mma(x.row(here + 32 * b * DP * 2 + TILE, ks), g[ks], d);
        }
        const int last = row.last - kt * BN - 4 * h;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i / 4) + i % 4 <= last) sum = fmaf(exp2_f(fmaf(p[i], c, -lse)), d[i], sum);
      }
    }
    D = other_half_sum(sum);
    wait_all_and_sync();
  }
  if (row.last < 0) D = 0.f;  // no gradient, whatever do holds
  if (row.stored && row.i < seq.lq && h == 0 && part == 0) back.delta[at_row] = D;
  // The first key that not all rows see, once others have to be wiped from there on;
  // marks: NaN for keys that had some, whose scores are NaN then where they are seen.
  int wiped = 0x7fffffff;
  float* marks = reinterpret_cast<float*>(smem + 4 * TILE + WORDS);  // [BN]
  auto step = [&](int kt, unsigned here, unsigned next) __attribute__((always_inline)) {
    const int k0 = kt * BN;
    wait_all_and_sync();
    const bool wiping = k0 + BN > wiped;
    if (wiping) {
      if (threadIdx.x < BN) marks[threadIdx.x] = 0.f;
      __syncthreads();
#pragma unroll 1
      for (int i = threadIdx.x; i < TILE / 16; i += NT)
        if (wipe<T>(lds0 + here, i)) marks[i / (DP / 8)] = __builtin_nanf("");
      __syncthreads();
    }
    if (kt + 1 < nk) tile.both(lds0 + next);
    if (k0 > most) return;
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const unsigned kb = here + 32 * b * DP * 2, vb = kb + TILE;
      f32x16 p = {}, d = {};
      {
        u32x4 f[2 * KS];
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) f[i] = x.row(i & 1 ? vb : kb, i / 2);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          p = Half<T>::mma(f[2 * ks], q[ks], p);
          d = Half<T>::mma(f[2 * ks + 1], g[ks], d);
        }
        constexpr int AHEAD = KS < 4 ? 2 * KS : 8;
        order<LDS_READ, AHEAD>();
#pragma unroll
        for (int i = 0; i < 2 * KS - AHEAD; ++i) {
          order<MFMA, 1>();
          order<LDS_READ, 1>();
        }
        order<MFMA, AHEAD>();
      }
      if (wiping) {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] += marks[32 * b + 8 * (i / 4) + 4 * h + i % 4];
      }
      const int last = row.last - k0 - 4 * h;
      if (k0 + 32 * b + 31 > least) {  // a dP of NaN in a masked place stays there
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * b + 8 * (i / 4) + i % 4 > last) {
            p[i] = NEG_INF;
            d[i] = 0.f;
          }
      }
      u32x4 f[2][DB];
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int db = 0; db < DB; ++db) f[kg][db] = x.column(kb + 16 * kg * DP * 2, db);
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
#pragma unroll
        for (int i = 8 * kg; i < 8 * kg + 8; ++i) {
          d[i] = exp2_f(fmaf(p[i], c, -lse)) * (d[i] - D);
          if (Half<T>::SCALED) d[i] *= ds;
        }
        const u32x4 w = pack8<T>(d, kg);
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = Half<T>::mma(f[kg][db], w, o[db]);
      }
      order<LDS_READ, 2 * DB>();
      order<VALU, 36>();
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        order<MFMA, 1>();
        order<LDS_READ, 2>();
        order<VALU, 36 / DB>();
      }
      order<MFMA, DB>();
    }
  };
  for (;;) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
    tile.init(a, seq, at.head, kt0 * BN, BN, wave, lane);
    if (kt0 < nk) tile.both(lds0);
    for (int kt = kt0; kt < nk; kt += 2) {
      step(kt, 0, 2 * TILE);
      if (kt + 1 < nk) step(kt + 1, 2 * TILE, 0);
    }
    if (!a.causal || wiped < 0x7fffffff) break;
    const bool others = row.last >= 0 && row.last < min(most / BN * BN + BN, seq.lk) - 1 && has_others(o);
    if (!any_wave<WAVES>(__any(others), reinterpret_cast<int*>(smem + 4 * TILE), wave)) break;
    wiped = uniform(row_of(a, seq, r0, G).last) + 1;
  }
  if (row.last < 0) {
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};
  }
  const float f = a.scale / ds;
  if (back.q_parts == 1) {
    store_columns<T, DB>(o, f, row.stored ? row_ptr<T>(a.dq, token, head) : nullptr, a.width, lane);
  } else {
    const int64_t at_sum = ((part * a.q_tokens + token) * a.heads + head) * DP;
    store_sums<DB>(o, f, row.stored ? back.dq + at_sum : nullptr, lane);
  }
}

// dk, dv: workgroup = 128 keys of one sequence and head over the rows of all the
// group's heads in tiles of 64; wave w has the keys 32 (w % 4) .. and the half
// w / 4 of every tile's rows, and the halves are added in LDS at the end.
//
// dk and dv take half of a wave's registers, so two waves a SIMD, without which
// the matrix cores wait for each exponential, leave no room for the keys' and
// values' operands beside them: those are read from LDS, in operand order (one
// wave a SIMD with them in registers 960 us, two 672, with the reads ahead of
// their products and the heaviest tiles first 478, without divisions a tile 469).
template <class T, int DP>
__global__ __launch_bounds__(2 * NT, 2) void packattn_dkv_kernel(PackedAttn a, int64_t tiles, Back back) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  typedef TileCopy<DP, BN, 2 * WAVES> C;
  constexpr int BK = 32 * WAVES, KS = DP / 16, DB = DP / 32, TILE = BN * DP * 2;
  const Place at = place(a.kv_heads, tiles);
  if (at.tile < 0) return;
  const int G = a.heads / a.kv_heads;
  int s;
  int64_t t;
  if (!find_work(a, at.tile, s, t)) return;
  const Seq seq = lane_seq(sequence(a, s, true), 0);
  const int have = a.fill ? seq.have : seq.lk;
  if (t * BK >= have) return;
  const int j0 = (int)t * BK;
  const int lane = threadIdx.x & 63, h = lane >> 5, wave = uniform(threadIdx.x >> 6);
  const int group = wave & 3, half = wave >> 2;
  const int j = j0 + 32 * group + (lane & 31);  // a lane's key
  const bool stored = j < have, live = j < seq.lk;
  const int64_t token = seq.k0 + min(j, have - 1);
  const int lag = seq.lk - seq.lq;  // query i sees keys up to i + lag
  const KeyRows seen = rows_of_keys(a.causal, j0, seq.lq, seq.lk, G, BN);
  const int sees = seen.blind;  // rows before see no key: taken as zeros
  const int part = blockIdx.y;
  const Part range = part_of_rows(seen, back.k_parts, part, BN);
  const int from = range.from, rows = range.to;
  float ds = 1.f;
  if (Half<T>::SCALED) {  // rows 32 x on of the sequence are dq's wave 4 q0 G / 128 + 4 s + x
    const int64_t wave0 = (seq.q0 * G / BK + s) * WAVES;
    const float g = largest(back.gmax + at.head * back.g_tiles + wave0 + from / 32, (rows - from + 31) / 32);
    const float v = largest(back.vmax + at.head * back.v_tiles + seq.k0 / NORM_KEYS + s,
                            rows > from ? (seq.lk + NORM_KEYS - 1) / NORM_KEYS : 0);
    ds = __builtin_bit_cast(float, uniform(__builtin_bit_cast(int, ds_scale(g, v))));
  }
  // P is made 2^SHIFT times as large in binary16
  constexpr float SHIFT = 2 * Half<T>::SHIFT;

  // the buffers (Q, do, and lse, D and the last key of their rows), then K, V
  constexpr int BUF = 2 * TILE + 3 * BN * 4, OPERANDS = KS * 1024;
  const unsigned lds0 = lds_addr(smem);
  const unsigned kop = lds0 + 2 * BUF + group * (2 * OPERANDS) + lane * 16;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks) {
    const u32x4 none = {0, 0, 0, 0};
    const HeadView& kv = half ? a.v : a.k;
    *(__attribute__((address_space(3))) u32x4*)(kop + half * OPERANDS + ks * 1024) =
        live ? load8(row_ptr<const T>(kv, token, at.head), 16 * ks + 8 * h, a.width) : none;
  }
  f32x16 dk[DB], dv[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) dk[db] = dv[db] = f32x16{};
  const float c = a.scale * LOG2E;

  int* others = reinterpret_cast<int*>(smem + 2 * BUF + 8 * OPERANDS);  // of a tile's rows, by buffer
  auto stats = [&](int buf) { return reinterpret_cast<float*>(smem + buf * BUF + 2 * TILE); };
  // Where 64 rows are whole tokens, the next tile's lie as this one's, so many
  // tokens on; elsewhere each tile divides its rows anew.
  const bool even = BN % G == 0;
  const int tokens = BN / G;
  auto offset = [&](const HeadView& v, int r, int i0, int i) {
    const int token_ = r / G, e = C::elem(i, wave, lane);
    return e < a.width ? (unsigned)((token_ - i0) * v.st + (r - token_ * G) * v.sh + e) * 2 : NOWHERE;
  };
  unsigned qo[C::PER], go[C::PER];
  const int i_from = from / G;
#pragma unroll
  for (int i = 0; i < C::PER; ++i) {
    const int r = from + C::row(i, wave, lane);
    qo[i] = offset(a.q, r, i_from, i);
    go[i] = offset(a.d_o, r, i_from, i);
  }
  uint64_t qp = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.q, seq.q0 + i_from, at.head * G));
  uint64_t gp = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.d_o, seq.q0 + i_from, at.head * G));
  const int64_t q_step = uniform64(tokens * a.q.st * 2), g_step = uniform64(tokens * a.d_o.st * 2);
  // the row whose lse, D and last key a thread of the first wave fetches
  int my_i = (from + (int)threadIdx.x) / G, my_g = from + (int)threadIdx.x - my_i * G;
  float n_lse = 0.f, n_delta = 0.f;
  int n_last = -1;
  auto issue = [&](int r0, int buf) __attribute__((always_inline)) {
    if (!even) {
      const int i0 = r0 / G;
      qp = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.q, seq.q0 + i0, at.head * G));
      gp = uniform64((int64_t)(uintptr_t)row_ptr<const T>(a.d_o, seq.q0 + i0, at.head * G));
#pragma unroll
      for (int i = 0; i < C::PER; ++i) {
        const int r = r0 + C::row(i, wave, lane);
        qo[i] = offset(a.q, r, i0, i);
        go[i] = offset(a.d_o, r, i0, i);
      }
      my_i = (r0 + (int)threadIdx.x) / G;
      my_g = r0 + (int)threadIdx.x - my_i * G;
    }
    if (wave == 0) {
      n_lse = -NEG_INF;
      n_delta = 0.f;
      n_last = -1;
      if (r0 + lane < rows) {
        const int64_t p = (int64_t)(at.head * G + my_g) * a.q_tokens + seq.q0 + my_i;
        n_lse = a.lse[p] * LOG2E;
        n_delta = back.delta[p];
        n_last = a.causal ? my_i + lag : seq.lk;
      }
    }
    const unsigned lds = lds0 + buf * BUF;
    const u32x4 qd = descriptor(qp), gd = descriptor(gp);
#pragma unroll
    for (int i = 0; i < C::PER; ++i) {
      if (!C::any(i, wave)) continue;
      const int r = r0 + C::row(i, wave, lane);
      const bool in = r >= sees && r < rows;
      copy16(in ? qo[i] : NOWHERE, qd, lds + C::dst(i, wave));
      copy16(in ? go[i] : NOWHERE, gd, lds + TILE + C::dst(i, wave));
    }
    qp += q_step;
    gp += g_step;
    my_i += tokens;
  };
  auto keep = [&](int buf) {
    if (wave == 0) {
      float* st = stats(buf);
      st[lane] = n_last < 0 ? -NEG_INF : n_lse;  // a row without a key: P = 0
      st[BN + lane] = n_delta;
      reinterpret_cast<int*>(st)[2 * BN + lane] = n_last;
      // a row of others in q or do has an lse or a D of them
      const bool other = n_last >= 0 && !(fabsf(n_delta) < -NEG_INF && n_lse == n_lse);
      if (a.causal) others[buf] = __any(other);
    }
  };
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  if (from < rows) {
    issue(from, 0);
    keep(0);
  }
  Operands<DP> ops;
  ops.init(lds0 + half * (32 * DP * 2), lane);
  // the first rows that see the first of the wave's keys, all of them, all of the workgroup's
  // (a division by G a tile for each comparison: 478 us, with a third one 488, so 469)
  const int some = j0 + 32 * group < seq.lk ? first_row(a.causal, j0 + 32 * group, seq.lq, seq.lk, G) : 0x7fffffff;
  const int every = first_row(a.causal, j0 + 32 * group + 31, seq.lq, seq.lk, G);
  const int whole = first_row(a.causal, j0 + BK - 1, seq.lq, seq.lk, G);
  auto step = [&](int r0, auto buf_) __attribute__((always_inline)) {
    constexpr int buf = decltype(buf_)::value;
    wait_all_and_sync();
    // Where some rows of the tile do not see all keys: others in rows that have any are
    // wiped, and P and dS of such a row are NaN where it sees.
    if (r0 < whole && uniform(others[buf])) {
#pragma unroll 1
      for (int i = 64 * wave + lane; i < 2 * TILE / 16; i += 2 * NT)
        if (wipe<T>(lds0 + buf * BUF, i)) stats(buf)[i % (TILE / 16) / (DP / 8)] = __builtin_nanf("");
      __syncthreads();
    }
    if (r0 + BN < rows) issue(r0 + BN, buf ^ 1);
    const int mine = r0 + 32 * half;  // the wave's rows of the tile
    const bool any = mine < rows && mine + 31 >= some;
    if (any) {
      const unsigned sb = lds0 + buf * BUF + 2 * TILE + 128 * half;
      const bool cut = mine < every;
      constexpr unsigned qb = buf * BUF, gb = qb + TILE;
      f32x16 p = {}, d = {};
      {
        u32x4 f[4 * KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          f[4 * ks] = ops.row(qb, ks);
          f[4 * ks + 1] = *(lds_u32x4*)(kop + ks * 1024);
          f[4 * ks + 2] = ops.row(gb, ks);
          f[4 * ks + 3] = *(lds_u32x4*)(kop + OPERANDS + ks * 1024);
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          p = Half<T>::mma(f[4 * ks], f[4 * ks + 1], p);
          d = Half<T>::mma(f[4 * ks + 2], f[4 * ks + 3], d);
        }
        constexpr int AHEAD = 1;  // steps of the width
        order<LDS_READ, 4 * AHEAD>();
#pragma unroll
        for (int i = 0; i < KS - AHEAD; ++i) {
          order<MFMA, 1>();
          order<LDS_READ, 2>();
          order<MFMA, 1>();
          order<LDS_READ, 2>();
        }
        order<MFMA, 2 * AHEAD>();
      }
      f32x4 lse[4], D[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const unsigned at_row = sb + (8 * x + 4 * h) * 4;
        lse[x] = *(lds_f32x4*)at_row;
        D[x] = *(lds_f32x4*)(at_row + BN * 4);
      }
      if (cut) {  // what a row holds that does not see the key stays there: P = dS = 0
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const u32x4 last = *(lds_u32x4*)(sb + (8 * x + 4 * h) * 4 + 2 * BN * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j > (int)last[i]) {
              p[4 * x + i] = d[4 * x + i] = D[x][i] = 0.f;
              lse[x][i] = -NEG_INF;
            }
        }
      }
      u32x4 fg[2][DB], fq[2][DB];
#pragma unroll
      for (int kg = 0; kg < 2; ++kg)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          fg[kg][db] = ops.column(gb + 16 * kg * DP * 2, db);
          fq[kg][db] = ops.column(qb + 16 * kg * DP * 2, db);
        }
#pragma unroll
      for (int kg = 0; kg < 2; ++kg) {
#pragma unroll
        for (int i = 8 * kg; i < 8 * kg + 8; ++i) {
          p[i] = exp2_f(fmaf(p[i], c, SHIFT - lse[i / 4][i % 4]));
          d[i] = p[i] * (d[i] - D[i / 4][i % 4]);
          if (Half<T>::SCALED) d[i] *= ds * (1.f / 16384.f);  // 2^-SHIFT
        }
        const u32x4 wp = pack8<T>(p, kg), wd = pack8<T>(d, kg);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          dv[db] = Half<T>::mma(fg[kg][db], wp, dv[db]);
          dk[db] = Half<T>::mma(fq[kg][db], wd, dk[db]);
        }
      }
      order<LDS_READ, 4>();
      order<VALU, 48>();
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        order<LDS_READ, 2>();
        order<MFMA, 1>();
        order<VALU, 48 / (2 * DB)>();
      }
#pragma unroll
      for (int i = 0; i < 2 * DB - 2; ++i) {
        order<LDS_READ, 2>();
        order<MFMA, 1>();
      }
      order<MFMA, 2>();
    }
    if (r0 + BN < rows) keep(buf ^ 1);
  };
  for (int r0 = from; r0 < rows; r0 += 2 * BN) {
    step(r0, std::integral_constant<int, 0>());
    if (r0 + BN < rows) step(r0 + BN, std::integral_constant<int, 1>());
  }
  // the second half's sums to the first: dk, then dv, in [group][element][lane]
  float* sums = reinterpret_cast<float*>(smem) + group * (DB * 16 * 64) + lane;
  auto join = [&](f32x16 (&x)[DB]) __attribute__((always_inline)) {
    __syncthreads();
    if (half) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) sums[(db * 16 + i) * 64] = x[db][i];
    }
    __syncthreads();
    if (!half) {
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) x[db][i] = live ? x[db][i] + sums[(db * 16 + i) * 64] : 0.f;
    }
  };
  join(dk);
  join(dv);
  if (half) return;
  const float fk = a.scale / ds, fv = Half<T>::SCALED ? 1.f / 16384.f : 1.f;
  if (back.k_parts == 1) {
    store_columns<T, DB>(dk, fk, stored ? row_ptr<T>(a.dk, token, at.head) : nullptr, a.width, lane);
    store_columns<T, DB>(dv, fv, stored ? row_ptr<T>(a.dv, token, at.head) : nullptr, a.width, lane);
  } else {
    const int64_t at_sum = ((part * a.k_tokens + token) * a.kv_heads + at.head) * DP;
    store_sums<DB>(dk, fk, stored ? back.dk + at_sum : nullptr, lane);
    store_sums<DB>(dv, fv, stored ? back.dv + at_sum : nullptr, lane);
  }
}

constexpr int SUM_TOKENS = 4;  // of a workgroup
// Bound by memory; 7 to 18 us where there are parts at all.
// The parts' sums of a few tokens of one sequence: blockIdx.y 0 of dq, 1 of dk, 2 of dv.
template <class T, int DP>
__global__ __launch_bounds__(NT) void packattn_sum_kernel(PackedAttn a, Back back) {
  const bool keys = blockIdx.y > 0;
  const int parts = keys ? back.k_parts : back.q_parts;
  if (parts == 1) return;
  const int64_t n = keys ? a.k_tokens : a.q_tokens;
  int s;
  const int64_t t = find_tile(keys ? a.k_off : a.q_off, a.sequences, n, 1, SUM_TOKENS, blockIdx.x, s);
  const Seq seq = lane_seq(sequence(a, s, keys), 0);
  const int have = a.fill ? seq.have : keys ? seq.lk : seq.lq, heads = keys ? a.kv_heads : a.heads;
  if (t < 0 || t * SUM_TOKENS >= have) return;
  const int count = (int)min((int64_t)SUM_TOKENS, have - t * SUM_TOKENS);
  const int64_t token0 = (keys ? seq.k0 : seq.q0) + t * SUM_TOKENS, stride = n * heads * DP;
  const float* sums = blockIdx.y == 0 ? back.dq : blockIdx.y == 1 ? back.dk : back.dv;
  const HeadView& out = blockIdx.y == 0 ? a.dq : blockIdx.y == 1 ? a.dk : a.dv;
  for (int i = threadIdx.x; i < count * heads * (DP / 4); i += NT) {
    const int e = i % (DP / 4) * 4, row = i / (DP / 4);
    if (e >= a.width) continue;
    const int64_t token = token0 + row / heads;
    const float* p = sums + (token0 * heads + row) * DP + e;
    float v[4] = {};
#pragma unroll 8
    for (int k = 0; k < parts; ++k) {
      const float4 x = *reinterpret_cast<const float4*>(p + k * stride);
      v[0] += x.x;
      v[1] += x.y;
      v[2] += x.z;
      v[3] += x.w;
    }
    Few<T, 4>::template store<false>(row_ptr<T>(out, token, row % heads) + e, v);
  }
}

// ------------------------------------------------------------------ launches
int64_t tiles_of(int64_t tokens, int unit, int tile, int sequences) {
  return tokens * unit / tile + sequences + 2;
}

template <class F, class T>
void by_width(const PackedAttn& a, T, F f) {
  if (a.width <= 32) f(T(), std::integral_constant<int, 32>());
  else if (a.width <= 64) f(T(), std::integral_constant<int, 64>());
  else f(T(), std::integral_constant<int, 128>());
}
template <class F>
void by_type(const PackedAttn& a, F f) {
  if (a.dtype == BC2N_F16) by_width(a, h16(), f);
  else by_width(a, bf16(), f);
  hip_check(hipGetLastError(), "attention launch");
}
// more than 64 KB of LDS has to be asked for
template <class K>
void with_lds(K* kernel, size_t bytes) {
  if (bytes > 64 * 1024)
    hip_check(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes),
            "hipFuncSetAttribute");
}

}  // namespace

namespace {

int padded(int width) { return width <= 32 ? 32 : width <= 64 ? 64 : 128; }

// Up to so many keys of all sequences one workgroup takes any sequence's.
constexpr int64_t UNSPLIT = 4096;

// Whether the rows go to the few-rows kernel: where a sequence has 32 rows or
// fewer, and where 128-row workgroups (`blocks` of them, each a sequence's keys
// long) would leave so many compute units idle that the other's overheads cost
// less.  A 128-row workgroup by itself on a unit takes 64 keys in 1.1 to 1.5 us;
// the stretches of all rows take a unit's share of the same in 1.65 times that, and
// their join some 20 us: they win where keys * (2/3 - blocks / units) is above 800
// (one sequence, 4 heads: of 4000 tokens 25 against 48 us, of 7900 200 against
// 133; three of 1800 61 against 34).  Without a join four waves share a
// sequence's keys, which from 1024 on pays as long as units are idle (one of 3000, 8
// heads 29 against 54 us; six of 512 25 against 16).
bool few_rows(const PackedAttn& a) {
  const int64_t rows = a.q_tokens * (a.heads / a.kv_heads), cus = device_cus();
  const int64_t live = std::max<int64_t>(1, std::min<int64_t>(a.sequences, a.q_tokens));
  if (rows <= 32 * live) return true;
  const int64_t blocks = std::max((rows + 127) / 128, live) * a.kv_heads, keys = a.k_tokens / live;
  if (a.k_tokens <= UNSPLIT) return 8 * blocks < 5 * cus || (keys >= 1024 && blocks < cus);
  return 3 * blocks < 2 * cus && keys * (2 * cus - 3 * blocks) > 3 * 800 * cus;
}
// Waves of it that the card holds, by their registers.
int64_t few_grid(const PackedAttn&) { return (int64_t)device_cus() * 8; }
// Stretches of a head of keys that fill it once.  A sequence with more than
// one has more blocks than a stretch, so all of those have at most twice as many.
int64_t few_goal(const PackedAttn& a) { return std::max<int64_t>(1, few_grid(a) / a.kv_heads); }
Split carve_split(const PackedAttn& a, char* p, size_t* bytes) {
  const size_t rows = (size_t)2 * few_goal(a) * a.kv_heads * 32;
  Split s;
  Sizer z;
  s.o = reinterpret_cast<float*>(p);
  z.take<float>(rows * padded(a.width));
  s.ml = reinterpret_cast<float2*>(p + z.off);
  z.take<float2>(rows);
  s.table = Table{};
  const size_t entries = (size_t)a.sequences + 2;
  if (entries > 64 * HELD) {
    int64_t** at[] = {&s.table.per, &s.table.items, &s.table.splits, &s.table.slots};
    for (int64_t** x : at) {
      *x = reinterpret_cast<int64_t*>(p + z.off);
      z.take<int64_t>(x == &s.table.per ? 1 : entries + 1);
    }
  }
  *bytes = z.off;
  return s;
}
bool may_split(const PackedAttn& a) { return a.q_tokens > 0 && few_rows(a) && a.k_tokens > UNSPLIT; }

}  // namespace

size_t packattn_fwd_work_bytes(const PackedAttn& a) {
  size_t n = 0;
  if (may_split(a)) carve_split(a, nullptr, &n);
  return n;
}

namespace {

// Parts of the sequences in the gradient's kernels: as many as make one round of
// workgroups, two a compute unit for dq and one for dk and dv, and no shorter than
// what a part costs by itself: 4 tiles of keys, 8 of rows (two sequences of 1262
// keys, 8 heads over one: 19 parts of 5 tiles 48 us, 9 of 10 34).
Back carve_back(const PackedAttn& a, char* base, size_t* bytes) {
  const int64_t G = a.heads / a.kv_heads, cus = device_cus(), DP = padded(a.width);
  const int64_t live = std::max<int64_t>(1, std::min<int64_t>(a.sequences, std::min(a.q_tokens, a.k_tokens)));
  auto parts = [&](int64_t room, int64_t items, int64_t tiles, int64_t shortest) {
    const int64_t blocks = std::max(live, (items + 127) / 128) * a.kv_heads;
    return (int)std::max<int64_t>(1, std::min<int64_t>({room / blocks, tiles / live / shortest, 64}));
  };
  Back b = {};
  b.q_parts = parts(2 * cus, a.q_tokens * G, a.k_tokens / BN, 4);
  b.k_parts = parts(cus, a.k_tokens, a.q_tokens * G / BN, 8);
  Sizer z;
  auto take = [&](int64_t n) {
    float* p = reinterpret_cast<float*>(base + z.off);
    z.take<float>((size_t)n);
    return p;
  };
  b.delta = take(a.heads * a.q_tokens);
  const bool scaled = a.dtype == BC2N_F16;
  b.v_tiles = tiles_of(a.k_tokens, 1, NORM_KEYS, a.sequences);
  b.g_tiles = tiles_of(a.q_tokens, (int)G, 32 * WAVES, a.sequences) * WAVES;
  b.vmax = take(scaled ? a.kv_heads * b.v_tiles : 0);
  b.gmax = take(scaled ? a.kv_heads * b.g_tiles : 0);
  b.dq = take(b.q_parts > 1 ? b.q_parts * a.q_tokens * a.heads * DP : 0);
  b.dk = take(b.k_parts > 1 ? b.k_parts * a.k_tokens * a.kv_heads * DP : 0);
  b.dv = take(b.k_parts > 1 ? b.k_parts * a.k_tokens * a.kv_heads * DP : 0);
  *bytes = z.off;
  return b;
}

}  // namespace

size_t packattn_bwd_work_bytes(const PackedAttn& a) {
  size_t n = 0;
  carve_back(a, nullptr, &n);
  return n;
}

void packattn_fwd(hipStream_t st, const PackedAttn& a, void* work) {
  if (a.q_tokens == 0) return;
  KTimed kt("attention.fwd", st);
  const int64_t G = a.heads / a.kv_heads;
  by_type(a, [&](auto v, auto dp) {
    typedef decltype(v) T;
    constexpr int DP = decltype(dp)::value;
    if (!few_rows(a)) {
      const int64_t tiles = tiles_of(a.q_tokens, G, 32 * WAVES, a.sequences);
      auto* kernel = &packattn_fwd_kernel<T, DP>;
      const size_t lds = 4 * BN * DP * 2 + WORDS;
      with_lds(kernel, lds);
      kernel<<<place_grid(a.kv_heads, tiles), NT, lds, st>>>(a, tiles);
      return;
    }
    const int64_t tiles = tiles_of(a.q_tokens, G, 32, a.sequences);
    if (!may_split(a)) {
      const int64_t items = std::min(tiles * a.kv_heads, 4 * (int64_t)device_cus());
      packattn_keys_kernel<T, DP, 4, false><<<(unsigned)items, 256, 0, st>>>(a, tiles, Split{});
      return;
    }
    size_t bytes = 0;
    const Split split = carve_split(a, reinterpret_cast<char*>(work), &bytes);
    const int64_t goal = few_goal(a);
    // items: a tile's first stretch each, and the further ones
    const int64_t items = (tiles + goal) * a.kv_heads;
    // a row's share of the waves, and of the stretches, were all sequences alike
    const int64_t rows = a.q_tokens * G, live = std::max<int64_t>(1, std::min<int64_t>(a.sequences, a.q_tokens));
    const int64_t x = std::min(live + rows / 32, goal) * a.kv_heads;
    const int64_t y = std::min<int64_t>(32, (rows + live - 1) / live);
    auto launch = [&](auto table) {
      constexpr bool TABLE = decltype(table)::value;
      packattn_keys_kernel<T, DP, 1, TABLE><<<(unsigned)std::min(items, few_grid(a)), 64, 0, st>>>(a, goal, split);
      // 16 waves a row where it has some 32 stretches (one sequence of 131 k, 8 rows a
      // head of keys: 12 us), one where it has fewer (7974 rows of three heads, two or
      // three stretches each: 592 us of 16 waves, 41 of one)
      if (goal >= 32 * std::max(live, rows / 32))
        packattn_join_kernel<T, DP, 16, TABLE><<<dim3((unsigned)x, (unsigned)y), 1024, 0, st>>>(a, goal, split);
      else
        packattn_join_kernel<T, DP, 1, TABLE><<<dim3((unsigned)x, (unsigned)(y + 3) / 4), NT, 0, st>>>(a, goal, split);
    };
    if (!split.table.per) {
      launch(std::false_type());
      return;
    }
    packattn_table_kernel<block_keys(DP)><<<1, 1024, 0, st>>>(a, goal, split.table);
    launch(std::true_type());
  });
}

void packattn_bwd(hipStream_t st, const PackedAttn& a, void* work) {
  if (a.q_tokens == 0 && a.k_tokens == 0) return;
  KTimed kt("attention.bwd", st);
  size_t bytes = 0;
  const Back back = carve_back(a, reinterpret_cast<char*>(work), &bytes);
  by_type(a, [&](auto v, auto dp) {
    typedef decltype(v) T;
    constexpr int DP = decltype(dp)::value;
    const int64_t q_tiles = tiles_of(a.q_tokens, a.heads / a.kv_heads, 32 * WAVES, a.sequences);
    const int64_t k_tiles = tiles_of(a.k_tokens, 1, 32 * WAVES, a.sequences);
    if constexpr (Half<T>::SCALED) {
      if (a.q_tokens && a.k_tokens) {
        const int64_t items = back.v_tiles * a.kv_heads;
        packattn_norms_kernel<T, DP><<<(unsigned)std::min<int64_t>(items, NORM_BLOCKS), NT, 0, st>>>(a, back.v_tiles,
                                                                                                    back.vmax);
      }
    }
    if (a.q_tokens) {
      auto* dq = &packattn_dq_kernel<T, DP>;
      const size_t lds = 4 * BN * DP * 2 + WORDS + BN * 4;
      with_lds(dq, lds);
      dq<<<dim3(place_grid(a.kv_heads, q_tiles), back.q_parts), NT, lds, st>>>(a, q_tiles, back);
    }
    if (a.k_tokens) {
      auto* dkv = &packattn_dkv_kernel<T, DP>;
      const size_t lds = 2 * (2 * BN * DP * 2 + 3 * BN * 4) + 2 * 32 * WAVES * DP * 2 + WORDS;
      with_lds(dkv, lds);
      dkv<<<dim3(place_grid(a.kv_heads, k_tiles), back.k_parts), 2 * NT, lds, st>>>(a, k_tiles, back);
    }
    if (back.q_parts > 1 || back.k_parts > 1) {
      const int64_t most = std::max(tiles_of(a.q_tokens, 1, SUM_TOKENS, a.sequences),
                                    tiles_of(a.k_tokens, 1, SUM_TOKENS, a.sequences));
      packattn_sum_kernel<T, DP><<<dim3((unsigned)most, 3), NT, 0, st>>>(a, back);
    }
  });
}

}  // namespace bc2n
