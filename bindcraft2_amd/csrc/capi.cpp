// The C ABI (include/bc2n.h): argument checks, weight lookup, error channel.
#include "../../include/bc2n.h"
#include "evoformer.h"
#include "gemm.h"
#include "gemm_f32.h"
#include "modules.h"
#include "tplembed.h"
#include "embed.h"
#include "heads.h"
#include "designstep.h"
#include "confidence.h"
#include "headnorm.h"
#include "logprobs.h"
#include "optim.h"
#include "packattn.h"
#include "sample.h"

#include <cmath>
#include <cstdio>
#include <map>
#include <tuple>

using namespace bc2n;

namespace {

// The library's scratch (arenas, detached and own save-sets, cotangent
// scales) is shared by every call on a GPU, so calls on different streams
// are ordered: each call records an event on its stream after its last
// launch, and a call arriving on another stream first waits for the
// previous call's event.  Calls on one stream pay one event record.  Under
// graph capture nothing is recorded or waited for (a captured graph runs on
// the capturing stream's order only).
struct StreamOrder {
  hipStream_t last = nullptr;
  hipEvent_t ev = nullptr;
  bool recorded = false;
};
std::mutex g_order_mu;
std::map<int, StreamOrder> g_order;
thread_local bool t_call_has_stream = false;
thread_local hipStream_t t_call_stream = nullptr;
thread_local int t_call_device = 0;

bool capturing(hipStream_t st) {
  hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(st, &cs) == hipSuccess && cs != hipStreamCaptureStatusNone;
}

hipStream_t as_stream(void* s) {
  hipStream_t st = reinterpret_cast<hipStream_t>(s);
  if (capturing(st)) return st;
  int dev = 0;
  BC2N_HIP(hipGetDevice(&dev));
  {
    std::lock_guard<std::mutex> lk(g_order_mu);
    StreamOrder& o = g_order[dev];
    if (o.recorded && o.last != st) BC2N_HIP(hipStreamWaitEvent(st, o.ev, 0));
  }
  t_call_has_stream = true;
  t_call_stream = st;
  t_call_device = dev;
  return st;
}

// For calls that use no library scratch: only their stream orders them, and
// they record no event (which costs a short call as much as its launch).
hipStream_t own_stream(void* s) { return reinterpret_cast<hipStream_t>(s); }

// after a call: mark the end of its work on its stream
void end_call() {
  if (!t_call_has_stream) return;
  t_call_has_stream = false;
  std::lock_guard<std::mutex> lk(g_order_mu);
  StreamOrder& o = g_order[t_call_device];
  if (!o.ev && hipEventCreateWithFlags(&o.ev, hipEventDisableTiming) != hipSuccess) return;
  if (hipEventRecord(o.ev, t_call_stream) == hipSuccess) {
    o.last = t_call_stream;
    o.recorded = true;
  }
}

template <class F>
int guarded(F f) {
  t_call_has_stream = false;
  int rc = 0;
  try {
    f();
  } catch (const std::exception& e) {
    set_error(e.what());
    rc = 1;
  } catch (...) {
    set_error("unknown error");
    rc = 1;
  }
  end_call();
  return rc;
}

std::mutex g_mu;
std::map<std::pair<std::string, std::string>, TriAttnW> g_triattn;

const TriAttnW& triattn_w(const char* dir, const char* prefix) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto key = std::make_pair(std::string(dir), std::string(prefix));
  auto it = g_triattn.find(key);
  if (it != g_triattn.end()) return it->second;
  TriAttnW w = triattn_weights(weights(dir), prefix);
  return g_triattn.emplace(key, w).first->second;
}

std::map<std::pair<std::string, std::string>, TriMulW> g_trimul;

const TriMulW& trimul_w(const char* dir, const char* prefix) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto key = std::make_pair(std::string(dir), std::string(prefix));
  auto it = g_trimul.find(key);
  if (it != g_trimul.end()) return it->second;
  TriMulW w = trimul_weights(weights(dir), prefix);
  return g_trimul.emplace(key, w).first->second;
}

template <class W, class F>
const W& cached(std::map<std::pair<std::string, std::string>, W>& m, const char* dir,
                const char* prefix, F make) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto key = std::make_pair(std::string(dir), std::string(prefix));
  auto it = m.find(key);
  if (it != m.end()) return it->second;
  W w = make(weights(dir), std::string(prefix));
  return m.emplace(key, w).first->second;
}
std::map<std::pair<std::string, std::string>, TransW> g_trans;
std::map<std::pair<std::string, std::string>, OpmW> g_opm;
std::map<std::pair<std::string, std::string>, MsaRowW> g_row;
std::map<std::pair<std::string, std::string>, MsaColW> g_col;
std::map<std::pair<std::string, std::string>, StackW> g_stack;

const StackW& stack_w(const char* dir, int depth, StackKind kind) {
  const char* kn = kind == StackKind::EVO ? ":evo" : kind == StackKind::PAIR_ONLY ? ":pair_only" : ":tpl";
  const std::string tag = std::to_string(depth) + kn;
  return cached(g_stack, dir, tag.c_str(), [&](WeightStore& ws, const std::string&) {
    return stack_weights(ws, depth, kind);
  });
}
StackKind evo_kind(int64_t pair_only) { return pair_only ? StackKind::PAIR_ONLY : StackKind::EVO; }

// Library-owned save-set for detached forwards (save=0) and own_save=1.
struct OwnSave {
  void* p = nullptr;
  size_t n = 0;
  void* get(hipStream_t st, size_t need) {
    if (need > n) {
      if (p) {
        BC2N_HIP(hipStreamSynchronize(st));
        BC2N_HIP(hipFree(p));
        p = nullptr;
      }
      BC2N_HIP(hipMalloc(&p, need));
      n = need;
    }
    return p;
  }
};
OwnSave g_own;
// Scratch of detached forwards (save = 0): one block's worth, reused.
OwnSave g_det;

void need(bool ok, const char* msg) {
  if (!ok) throw std::invalid_argument(msg);
}

}  // namespace

extern "C" {

const char* bc2n_last_error(void) { return last_error(); }
int bc2n_abi_version(void) { return 4; }

size_t bc2n_triattn_save_bytes(int N, int C, int H) { return triattn_save_bytes(N, C, H); }

int bc2n_triattn_fwd(void* stream, const char* weights_dir, const char* prefix, int per_column,
                     int N, const float* pair, const float* pair_mask, const float* drop_tbl,
                     float* pair_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix, "weights_dir/prefix required");
    need(pair && pair_mask && pair_out && save, "null operand");
    need(pair_out != pair, "triattn: pair_out must not alias pair");
    const TriAttnW& w = triattn_w(weights_dir, prefix);
    triattn_fwd(as_stream(stream), w, per_column != 0, N, pair, pair_mask, drop_tbl, pair_out,
                save);
  });
}

int bc2n_triattn_fwd_noalloc(void* stream, const char* weights_dir, const char* prefix,
                             int per_column, int N, const float* pair, const float* pair_mask,
                             const float* drop_tbl, float* pair_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix, "weights_dir/prefix required");
    need(pair && pair_mask && pair_out && save, "null operand");
    need(pair_out != pair, "triattn: pair_out must not alias pair");
    const TriAttnW* w = nullptr;
    {
      // only weights already on the device: loading would allocate
      std::lock_guard<std::mutex> lk(g_mu);
      auto it = g_triattn.find(std::make_pair(std::string(weights_dir), std::string(prefix)));
      if (it != g_triattn.end()) w = &it->second;
    }
    need(w != nullptr,
         "triattn_fwd_noalloc: weights not resident; call bc2n_triattn_fwd once with this "
         "weights_dir and prefix first");
    triattn_fwd_noalloc(as_stream(stream), *w, per_column != 0, N, pair, pair_mask, drop_tbl,
                        pair_out, save);
  });
}

int bc2n_triattn_bwd(void* stream, const char* weights_dir, const char* prefix, int per_column,
                     int N, const float* pair, const float* pair_mask, const float* drop_tbl,
                     const void* save, const float* dpair_out, float* dpair_in) {
  return guarded([&] {
    need(weights_dir && prefix, "weights_dir/prefix required");
    need(pair && pair_mask && save && dpair_out && dpair_in, "null operand");
    const TriAttnW& w = triattn_w(weights_dir, prefix);
    triattn_bwd(as_stream(stream), w, per_column != 0, N, pair, pair_mask, drop_tbl, save,
                dpair_out, dpair_in);
  });
}

size_t bc2n_trimul_save_bytes(int N, int C, int I) { return trimul_save_bytes(N, C, I); }

int bc2n_trimul_fwd(void* stream, const char* weights_dir, const char* prefix, int outgoing,
                    int N, const float* pair, const float* pair_mask, const float* drop_tbl,
                    float* pair_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix, "weights_dir/prefix required");
    need(pair && pair_mask && pair_out && save, "null operand");
    need(pair_out != pair, "trimul: pair_out must not alias pair");
    const TriMulW& w = trimul_w(weights_dir, prefix);
    trimul_fwd(as_stream(stream), w, outgoing != 0, N, pair, pair_mask, drop_tbl, pair_out, save);
  });
}

int bc2n_trimul_bwd(void* stream, const char* weights_dir, const char* prefix, int outgoing,
                    int N, const float* pair, const float* pair_mask, const float* drop_tbl,
                    const void* save, const float* dpair_out, float* dpair_in) {
  return guarded([&] {
    need(weights_dir && prefix, "weights_dir/prefix required");
    need(pair && pair_mask && save && dpair_out && dpair_in, "null operand");
    const TriMulW& w = trimul_w(weights_dir, prefix);
    trimul_bwd(as_stream(stream), w, outgoing != 0, N, pair, pair_mask, drop_tbl, save, dpair_out,
               dpair_in);
  });
}

size_t bc2n_transition_save_bytes(long rows, int C, int factor) {
  return transition_save_bytes(rows, C, factor);
}

int bc2n_transition_fwd(void* stream, const char* weights_dir, const char* prefix, long rows,
                        int N, const float* act, const float* drop_tbl, float* act_out,
                        void* save) {
  return guarded([&] {
    need(weights_dir && prefix && act && act_out && save, "null operand");
    need(act_out != act, "transition: act_out must not alias act");
    need(rows > 0 && N > 0 && rows % N == 0, "transition: rows must be a multiple of N");
    const TransW& w = cached(g_trans, weights_dir, prefix, transition_weights);
    transition_fwd(as_stream(stream), w, rows, N, act, drop_tbl, act_out, save);
  });
}

int bc2n_transition_bwd(void* stream, const char* weights_dir, const char* prefix, long rows,
                        int N, const float* act, const float* drop_tbl, const void* save,
                        const float* dact_out, float* dact_in) {
  return guarded([&] {
    need(weights_dir && prefix && act && save && dact_out && dact_in, "null operand");
    const TransW& w = cached(g_trans, weights_dir, prefix, transition_weights);
    transition_bwd(as_stream(stream), w, rows, N, act, drop_tbl, save, dact_out, dact_in);
  });
}

size_t bc2n_opm_save_bytes(int S, int N, int O, int C) { return opm_save_bytes(S, N, O, C); }

int bc2n_opm_fwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                 const float* msa, const float* msa_mask, const float* pair,
                 const float* drop_tbl, float* pair_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && pair && pair_out && save, "null operand");
    need(pair_out != pair, "opm: pair_out must not alias pair");
    const OpmW& w = cached(g_opm, weights_dir, prefix, opm_weights);
    opm_fwd(as_stream(stream), w, S, N, msa, msa_mask, pair, drop_tbl, pair_out, save);
  });
}

int bc2n_opm_bwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                 const float* msa, const float* msa_mask, const float* drop_tbl, const void* save,
                 const float* dpair, const float* dmsa_out, float* dmsa_in) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && save && dpair && dmsa_out && dmsa_in,
         "null operand");
    const OpmW& w = cached(g_opm, weights_dir, prefix, opm_weights);
    opm_bwd(as_stream(stream), w, S, N, msa, msa_mask, drop_tbl, save, dpair, dmsa_out, dmsa_in);
  });
}

size_t bc2n_msarow_save_bytes(int S, int N, int Cm, int H) { return msarow_save_bytes(S, N, Cm, H); }

int bc2n_msarow_fwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                    const float* msa, const float* msa_mask, const float* pair,
                    const float* drop_tbl, float* msa_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && pair && msa_out && save, "null operand");
    need(msa_out != msa, "msarow: msa_out must not alias msa");
    const MsaRowW& w = cached(g_row, weights_dir, prefix, msarow_weights);
    msarow_fwd(as_stream(stream), w, S, N, msa, msa_mask, pair, drop_tbl, msa_out, save);
  });
}

int bc2n_msarow_bwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                    const float* msa, const float* msa_mask, const float* pair,
                    const float* drop_tbl, const void* save, const float* dmsa_out,
                    float* dmsa_in, float* dpair) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && pair && save && dmsa_out && dmsa_in && dpair,
         "null operand");
    const MsaRowW& w = cached(g_row, weights_dir, prefix, msarow_weights);
    msarow_bwd(as_stream(stream), w, S, N, msa, msa_mask, pair, drop_tbl, save, dmsa_out, dmsa_in,
               dpair);
  });
}

size_t bc2n_msacol_save_bytes(int S, int N, int Cm, int H) { return msacol_save_bytes(S, N, Cm, H); }

int bc2n_msacol_fwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                    const float* msa, const float* msa_mask, const float* drop_tbl,
                    float* msa_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && msa_out && save, "null operand");
    need(msa_out != msa, "msacol: msa_out must not alias msa");
    const MsaColW& w = cached(g_col, weights_dir, prefix, msacol_weights);
    msacol_fwd(as_stream(stream), w, S, N, msa, msa_mask, drop_tbl, msa_out, save);
  });
}

std::map<std::pair<std::string, std::string>, MsaGlobW> g_glob;

size_t bc2n_msaglobal_save_bytes(const char* weights_dir, const char* prefix, int S, int N) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir && prefix && S > 0 && N > 0, "bad arguments");
        const MsaGlobW& w = cached(g_glob, weights_dir, prefix, msaglobal_weights);
        n = msaglobal_save_bytes(w, S, N);
      }) != 0)
    return 0;
  return n;
}

int bc2n_msaglobal_fwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                       const float* msa, const float* msa_mask, const float* drop_tbl,
                       float* msa_out, void* save) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && msa_out && save, "null operand");
    need(msa_out != msa, "msaglobal: msa_out must not alias msa");
    const MsaGlobW& w = cached(g_glob, weights_dir, prefix, msaglobal_weights);
    msaglobal_fwd(as_stream(stream), w, S, N, msa, msa_mask, drop_tbl, msa_out, save);
  });
}

int bc2n_msaglobal_bwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                       const float* msa, const float* msa_mask, const float* drop_tbl,
                       const void* save, const float* dmsa_out, float* dmsa_in) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && save && dmsa_out && dmsa_in, "null operand");
    const MsaGlobW& w = cached(g_glob, weights_dir, prefix, msaglobal_weights);
    msaglobal_bwd(as_stream(stream), w, S, N, msa, msa_mask, drop_tbl, save, dmsa_out, dmsa_in);
  });
}

int bc2n_msacol_bwd(void* stream, const char* weights_dir, const char* prefix, int S, int N,
                    const float* msa, const float* msa_mask, const float* drop_tbl,
                    const void* save, const float* dmsa_out, float* dmsa_in) {
  return guarded([&] {
    need(weights_dir && prefix && msa && msa_mask && save && dmsa_out && dmsa_in, "null operand");
    const MsaColW& w = cached(g_col, weights_dir, prefix, msacol_weights);
    msacol_bwd(as_stream(stream), w, S, N, msa, msa_mask, drop_tbl, save, dmsa_out, dmsa_in);
  });
}

// ------------------------------------------------------------ the stack

size_t bc2n_evoformer_save_bytes(const char* weights_dir, int N, int S, int64_t depth,
                                 int64_t pair_only) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        const StackW& w = stack_w(weights_dir, (int)depth, evo_kind(pair_only));
        n = stack_save_bytes(w, N, S, (int)depth) + 256;
      }) != 0)
    return 0;
  return n;
}

size_t bc2n_evoformer_detached_bytes(const char* weights_dir, int N, int S, int64_t depth,
                                     int64_t pair_only) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        const StackW& w = stack_w(weights_dir, (int)depth, evo_kind(pair_only));
        n = stack_detached_bytes(w, N, S, (int)depth) + 256;
      }) != 0)
    return 0;
  return n;
}

int bc2n_set_save_policy(int policy) { return set_save_policy(policy); }

int bc2n_set_msa_overlap(int on) { return set_msa_overlap(on != 0) ? 1 : 0; }

int bc2n_evoformer_replays(const char* weights_dir, int N, int S, int64_t depth,
                           int64_t pair_only) {
  int r = -1;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        const StackW& w = stack_w(weights_dir, (int)depth, evo_kind(pair_only));
        r = stack_replays(w, N, S, (int)depth) ? 1 : 0;
      }) != 0)
    return -1;
  return r;
}

static const uint32_t* stack_key(hipStream_t st, const uint32_t* seed, int seed_len,
                                 uint32_t* scratch) {
  if (seed_len == 3) return seed;  // [k0, k1, enabled]: jax.random.key_data
  key_from_bits(st, seed, scratch);  // [bits, enabled]: PRNGKey(bits)
  return scratch;
}

int bc2n_evoformer_fwd(void* stream, const float* pair, const float* msa, const float* pair_mask,
                       const float* msa_mask, const uint32_t* seed, int seed_len, int N, int S,
                       int Cm, int64_t depth, int64_t save, int64_t pair_only, int64_t own_save,
                       int64_t opm_first, int64_t dropout, const char* weights_dir,
                       float* pair_out, float* msa_out, void* psave, void* msave) {
  (void)msave;
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && pair && pair_mask && pair_out, "null operand");
    need(opm_first == 1, "evoformer: only outer_product_mean.first=True (AF2-multimer) is built");
    need(seed_len == 2 || seed_len == 3, "evoformer: seed must be u32[2] or u32[3]");
    need(!dropout || seed, "evoformer: dropout needs the seed operand");
    need(pair_only || (msa && msa_mask && msa_out), "evoformer: msa operands required");
    need(pair_out != pair && (pair_only || msa_out != msa), "evoformer: outputs must not alias inputs");
    const StackW& w = stack_w(weights_dir, (int)depth, evo_kind(pair_only));
    if (!pair_only) need(Cm == w.blocks[0].row.a.Cin, "evoformer: msa channel width mismatch");
    // save = 0: a detached forward (no backward follows), one block's scratch
    const bool detached = (save == 0);
    const size_t bytes = (detached ? stack_detached_bytes(w, N, S, (int)depth)
                                   : stack_save_bytes(w, N, S, (int)depth)) + 256;
    void* sv = detached ? g_det.get(st, bytes)
               : (own_save != 0 || psave == nullptr) ? g_own.get(st, bytes) : psave;
    uint32_t* keyslot = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(sv) + bytes - 256);
    const uint32_t* key = dropout ? stack_key(st, seed, seed_len, keyslot) : nullptr;
    const uint32_t* enabled = dropout ? seed + (seed_len - 1) : nullptr;
    stack_fwd(st, w, N, S, (int)depth, pair, msa, pair_mask, msa_mask, key, enabled, dropout != 0,
              pair_out, msa_out, sv, detached);
    if (pair_only && msa && msa_out && msa_out != msa && Cm > 0)
      BC2N_HIP(hipMemcpyAsync(msa_out, msa, (size_t)S * N * Cm * 4, hipMemcpyDeviceToDevice, st));
  });
}

int bc2n_evoformer_bwd(void* stream, const float* ct_pair, const float* ct_msa,
                       const float* pair_mask, const float* msa_mask, const void* psave,
                       const void* msave, const uint32_t* seed, int seed_len, int N, int S,
                       int Cm, int64_t depth, int64_t pair_only, int64_t own_save,
                       int64_t opm_first, int64_t dropout, const char* weights_dir,
                       float* dpair, float* dmsa) {
  (void)msave;
  (void)seed;
  (void)seed_len;
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && ct_pair && pair_mask && dpair, "null operand");
    need(opm_first == 1, "evoformer: only outer_product_mean.first=True (AF2-multimer) is built");
    need(pair_only || (ct_msa && msa_mask && dmsa), "evoformer: msa operands required");
    const StackW& w = stack_w(weights_dir, (int)depth, evo_kind(pair_only));
    const size_t bytes = stack_save_bytes(w, N, S, (int)depth) + 256;
    const void* sv = (own_save != 0 || psave == nullptr) ? g_own.get(st, bytes) : psave;
    stack_bwd(st, w, N, S, (int)depth, pair_mask, msa_mask, dropout != 0, sv, ct_pair, ct_msa,
              dpair, dmsa);
    if (pair_only && dmsa && ct_msa && dmsa != ct_msa && Cm > 0)
      BC2N_HIP(hipMemcpyAsync(dmsa, ct_msa, (size_t)S * N * Cm * 4, hipMemcpyDeviceToDevice, st));
  });
}

// ------------------------------------------------------------ preallocation
// Called before the first real call (the reference calls its counterparts at
// trace time, before XLA has allocated): upload the component's weights and
// grow every scratch arena to what its calls at these shapes need, so that
// no call allocates afterwards.  The arenas' needs depend on the shapes, not
// on the depth, so one forward and backward of the first block on zero
// inputs (on the null stream, synchronised) grows them exactly; detached
// forwards' scratch is grown to its size as well.  Prints what it took.

namespace {

struct DevBuf {
  void* p = nullptr;
  explicit DevBuf(size_t n) {
    BC2N_HIP(hipMalloc(&p, n < 256 ? 256 : n));
    BC2N_HIP(hipMemset(p, 0, n < 256 ? 256 : n));
  }
  ~DevBuf() { if (p) (void)hipFree(p); }
  float* f() const { return static_cast<float*>(p); }
};

size_t free_bytes(size_t* total = nullptr) {
  size_t f = 0, t = 0;
  BC2N_HIP(hipMemGetInfo(&f, &t));
  if (total) *total = t;
  return f;
}

void report(const char* what, const std::string& shape, size_t f0) {
  size_t t = 0;
  const size_t f1 = free_bytes(&t);
  fprintf(stderr, "bc2n: prealloc %s %s took %.2f GB (%.2f of %.2f GB free after)\n", what,
          shape.c_str(), (double)((f0 > f1) ? f0 - f1 : 0) / 1e9, (double)f1 / 1e9,
          (double)t / 1e9);
}

void stack_dry_run(const StackW& w, int N, int S) {
  const long M = (long)N * N;
  const int Cz = w.blocks[0].tmo.C, Cm = w.pair_only ? 64 : w.blocks[0].row.a.Cin;
  const size_t sb = stack_save_bytes(w, N, S, 1);
  DevBuf pair(M * Cz * 4), pair_out(M * Cz * 4), dpair(M * Cz * 4), pmask(M * 4);
  DevBuf msa((size_t)S * N * Cm * 4), msa_out((size_t)S * N * Cm * 4),
      dmsa((size_t)S * N * Cm * 4), mmask((size_t)S * N * 4), save(sb);
  hipStream_t st = nullptr;
  stack_fwd(st, w, N, S, 1, pair.f(), w.pair_only ? nullptr : msa.f(),
            pmask.f(), mmask.f(), nullptr, nullptr, false, pair_out.f(),
            w.pair_only ? nullptr : msa_out.f(), save.p);
  stack_bwd(st, w, N, S, 1, pmask.f(), mmask.f(), false, save.p,
            pair_out.f(), w.pair_only ? nullptr : msa_out.f(), dpair.f(),
            w.pair_only ? nullptr : dmsa.f());
  BC2N_HIP(hipDeviceSynchronize());
}

}  // namespace

int bc2n_stack_prealloc(int N, int S, int depth, const char* weights_dir, int pair_only,
                        int opm_first, int dropout) {
  (void)dropout;
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    need(opm_first == 1, "evoformer: only outer_product_mean.first=True (AF2-multimer) is built");
    const size_t f0 = free_bytes();
    const StackW& w = stack_w(weights_dir, depth, evo_kind(pair_only));
    stack_dry_run(w, N, S);
    (void)g_det.get(nullptr, stack_detached_bytes(w, N, S, depth) + 256);
    BC2N_HIP(hipDeviceSynchronize());
    report("stack", "N=" + std::to_string(N) + " S=" + std::to_string(S) + " depth=" +
           std::to_string(depth) + " pair_only=" + std::to_string(pair_only), f0);
  });
}

int bc2n_tplstack_prealloc(int N, int depth, const char* weights_dir) {
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    const size_t f0 = free_bytes();
    stack_dry_run(stack_w(weights_dir, depth, StackKind::TEMPLATE), N, 1);
    report("tplstack", "N=" + std::to_string(N) + " depth=" + std::to_string(depth), f0);
  });
}

// (the structure-module and template-embedding counterparts follow their
// weight caches below)

int bc2n_save_slots_probe(const char* weights_dir, int depth, int N, int S, int pair_only) {
  int slots = -1;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        const StackW& w = stack_w(weights_dir, depth, evo_kind(pair_only));
        const size_t bytes = stack_save_bytes(w, N, S, depth) + 256;
        const size_t slot = (size_t)N * N * 128 * 2;  // one bf16 [N,N,128] slot
        slots = (int)((bytes + slot - 1) / slot);
      }) != 0)
    return -1;
  return slots;
}

// ------------------------------------------------------ template pair stack

size_t bc2n_tplstack_save_bytes(const char* weights_dir, int N, int64_t depth) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        const StackW& w = stack_w(weights_dir, (int)depth, StackKind::TEMPLATE);
        n = stack_save_bytes(w, N, 1, (int)depth) + 256;
      }) != 0)
    return 0;
  return n;
}

int bc2n_tplstack_fwd(void* stream, const float* pair, const float* pair_mask,
                      const uint32_t* seed, int seed_len, int N, int64_t depth, int64_t dropout,
                      const char* weights_dir, float* out, void* save) {
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && pair && pair_mask && out && save, "null operand");
    need(out != pair, "tplstack: out must not alias pair");
    need(seed_len == 2 || seed_len == 3, "tplstack: seed must be u32[2] or u32[3]");
    need(!dropout || seed, "tplstack: dropout needs the seed operand");
    const StackW& w = stack_w(weights_dir, (int)depth, StackKind::TEMPLATE);
    const size_t bytes = stack_save_bytes(w, N, 1, (int)depth) + 256;
    uint32_t* keyslot = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(save) + bytes - 256);
    const uint32_t* key = dropout ? stack_key(st, seed, seed_len, keyslot) : nullptr;
    const uint32_t* enabled = dropout ? seed + (seed_len - 1) : nullptr;
    stack_fwd(st, w, N, 1, (int)depth, pair, nullptr, pair_mask, nullptr, key, enabled,
              dropout != 0, out, nullptr, save);
  });
}

int bc2n_tplstack_bwd(void* stream, const float* ct, const float* pair_mask, const void* save,
                      const uint32_t* seed, int seed_len, int N, int64_t depth, int64_t dropout,
                      const char* weights_dir, float* dpair) {
  (void)seed;
  (void)seed_len;
  return guarded([&] {
    need(weights_dir && ct && pair_mask && save && dpair, "null operand");
    const StackW& w = stack_w(weights_dir, (int)depth, StackKind::TEMPLATE);
    stack_bwd(as_stream(stream), w, N, 1, (int)depth, pair_mask, nullptr, dropout != 0, save, ct,
              nullptr, dpair, nullptr);
  });
}

// --------------------------------------------------------- template embedding

namespace {
std::map<std::pair<std::string, std::string>, TplEmbedW> g_te;
const TplEmbedW& te_w(const char* dir, int depth) {
  return cached(g_te, dir, std::to_string(depth).c_str(), [&](WeightStore& ws, const std::string&) {
    return tplembed_weights(ws, depth);
  });
}
}  // namespace

int bc2n_tplembed_prealloc(int N, int depth, const char* weights_dir) {
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    const size_t f0 = free_bytes();
    const TplEmbedW& w = te_w(weights_dir, depth);
    const long M = (long)N * N;
    DevBuf query(M * 128 * 4), act_const(M * 64 * 4), pmask(M * 4), out(M * 128 * 4),
        dq(M * 128 * 4), save(tplembed_save_bytes(w, N) + 256);
    tplembed_fwd(nullptr, w, N, query.f(), act_const.f(), pmask.f(),
                 nullptr, nullptr, false, out.f(), save.p);
    tplembed_bwd(nullptr, w, N, query.f(), pmask.f(), false, save.p,
                 out.f(), dq.f());
    BC2N_HIP(hipDeviceSynchronize());
    report("tplembed", "N=" + std::to_string(N) + " depth=" + std::to_string(depth), f0);
  });
}

size_t bc2n_tplembed_save_bytes(const char* weights_dir, int N, int64_t depth) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        n = tplembed_save_bytes(te_w(weights_dir, (int)depth), N) + 256;
      }) != 0)
    return 0;
  return n;
}

int bc2n_tplembed_fwd(void* stream, const float* query, const float* act_const,
                      const float* pair_mask, const uint32_t* seed, int seed_len, int N,
                      int64_t depth, int64_t dropout, const char* weights_dir, float* out,
                      void* save) {
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && query && act_const && pair_mask && out && save, "null operand");
    need(seed_len == 2 || seed_len == 3, "tplembed: seed must be u32[2] or u32[3]");
    need(!dropout || seed, "tplembed: dropout needs the seed operand");
    const TplEmbedW& w = te_w(weights_dir, (int)depth);
    const size_t bytes = tplembed_save_bytes(w, N) + 256;
    uint32_t* keyslot = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(save) + bytes - 256);
    const uint32_t* key = dropout ? stack_key(st, seed, seed_len, keyslot) : nullptr;
    const uint32_t* enabled = dropout ? seed + (seed_len - 1) : nullptr;
    tplembed_fwd(st, w, N, query, act_const, pair_mask, key, enabled, dropout != 0, out, save);
  });
}

int bc2n_tplembed_bwd(void* stream, const float* ct, const float* query, const float* act_const,
                      const float* pair_mask, const void* save, const uint32_t* seed, int seed_len,
                      int N, int64_t depth, int64_t dropout, const char* weights_dir,
                      float* dquery) {
  (void)act_const;
  (void)seed;
  (void)seed_len;
  return guarded([&] {
    need(weights_dir && ct && query && pair_mask && save && dquery, "null operand");
    const TplEmbedW& w = te_w(weights_dir, (int)depth);
    tplembed_bwd(as_stream(stream), w, N, query, pair_mask, dropout != 0, save, ct, dquery);
  });
}

// ------------------------------------------------------------------ embedder

namespace {
std::map<std::pair<std::string, std::string>, EmbedW> g_emb;
const EmbedW& emb_w(const char* dir) {
  return cached(g_emb, dir, "", [&](WeightStore& ws, const std::string&) { return embed_weights(ws); });
}
}  // namespace

int bc2n_embedder_fwd(void* stream, const float* target_feat, const float* msa_feat,
                      const float* residue_index, const float* asym_id, const float* entity_id,
                      const float* sym_id, const int32_t* offset, int N, int S,
                      const char* weights_dir, float* msa, float* pair) {
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    embed_fwd(as_stream(stream), emb_w(weights_dir), N, S, target_feat, msa_feat, residue_index,
              asym_id, entity_id, sym_id, offset, msa, pair);
  });
}

int bc2n_embedder_bwd(void* stream, const float* dmsa, const float* dpair, const float* target_feat,
                      int N, int S, const char* weights_dir, float* dtarget_feat, float* dmsa_feat) {
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    embed_bwd(as_stream(stream), emb_w(weights_dir), N, S, dmsa, dpair, target_feat, dtarget_feat,
              dmsa_feat);
  });
}

// ------------------------------------------------ structure module folding

namespace {
std::map<std::string, FoldW> g_fold;
const FoldW& fold_w(const char* dir) {
  std::lock_guard<std::mutex> lk(g_mu);
  auto it = g_fold.find(dir);
  if (it != g_fold.end()) return it->second;
  FoldW w = fold_weights(weights(dir));
  return g_fold.emplace(dir, w).first->second;
}
}  // namespace

size_t bc2n_fold_save_bytes(const char* weights_dir, int N, int64_t depth) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        need(N > 0 && N <= 1024 && depth > 0, "fold: bad shape");
        (void)fold_w(weights_dir);
        n = fold_save_bytes(N, (int)depth) + 256;
      }) != 0)
    return 0;
  return n;
}

int bc2n_fold_fwd(void* stream, const float* single, const float* pair, const float* seq_mask,
                  const uint32_t* seed, int seed_len, int N, int64_t depth, int64_t dropout,
                  const char* weights_dir, float* act, float* traj, void* save) {
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && single && pair && seq_mask && act && traj && save, "null operand");
    need(N > 0 && N <= 1024 && depth > 0, "fold: bad shape");
    need(seed_len == 2 || seed_len == 3, "fold: seed must be u32[2] or u32[3]");
    need(!dropout || seed, "fold: dropout needs the seed operand");
    const FoldW& w = fold_w(weights_dir);
    const size_t bytes = fold_save_bytes(N, (int)depth) + 256;
    uint32_t* keyslot = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(save) + bytes - 256);
    const uint32_t* key = dropout ? stack_key(st, seed, seed_len, keyslot) : nullptr;
    const uint32_t* enabled = dropout ? seed + (seed_len - 1) : nullptr;
    fold_fwd(st, w, N, (int)depth, single, pair, seq_mask, key, enabled, dropout != 0, act, traj,
             save);
  });
}

int bc2n_fold_bwd(void* stream, const float* d_act, const float* d_traj, const float* single,
                  const float* pair, const float* seq_mask, const void* save, int N,
                  int64_t depth, int64_t dropout, const char* weights_dir, float* dsingle,
                  float* dpair) {
  return guarded([&] {
    need(weights_dir && single && pair && seq_mask && save && dsingle && dpair, "null operand");
    need(N > 0 && N <= 1024 && depth > 0, "fold: bad shape");
    const FoldW& w = fold_w(weights_dir);
    fold_bwd(as_stream(stream), w, N, (int)depth, single, pair, seq_mask, dropout != 0, save,
             d_act, d_traj, dsingle, dpair);
  });
}

// ------------------------------------------------ structure module + heads

namespace {
std::map<std::pair<std::string, std::string>, StructHeadsW> g_sh;
const StructHeadsW& sh_w(const char* dir) {
  return cached(g_sh, dir, "", [&](WeightStore& ws, const std::string&) { return structheads_weights(ws); });
}
}  // namespace

int bc2n_sm_prealloc(int N, int depth, const char* weights_dir) {
  return guarded([&] {
    need(weights_dir != nullptr, "weights_dir required");
    need(N > 0 && N <= 1024 && depth > 0, "structure heads: bad shape");
    const size_t f0 = free_bytes();
    const StructHeadsW& w = sh_w(weights_dir);
    const long M = (long)N * N;
    DevBuf single((size_t)N * 384 * 4), pair(M * 128 * 4), seq_mask((size_t)N * 4),
        aatype((size_t)N * 4), atom14((size_t)N * 14 * 3 * 4), dgram(M * 64 * 4),
        pae(M * 64 * 4), plddt((size_t)N * 50 * 4), expres((size_t)N * 37 * 4),
        dsingle((size_t)N * 384 * 4), dpair(M * 128 * 4),
        save(structheads_save_bytes(N, 1) + 256);
    structheads_fwd(nullptr, w, N, 1, single.f(), pair.f(), seq_mask.f(),
                    aatype.f(), nullptr, nullptr, false, atom14.f(),
                    dgram.f(), pae.f(), plddt.f(), expres.f(),
                    save.p);
    structheads_bwd(nullptr, w, N, 1, single.f(), pair.f(), seq_mask.f(),
                    aatype.f(), false, save.p, atom14.f(), dgram.f(),
                    pae.f(), plddt.f(), expres.f(), dsingle.f(),
                    dpair.f());
    BC2N_HIP(hipDeviceSynchronize());
    report("structure module", "N=" + std::to_string(N) + " depth=" + std::to_string(depth), f0);
  });
}

size_t bc2n_structure_heads_save_bytes(const char* weights_dir, int N, int64_t depth) {
  size_t n = 0;
  if (guarded([&] {
        need(weights_dir != nullptr, "weights_dir required");
        need(N > 0 && N <= 1024 && depth > 0, "structure heads: bad shape");
        (void)sh_w(weights_dir);
        n = structheads_save_bytes(N, (int)depth) + 256;
      }) != 0)
    return 0;
  return n;
}

int bc2n_structure_heads_fwd(void* stream, const float* single, const float* pair,
                             const float* seq_mask, const float* aatype, const uint32_t* seed,
                             int seed_len, int N, int64_t depth, int64_t dropout,
                             const char* weights_dir, float* atom14, float* distogram, float* pae,
                             float* plddt, float* expres, void* save) {
  return guarded([&] {
    hipStream_t st = as_stream(stream);
    need(weights_dir && single && pair && seq_mask && aatype && save, "null operand");
    need(atom14 && distogram && pae && plddt && expres, "null output");
    need(N > 0 && N <= 1024 && depth > 0, "structure heads: bad shape");
    need(seed_len == 2 || seed_len == 3, "structure heads: seed must be u32[2] or u32[3]");
    need(!dropout || seed, "structure heads: dropout needs the seed operand");
    const StructHeadsW& w = sh_w(weights_dir);
    const size_t bytes = structheads_save_bytes(N, (int)depth) + 256;
    uint32_t* keyslot = reinterpret_cast<uint32_t*>(reinterpret_cast<char*>(save) + bytes - 256);
    const uint32_t* key = dropout ? stack_key(st, seed, seed_len, keyslot) : nullptr;
    const uint32_t* enabled = dropout ? seed + (seed_len - 1) : nullptr;
    structheads_fwd(st, w, N, (int)depth, single, pair, seq_mask, aatype, key, enabled,
                    dropout != 0, atom14, distogram, pae, plddt, expres, save);
  });
}

int bc2n_structure_heads_bwd(void* stream, const float* single, const float* pair,
                             const float* seq_mask, const float* aatype, const float* d_atom14,
                             const float* d_distogram, const float* d_pae, const float* d_plddt,
                             const float* d_expres, void* save, int N, int64_t depth,
                             int64_t dropout, const char* weights_dir, float* dsingle,
                             float* dpair) {
  return guarded([&] {
    need(weights_dir && single && pair && seq_mask && aatype && save && dsingle && dpair,
         "null operand");
    need(N > 0 && N <= 1024 && depth > 0, "structure heads: bad shape");
    const StructHeadsW& w = sh_w(weights_dir);
    structheads_bwd(as_stream(stream), w, N, (int)depth, single, pair, seq_mask, aatype,
                    dropout != 0, save, d_atom14, d_distogram, d_pae, d_plddt, d_expres, dsingle,
                    dpair);
  });
}

// ------------------------------------------------------- one-call design step

namespace {
std::map<std::string, DesignStepW> g_ds;
// The recycle terms' weights live in the embedder's directory
// (native/design_step.cuh:884, bindcraft/af/native.py:515-527).
RecycleW recycle_w(WeightStore& ews) {
  auto rec = [&](const char* name, size_t n) {
    const std::string k = std::string("param/") + name;
    if (ews.host(k).data.size() != n)
      throw std::runtime_error(std::string("recycle terms: ") + k + " has the wrong size");
    return ews.f32(k);
  };
  RecycleW r;
  r.wpp = rec("prev_pos_linear/weights", 15 * 128);
  r.bpp = rec("prev_pos_linear/bias", 128);
  r.s_msa = rec("prev_msa_first_row_norm/scale", 256);
  r.o_msa = rec("prev_msa_first_row_norm/offset", 256);
  r.s_pair = rec("prev_pair_norm/scale", 128);
  r.o_pair = rec("prev_pair_norm/offset", 128);
  return r;
}

const DesignStepW& ds_w(const char* emb, const char* tpl, const char* extra, const char* main,
                        const char* post, int64_t dt, int64_t de, int64_t dm, int64_t df) {
  need(emb && tpl && extra && main && post, "design step: five weights directories required");
  const std::string key = std::string(emb) + "|" + tpl + "|" + extra + "|" + main + "|" + post +
                          "|" + std::to_string(dt) + "," + std::to_string(de) + "," +
                          std::to_string(dm) + "," + std::to_string(df);
  {
    std::lock_guard<std::mutex> lk(g_mu);
    auto it = g_ds.find(key);
    if (it != g_ds.end()) return it->second;
  }
  DesignStepW w;
  w.d_tpl = (int)dt; w.d_extra = (int)de; w.d_main = (int)dm; w.d_fold = (int)df;
  w.emb = emb_w(emb);
  WeightStore& ews = weights(emb);
  w.wsa = ews.f32("param/single_activations/weights");
  w.bsa = ews.f32("param/single_activations/bias");
  if (ews.host("param/single_activations/weights").data.size() != 256u * 384u)
    throw std::runtime_error("design step: single_activations must be [256,384]");
  w.rec = recycle_w(ews);
  w.tpl = te_w(tpl, (int)dt);
  w.extra = stack_w(extra, (int)de, StackKind::PAIR_ONLY);
  w.main = stack_w(main, (int)dm, StackKind::EVO);
  w.sh = sh_w(post);
  WeightStore& pws = weights(post);
  // the template's MSA row: Linears in the embedder's directory, chi tables
  // in the structure module's (both optional; the row needs all six)
  auto opt = [](WeightStore& ws, const char* name, size_t n) -> const float* {
    if (!ws.has(name)) return nullptr;
    if (ws.host(name).data.size() != n)
      throw std::runtime_error(std::string("design step: ") + name + " has the wrong size");
    return ws.f32(name);
  };
  w.trow.w1 = opt(ews, "param/template_single_embedding/weights", 34 * 256);
  w.trow.b1 = opt(ews, "param/template_single_embedding/bias", 256);
  w.trow.w2 = opt(ews, "param/template_projection/weights", 256 * 256);
  w.trow.b2 = opt(ews, "param/template_projection/bias", 256);
  w.trow.chi_idx = opt(pws, "const/chi_atom_indices", 21 * 16);
  w.trow.chi_mask = opt(pws, "const/chi_angles_mask", 21 * 4);
  if (pws.has("const/atom37_to_atom14") && pws.has("const/atom37_mask")) {
    if (pws.host("const/atom37_to_atom14").data.size() != 21u * 37u ||
        pws.host("const/atom37_mask").data.size() != 21u * 37u)
      throw std::runtime_error("design step: the atom37 tables must be [21,37]");
    w.a37_14 = pws.f32("const/atom37_to_atom14");
    w.a37_mask = pws.f32("const/atom37_mask");
  }
  std::lock_guard<std::mutex> lk(g_mu);
  return g_ds.emplace(key, w).first->second;
}
}  // namespace

size_t bc2n_design_step_save_bytes(const char* emb_dir, const char* tpl_dir,
                                   const char* extra_dir, const char* main_dir,
                                   const char* post_dir, int N, int S, int64_t d_tpl,
                                   int64_t d_extra, int64_t d_main, int64_t d_fold) {
  size_t n = 0;
  if (guarded([&] {
        const DesignStepW& w =
            ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
        need(N > 0 && S > 0, "design step: bad shape");
        n = design_step_save_bytes(w, N, S);
      }) != 0)
    return 0;
  return n;
}

int bc2n_design_step_fwd(void* stream, const float* target_feat, const float* msa_feat,
                         const float* residue_index, const float* asym_id,
                         const float* entity_id, const float* sym_id, const int32_t* offset,
                         const float* seq_mask, const float* act_const, const float* aatype,
                         const uint32_t* seeds, int N, int S, int64_t d_tpl, int64_t d_extra,
                         int64_t d_main, int64_t d_fold, int64_t dropout, int64_t recycles,
                         const char* emb_dir, const char* tpl_dir, const char* extra_dir,
                         const char* main_dir, const char* post_dir, float* atom14,
                         float* distogram, float* pae, float* plddt, float* expres, void* save) {
  return guarded([&] {
    need(target_feat && msa_feat && residue_index && asym_id && entity_id && sym_id && seq_mask &&
             aatype && save, "null operand");
    need(atom14 && distogram && pae && plddt && expres, "null output");
    need(!dropout || seeds, "design step: dropout needs the seeds operand");
    const DesignStepW& w =
        ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
    design_step_fwd(as_stream(stream), w, N, S, target_feat, msa_feat, residue_index, asym_id,
                    entity_id, sym_id, offset, seq_mask, act_const, aatype, seeds, dropout != 0,
                    (int)recycles, atom14, distogram, pae, plddt, expres, save);
  });
}

int bc2n_design_step_bwd(void* stream, const float* target_feat, const float* seq_mask,
                         const float* aatype, int64_t with_template, const float* d_atom14,
                         const float* d_distogram, const float* d_pae, const float* d_plddt,
                         const float* d_expres, void* save, int N, int S, int64_t d_tpl,
                         int64_t d_extra, int64_t d_main, int64_t d_fold, int64_t dropout,
                         const char* emb_dir, const char* tpl_dir, const char* extra_dir,
                         const char* main_dir, const char* post_dir, float* d_target_feat,
                         float* d_msa_feat) {
  return guarded([&] {
    need(target_feat && seq_mask && aatype && save && d_target_feat && d_msa_feat, "null operand");
    const DesignStepW& w =
        ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
    design_step_bwd(as_stream(stream), w, N, S, target_feat, seq_mask, with_template != 0, aatype,
                    dropout != 0, save, d_atom14, d_distogram, d_pae, d_plddt, d_expres,
                    d_target_feat, d_msa_feat);
  });
}

int bc2n_seqfeat_fwd(void* stream, const float* logits, const uint8_t* flags, const float* aa_bias,
                     float softmax_weight, float one_hot_weight, float temperature,
                     float logit_scale, float omitted_half, const float* scalars, int N,
                     float* feat, float* prof) {
  return guarded([&] {
    need(logits && flags && feat && prof, "null operand");
    need(N > 0, "seqfeat: N must be positive");
    need(scalars || temperature != 0.f, "seqfeat: temperature must be non-zero");
    seqfeat_fwd(as_stream(stream), logits, flags, aa_bias,
                SeqScalars{softmax_weight, one_hot_weight, temperature, logit_scale}, scalars,
                omitted_half, N, feat, prof);
  });
}

int bc2n_seqfeat_bwd(void* stream, const float* logits, const uint8_t* flags, const float* aa_bias,
                     const float* d_feat, const float* d_prof, float softmax_weight,
                     float one_hot_weight, float temperature, float logit_scale,
                     float omitted_half, const float* scalars, int N, float* d_logits) {
  return guarded([&] {
    need(logits && flags && d_feat && d_prof && d_logits, "null operand");
    need(N > 0, "seqfeat: N must be positive");
    need(scalars || temperature != 0.f, "seqfeat: temperature must be non-zero");
    seqfeat_bwd(as_stream(stream), logits, flags, aa_bias,
                SeqScalars{softmax_weight, one_hot_weight, temperature, logit_scale}, scalars,
                omitted_half, N, d_feat, d_prof, d_logits);
  });
}

int bc2n_design_inputs_fwd(void* stream, const float* feat, const float* prof, int N,
                           float* target_feat, float* msa_feat, float* aatype) {
  return guarded([&] {
    need(feat && prof && target_feat && msa_feat && aatype, "null operand");
    need(N > 0, "design inputs: N must be positive");
    design_inputs_fwd(as_stream(stream), feat, prof, N, target_feat, msa_feat, aatype);
  });
}

int bc2n_design_inputs_bwd(void* stream, const float* d_target_feat, const float* d_msa_feat,
                           int N, float* d_feat, float* d_prof) {
  return guarded([&] {
    need(d_target_feat && d_msa_feat && d_feat && d_prof, "null operand");
    need(N > 0, "design inputs: N must be positive");
    design_inputs_bwd(as_stream(stream), d_target_feat, d_msa_feat, N, d_feat, d_prof);
  });
}

size_t bc2n_design_step_seq_save_bytes(const char* emb_dir, const char* tpl_dir,
                                       const char* extra_dir, const char* main_dir,
                                       const char* post_dir, int N, int64_t d_tpl,
                                       int64_t d_extra, int64_t d_main, int64_t d_fold) {
  size_t n = 0;
  if (guarded([&] {
        const DesignStepW& w =
            ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
        need(N > 0, "design step: bad shape");
        n = design_step_seq_save_bytes(w, N);
      }) != 0)
    return 0;
  return n;
}

int bc2n_design_step_seq_fwd(void* stream, const float* logits, const uint8_t* flags,
                             const float* aa_bias, const float* scalars, float omitted_half,
                             const float* residue_index, const float* asym_id,
                             const float* entity_id, const float* sym_id, const int32_t* offset,
                             const float* seq_mask, const float* act_const,
                             const uint32_t* seeds, int N, const int32_t* n, int64_t d_tpl,
                             int64_t d_extra, int64_t d_main, int64_t d_fold, int64_t dropout,
                             int64_t recycles, int64_t cyclic_mode, float flexibility,
                             const char* emb_dir, const char* tpl_dir,
                             const char* extra_dir, const char* main_dir, const char* post_dir,
                             float* atom14, float* distogram, float* pae, float* plddt,
                             float* expres, const float* tpl_atoms37, const float* tpl_mask37,
                             float* atom37,
                             float* atom37_mask, const int32_t* interface_asym,
                             float* conf_plddt, float* conf_pae, float* ptm, float* iptm,
                             float* iptm_per_residue, float* expres_ca, void* save) {
  return guarded([&] {
    need(logits && flags && scalars && residue_index && asym_id && entity_id && sym_id &&
             seq_mask && save, "null operand");
    need(atom14 && distogram && pae && plddt && expres, "null output");
    need(!dropout || seeds, "design step: dropout needs the seeds operand");
    need(!conf_plddt || (interface_asym && conf_pae && ptm && iptm && iptm_per_residue && expres_ca),
         "design step: the confidence outputs come together, with interface_asym");
    const DesignStepW& w =
        ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
    design_step_seq_fwd(as_stream(stream), w, N, n, logits, flags, aa_bias, scalars, omitted_half,
                        residue_index, asym_id, entity_id, sym_id, offset, seq_mask, act_const,
                        seeds, dropout != 0, (int)recycles, (int)cyclic_mode, flexibility,
                        atom14, distogram, pae, plddt, expres,
                        AtomsOut{tpl_atoms37, tpl_mask37, atom37, atom37_mask},
                        ConfOut{interface_asym, conf_plddt, conf_pae, ptm, iptm, iptm_per_residue,
                                expres_ca},
                        save);
  });
}

int bc2n_design_step_seq_bwd(void* stream, const float* logits, const uint8_t* flags,
                             const float* aa_bias, const float* scalars, float omitted_half,
                             const float* seq_mask, int64_t with_template,
                             const float* d_atom14, const float* d_distogram, const float* d_pae,
                             const float* d_plddt, const float* d_expres, const float* d_atom37,
                             const int32_t* interface_asym, const float* d_conf_plddt,
                             const float* d_conf_pae, const float* d_ptm, const float* d_iptm,
                             const float* d_iptm_per_residue, const float* d_expres_ca, void* save,
                             int N, const int32_t* n, int64_t d_tpl, int64_t d_extra, int64_t d_main, int64_t d_fold,
                             int64_t dropout, const char* emb_dir, const char* tpl_dir,
                             const char* extra_dir, const char* main_dir, const char* post_dir,
                             float* d_logits) {
  return guarded([&] {
    need(logits && flags && scalars && seq_mask && save && d_logits, "null operand");
    const DesignStepW& w =
        ds_w(emb_dir, tpl_dir, extra_dir, main_dir, post_dir, d_tpl, d_extra, d_main, d_fold);
    design_step_seq_bwd(as_stream(stream), w, N, n, logits, flags, aa_bias, scalars, omitted_half,
                        seq_mask, with_template != 0, dropout != 0, save, d_atom14, d_distogram,
                        d_pae, d_plddt, d_expres, d_atom37,
                        ConfCt{interface_asym, d_conf_plddt, d_conf_pae, d_ptm, d_iptm,
                               d_iptm_per_residue, d_expres_ca},
                        d_logits);
  });
}

size_t bc2n_confidence_save_bytes(int N) { return N > 0 ? confidence_save_bytes(N) : 0; }

int bc2n_confidence_fwd(void* stream, const float* plddt_logits, const float* pae_logits,
                        const float* expres_logits, const float* seq_mask,
                        const int32_t* interface_asym, int N, float* plddt, float* pae,
                        float* ptm, float* iptm, float* iptm_per_residue, float* expres_ca,
                        void* save) {
  return guarded([&] {
    need(plddt_logits && pae_logits && expres_logits && seq_mask && interface_asym && save,
         "null operand");
    need(plddt && pae && ptm && iptm && iptm_per_residue && expres_ca, "null output");
    confidence_fwd(as_stream(stream), plddt_logits, pae_logits, expres_logits, seq_mask,
                   interface_asym, N, plddt, pae, ptm, iptm, iptm_per_residue, expres_ca, save);
  });
}

int bc2n_confidence_bwd(void* stream, const float* plddt_logits, const float* pae_logits,
                        const float* expres_logits, const float* seq_mask,
                        const int32_t* interface_asym, const void* save, const float* d_plddt,
                        const float* d_pae, const float* d_ptm, const float* d_iptm,
                        const float* d_iptm_per_residue, const float* d_expres_ca, int N,
                        float* d_plddt_logits, float* d_pae_logits, float* d_expres_logits) {
  return guarded([&] {
    need(plddt_logits && pae_logits && expres_logits && seq_mask && interface_asym && save,
         "null operand");
    need(d_plddt_logits && d_pae_logits && d_expres_logits, "null output");
    confidence_bwd(as_stream(stream), plddt_logits, pae_logits, expres_logits, seq_mask,
                   interface_asym, N, save, d_plddt, d_pae, d_ptm, d_iptm, d_iptm_per_residue,
                   d_expres_ca, d_plddt_logits, d_pae_logits, d_expres_logits);
  });
}

namespace {
void aligned(const void* p, int to, const char* what) {
  if (p && reinterpret_cast<uintptr_t>(p) % (uintptr_t)to)
    throw std::invalid_argument(std::string("unaligned ") + what);
}
LogProbs lp_operands(int dtype, const void* logits, int64_t ld, int64_t rows, int classes,
                     const void* targets, int target_bits) {
  need(dtype == BC2N_F32 || dtype == BC2N_F16 || dtype == BC2N_BF16, "logprobs: bad dtype");
  need(rows >= 0 && rows < (int64_t(1) << 31), "logprobs: bad number of rows");
  need(classes > 0 && classes <= (1 << 28), "logprobs: bad number of classes");
  need(ld >= classes, "logprobs: the row stride is below the number of classes");
  need(!targets || target_bits == 32 || target_bits == 64, "logprobs: targets are i32 or i64");
  need(rows == 0 || logits, "null operand");
  aligned(logits, dtype == BC2N_F32 ? 4 : 2, "logits");
  if (targets) aligned(targets, target_bits / 8, "targets");
  LogProbs a;
  a.dtype = dtype;
  a.x = logits;
  a.ld = ld;
  a.rows = a.total = rows;
  a.V = classes;
  a.target = targets;
  a.target64 = target_bits == 64;
  return a;
}
void lp_top(LogProbs& a, int top) {
  need(top >= 0 && top <= LP_MAX_TOP && top <= a.V,
       "logprobs: top must be 0..32 and at most the number of classes");
  a.K = top;
}
void lp_gradient(LogProbs& a, void* d_logits, int64_t d_ld) {
  need(a.rows == 0 || d_logits, "null output");
  need(d_ld >= a.V, "logprobs: the gradient's row stride is below the number of classes");
  need(d_logits != a.x || d_ld == a.ld, "logprobs: a gradient in place has the logits' row stride");
  const int64_t w = a.dtype == BC2N_F32 ? 4 : 2;
  aligned(d_logits, (int)w, "d_logits");
  if (d_logits != a.x && a.rows > 0) {
    // apart, or columns of one buffer that no class shares
    const intptr_t x = reinterpret_cast<intptr_t>(a.x), d = reinterpret_cast<intptr_t>(d_logits);
    const bool apart = d >= x + ((a.rows - 1) * a.ld + a.V) * w ||
                       x >= d + ((a.rows - 1) * d_ld + a.V) * w;
    const int64_t column = (((d - x) / w) % a.ld + a.ld) % a.ld;
    need(apart || (d_ld == a.ld && column >= a.V && column + a.V <= a.ld),
         "logprobs: the gradient overlaps the logits");
  }
  a.d = d_logits;
  a.d_ld = d_ld;
}
TensorList& list_of(void* list) {
  TensorList* l = reinterpret_cast<TensorList*>(list);
  need(l && l->magic == TensorList::MAGIC, "list: not a list of tensors");
  return *l;
}
void list_work(const TensorList& l, const void* work) {
  need(work || l.work_bytes() == 0, "list: null work");
  aligned(work, 16, "work");
}
hipStream_t list_stream(void* s, TensorList& l) {
  if (l.dev && capturing(own_stream(s))) l.keep_table();
  return own_stream(s);
}
bool known_type(int t) { return t == BC2N_F32 || t == BC2N_F16 || t == BC2N_BF16; }
}  // namespace

size_t bc2n_logprobs_save_bytes(int64_t rows) { return rows > 0 ? (size_t)rows * 16 : 0; }

size_t bc2n_logprobs_work_bytes(int dtype, int64_t rows, int classes, int top) {
  size_t n = 0;
  guarded([&] {
    LogProbs a = lp_operands(dtype, &n, classes, rows, classes, nullptr, 0);
    lp_top(a, top);
    n = logprobs_work_bytes(dtype, rows, classes, top);
  });
  return n;
}

int bc2n_logprobs_fwd(void* stream, int dtype, const void* logits, int64_t ld, int64_t rows,
                      int classes, const void* targets, int target_bits, int top, float* logp,
                      float* entropy, float* top_logp, int32_t* top_index, void* save,
                      void* work) {
  return guarded([&] {
    LogProbs a = lp_operands(dtype, logits, ld, rows, classes, targets, target_bits);
    lp_top(a, top);
    need(!logp || targets, "logprobs: logp needs targets");
    need(top == 0 || rows == 0 || (top_logp && top_index), "null output");
    need(work || logprobs_work_bytes(dtype, rows, classes, top) == 0, "logprobs: null work");
    aligned(work, 16, "work");
    aligned(save, 16, "save");
    a.logp = logp;
    a.entropy = entropy;
    a.top_logp = top_logp;
    a.top_index = top_index;
    a.save = reinterpret_cast<float*>(save);
    logprobs_fwd(own_stream(stream), a, work);
  });
}

int bc2n_logprobs_bwd(void* stream, int dtype, const void* logits, int64_t ld, int64_t rows,
                      int classes, const void* targets, int target_bits, int top,
                      const int32_t* top_index, const void* save, const float* d_logp,
                      const float* d_entropy, const float* d_top_logp, void* d_logits,
                      int64_t d_ld) {
  return guarded([&] {
    LogProbs a = lp_operands(dtype, logits, ld, rows, classes, targets, target_bits);
    lp_top(a, top);
    lp_gradient(a, d_logits, d_ld);
    need(rows == 0 || save, "null operand");
    aligned(save, 16, "save");
    need(!d_logp || targets, "logprobs: d_logp needs targets");
    need(!d_top_logp || (top > 0 && top_index), "logprobs: d_top_logp needs top_index");
    a.top_index = const_cast<int32_t*>(top_index);
    a.save = reinterpret_cast<float*>(const_cast<void*>(save));
    a.d_logp = d_logp;
    a.d_entropy = d_entropy;
    a.d_top = d_top_logp;
    logprobs_bwd(own_stream(stream), a);
  });
}

int bc2n_logprobs_grad(void* stream, int dtype, const void* logits, int64_t ld, int64_t rows,
                       int classes, const void* targets, int target_bits, const float* d_logp,
                       const float* d_entropy, float* logp, float* entropy, void* d_logits,
                       int64_t d_ld, void* work) {
  return guarded([&] {
    LogProbs a = lp_operands(dtype, logits, ld, rows, classes, targets, target_bits);
    lp_gradient(a, d_logits, d_ld);
    need((!logp && !d_logp) || targets, "logprobs: logp needs targets");
    need(work || logprobs_work_bytes(dtype, rows, classes, 0) == 0, "logprobs: null work");
    aligned(work, 16, "work");
    a.logp = logp;
    a.entropy = entropy;
    a.d_logp = d_logp;
    a.d_entropy = d_entropy;
    logprobs_grad(own_stream(stream), a, work);
  });
}

namespace {
// A [tokens][heads][width] operand and the bytes that it takes.
struct Span {
  intptr_t p;
  int64_t st, row, total;  // bytes: token stride, of one token's heads, of all
  bool by_token;           // a token's heads lie before the next token's
};
Span span_of(const HeadView& v, int64_t tokens, int heads, int width, int64_t es) {
  Span s;
  s.p = reinterpret_cast<intptr_t>(v.p);
  s.st = v.st * es;
  s.row = ((heads - 1) * v.sh + width) * es;
  s.total = (tokens - 1) * s.st + s.row;
  s.by_token = tokens == 1 || s.st >= s.row;
  return s;
}
// no element in both: ranges apart, or slices of the same tokens
bool apart(const Span& a, const Span& b) {
  if (b.p >= a.p + a.total || a.p >= b.p + b.total) return true;
  if (!a.by_token || !b.by_token || a.st != b.st) return false;
  const int64_t at = ((b.p - a.p) % a.st + a.st) % a.st;
  return at >= a.row && at + b.row <= a.st;
}
struct Heads {
  HeadView v;
  int64_t tokens;
  int heads, width;
  int64_t es;
  const char* what;
  bool empty() const { return tokens == 0 || heads == 0; }
  Span span() const { return span_of(v, tokens, heads, width, es); }
};
void refuse_unless(bool ok, const char* what, const char* msg) {
  if (!ok) throw std::invalid_argument(std::string(what) + msg);
}
Heads heads_of(const char* what, const void* p, int64_t st, int64_t sh, int64_t tokens, int heads,
               int width, int dtype, int align, bool written) {
  Heads h;
  h.v.p = p;
  h.v.st = st;
  h.v.sh = sh;
  h.tokens = tokens;
  h.heads = heads;
  h.width = width;
  h.es = dtype == BC2N_F32 ? 4 : 2;
  h.what = what;
  if (h.empty()) return h;
  if (tokens == 1) h.v.st = st = width;  // no call steps by these
  if (heads == 1) h.v.sh = sh = width;
  refuse_unless(p, what, ": null operand");
  aligned(p, align, what);
  refuse_unless(st >= 0 && sh >= 0, what, ": negative stride");
  refuse_unless(st < (int64_t(1) << 40) && sh < (int64_t(1) << 40), what, ": stride too large");
  refuse_unless((st * h.es) % align == 0 && (sh * h.es) % align == 0, what,
                ": strides have to keep the alignment");
  refuse_unless((tokens - 1) * (double)st + (heads - 1) * (double)sh < 0x1p56, what, ": stride too large");
  if (written) {
    const bool by_token = (heads == 1 || sh >= width) && (tokens == 1 || st >= (heads - 1) * sh + width);
    const bool by_head = (tokens == 1 || st >= width) && (heads == 1 || sh >= (tokens - 1) * st + width);
    refuse_unless(by_token || by_head, what, ": elements overlap");
  }
  return h;
}
// every written operand apart from all others, but (in_place) for the one that is
// read in the same place of each as many
void all_apart(const std::vector<Heads>& written, const std::vector<Heads>& read, bool in_place) {
  for (size_t i = 0; i < written.size(); ++i) {
    const Heads& w = written[i];
    if (w.empty()) continue;
    for (size_t j = 0; j < written.size() + read.size(); ++j) {
      const Heads& o = j < written.size() ? written[j] : read[j - written.size()];
      if (o.empty() || j == i) continue;
      const bool same = in_place && j >= written.size() && j % written.size() == i && o.v.p == w.v.p && o.heads == w.heads &&
                        (o.v.st == w.v.st || o.tokens == 1) && (o.v.sh == w.v.sh || o.heads == 1);
      if (!same && !apart(w.span(), o.span()))
        throw std::invalid_argument(std::string(w.what) + " overlaps " + o.what);
    }
  }
}

HeadNorm headnorm_operands(int dtype, int64_t tokens, int heads, int kv_heads, int width, int rotated,
                           int interleaved, const void* positions, int position_bits,
                           const float* freq, const void* q_weight, const void* k_weight,
                           int weight_dtype, float eps) {
  need(known_type(dtype), "headnorm: bad dtype");
  need(weight_dtype == BC2N_F32 || weight_dtype == dtype,
       "headnorm: weights are f32 or of the operands' type");
  need(tokens >= 0 && tokens < (int64_t(1) << 26), "headnorm: bad number of tokens");
  need(heads >= 0 && kv_heads >= 0 && heads + kv_heads > 0 && heads <= 65536 && kv_heads <= 65536,
       "headnorm: bad number of heads");
  need(width >= 2 && width % 2 == 0, "headnorm: the width has to be even");
  need(rotated >= 0 && rotated <= width && rotated % 2 == 0,
       "headnorm: the rotated elements are an even number up to the width");
  need(headnorm_vector(dtype, width, rotated, interleaved) > 0,
       "headnorm: no layout for this width (64 vectors of a pair's elements at most)");
  need(tokens == 0 || rotated == 0 || (positions && freq), "headnorm: null positions or frequencies");
  need(position_bits == 32 || position_bits == 64, "headnorm: positions are i32 or i64");
  need(heads == 0 || q_weight, "headnorm: null q_weight");
  need(kv_heads == 0 || k_weight, "headnorm: null k_weight");
  need(eps >= 0 && std::isfinite(eps), "headnorm: bad eps");
  if (positions) aligned(positions, position_bits / 8, "positions");
  if (freq) aligned(freq, 4, "frequencies");
  for (const void* w : {q_weight, k_weight})
    if (w) aligned(w, weight_dtype == BC2N_F32 ? 4 : 2, "weight");
  HeadNorm a;
  a.dtype = dtype;
  a.weight_dtype = weight_dtype;
  a.tokens = tokens;
  a.heads[0] = heads;
  a.heads[1] = kv_heads;
  a.width = width;
  a.rotated = rotated;
  a.interleaved = interleaved != 0;
  a.pos = positions;
  a.pos64 = position_bits == 64;
  a.freq = freq;
  a.weight[0] = q_weight;
  a.weight[1] = k_weight;
  a.eps = eps;
  return a;
}

PackedAttn attention_operands(int dtype, int causal, int sequences, int64_t q_tokens, int64_t k_tokens,
                              int heads, int kv_heads, int width, float scale,
                              const int32_t* q_offsets, const int32_t* k_offsets,
                              const int32_t* q_lengths, const int32_t* k_lengths) {
  need(dtype == BC2N_F16 || dtype == BC2N_BF16, "attention: f16 or bf16");
  need(sequences >= 0 && sequences <= (1 << 24), "attention: bad number of sequences");
  need(heads > 0 && kv_heads > 0 && heads % kv_heads == 0 && heads < 65536,
       "attention: the heads have to be a multiple of the keys' heads");
  need(width > 0 && width % 8 == 0 && width <= PA_MAX_WIDTH,
       "attention: the width has to be a multiple of 8 up to 128");
  const int64_t G = heads / kv_heads, most = (int64_t(1) << 31) - (1 << 14);
  need(q_tokens >= 0 && k_tokens >= 0 && q_tokens * G < most && k_tokens * G < most,
       "attention: bad number of tokens");
  need(scale > 0 && std::isfinite(scale), "attention: the scale has to be positive");
  need(q_offsets && k_offsets, "attention: null offsets");
  for (const void* p : {q_offsets, k_offsets, q_lengths, k_lengths})
    if (p) aligned(p, 4, "offsets");
  PackedAttn a;
  a.dtype = dtype;
  a.causal = causal != 0;
  a.sequences = sequences;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.width = width;
  a.q_tokens = q_tokens;
  a.k_tokens = k_tokens;
  a.scale = scale;
  a.q_off = q_offsets;
  a.k_off = k_offsets;
  a.q_len = q_lengths;
  a.k_len = k_lengths;
  return a;
}
// 64 tokens of all heads of a group within 2 GiB: the copies' offsets have 32 bits
void near_enough(const Heads& h, int group) {
  if (h.empty()) return;
  refuse_unless(66 * h.v.st + (group + 1) * h.v.sh + h.width < (int64_t(1) << 30), h.what,
                ": stride too large");
}
}  // namespace

int bc2n_headnorm_fwd(void* stream, int dtype, int64_t tokens, int heads, int kv_heads, int width,
                      int rotated, int interleaved, const void* q, int64_t q_st, int64_t q_sh,
                      const void* k, int64_t k_st, int64_t k_sh, const void* positions,
                      int position_bits, const float* freq, const void* q_weight,
                      const void* k_weight, int weight_dtype, float eps, void* q_out, int64_t qo_st,
                      int64_t qo_sh, void* k_out, int64_t ko_st, int64_t ko_sh) {
  return guarded([&] {
    HeadNorm a = headnorm_operands(dtype, tokens, heads, kv_heads, width, rotated, interleaved, positions,
                                   position_bits, freq, q_weight, k_weight, weight_dtype, eps);
    const int es = dtype == BC2N_F32 ? 4 : 2;
    auto view = [&](const char* what, const void* p, int64_t st, int64_t sh, int n, bool w) {
      return heads_of(what, p, st, sh, tokens, n, width, dtype, es, w);
    };
    const Heads x[2] = {view("q", q, q_st, q_sh, heads, false), view("k", k, k_st, k_sh, kv_heads, false)};
    const Heads y[2] = {view("q_out", q_out, qo_st, qo_sh, heads, true),
                        view("k_out", k_out, ko_st, ko_sh, kv_heads, true)};
    all_apart({y[0], y[1]}, {x[0], x[1]}, true);
    for (int i = 0; i < 2; ++i) {
      a.x[i] = x[i].v;
      a.out[i] = y[i].v;
    }
    headnorm_fwd(own_stream(stream), a);
  });
}

size_t bc2n_headnorm_work_bytes(int64_t tokens, int width) {
  return tokens > 0 && width > 0 ? headnorm_work_bytes(tokens, width) : 0;
}

int bc2n_headnorm_bwd(void* stream, int dtype, int64_t tokens, int heads, int kv_heads, int width,
                      int rotated, int interleaved, const void* d_q, int64_t dq_st, int64_t dq_sh,
                      const void* d_k, int64_t dk_st, int64_t dk_sh, const void* q, int64_t q_st,
                      int64_t q_sh, const void* k, int64_t k_st, int64_t k_sh, const void* positions,
                      int position_bits, const float* freq, const void* q_weight,
                      const void* k_weight, int weight_dtype, float eps, void* q_grad, int64_t qg_st,
                      int64_t qg_sh, void* k_grad, int64_t kg_st, int64_t kg_sh, float* d_q_weight,
                      float* d_k_weight, void* work) {
  return guarded([&] {
    HeadNorm a = headnorm_operands(dtype, tokens, heads, kv_heads, width, rotated, interleaved, positions,
                                   position_bits, freq, q_weight, k_weight, weight_dtype, eps);
    const int es = dtype == BC2N_F32 ? 4 : 2;
    auto view = [&](const char* what, const void* p, int64_t st, int64_t sh, int n, bool w) {
      return heads_of(what, p, st, sh, tokens, n, width, dtype, es, w);
    };
    const Heads x[2] = {view("q", q, q_st, q_sh, heads, false), view("k", k, k_st, k_sh, kv_heads, false)};
    const Heads d[2] = {view("d_q", d_q, dq_st, dq_sh, heads, false),
                        view("d_k", d_k, dk_st, dk_sh, kv_heads, false)};
    const Heads y[2] = {view("q_grad", q_grad, qg_st, qg_sh, heads, true),
                        view("k_grad", k_grad, kg_st, kg_sh, kv_heads, true)};
    all_apart({y[0], y[1]}, {x[0], x[1], d[0], d[1]}, true);
    need(tokens == 0 || work, "headnorm: null work");
    aligned(work, 16, "work");
    for (int i = 0; i < 2; ++i) {
      a.x[i] = x[i].v;
      a.d[i] = d[i].v;
      a.out[i] = y[i].v;
    }
    a.d_weight[0] = d_q_weight;
    a.d_weight[1] = d_k_weight;
    headnorm_bwd(own_stream(stream), a, work);
  });
}

size_t bc2n_attention_fwd_work_bytes(int dtype, int causal, int sequences, int64_t q_tokens,
                                     int64_t k_tokens, int heads, int kv_heads, int width) {
  size_t n = 0;
  guarded([&] {
    const int32_t none = 0;
    n = packattn_fwd_work_bytes(attention_operands(dtype, causal, sequences, q_tokens, k_tokens, heads,
                                                   kv_heads, width, 1.f, &none, &none, nullptr, nullptr));
  });
  return n;
}
size_t bc2n_attention_bwd_work_bytes(int dtype, int causal, int sequences, int64_t q_tokens,
                                     int64_t k_tokens, int heads, int kv_heads, int width) {
  size_t n = 0;
  guarded([&] {
    const int32_t none = 0;
    n = packattn_bwd_work_bytes(attention_operands(dtype, causal, sequences, q_tokens, k_tokens, heads,
                                                   kv_heads, width, 1.f, &none, &none, nullptr, nullptr));
  });
  return n;
}

int bc2n_attention_fwd(void* stream, int dtype, int causal, int sequences, int64_t q_tokens,
                       int64_t k_tokens, int heads, int kv_heads, int width, float scale,
                       const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* q_lengths,
                       const int32_t* k_lengths, const void* q, int64_t q_st, int64_t q_sh,
                       const void* k, int64_t k_st, int64_t k_sh, const void* v, int64_t v_st,
                       int64_t v_sh, int fill, void* out, int64_t o_st, int64_t o_sh, float* lse,
                       void* work) {
  return guarded([&] {
    PackedAttn a = attention_operands(dtype, causal, sequences, q_tokens, k_tokens, heads, kv_heads, width,
                                      scale, q_offsets, k_offsets, q_lengths, k_lengths);
    const Heads hq = heads_of("q", q, q_st, q_sh, q_tokens, heads, width, dtype, 16, false);
    const Heads hk = heads_of("k", k, k_st, k_sh, k_tokens, kv_heads, width, dtype, 16, false);
    const Heads hv = heads_of("v", v, v_st, v_sh, k_tokens, kv_heads, width, dtype, 16, false);
    const Heads ho = heads_of("out", out, o_st, o_sh, q_tokens, heads, width, dtype, 16, true);
    for (const Heads* h : {&hk, &hv}) {
      near_enough(*h, 1);
      refuse_unless(h->tokens <= 1 || h->v.st >= width, h->what, ": tokens overlap");
    }
    all_apart({ho}, {hq, hk, hv}, false);
    need(q_tokens == 0 || lse, "attention: null lse");
    aligned(lse, 4, "lse");
    need(work || packattn_fwd_work_bytes(a) == 0, "attention: null work");
    aligned(work, 16, "work");
    a.fill = fill != 0;
    a.q = hq.v;
    a.k = hk.v;
    a.v = hv.v;
    a.o = ho.v;
    a.lse = lse;
    packattn_fwd(own_stream(stream), a, work);
  });
}

int bc2n_attention_bwd(void* stream, int dtype, int causal, int sequences, int64_t q_tokens,
                       int64_t k_tokens, int heads, int kv_heads, int width, float scale,
                       const int32_t* q_offsets, const int32_t* k_offsets, const int32_t* q_lengths,
                       const int32_t* k_lengths, const void* d_out, int64_t do_st, int64_t do_sh,
                       const void* q, int64_t q_st, int64_t q_sh, const void* k, int64_t k_st,
                       int64_t k_sh, const void* v, int64_t v_st, int64_t v_sh, const void* out,
                       int64_t o_st, int64_t o_sh, const float* lse, int fill, void* d_q, int64_t dq_st,
                       int64_t dq_sh, void* d_k, int64_t dk_st, int64_t dk_sh, void* d_v, int64_t dv_st,
                       int64_t dv_sh, void* work) {
  return guarded([&] {
    PackedAttn a = attention_operands(dtype, causal, sequences, q_tokens, k_tokens, heads, kv_heads, width,
                                      scale, q_offsets, k_offsets, q_lengths, k_lengths);
    auto rows = [&](const char* what, const void* p, int64_t st, int64_t sh, bool w) {
      return heads_of(what, p, st, sh, q_tokens, heads, width, dtype, 16, w);
    };
    auto keys = [&](const char* what, const void* p, int64_t st, int64_t sh, bool w) {
      return heads_of(what, p, st, sh, k_tokens, kv_heads, width, dtype, 16, w);
    };
    const Heads hq = rows("q", q, q_st, q_sh, false), hg = rows("d_out", d_out, do_st, do_sh, false);
    const Heads ho = rows("out", out, o_st, o_sh, false), hdq = rows("d_q", d_q, dq_st, dq_sh, true);
    const Heads hk = keys("k", k, k_st, k_sh, false), hv = keys("v", v, v_st, v_sh, false);
    const Heads hdk = keys("d_k", d_k, dk_st, dk_sh, true), hdv = keys("d_v", d_v, dv_st, dv_sh, true);
    for (const Heads* h : {&hk, &hv}) {
      near_enough(*h, 1);
      refuse_unless(h->tokens <= 1 || h->v.st >= width, h->what, ": tokens overlap");
    }
    for (const Heads* h : {&hq, &hg}) near_enough(*h, heads / kv_heads);
    all_apart({hdq, hdk, hdv}, {hq, hk, hv, ho, hg}, false);
    need(q_tokens == 0 || lse, "attention: null lse");
    aligned(lse, 4, "lse");
    need(work || packattn_bwd_work_bytes(a) == 0, "attention: null work");
    aligned(work, 16, "work");
    a.fill = fill != 0;
    a.q = hq.v;
    a.k = hk.v;
    a.v = hv.v;
    a.o = ho.v;
    a.lse = const_cast<float*>(lse);
    a.d_o = hg.v;
    a.dq = hdq.v;
    a.dk = hdk.v;
    a.dv = hdv.v;
    packattn_bwd(own_stream(stream), a, work);
  });
}

int bc2n_sample(void* stream, int dtype, const void* logits, int64_t ld, int64_t rows, int classes,
                const float* uniforms, double temperature, const float* temperatures, int64_t top_k,
                const int32_t* top_ks, double top_p, const float* top_ps, double min_p,
                const float* min_ps, int32_t* index, float* logp) {
  return guarded([&] {
    need(known_type(dtype), "sample: bad dtype");
    need(rows >= 0 && rows < (int64_t(1) << 31), "sample: bad number of rows");
    need(classes > 0 && classes <= (1 << 28), "sample: bad number of classes");
    need(rows <= 1 || ld >= classes, "sample: the row stride is below the number of classes");
    need(rows == 0 || (logits && uniforms), "null operand");
    need(rows == 0 || index, "null output");
    need(temperatures || (temperature >= 0 && std::isfinite(temperature)),
         "sample: the temperature has to be finite and not negative");
    need(top_ks || top_k >= 0, "sample: top_k must not be negative");
    need(top_ps || !std::isnan(top_p), "sample: top_p is NaN");
    need(min_ps || !std::isnan(min_p), "sample: min_p is NaN");
    aligned(logits, dtype == BC2N_F32 ? 4 : 2, "logits");
    for (const void* p : {(const void*)uniforms, (const void*)temperatures, (const void*)top_ks,
                          (const void*)top_ps, (const void*)min_ps, (const void*)index, (const void*)logp})
      aligned(p, 4, "sample operand");
    Sample a;
    a.dtype = dtype;
    a.x = logits;
    a.ld = ld;
    a.rows = rows;
    a.V = classes;
    a.u = uniforms;
    a.temperature.v = temperature;
    a.temperature.row = temperatures;
    a.top_p.v = top_p;
    a.top_p.row = top_ps;
    a.min_p.v = min_p;
    a.min_p.row = min_ps;
    a.top_k = top_k;
    a.top_k_row = top_ks;
    a.index = index;
    a.logp = logp;
    sample(own_stream(stream), a);
  });
}

void* bc2n_grad_list(int count, const void* const* grads, const int64_t* sizes, const int* dtypes,
                     void* const* out) {
  TensorList* l = nullptr;
  guarded([&] {
    need(count >= 0 && (count == 0 || (grads && sizes && dtypes)), "list: null operand");
    std::vector<ListEntry> e((size_t)count);
    for (int i = 0; i < count; ++i) {
      need(known_type(dtypes[i]), "list: bad dtype");
      e[i].g = grads[i];
      e[i].n = sizes[i];
      e[i].g_type = dtypes[i];
      if (out) {
        need(out[i] || sizes[i] == 0, "list: null output");
        e[i].g_out = out[i];
      }
    }
    l = new TensorList(std::move(e), out != nullptr, false);
  });
  return l;
}

void* bc2n_adam_list(int count, const int64_t* sizes, const void* const* params,
                     const int* param_dtypes, const void* const* grads, const int* grad_dtypes,
                     const float* const* avg, const float* const* avg_sq, void* const* params_out,
                     float* const* avg_out, float* const* avg_sq_out) {
  TensorList* l = nullptr;
  guarded([&] {
    need(count >= 0 && (count == 0 || (sizes && params && param_dtypes && grads && grad_dtypes &&
                                       avg && avg_sq && params_out && avg_out && avg_sq_out)),
         "list: null operand");
    std::vector<ListEntry> e((size_t)count);
    for (int i = 0; i < count; ++i) {
      need(known_type(param_dtypes[i]) && known_type(grad_dtypes[i]), "list: bad dtype");
      e[i].n = sizes[i];
      e[i].g = grads[i];
      e[i].g_type = grad_dtypes[i];
      e[i].p = params[i];
      e[i].p_type = param_dtypes[i];
      e[i].m = avg[i];
      e[i].v = avg_sq[i];
      e[i].p_out = params_out[i];
      e[i].m_out = avg_out[i];
      e[i].v_out = avg_sq_out[i];
    }
    l = new TensorList(std::move(e), false, true);
  });
  return l;
}

int bc2n_list_free(void* list) {
  return guarded([&] {
    if (list) delete &list_of(list);
  });
}

size_t bc2n_list_work_bytes(void* list) {
  size_t n = 0;
  guarded([&] { n = list_of(list).work_bytes(); });
  return n;
}

int bc2n_grad_norm(void* stream, void* list, float* norm, void* work) {
  return guarded([&] {
    TensorList& l = list_of(list);
    need(norm, "null operand");
    list_work(l, work);
    grad_norm(list_stream(stream, l), l, norm, work);
  });
}

int bc2n_grad_clip(void* stream, void* list, float max_norm, float* norm, void* work) {
  return guarded([&] {
    TensorList& l = list_of(list);
    need(l.clips, "grad_clip: the list has no outputs");
    need(max_norm > 0.f, "grad_clip: max_norm must be positive");
    list_work(l, work);
    grad_clip(list_stream(stream, l), l, max_norm, norm, work);
  });
}

int bc2n_adam_step(void* stream, void* list, double lr, double beta1, double beta2, double eps,
                   double weight_decay, int64_t step, double max_norm, const float* scalars,
                   float* norm, void* work) {
  return guarded([&] {
    TensorList& l = list_of(list);
    need(l.adam, "adam_step: not a list of parameters");
    need(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1, "adam_step: betas must be in [0, 1)");
    need((float)eps > 0 && std::isfinite((float)eps),
         "adam_step: eps must be positive and finite in f32");
    need(weight_decay >= 0 && std::isfinite(weight_decay),
         "adam_step: weight_decay must be finite and not negative");
    need(scalars || (step >= 1 && std::isfinite(lr)), "adam_step: step counts from 1, lr is finite");
    need(max_norm >= 0, "adam_step: max_norm must be positive, or 0 for none");
    list_work(l, work);
    AdamScalars s;
    s.lr = lr;
    s.beta1 = beta1;
    s.beta2 = beta2;
    s.eps = eps;
    s.decay = weight_decay;
    s.step = step;
    s.max_norm = max_norm;
    s.device = scalars;
    adam_step(list_stream(stream, l), l, s, norm, work);
  });
}

int bc2n_dropout_table(void* stream, float* tbl, int B, int C, uint32_t k0, uint32_t k1,
                       float rate) {
  return guarded([&] {
    need(tbl && B > 0 && C > 0, "bad table shape");
    need(rate >= 0.f && rate < 1.f, "rate must be in [0,1)");
    const float keep = 1.0f - rate;
    dropout_table(as_stream(stream), tbl, B, C, k0, k1, keep);
  });
}

int bc2n_bernoulli_bits(void* stream, uint8_t* out, long n, uint32_t k0, uint32_t k1,
                        float rate) {
  return guarded([&] {
    need(out && n > 0, "bad output");
    need(rate >= 0.f && rate < 1.f, "rate must be in [0,1)");
    bernoulli_bits(as_stream(stream), out, n, k0, k1, 1.0f - rate);
  });
}

int bc2n_stack_keys(void* stream, const uint32_t* seed, int depth, uint32_t* out) {
  return guarded([&] {
    need(seed && out && depth > 0, "bad arguments");
    stack_keys(as_stream(stream), seed, depth, out);
  });
}

int bc2n_prof_enable(int on) {
  return guarded([&] { kprof_enable(on != 0); });
}

int bc2n_prof_filter(const char* name) {
  return guarded([&] { kprof_filter(name); });
}

int bc2n_prof_read(char* names, int name_len, double* ms, int* counts, int cap) {
  int n = -1;
  if (guarded([&] { n = kprof_read(names, name_len, ms, counts, cap); }) != 0) return -1;
  return n;
}

int bc2n_probe_gemm(void* stream, int M, int N, int K, const uint16_t* A, const uint16_t* B,
                    float* C) {
  return guarded([&] {
    need(A && B && C, "null operand");
    GemmArgs g;
    g.M = M; g.N = N; g.K = K;
    g.A = reinterpret_cast<const h16*>(A); g.a_sm = K; g.a_sk = 1;
    g.B = reinterpret_cast<const h16*>(B); g.b_sn = K; g.b_sk = 1;
    gemm<128, 128>(as_stream(stream), g, EpiStore<float>{C, N, 0, nullptr, N});
  });
}

double bc2n_probe_mfma(void* stream, int form, int blocks, int iters, float* out) {
  double flops = -1.0;
  if (guarded([&] { flops = probe_mfma_rate(as_stream(stream), form, blocks, iters, out); }) != 0)
    return -1.0;
  return flops;
}

int bc2n_probe_gemm_f32(void* stream, int M, int N, int K, int batch, const float* A,
                        long a_sm, long a_sk, long a_sb, const float* B, long b_sk, long b_sn,
                        long b_sb, float* C, long c_sm, long c_sn, long c_sb) {
  return guarded([&] {
    GemmF32 g;
    g.M = M; g.N = N; g.K = K; g.batch = batch;
    g.A = A; g.a_sm = a_sm; g.a_sk = a_sk; g.a_sb = a_sb;
    g.B = B; g.b_sk = b_sk; g.b_sn = b_sn; g.b_sb = b_sb;
    g.C = C; g.c_sm = c_sm; g.c_sn = c_sn; g.c_sb = c_sb;
    gemm_f32(as_stream(stream), g, "probe.gemm_f32");
  });
}

int bc2n_probe_recycle(void* stream, int N, const char* emb_dir, const float* aatype,
                       const float* prev_atom14, const float* prev_pair, const float* prev_msa0,
                       float* pair, float* msa0) {
  return guarded([&] {
    need(emb_dir && pair && msa0, "null operand");
    RecycleW r = recycle_w(weights(emb_dir));
    recycle_terms(as_stream(stream), r, N, aatype, prev_atom14, prev_pair, prev_msa0, pair, msa0);
  });
}

int bc2n_probe_layernorm(void* stream, long M, int C, const float* x, const float* gamma,
                         const float* beta, int fast, uint16_t* y, float* mean, float* rstd) {
  return guarded([&] {
    need(x && gamma && beta && y && mean && rstd, "null operand");
    ln_fwd_f32(as_stream(stream), x, M, C, 0, gamma, beta, reinterpret_cast<h16*>(y), mean,
               rstd, fast != 0, 0, nullptr, nullptr);
  });
}

}  // extern "C"
