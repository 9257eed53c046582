// Log probabilities of given tokens with the entropy of each row's distribution
// and its k most likely tokens, and the gradient of log probability and
// entropy, for rows of fp32 / bf16 / fp16 logits.
//
//   m = max x,  s = sum e^(x - m),  q = sum e^(x - m) (x - m)
//   logp_t  = (x_t - m) - ln s
//   entropy = ln s - q / s                       (= -sum p ln p; 0 ln 0 = 0)
//   dx_j    = -p_j (g_logp + g_entropy (logp_j + entropy)) + g_logp [j == t]
//
// Forward reads the logits once: every thread keeps a running (m, s, q),
// rescaled when m grows (s' = s e^d, q' = e^d (q + d s) with d = m - m'), and
// the same loads feed the top-k filter.  Backward reads them once more and
// writes dx.  Both are bound by memory; few rows are split over blocks (each
// split writes its (m, s, q) and its sorted k keys, a second launch joins them).
//
// Differences x - m are formed before the scaling to base 2, so the error of
// e^(x - m) does not grow with |m|; m and ln s are kept apart for the backward
// for the same reason.
//
// Top k: a wave holds its k best keys sorted, one per lane.  A key is the
// order-preserving image of the value with the complement of the place under
// it, so equal values rank by the lower place and no two keys are equal.
// Values above the k-th key (a compare per element, nearly always false) are
// collected in LDS, up to 64, and merged by rank: a key's place is the number
// of greater ones.  When one 512-element tile has more candidates than the
// buffer takes, the k-th largest of its lane maxima (a binary search with
// ballots) raises the threshold first, so a rising row costs a merge per tile
// and not one per element.
//
// Rows: all -inf -> logp -inf, entropy 0, gradient 0.  A NaN or +inf -> NaN.
// The ignored index: logp 0 and no gradient from it.  Any other token outside
// [0, V): logp NaN and a NaN gradient row.
#include "rows.h"

namespace {

typedef unsigned long long u64;

constexpr int kNT = 256;
constexpr float kL2E = 1.44269504088896340736f;
constexpr float kLow = -1e30f;  // stands for -inf where it is multiplied by a 0
constexpr int kMaxSplits = 64;
constexpr int kMaxTop = 64;

__device__ __forceinline__ float exp_d(float d) { return __builtin_amdgcn_exp2f(d * kL2E); }

// ---- running softmax statistics -------------------------------------------
struct Stat {
  float m, s, q;
};

__device__ __forceinline__ void stat_add8(Stat& a, const float (&x)[8]) {
  const float v = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                        fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
  const float m = fmaxf(a.m, v);
  const float ms = m == -INFINITY ? 0.f : m;
  const float d0 = a.m - ms, c = exp_d(d0);
  a.q = (a.q + fmaxf(d0, kLow) * a.s) * c;
  a.s *= c;
  a.m = m;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float d = x[i] - ms, e = exp_d(d);  // d = -inf: e = 0; NaN: e = NaN
    a.s += e;
    a.q += e * fmaxf(d, kLow);
  }
}

__device__ __forceinline__ Stat stat_join(const Stat& a, const Stat& b) {
  const float m = fmaxf(a.m, b.m);
  const float ms = m == -INFINITY ? 0.f : m;
  const float da = a.m - ms, db = b.m - ms, ca = exp_d(da), cb = exp_d(db);
  Stat r;
  r.m = m;
  r.s = a.s * ca + b.s * cb;
  r.q = (a.q + fmaxf(da, kLow) * a.s) * ca + (b.q + fmaxf(db, kLow) * b.s) * cb;
  return r;
}

__device__ __forceinline__ Stat stat_wave(Stat a) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) {
    const Stat b{__shfl_xor(a.m, off, 64), __shfl_xor(a.s, off, 64), __shfl_xor(a.q, off, 64)};
    a = stat_join(a, b);
  }
  return a;
}

// ---- top k ------------------------------------------------------------------
// Greater floats have greater images; -0 = +0, every NaN ranks above +inf, and
// 0 is below all of them (an empty slot).
__device__ __forceinline__ uint32_t order_of(float f) {
  const uint32_t u = __float_as_uint(f + 0.f);
  return f != f ? 0xffffffffu : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float((o & 0x80000000u) ? o ^ 0x80000000u : ~o);
}

__device__ __forceinline__ u64 lane64(u64 v, int l) {
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, l);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l);
  return ((u64)hi << 32) | lo;
}

// The LDS of a wave is written and read by that wave only: its accesses keep
// their order, the compiler must too.
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

struct Top {
  u64 best;   // lane i: the i-th greatest key so far (0: none)
  u64 least;  // a key must exceed this one to matter (wave-uniform)
  int fill;   // keys waiting in buf (wave-uniform)
  int k;
  u64* buf;   // LDS: 64 waiting keys
  u64* tmp;   // LDS: 64 slots of the merge
};

// Merge lane i's key `b` (i < n) into the sorted list.
__device__ __forceinline__ void top_merge(Top& t, u64 b, int n) {
  const int lane = threadIdx.x & 63;
  b = lane < n ? b : 0;
  int rl = lane, rb = 0;  // the list is sorted: its own greater keys are the lanes below
  for (int i = 0; i < n; ++i) {
    const u64 o = lane64(b, i);
    rl += o > t.best;
    rb += o > b;
  }
  for (int i = 0; i < t.k; ++i) rb += lane64(t.best, i) > b;
  t.tmp[lane] = 0;
  wave_fence();
  if (t.best != 0 && rl < t.k) t.tmp[rl] = t.best;
  if (b != 0 && rb < t.k) t.tmp[rb] = b;
  wave_fence();
  t.best = t.tmp[lane];
  wave_fence();
  const u64 last = lane64(t.best, t.k - 1);
  t.least = last > t.least ? last : t.least;
}

__device__ __forceinline__ void top_flush(Top& t) {
  if (t.fill == 0) return;
  wave_fence();
  const u64 b = t.buf[threadIdx.x & 63];
  top_merge(t, b, t.fill);
  t.fill = 0;
}

// Eight elements per lane, places base .. base + n - 1; places rise from tile
// to tile of a wave, so a value equal to the list's last never enters later.
__device__ __forceinline__ void top_add8(Top& t, const float (&x)[8], int base, int n) {
  uint32_t o[8], top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o[j] = j < n ? order_of(x[j]) : 0u;
    top = o[j] > top ? o[j] : top;
  }
  uint32_t least = (uint32_t)(t.least >> 32);
  if (__ballot(top > least) == 0) return;
  int count = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) count += __popcll(__ballot(o[j] > least));
  if (t.fill + count > 64) {
    // at least k values of this tile are >= the k-th largest lane maximum
    uint32_t kth = 0;
    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
      if (__popcll(__ballot(top >= (kth | bit))) >= t.k) kth |= bit;
    if (kth > least) t.least = ((u64)(kth - 1) << 32) | 0xffffffffull;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const u64 key = o[j] ? ((u64)o[j] << 32) | (uint32_t)~(uint32_t)(base + j) : 0;
    u64 in = __ballot(key > t.least);
    if (in == 0) continue;
    if (t.fill + __popcll(in) > 64) {
      top_flush(t);
      in = __ballot(key > t.least);
    }
    const int at = t.fill + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32),
                                                      __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
    if (key > t.least) t.buf[at] = key;
    t.fill += __popcll(in);
  }
}

struct LpArgs {
  const void* x;            // [rows][xs]
  const long long* tokens;  // [rows]
  float* logp;              // [rows]
  float* entropy;           // [rows]
  float* stats;             // [rows][3]: m, ln s, entropy (or null)
  float* top_logp;          // [rows][k]
  long long* top_ids;       // [rows][k]
  float* pstat;             // [rows][splits][4]
  u64* pkeys;               // [rows][splits][k]
  const float* g_logp;      // backward: [rows] or null
  const float* g_entropy;   // [rows] or null
  void* dx;                 // [rows][V]
  long long rows, row0, xs, ignore;
  int V, k, splits, chunk;
};

// One thread's answer for the row from its statistics.
template <int DT>
__device__ __forceinline__ float lp_finish(const LpArgs& a, long long row, const Stat& t) {
  const bool none = t.m == -INFINITY && t.s == 0.f;
  const float ls = none ? 0.f : logf(t.s);
  const float h = none ? 0.f : ls - t.q / t.s;
  const long long tok = a.tokens[row];
  float lp;
  if (tok == a.ignore) {
    lp = 0.f;
  } else if (tok >= 0 && tok < a.V) {
    const float xt = Elem<DT>::up(
        reinterpret_cast<const typename Elem<DT>::raw*>(a.x)[row * a.xs + tok]);
    lp = none ? -INFINITY : (xt - t.m) - ls;
  } else {
    lp = NAN;
  }
  a.logp[row] = lp;
  a.entropy[row] = h;
  if (a.stats) {
    a.stats[row * 3] = t.m;
    a.stats[row * 3 + 1] = ls;
    a.stats[row * 3 + 2] = h;
  }
  return ls;
}

__device__ __forceinline__ void top_write(const LpArgs& a, long long row, u64 key, float m,
                                          float ls) {
  const int lane = threadIdx.x & 63;
  if (lane < a.k) {
    const float v = value_of((uint32_t)(key >> 32));
    // a row of -inf: m = -inf, and every alternative's log probability is -inf
    a.top_logp[row * a.k + lane] = m == -INFINITY && ls == 0.f ? v : (v - m) - ls;
    a.top_ids[row * a.k + lane] = (long long)(uint32_t)~(uint32_t)key;
  }
}

// WPR waves per row and split: 1 (four rows per block) or 4 (the block).
template <int DT, bool TOP, int WPR>
__global__ __launch_bounds__(kNT) void lp_fwd_kernel(LpArgs a) {
  typedef typename Elem<DT>::raw raw;
  __shared__ u64 lds[TOP ? 4 * 128 : 1];
  __shared__ Stat joined[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long unit = WPR == 1 ? (long long)blockIdx.x * 4 + wave : blockIdx.x;
  const long long row = a.row0 + (WPR == 1 ? unit : unit / a.splits);
  if (row >= a.rows) return;  // WPR = 1 only (no barrier below), or past the last row as a block
  const int split = WPR == 1 ? 0 : (int)(unit % a.splits);
  const int lo = split * a.chunk, hi = min(a.V, lo + a.chunk);
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  Stat st{-INFINITY, 0.f, 0.f};
  Top top{0, 0, 0, a.k, lds + (TOP ? wave * 128 : 0), lds + (TOP ? wave * 128 + 64 : 0)};
  const int w = WPR == 1 ? 0 : wave;
  for (int c0 = lo + w * 512; c0 < hi; c0 += WPR * 512) {  // wave-uniform
    const int c = c0 + lane * 8;
    float f[8];
    load8_n<DT>(x + c, hi - c, -INFINITY, f);
    stat_add8(st, f);
    if constexpr (TOP) top_add8(top, f, c, hi - c);
  }
  st = stat_wave(st);
  if constexpr (TOP) top_flush(top);
  if constexpr (WPR == 4) {
    if (lane == 0) joined[wave] = st;
    if constexpr (TOP) {
      wave_fence();
      top.buf[lane] = top.best;
    }
    __syncthreads();
    if (wave != 0) return;
    st = stat_join(stat_join(joined[0], joined[1]), stat_join(joined[2], joined[3]));
    if constexpr (TOP) {
#pragma unroll 1
      for (int o = 1; o < 4; ++o) {
        const u64 b = lds[o * 128 + lane];
        const u64 in = __ballot(b > top.least);  // sorted: the first lanes
        if (in) top_merge(top, b, __popcll(in));
      }
    }
    if (a.splits > 1) {
      const long long p = row * a.splits + split;
      if (lane == 0) {
        a.pstat[p * 4] = st.m;
        a.pstat[p * 4 + 1] = st.s;
        a.pstat[p * 4 + 2] = st.q;
      }
      if (TOP && lane < a.k) a.pkeys[p * a.k + lane] = top.best;
      return;
    }
  }
  float ls = 0.f;
  if (lane == 0) ls = lp_finish<DT>(a, row, st);
  if constexpr (TOP) top_write(a, row, top.best, __shfl(st.m, 0, 64), __shfl(ls, 0, 64));
}

// Joins the splits of a row: statistics in one wave, keys in 16 waves of up to
// four lists each and then in one.
template <int DT, bool TOP>
__global__ __launch_bounds__(TOP ? 1024 : 64) void lp_join_kernel(LpArgs a) {
  __shared__ u64 lds[TOP ? 16 * 128 : 1];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long row = a.row0 + blockIdx.x;
  Top top{0, 0, 0, a.k, lds + (TOP ? wave * 128 : 0), lds + (TOP ? wave * 128 + 64 : 0)};
  if constexpr (TOP) {
    u64 b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int sp = wave + 16 * i;
      b[i] = sp < a.splits && lane < a.k ? a.pkeys[(row * a.splits + sp) * a.k + lane] : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u64 in = __ballot(b[i] > top.least);
      if (in) top_merge(top, b[i], __popcll(in));
    }
    top.buf[lane] = top.best;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll 1
    for (int o = 1; o < 16; ++o) {
      const u64 c = lds[o * 128 + lane];
      const u64 in = __ballot(c > top.least);
      if (in) top_merge(top, c, __popcll(in));
    }
  }
  Stat st{-INFINITY, 0.f, 0.f};
  if (lane < a.splits) {
    const float* p = a.pstat + (row * a.splits + lane) * 4;
    st = Stat{p[0], p[1], p[2]};
  }
  st = stat_wave(st);
  float ls = 0.f;
  if (lane == 0) ls = lp_finish<DT>(a, row, st);
  if constexpr (TOP) top_write(a, row, top.best, __shfl(st.m, 0, 64), __shfl(ls, 0, 64));
}

// WPR = 4: a block takes `chunk` elements of a row; 1: a wave takes a row.
template <int DT, int WPR>
__global__ __launch_bounds__(kNT) void lp_bwd_kernel(LpArgs a) {
  typedef typename Elem<DT>::raw raw;
  const int wave = threadIdx.x >> 6;
  const long long unit = WPR == 1 ? (long long)blockIdx.x * 4 + wave : blockIdx.x;
  const long long row = a.row0 + (WPR == 1 ? unit : unit / a.splits);
  if (row >= a.rows) return;
  const int split = WPR == 1 ? 0 : (int)(unit % a.splits);
  const int lo = split * a.chunk, hi = min(a.V, lo + a.chunk);
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  raw* dx = reinterpret_cast<raw*>(a.dx) + row * a.V;
  const float m = a.stats[row * 3], ls = a.stats[row * 3 + 1], h = a.stats[row * 3 + 2];
  const long long tok = a.tokens[row];
  float gl = a.g_logp ? a.g_logp[row] : 0.f;
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const bool in = tok >= 0 && tok < a.V;
  if (tok == a.ignore) gl = 0.f;
  else if (!in) gl = NAN;
  const bool none = m == -INFINITY && ls == 0.f;
  const float ga = gl + gh * h;
  const int t = in ? (int)tok : -1;
  const int l = WPR == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  for (int c = lo + l * 8; c < hi; c += WPR * 512) {
    float f[8];
    load8_n<DT>(x + c, hi - c, 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float lp = (f[i] - m) - ls;
      const float r = -exp_d(lp) * (ga + gh * fmaxf(lp, kLow));
      f[i] = none ? 0.f : (c + i == t ? r + gl : r);
    }
    store8_n<DT>(dx + c, hi - c, f);
  }
}

// Splits of the forward: enough blocks for the chip when rows are few, at
// least 2048 elements (one tile per wave) each.
int fwd_splits(long long rows, int V) {
  if (V <= 2048) return 1;
  const long long most = (V + 2047LL) / 2048;
  long long s = (1024 + rows - 1) / rows;
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  if (s <= 1) return 1;
  const long long chunk = ((V + s - 1) / s + 2047) / 2048 * 2048;
  return (int)((V + chunk - 1) / chunk);
}

constexpr long long kUnitsPerLaunch = 1LL << 22;  // blocks: a grid holds under 2^32 threads

template <int DT, bool TOP>
int lp_fwd(LpArgs a, hipStream_t st) {
  const long long step = kUnitsPerLaunch / a.splits;
  const long long last = a.rows;
  for (a.row0 = 0; a.row0 < last; a.row0 += step) {
    const long long n = last - a.row0 < step ? last - a.row0 : step;
    a.rows = a.row0 + n;
    if (a.V <= 2048) {
      hipLaunchKernelGGL((lp_fwd_kernel<DT, TOP, 1>), dim3((unsigned)((n + 3) / 4)), dim3(kNT), 0,
                         st, a);
    } else {
      hipLaunchKernelGGL((lp_fwd_kernel<DT, TOP, 4>), dim3((unsigned)(n * a.splits)), dim3(kNT), 0,
                         st, a);
      if (a.splits > 1)
        hipLaunchKernelGGL((lp_join_kernel<DT, TOP>), dim3((unsigned)n), dim3(TOP ? 1024 : 64), 0,
                           st, a);
    }
    ZK_CHECK_LAUNCH();
  }
  return 0;
}

template <int DT>
int lp_bwd(LpArgs a, hipStream_t st) {
  const long long step = kUnitsPerLaunch / a.splits;
  const long long last = a.rows;
  for (a.row0 = 0; a.row0 < last; a.row0 += step) {
    const long long n = last - a.row0 < step ? last - a.row0 : step;
    a.rows = a.row0 + n;
    if (a.V <= 2048)
      hipLaunchKernelGGL((lp_bwd_kernel<DT, 1>), dim3((unsigned)((n + 3) / 4)), dim3(kNT), 0, st, a);
    else
      hipLaunchKernelGGL((lp_bwd_kernel<DT, 4>), dim3((unsigned)(n * a.splits)), dim3(kNT), 0, st,
                         a);
    ZK_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

// Workspace bytes of zk_token_logprobs_fwd (0: none).
ZK_EXPORT long long zk_token_logprobs_ws_bytes(long long rows, int V, int k) {
  if (rows < 1 || V < 1 || k < 0 || k > kMaxTop) return 0;
  const long long s = fwd_splits(rows, V);
  return s > 1 ? rows * s * (16 + 8LL * k) : 0;
}

// x [rows][xs] logits, tokens [rows] int64 -> logp, entropy [rows] fp32; with
// k > 0 top_logp [rows][k] fp32 and top_ids [rows][k] int64; stats [rows][3]
// fp32 for the backward, or null.  dt: 0 fp32, 1 bf16, 2 fp16.
ZK_EXPORT int zk_token_logprobs_fwd(const void* x, const void* tokens, void* logp, void* entropy,
                                    void* stats, void* top_logp, void* top_ids, void* ws,
                                    long long ws_bytes, long long rows, int V, long long xs, int k,
                                    long long ignore, int dt, hipStream_t st) {
  if (rows < 0 || V < 1 || V >= 0x7fff0000 || xs < 0 || k < 0 || k > kMaxTop || k > V || dt < 0 ||
      dt > 2)
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  if (k > 0 && (!top_logp || !top_ids)) return (int)hipErrorInvalidValue;
  const int splits = fwd_splits(rows, V);
  const long long need = zk_token_logprobs_ws_bytes(rows, V, k);
  if (need > 0 && (!ws || ws_bytes < need)) return (int)hipErrorInvalidValue;
  LpArgs a{};
  a.x = x;
  a.tokens = (const long long*)tokens;
  a.logp = (float*)logp;
  a.entropy = (float*)entropy;
  a.stats = (float*)stats;
  a.top_logp = (float*)top_logp;
  a.top_ids = (long long*)top_ids;
  a.pkeys = (u64*)ws;  // keys first: 8-byte aligned
  a.pstat = (float*)((char*)ws + rows * splits * 8LL * k);
  a.rows = rows;
  a.xs = xs;
  a.ignore = ignore;
  a.V = V;
  a.k = k;
  a.splits = splits;
  a.chunk = splits > 1 ? (int)((((long long)V + splits - 1) / splits + 2047) / 2048 * 2048) : V;
#define ZK_LP(T) return k > 0 ? lp_fwd<T, true>(a, st) : lp_fwd<T, false>(a, st)
  if (dt == 0) ZK_LP(0);
  if (dt == 1) ZK_LP(1);
  ZK_LP(2);
#undef ZK_LP
}

// dx [rows][V] from the forward's stats; g_logp / g_entropy [rows] fp32, either
// may be null (no gradient from it).
ZK_EXPORT int zk_token_logprobs_bwd(const void* x, const void* tokens, const void* stats,
                                    const void* g_logp, const void* g_entropy, void* dx,
                                    long long rows, int V, long long xs, long long ignore, int dt,
                                    hipStream_t st) {
  if (rows < 0 || V < 1 || V >= 0x7fff0000 || xs < 0 || dt < 0 || dt > 2)
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  LpArgs a{};
  a.x = x;
  a.tokens = (const long long*)tokens;
  a.stats = (float*)const_cast<void*>(stats);
  a.g_logp = (const float*)g_logp;
  a.g_entropy = (const float*)g_entropy;
  a.dx = dx;
  a.rows = rows;
  a.xs = xs;
  a.ignore = ignore;
  a.V = V;
  a.chunk = V <= 2048 ? V : 8192;
  a.splits = (int)(((long long)V + a.chunk - 1) / a.chunk);
  if (dt == 0) return lp_bwd<0>(a, st);
  if (dt == 1) return lp_bwd<1>(a, st);
  return lp_bwd<2>(a, st);
}
