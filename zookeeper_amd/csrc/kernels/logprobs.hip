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
// writes dx.  Both are bound by memory (8192 x 131072 bf16: 0.38 and 0.76 ms back to back
// with themselves, 5.6 TB/s);
// few rows are split over blocks, at least 2048 elements each (each split writes its
// (m, s, q) and its waves' sorted k keys, a second launch joins them: 1 x 129000 bf16
// 5.6 us, 12 with k = 20).  Rows of up to 2048 elements take a wave each, four to a
// block, without LDS joins (1536 x 1000 fp32: 4 us, 7 with k = 5).
//
// Differences x - m are formed before the scaling to base 2, so the error of
// e^(x - m) does not grow with |m|; m and ln s are kept apart for the backward
// for the same reason.
//
// Top k: a wave holds its k best keys sorted, one per lane.  A key is the
// order-preserving image of the value with the complement of the place under
// it, so equal values rank by the lower place and no two keys are equal.
// A tile of 512 elements is passed over when its lanes' maxima (which the running
// statistics need anyway) stay at or under the k-th value.  Else its greater values
// are collected in LDS, up to 64, and merged by rank: a key's place is the number of
// greater ones.  When a tile has more candidates than the buffer takes, the k-th
// largest of its lane maxima (a binary search with ballots) raises the threshold
// first, so a rising row costs a merge per tile and not one per element.
//
// Joining lists (of the waves of a block, of the splits of a row): with j = ceil(k /
// lists), the ceil(k / j)-th largest of the lists' j-th keys has at least k keys at or
// above it; only those are merged, some 1.5 k of a list each times k.  (Merging list
// by list instead took 30 of the 36 us of one row of 129000 with k = 20.)
//
// Rows: all -inf -> logp -inf, entropy 0, gradient 0.  A NaN or +inf -> NaN.
// The ignored index: logp 0 and no gradient from it.  Any other token outside
// [0, V): logp NaN, and a NaN gradient row if logp has a gradient.
#include "rows.h"

namespace {

typedef unsigned long long u64;

constexpr int kNT = 256;
constexpr float kL2E = 1.44269504088896340736f;
constexpr float kLow = -1e4f;  // for differences where e^d is 0: finite times 0 is 0
constexpr int kMaxSplits = 64;
constexpr int kMaxTop = 64;

__device__ __forceinline__ float exp_d(float d) { return __builtin_amdgcn_exp2f(d * kL2E); }

// ---- running softmax statistics -------------------------------------------
struct Stat {
  float m, s, q;
};

// the greatest of 8; NaN if one is
__device__ __forceinline__ float max8(const float (&x)[8]) {
  float v = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) v = __builtin_elementwise_maximum(v, x[i]);
  return v;
}

// v: max8(x).  A NaN reaches s through its own term, so m may drop it.
__device__ __forceinline__ void stat_add8(Stat& a, const float (&x)[8], float v) {
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
  float thr;  // ... as a value; NaN while anything may enter
  int fill;   // keys waiting in buf (wave-uniform)
  int k;
  u64* buf;   // LDS: 64 waiting keys
  u64* lst;   // LDS: 64 slots of the merge
};

__device__ __forceinline__ Top top_new(int k, u64* lds) {
  return Top{0, 0, NAN, 0, k, lds, lds + 64};
}

__device__ __forceinline__ void top_raise(Top& t, u64 least) {
  if (least > t.least) {
    t.least = least;
    t.thr = value_of((uint32_t)(least >> 32));
  }
}

// Merge the n keys in buf (any order) into the sorted list.
__device__ __forceinline__ void top_merge(Top& t, int n) {
  typedef u64 u64x2 __attribute__((ext_vector_type(2)));
  const int lane = threadIdx.x & 63;
  if (lane >= n) t.buf[lane] = 0;
  t.lst[lane] = t.best;
  wave_fence();
  const u64 b = t.buf[lane];
  int rl = lane, rb = 0;  // the list is sorted: its own greater keys are the lanes below
  for (int i = 0; i < n; i += 4) {
    const u64x2 p = *reinterpret_cast<const u64x2*>(t.buf + i);
    const u64x2 q = *reinterpret_cast<const u64x2*>(t.buf + i + 2);
    rl += (p[0] > t.best) + (p[1] > t.best) + (q[0] > t.best) + (q[1] > t.best);
    rb += (p[0] > b) + (p[1] > b) + (q[0] > b) + (q[1] > b);
  }
  if (lane64(t.best, 0) != 0) {
    for (int i = 0; i < t.k; i += 4) {  // behind k: zeros
      const u64x2 p = *reinterpret_cast<const u64x2*>(t.lst + i);
      const u64x2 q = *reinterpret_cast<const u64x2*>(t.lst + i + 2);
      rb += (p[0] > b) + (p[1] > b) + (q[0] > b) + (q[1] > b);
    }
  }
  wave_fence();
  t.lst[lane] = 0;
  wave_fence();
  if (t.best != 0 && rl < t.k) t.lst[rl] = t.best;
  if (b != 0 && rb < t.k) t.lst[rb] = b;
  wave_fence();
  t.best = t.lst[lane];
  wave_fence();
  top_raise(t, lane64(t.best, t.k - 1));
}

__device__ __forceinline__ void top_flush(Top& t) {
  if (t.fill == 0) return;
  wave_fence();
  top_merge(t, t.fill);
  t.fill = 0;
}

// One key per lane (0: none) into the waiting ones.
__device__ __forceinline__ void top_push(Top& t, u64 key) {
  u64 in = __ballot(key > t.least);
  if (in == 0) return;
  if (t.fill + __popcll(in) > 64) {
    top_flush(t);
    in = __ballot(key > t.least);
  }
  const int at = t.fill + __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32),
                                                    __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
  if (key > t.least) t.buf[at] = key;
  t.fill += __popcll(in);
}

// Eight elements per lane, places base .. base + n - 1, v = max8 of them; places
// rise from tile to tile of a wave, so a value equal to the list's last never enters
// later.
__device__ __forceinline__ void top_add8(Top& t, const float (&x)[8], float v, int base, int n) {
  if (__ballot(!(v <= t.thr)) == 0) return;
  uint32_t o[8], top = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o[j] = j < n ? order_of(x[j]) : 0u;
    top = o[j] > top ? o[j] : top;
  }
  // many lanes with a candidate: at least k values of this tile are >= the k-th
  // largest lane maximum
  if (__popcll(__ballot(top > (uint32_t)(t.least >> 32))) > 24) {
    uint32_t kth = 0;
    for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
      if (__popcll(__ballot(top >= (kth | bit))) >= t.k) kth |= bit;
    if (kth > 0) top_raise(t, ((u64)(kth - 1) << 32) | 0xffffffffull);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)
    top_push(t, o[j] ? ((u64)o[j] << 32) | (uint32_t)~(uint32_t)(base + j) : 0);
  // a merge lowers the number of later tiles that get here
  if (t.fill >= 16 || t.fill >= t.k) top_flush(t);
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
  u64* pkeys;               // [rows][splits * 4][k]: a list per wave
  const float* g_logp;      // backward: [rows] or null
  const float* g_entropy;   // [rows] or null
  void* dx;                 // [rows][V]
  long long rows, row0, xs, ignore;
  int V, k, splits, chunk;
};

// The last of 64 splits, each rounded up to 2048, may reach past 2^31 - 1.
__device__ __forceinline__ int split_end(const LpArgs& a, int lo) {
  return a.V - lo < a.chunk ? a.V : lo + a.chunk;
}

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

// WPR waves per row and split: 1 (four rows per block) or 4 (the block).  Eight waves
// per SIMD: with the 110 registers that the filter would take, 4095 x 50001, k = 5
// ran 160 us instead of 124.
template <int DT, bool TOP, int WPR>
__global__ __launch_bounds__(kNT, 8) void lp_fwd_kernel(LpArgs a) {
  typedef typename Elem<DT>::raw raw;
  __shared__ __attribute__((aligned(16))) u64 lds[TOP ? 4 * 128 : 1];
  __shared__ u64 keys[TOP && WPR == 4 ? 4 * 64 : 1];
  __shared__ Stat joined[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const long long unit = WPR == 1 ? (long long)blockIdx.x * 4 + wave : blockIdx.x;
  const long long row = a.row0 + (WPR == 1 ? unit : unit / a.splits);
  if (row >= a.rows) return;  // WPR = 1 only (no barrier below), or past the last row as a block
  const int split = WPR == 1 ? 0 : (int)(unit % a.splits);
  const int lo = split * a.chunk, hi = split_end(a, lo);
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  Stat st{-INFINITY, 0.f, 0.f};
  Top top = top_new(a.k, lds + (TOP ? wave * 128 : 0));
  const int w = WPR == 1 ? 0 : wave;
  int c0 = lo + w * 512;
  Raw8<DT> next = raw8<DT>(x + c0 + lane * 8, hi - c0 - lane * 8);
  for (; c0 < hi; c0 += WPR * 512) {  // wave-uniform
    const int c = c0 + lane * 8, cn = c + WPR * 512;
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = raw_at<DT>(next, i);
    next = raw8<DT>(x + cn, hi - cn);
    if (hi - c < 8) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i >= hi - c) f[i] = -INFINITY;
    }
    const float v = max8(f);
    stat_add8(st, f, v);
    if constexpr (TOP) top_add8(top, f, v, c, hi - c);
  }
  st = stat_wave(st);
  if constexpr (TOP) top_flush(top);
  if constexpr (WPR == 4) {
    if (lane == 0) joined[wave] = st;
    if constexpr (TOP) {
      if (a.splits > 1) {
        if (lane < a.k)
          a.pkeys[((row * a.splits + split) * 4 + wave) * a.k + lane] = top.best;
      } else {
        keys[wave * 64 + lane] = top.best;
      }
    }
    __syncthreads();
    if (wave != 0) return;
    st = stat_join(stat_join(joined[0], joined[1]), stat_join(joined[2], joined[3]));
    if (a.splits > 1) {
      if (lane == 0) {
        float* p = a.pstat + (row * a.splits + split) * 4;
        p[0] = st.m;
        p[1] = st.s;
        p[2] = st.q;
      }
      return;
    }
    if constexpr (TOP) {
      // the least of the four lists' ceil(k / 4)-th keys has k keys at or above it
      const int j = (a.k + 3) / 4 - 1;
      u64 t = keys[j];
#pragma unroll
      for (int o = 1; o < 4; ++o) t = keys[o * 64 + j] < t ? keys[o * 64 + j] : t;
      if (t > 0) top_raise(top, t - 1);
#pragma unroll 1
      for (int o = 1; o < 4; ++o) top_push(top, keys[o * 64 + lane]);
      top_flush(top);
    }
  }
  float ls = 0.f;
  if (lane == 0) ls = lp_finish<DT>(a, row, st);
  if constexpr (TOP) top_write(a, row, top.best, __shfl(st.m, 0, 64), __shfl(ls, 0, 64));
}

// Joins the splits of a row: statistics in one wave; keys of up to 256 lists.
constexpr int kJoinNT = 1024;
template <int DT, bool TOP>
__global__ __launch_bounds__(TOP ? kJoinNT : 64) void lp_join_kernel(LpArgs a) {
  constexpr int MAXC = kMaxTop * kMaxTop;  // keys that can be at or above the threshold
  __shared__ __attribute__((aligned(16))) u64 lds[TOP ? 128 : 1];
  __shared__ u64 cand[TOP ? MAXC : 1];
  __shared__ u64 bound;
  __shared__ int count;
  const int lane = threadIdx.x & 63;
  const long long row = a.row0 + blockIdx.x;
  const int lists = a.splits * 4;
  if constexpr (TOP) {
    // this thread's share of the keys: in flight while the threshold is searched
    const u64* src = a.pkeys + row * lists * a.k;
    const int total = lists * a.k;
    u64 mine[kMaxSplits * 4 * kMaxTop / kJoinNT];
    constexpr int MINE = sizeof(mine) / 8;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int at = i * kJoinNT + (int)threadIdx.x;
      mine[i] = at < total ? src[at] : 0;
    }
    if (threadIdx.x < 64) {
      const int j = (a.k + lists - 1) / lists, need = (a.k + j - 1) / j;
      u64 head[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int l = i * 64 + lane;
        head[i] = l < lists ? src[l * a.k + j - 1] : 0;
      }
      // the need-th largest: by value, and where equal values leave more, by place
      uint32_t hi = 0;
      int n = 0, above = 0;
      for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
        n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          n += __popcll(__ballot((uint32_t)(head[i] >> 32) >= (hi | bit)));
        if (n >= need) hi |= bit, above = n;
      }
      u64 t = (u64)hi << 32;
      if (hi != 0 && above > need) {
        for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
          n = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) n += __popcll(__ballot(head[i] >= (t | bit)));
          if (n >= need) t |= bit;
        }
      }
      if (lane == 0) {
        bound = t;  // 0: lists that are not full
        count = 0;
      }
    }
    __syncthreads();
    const u64 t = bound > 0 ? bound : 1;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (mine[i] >= t) {
        const int at = atomicAdd(&count, 1);  // any order: the merge sorts
        if (at < MAXC) cand[at] = mine[i];
      }
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
  }
  Top top = top_new(a.k, lds);
  if constexpr (TOP) {
    const int n = min(count, MAXC);
    for (int i = 0; i < n; i += 64) top_push(top, i + lane < n ? cand[i + lane] : 0);
    top_flush(top);
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
  const int lo = split * a.chunk, hi = split_end(a, lo);
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  raw* dx = reinterpret_cast<raw*>(a.dx) + row * a.V;
  const float m = a.stats[row * 3], ls = a.stats[row * 3 + 1], h = a.stats[row * 3 + 2];
  const long long tok = a.tokens[row];
  float gl = a.g_logp ? a.g_logp[row] : 0.f;
  const float gh = a.g_entropy ? a.g_entropy[row] : 0.f;
  const bool in = tok >= 0 && tok < a.V;
  if (tok == a.ignore) gl = 0.f;
  else if (!in && a.g_logp) gl = NAN;
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
        hipLaunchKernelGGL((lp_join_kernel<DT, TOP>), dim3((unsigned)n), dim3(TOP ? kJoinNT : 64),
                           0,
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
      hipLaunchKernelGGL((lp_bwd_kernel<DT, 1>), dim3((unsigned)((n + 3) / 4)), dim3(kNT), 0, st,
                         a);
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
  return s > 1 ? rows * s * (16 + 4 * 8LL * k) : 0;
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
  a.pstat = (float*)((char*)ws + rows * splits * 4 * 8LL * k);
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
