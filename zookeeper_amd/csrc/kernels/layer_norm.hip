// Layer normalisation over the last dimension, forward and backward, for
// fp32 / bf16 / fp16 rows with fp32 weight and bias.
//
//   forward   mean = sum x / D,  var = sum (x - mean)^2 / D,
//             rstd = 1 / sqrt(var + eps),  xhat = (x - mean) * rstd,
//             y = xhat * w + b
//   backward  g = dy * w,
//             dx = rstd * (g - sum(g) / D - xhat * sum(g * xhat) / D),
//             dw = sum_rows dy * xhat,  db = sum_rows dy
//
// All arithmetic is fp32; the variance is centred (a second pass over the
// registers, no E[x^2] - mean^2).  Both passes are bound by memory: forward
// x + y, backward x + dy + dx, everything else stays in registers.  A row
// belongs to G lanes that hold it whole: NV vectors of 8 elements per lane.
// Measured, 32768 x 2048 bf16: forward 52 us (5.1 TB/s), backward 84 us (4.8 TB/s, of
// which 5 us for the join of dw / db); 4096 x 16384 51 and 92 us; 1000000 x 16 fp32 23
// and 37 us; a device copy runs at 5.2 TB/s.
//
// Rows over 16384 elements take the looping kernels: three sweeps of x forward, three
// of x and dy backward, which the L2s hold in part only.  4096 x 32768 bf16 180 and 372 us
// (3.0 and 2.2 TB/s of x + y and x + dy + dx), fp32 394 and 661 us; 512 x 65536 bf16 55
// and 107 us.
//
// dw / db: blocks walk rows with a fixed stride and keep their columns' sums in
// registers; the lane groups of a block are joined through LDS, each block
// writes one partial row pair, and a second launch adds the partials in block
// order.  No atomics: the result depends on the sizes alone.
#include "rows.h"

namespace {

constexpr int kNT = 256;       // threads per block (rows of G > 256 lanes: G)
constexpr int kMaxD = 16384;   // widest row kept in registers

constexpr int block_of(int g) { return g > kNT ? g : kNT; }

struct LnArgs {
  const void* x;       // [rows][xs]
  const void* dy;      // [rows][dys] (backward)
  const float* w;      // [D] or null (ones)
  const float* b;      // [D] or null (zeros)
  void* out;           // y / dx, [rows][D]; dx may be null (only dw / db wanted)
  float* mean;         // [rows] (forward: may be null)
  float* rstd;
  float* part;         // backward: [blocks][2][D] partials, or null (no dw / db)
  long long rows, xs, dys, row0;  // row0: first row of this launch
  int D;
  float eps;
};

// Sums over the G lanes of a row: groups inside a wave, or a block of G / 64 waves
// (red: 2 * G / 64 floats that nobody reads any more).
template <int G>
__device__ __forceinline__ float row_sum(float v, float* red) {
  if constexpr (G <= 64) {
    return group_sum<G>(v);
  } else {
    v = group_sum<64>(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = red[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) s += red[i];
    return s;
  }
}

template <int G>
__device__ __forceinline__ void row_sum2(float& a, float& b, float* red) {
  if constexpr (G <= 64) {
    a = group_sum<G>(a);
    b = group_sum<G>(b);
  } else {
    constexpr int W = G / 64;
    a = group_sum<64>(a);
    b = group_sum<64>(b);
    if ((threadIdx.x & 63) == 0) {
      red[threadIdx.x >> 6] = a;
      red[W + (threadIdx.x >> 6)] = b;
    }
    __syncthreads();
    a = red[0];
    b = red[W];
#pragma unroll
    for (int i = 1; i < W; ++i) {
      a += red[i];
      b += red[W + i];
    }
  }
}

__device__ __forceinline__ void load_param(const float* p, int c, int n, float fill,
                                           float (&f)[8]) {
  if (p) {
    load8_n<0>(p + c, n, fill, f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fill;
  }
}

template <int DT, int G, int NV>
__global__ __launch_bounds__(block_of(G)) void ln_fwd_kernel(LnArgs a) {
  typedef typename Elem<DT>::raw raw;
  __shared__ float red[2][16];
  const int l = threadIdx.x % G;
  const long long row = a.row0 + (long long)blockIdx.x * (block_of(G) / G) + threadIdx.x / G;
  if (row >= a.rows) return;  // G >= 256: never (one row per block)
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  raw* y = reinterpret_cast<raw*>(a.out) + row * a.D;
  float v[NV][8];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * G + l) * 8;
    load8_n<DT>(x + c, a.D - c, 0.f, v[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[k][i];
  }
  const float invd = 1.f / (float)a.D;
  const float mean = row_sum<G>(s, red[0]) * invd;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int n = a.D - (k * G + l) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[k][i] -= mean;
      if (i < n) q += v[k][i] * v[k][i];
    }
  }
  const float rstd = rsqrtf(row_sum<G>(q, red[1]) * invd + a.eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * G + l) * 8, n = a.D - c;
    if (n > 0) {
      float w[8], b[8];
      load_param(a.w, c, n, 1.f, w);
      load_param(a.b, c, n, 0.f, b);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * rstd * w[i] + b[i];
      store8_n<DT>(y + c, n, v[k]);
    }
  }
  if (a.mean && l == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// Any row length: the row is read three times (mean, variance, output).
template <int DT>
__global__ __launch_bounds__(kNT) void ln_fwd_loop_kernel(LnArgs a) {
  typedef typename Elem<DT>::raw raw;
  __shared__ float red[2][16];
  const long long row = a.row0 + blockIdx.x;
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  raw* y = reinterpret_cast<raw*>(a.out) + row * a.D;
  const float invd = 1.f / (float)a.D;
  float f[8], s = 0.f, q = 0.f;
  for (long long c = threadIdx.x * 8; c < a.D; c += kNT * 8) {
    load8_n<DT>(x + c, (int)min(8LL, a.D - c), 0.f, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) s += f[i];
  }
  const float mean = row_sum<kNT>(s, red[0]) * invd;
  for (long long c = threadIdx.x * 8; c < a.D; c += kNT * 8) {
    load8_n<DT>(x + c, (int)min(8LL, a.D - c), mean, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) q += (f[i] - mean) * (f[i] - mean);
  }
  const float rstd = rsqrtf(row_sum<kNT>(q, red[1]) * invd + a.eps);
  for (long long c = threadIdx.x * 8; c < a.D; c += kNT * 8) {
    const int n = (int)min(8LL, a.D - c);
    float w[8], b[8];
    load8_n<DT>(x + c, n, 0.f, f);
    load_param(a.w, (int)c, n, 1.f, w);
    load_param(a.b, (int)c, n, 0.f, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (f[i] - mean) * rstd * w[i] + b[i];
    store8_n<DT>(y + c, n, f);
  }
  if (a.mean && threadIdx.x == 0) {
    a.mean[row] = mean;
    a.rstd[row] = rstd;
  }
}

// Blocks walk the rows; a lane group keeps the sums of its columns.  The next row's
// loads are in flight while a row is reduced and written (without them bf16 rows
// ran at 3.1 TB/s: too few bytes in flight, 32768 x 2048 112 us).
template <int DT, int G, int NV>
__global__ __launch_bounds__(block_of(G)) void ln_bwd_kernel(LnArgs a) {
  typedef typename Elem<DT>::raw raw;
  constexpr int NT = block_of(G), RPB = NT / G;  // RPB: rows of a block at a time
  constexpr bool AHEAD = G < 1024;  // 16 waves leave 128 registers each: none to spare
  __shared__ float red[2][32];
  const int l = threadIdx.x % G, grp = threadIdx.x / G;
  const float invd = 1.f / (float)a.D;
  float w[NV][8], dw[NV][8], db[NV][8];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * G + l) * 8;
    load_param(a.w, c, a.D - c, 1.f, w[k]);
#pragma unroll
    for (int i = 0; i < 8; ++i) dw[k][i] = db[k][i] = 0.f;
  }
  const long long stride = (long long)gridDim.x * RPB;
  long long row = (long long)blockIdx.x * RPB + grp;
  Raw8<DT> nx[NV], ny[NV];
  float nm = 0.f, nr = 0.f;
  auto load = [&](long long r) {
    const raw* x = reinterpret_cast<const raw*>(a.x) + r * a.xs;
    const raw* dy = reinterpret_cast<const raw*>(a.dy) + r * a.dys;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * G + l) * 8;
      nx[k] = raw8<DT>(x + c, a.D - c);
      ny[k] = raw8<DT>(dy + c, a.D - c);  // zeros behind D
    }
    nm = a.mean[r];
    nr = a.rstd[r];
  };
  if (AHEAD && row < a.rows) load(row);
  // G > 64: the trip count is the same for the whole block (row_sum2's barrier; its
  // buffers alternate, so one barrier per row is enough)
  for (int it = 0; row < a.rows; row += stride, it ^= 1) {
    if (!AHEAD) load(row);
    float xh[NV][8], g[NV][8];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        xh[k][i] = raw_at<DT>(nx[k], i);
        g[k][i] = raw_at<DT>(ny[k], i);
      }
    const float mean = nm, rstd = nr;
    // behind D: xhat 0 (a zero's own could overflow, and 0 * inf reach the sums)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int n = a.D - (k * G + l) * 8;
      if (n < 8)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i >= n) xh[k][i] = mean;
    }
    if (AHEAD && row + stride < a.rows) load(row + stride);
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float h = (xh[k][i] - mean) * rstd, d = g[k][i];
        dw[k][i] += d * h;
        db[k][i] += d;
        const float gw = d * w[k][i];
        s1 += gw;
        s2 += gw * h;
        xh[k][i] = h;
        g[k][i] = gw;
      }
    if (a.out) {
      row_sum2<G>(s1, s2, red[it]);
      s1 *= invd;
      s2 *= invd;
      raw* dx = reinterpret_cast<raw*>(a.out) + row * a.D;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * G + l) * 8, n = a.D - c;
#pragma unroll
        for (int i = 0; i < 8; ++i) g[k][i] = rstd * (g[k][i] - s1 - xh[k][i] * s2);
        if (n > 0) store8_n<DT>(dx + c, n, g[k]);
      }
    }
  }
  if (!a.part) return;
  // join the lane groups of a wave, then the waves (through LDS, wave order)
  if constexpr (G < 64) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int off = G; off < 64; off <<= 1) {
          dw[k][i] += __shfl_xor(dw[k][i], off, 64);
          db[k][i] += __shfl_xor(db[k][i], off, 64);
        }
      }
  }
  float* pw = a.part + (long long)blockIdx.x * 2 * a.D;
  float* pb = pw + a.D;
  if constexpr (G <= 64) {
    __shared__ float joined[3][2][G * 8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      __syncthreads();
      if (wave > 0 && lane < G)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          joined[wave - 1][0][i * G + lane] = dw[k][i];
          joined[wave - 1][1][i * G + lane] = db[k][i];
        }
      __syncthreads();
      if (wave == 0 && lane < G) {
        const int c = (k * G + lane) * 8, n = a.D - c;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
          for (int o = 0; o < 3; ++o) {
            dw[k][i] += joined[o][0][i * G + lane];
            db[k][i] += joined[o][1][i * G + lane];
          }
        }
        if (n > 0) {
          store8_n<0>(pw + c, n, dw[k]);
          store8_n<0>(pb + c, n, db[k]);
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * G + l) * 8, n = a.D - c;
      if (n > 0) {
        store8_n<0>(pw + c, n, dw[k]);
        store8_n<0>(pb + c, n, db[k]);
      }
    }
  }
}

// Any row length, dx only: two sweeps of the row.
template <int DT>
__global__ __launch_bounds__(kNT) void ln_bwd_loop_kernel(LnArgs a) {
  typedef typename Elem<DT>::raw raw;
  __shared__ float red[8];
  const long long row = a.row0 + blockIdx.x;
  const raw* x = reinterpret_cast<const raw*>(a.x) + row * a.xs;
  const raw* dy = reinterpret_cast<const raw*>(a.dy) + row * a.dys;
  raw* dx = reinterpret_cast<raw*>(a.out) + row * a.D;
  const float invd = 1.f / (float)a.D, mean = a.mean[row], rstd = a.rstd[row];
  float xv[8], g[8], w[8], s1 = 0.f, s2 = 0.f;
  for (long long c = threadIdx.x * 8; c < a.D; c += kNT * 8) {
    const int n = (int)min(8LL, a.D - c);
    load8_n<DT>(x + c, n, mean, xv);
    load8_n<DT>(dy + c, n, 0.f, g);
    load_param(a.w, (int)c, n, 1.f, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float gw = g[i] * w[i];
      s1 += gw;
      s2 += gw * ((xv[i] - mean) * rstd);
    }
  }
  row_sum2<kNT>(s1, s2, red);
  s1 *= invd;
  s2 *= invd;
  for (long long c = threadIdx.x * 8; c < a.D; c += kNT * 8) {
    const int n = (int)min(8LL, a.D - c);
    load8_n<DT>(x + c, n, mean, xv);
    load8_n<DT>(dy + c, n, 0.f, g);
    load_param(a.w, (int)c, n, 1.f, w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      g[i] = rstd * (g[i] * w[i] - s1 - (xv[i] - mean) * rstd * s2);
    store8_n<DT>(dx + c, n, g);
  }
}

// Any row length, dw / db partials: block (cx, p) owns 2048 columns and every
// gridDim.y-th row from p.
template <int DT>
__global__ __launch_bounds__(kNT) void ln_cols_kernel(LnArgs a) {
  typedef typename Elem<DT>::raw raw;
  const long long c = ((long long)blockIdx.x * kNT + threadIdx.x) * 8;
  if (c >= a.D) return;
  const int n = (int)min(8LL, a.D - c);
  float dw[8], db[8], xv[8], g[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) dw[i] = db[i] = 0.f;
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float mean = a.mean[row], rstd = a.rstd[row];
    load8_n<DT>(reinterpret_cast<const raw*>(a.x) + row * a.xs + c, n, mean, xv);
    load8_n<DT>(reinterpret_cast<const raw*>(a.dy) + row * a.dys + c, n, 0.f, g);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      dw[i] += g[i] * ((xv[i] - mean) * rstd);
      db[i] += g[i];
    }
  }
  float* pw = a.part + (long long)blockIdx.y * 2 * a.D;
  store8_n<0>(pw + c, n, dw);
  store8_n<0>(pw + a.D + c, n, db);
}

// out[c] (+)= sum over p of part[p][c], c < n2 = 2 D (dw then db); 16 slices of
// the partials in parallel, each in order, joined in order.
__global__ __launch_bounds__(1024) void ln_part_sum_kernel(const float* __restrict__ part,
                                                           int parts, int D, float* dw, float* db,
                                                           int add) {
  __shared__ float red[16][64];
  const int col = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const long long n2 = 2LL * D;
  const long long c = (long long)blockIdx.x * 64 + col;
  float s = 0.f;
  if (c < n2) {
    const float* p = part + sl * n2 + c;
    int k = sl;
    for (; k + 112 < parts; k += 128, p += 128 * n2) {  // eight loads in flight
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = p[16 * i * n2];
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[i];
    }
    for (; k < parts; k += 16, p += 16 * n2) s += *p;
  }
  red[sl][col] = s;
  __syncthreads();
  if (sl == 0 && c < n2) {
#pragma unroll
    for (int o = 1; o < 16; ++o) s += red[o][col];
    float* out = c < D ? dw : db;
    if (out) {
      const long long i = c < D ? c : c - D;
      out[i] = (add & (c < D ? 1 : 2)) ? out[i] + s : s;
    }
  }
}

// Lanes and vectors of a row by its length: at most two vectors per lane (the
// backward holds 40 registers for each), few idle lanes.
#define ZK_LN_SHAPES(D, RUN)      \
  do {                            \
    if ((D) <= 8) RUN(1, 1);      \
    else if ((D) <= 16) RUN(2, 1);   \
    else if ((D) <= 32) RUN(4, 1);   \
    else if ((D) <= 64) RUN(8, 1);   \
    else if ((D) <= 128) RUN(16, 1); \
    else if ((D) <= 256) RUN(32, 1); \
    else if ((D) <= 512) RUN(64, 1); \
    else if ((D) <= 1024) RUN(64, 2);   \
    else if ((D) <= 2048) RUN(256, 1);  \
    else if ((D) <= 4096) RUN(256, 2);  \
    else if ((D) <= 8192) RUN(512, 2);  \
    else RUN(1024, 2);               \
  } while (0)

// Blocks of the backward: as many as the chip holds at a time, but each lane group
// has at least four rows (its partial sums are two fp32 rows to write and read
// again), if that leaves 64 blocks.
int bwd_blocks(long long rows, int D) {
  long long rpb = 1, cap = 1024;
#define ZK_LN_RPB(G, NV)            \
  do {                              \
    rpb = block_of(G) / G;          \
    cap = 1024 / (block_of(G) / kNT); \
  } while (0)
  ZK_LN_SHAPES(D, ZK_LN_RPB);
#undef ZK_LN_RPB
  const long long all = (rows + rpb - 1) / rpb;
  long long nb = rows / (4 * rpb);
  if (nb < 64) nb = 64;
  if (nb > cap) nb = cap;
  return (int)(nb < all ? nb : all);
}

int loop_parts(long long rows) { return (int)(rows < 64 ? rows : 64); }

// Rows of one launch of the kernels that give a row to a block: a grid holds
// fewer than 2^32 threads.
constexpr long long kRowsPerLaunch = 1LL << 21;

template <int DT>
int fwd_dispatch(LnArgs a, hipStream_t st) {
  for (a.row0 = 0; a.row0 < a.rows; a.row0 += kRowsPerLaunch) {
    const long long left = a.rows - a.row0;
    const unsigned r = (unsigned)(left < kRowsPerLaunch ? left : kRowsPerLaunch);
#define ZK_LN_FWD(G, NV)                                                                    \
  hipLaunchKernelGGL((ln_fwd_kernel<DT, G, NV>),                                            \
                     dim3((r + block_of(G) / G - 1) / (block_of(G) / G)), dim3(block_of(G)), \
                     0, st, a)
    if (a.D > kMaxD) hipLaunchKernelGGL(ln_fwd_loop_kernel<DT>, dim3(r), dim3(kNT), 0, st, a);
    else ZK_LN_SHAPES(a.D, ZK_LN_FWD);
#undef ZK_LN_FWD
    ZK_CHECK_LAUNCH();
  }
  return 0;
}

template <int DT>
int bwd_dispatch(const LnArgs& a, int blocks, hipStream_t st) {
#define ZK_LN_BWD(G, NV)                                                                     \
  hipLaunchKernelGGL((ln_bwd_kernel<DT, G, NV>), dim3(blocks), dim3(block_of(G)), 0, st, a)
  ZK_LN_SHAPES(a.D, ZK_LN_BWD);
#undef ZK_LN_BWD
  return (int)hipGetLastError();
}

}  // namespace

// x [rows][xs] (unit stride inside a row) -> y [rows][D]; mean / rstd [rows]
// fp32, or both null; w / b [D] fp32 or null; dt: 0 fp32, 1 bf16, 2 fp16.
ZK_EXPORT int zk_layer_norm_fwd(const void* x, const void* w, const void* b, void* y, void* mean,
                                void* rstd, long long rows, int D, long long xs, float eps,
                                int dt, hipStream_t st) {
  if (rows < 0 || D < 1 || xs < 0 || rows >= (1LL << 31) || dt < 0 || dt > 2)
    return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  LnArgs a{x, nullptr, (const float*)w, (const float*)b, y, (float*)mean, (float*)rstd, nullptr,
           rows, xs, 0, 0, D, eps};
  return dt == 0 ? fwd_dispatch<0>(a, st) : dt == 1 ? fwd_dispatch<1>(a, st)
                                                    : fwd_dispatch<2>(a, st);
}

// Bytes of the workspace of zk_layer_norm_bwd when dw or db is wanted.
ZK_EXPORT long long zk_layer_norm_bwd_ws_bytes(long long rows, int D) {
  if (rows < 1 || D < 1) return 0;
  const long long p = D <= kMaxD ? bwd_blocks(rows, D) : loop_parts(rows);
  return p * 2 * D * 4;
}

// dx [rows][D] (or null), dw / db [D] fp32 (or null).  add: bit 0 dw, bit 1
// db are accumulated into instead of written.
ZK_EXPORT int zk_layer_norm_bwd(const void* dy, const void* x, const void* w, const void* mean,
                                const void* rstd, void* dx, void* dw, void* db, void* ws,
                                long long ws_bytes, long long rows, int D, long long xs,
                                long long dys, int dt, int add, hipStream_t st) {
  if (rows < 1 || D < 1 || xs < 0 || dys < 0 || rows >= (1LL << 31) || dt < 0 || dt > 2)
    return (int)hipErrorInvalidValue;
  const bool cols = dw || db;
  if (cols && (!ws || ws_bytes < zk_layer_norm_bwd_ws_bytes(rows, D)))
    return (int)hipErrorInvalidValue;
  if (!cols && !dx) return 0;
  LnArgs a{x, dy, (const float*)w, nullptr, dx, (float*)const_cast<void*>(mean),
           (float*)const_cast<void*>(rstd), cols ? (float*)ws : nullptr, rows, xs, dys, 0, D, 0.f};
  int parts;
  if (D <= kMaxD) {
    parts = bwd_blocks(rows, D);
    const int e = dt == 0 ? bwd_dispatch<0>(a, parts, st)
                          : dt == 1 ? bwd_dispatch<1>(a, parts, st) : bwd_dispatch<2>(a, parts, st);
    if (e) return e;
  } else {
    parts = loop_parts(rows);
    const dim3 gc((unsigned)((D + kNT * 8LL - 1) / (kNT * 8LL)), (unsigned)parts);
#define ZK_LN_LOOP(T)                                                                         \
  do {                                                                                        \
    for (a.row0 = 0; dx && a.row0 < rows; a.row0 += kRowsPerLaunch) {                          \
      const long long left = rows - a.row0;                                                   \
      hipLaunchKernelGGL(ln_bwd_loop_kernel<T>,                                               \
                         dim3((unsigned)(left < kRowsPerLaunch ? left : kRowsPerLaunch)),     \
                         dim3(kNT), 0, st, a);                                                \
    }                                                                                         \
    if (cols) hipLaunchKernelGGL(ln_cols_kernel<T>, gc, dim3(kNT), 0, st, a);                  \
  } while (0)
    if (dt == 0) ZK_LN_LOOP(0);
    else if (dt == 1) ZK_LN_LOOP(1);
    else ZK_LN_LOOP(2);
#undef ZK_LN_LOOP
    ZK_CHECK_LAUNCH();
  }
  if (cols) {
    hipLaunchKernelGGL(ln_part_sum_kernel, dim3((unsigned)((2LL * D + 63) / 64)), dim3(1024), 0, st,
                       (const float*)ws, parts, D, (float*)dw, (float*)db, add);
    ZK_CHECK_LAUNCH();
  }
  return 0;
}
