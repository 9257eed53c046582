// Activations kept in 8 bits for the backward pass, and the passes that use
// them: pack / unpack, GELU forward and backward, weight and bias gradient of a
// dense layer.
//
// Form.  A row is cut into blocks of 32 values; a block has one scale byte E and
// a signed 8-bit code per value, value = code * 2^(E - 133) (the layout of the
// OCP MXINT8 format).  E - 127 = floor(log2(max |x|)), one more where the largest
// value would round to code 128 (so every value is within half a step; only E =
// 254 clamps), never under E = 7 (step 2^-126: the smallest normal).  A block
// that holds an infinity or a NaN has E = 255 and decodes to NaN.  E under 7, which
// pack does not write but a form from elsewhere may hold (zeroed memory, for one),
// decodes to its subnormal step; whole steps of that are exact in bf16 too.
//
// Why whole steps of a power of two and not e4m3: codes up to 127 and a sign are
// exact in bf16, so a decoded tile feeds the bf16 matrix instructions without a
// further rounding, and the error is 1 / 127.5 of the block's largest value at
// most where e4m3's is 2^-4 of each value.
//
// All elementwise kernels are bound by memory.  A lane owns 8 values, the four
// lanes of a quad a block: the block's maximum takes two DPP moves.  Measured, 16384 x
// 8192 bf16, each back to back with itself: pack 76 us, unpack 72 us (5.4 TB/s), GELU
// with its kept input 128 us, GELU backward 165 us (4.1 TB/s: its 31 instructions a value,
// two of them transcendental, take nearly as long; fp32 208 and 207 us, 5.8 TB/s).  The
// two passes of GELU in turn take 275 us.
#include <atomic>

#include "mfma_common.h"
#include "rows.h"

namespace {

typedef unsigned long long u64_t;

constexpr int kNT = 256;

// max over the quad of lanes that shares a 32-value block
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  const uint32_t a = __builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true);
  v = a > v ? a : v;
  const uint32_t b = __builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true);
  return b > v ? b : v;
}

__device__ __forceinline__ float step_of(uint32_t E) {  // 2^(E - 133); E = 255: NaN
  return E == 255u ? NAN : __uint_as_float(E < 7u ? 0x10000u << E : (E - 6u) << 23);
}

// The quad's block of 32: scale byte and this lane's 8 codes.
__device__ __forceinline__ uint32_t encode8(const float (&x)[8], uint32_t (&code)[2]) {
  float t = fabsf(x[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) t = __builtin_elementwise_maximum(t, fabsf(x[i]));  // keeps a NaN
  const uint32_t top = quad_max(__float_as_uint(t) & 0x7fffffffu);  // NaN > inf > numbers
  uint32_t E = top >> 23;
  if (E == 255u) {
    code[0] = code[1] = 0u;
    return 255u;
  }
  E = E < 7u ? 7u : E;
  // 1 / step = 2^(133 - E): products with it are exact
  const float most = __uint_as_float(top) * __uint_as_float((260u - E) << 23);
  if (__builtin_rintf(most) >= 128.f && E < 254u) ++E;
  const float inv = __uint_as_float((260u - E) << 23);
  uint32_t c[8];
  // adding 1.5 * 2^23 rounds to a whole number (ties to even) whose two's complement
  // is in the low byte; only at E = 254 can it be 128
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = __float_as_uint(__builtin_fmaf(x[i], inv, 12582912.f));
  if (E == 254u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      c[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[i] * inv, -127.f, 127.f) + 12582912.f);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {  // low bytes of four words: v_perm_b32
    const uint32_t lo = __builtin_amdgcn_perm(c[4 * i + 1], c[4 * i], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(c[4 * i + 3], c[4 * i + 2], 0x04000c0cu);
    code[i] = lo | hi;
  }
  return E;
}

__device__ __forceinline__ float code_at(uint32_t w, int i) {
  return (float)(int8_t)(uint8_t)(w >> (8 * i));
}

__device__ __forceinline__ void decode8(const uint32_t (&code)[2], uint32_t E, float (&x)[8]) {
  const float s = step_of(E);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = code_at(code[i >> 2], i & 3) * s;
}

// Phi(-|x|) = t P(t) e^(-x^2 / 2) with t = 1 / (1 + 0.305 |x|) and P of degree 7,
// fitted here to erfcx(|x| / sqrt 2) / 2 on [0, 14] (least squares, reweighted to
// an even relative error: 1e-7).  The exponential is the normal density's too.
__device__ __forceinline__ void normal_of(float x, float& cdf, float& e) {
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.305f, fabsf(x), 1.f));
  e = __builtin_amdgcn_exp2f(x * (x * -0.72134752044448170368f));
  float p = 0.036698496726864566f;
  p = __builtin_fmaf(p, t, -0.1529855293523711f);
  p = __builtin_fmaf(p, t, 0.18571227887536676f);
  p = __builtin_fmaf(p, t, -0.03797271523729383f);
  p = __builtin_fmaf(p, t, 0.1210195686418104f);
  p = __builtin_fmaf(p, t, 0.10342148895084405f);
  p = __builtin_fmaf(p, t, 0.12246671928545089f);
  p = __builtin_fmaf(p, t, 0.121639738931009f);
  const float q = p * t * e;
  cdf = x < 0.f ? q : 1.f - q;  // NaN: q is NaN
}

struct A8Args {
  const void* in;     // x (pack, gelu fwd) / dy (gelu bwd), [rows][is]
  void* out;          // y / dx / unpacked, [rows][D]
  int8_t* codes;      // [rows][D]
  uint8_t* scales;    // [rows][blocks]
  long long rows, D, is, nv, total;  // nv: 8-value vectors of a row, padded to whole blocks
};

enum { kPack = 0, kUnpack = 1, kGeluFwd = 2, kGeluKeep = 3, kGeluBwd = 4 };

template <int DT, int OP>
__global__ __launch_bounds__(kNT) void act8_kernel(A8Args a) {
  typedef typename Elem<DT>::raw raw;
  const long long step = (long long)gridDim.x * kNT;
  for (long long id = (long long)blockIdx.x * kNT + threadIdx.x; id < a.total; id += step) {
    long long row = 0, v = id;
    if (a.rows > 1) {  // uniform
      if (a.total < (1LL << 31)) {
        row = (uint32_t)id / (uint32_t)a.nv;
      } else {
        row = id / a.nv;
      }
      v = id - row * a.nv;
    }
    const long long c = v * 8;
    const int n = (int)(a.D - c < 8 ? a.D - c : 8);  // <= 0 behind the row's end
    const long long at = row * a.D + c;
    const long long sc = row * (a.nv >> 2) + (v >> 2);
    float x[8];
    if constexpr (OP != kUnpack) {
      load8_n<DT>(reinterpret_cast<const raw*>(a.in) + row * a.is + c, n, 0.f, x);
    }
    if constexpr (OP == kPack || OP == kGeluKeep) {
      uint32_t w[2];
      const uint32_t E = encode8(x, w);
      if (n >= 8) {
        Bytes8 b;
        b[0] = w[0];
        b[1] = w[1];
        *reinterpret_cast<Bytes8*>(a.codes + at) = b;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) a.codes[at + i] = (int8_t)(uint8_t)(w[i >> 2] >> (8 * (i & 3)));
      }
      if ((v & 3) == 0) a.scales[sc] = (uint8_t)E;
    }
    if constexpr (OP == kUnpack || OP == kGeluBwd) {
      uint32_t w[2] = {0u, 0u};
      if (n >= 8) {
        const Bytes8 b = *reinterpret_cast<const Bytes8*>(a.codes + at);
        w[0] = b[0];
        w[1] = b[1];
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < n) w[i >> 2] |= (uint32_t)(uint8_t)a.codes[at + i] << (8 * (i & 3));
      }
      float k[8];
      decode8(w, a.scales[sc], k);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if constexpr (OP == kUnpack) {
          x[i] = k[i];
        } else {
          float cdf, e;
          normal_of(k[i], cdf, e);
          x[i] *= cdf + k[i] * e * 0.39894228040143267794f;
        }
      }
    }
    if constexpr (OP == kGeluFwd || OP == kGeluKeep) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float cdf, e;
        normal_of(x[i], cdf, e);
        x[i] *= cdf;
      }
    }
    if constexpr (OP != kPack) {
      if (n > 0) store8_n<DT>(reinterpret_cast<raw*>(a.out) + at, n, x);
    }
  }
}

template <int OP>
int act8_launch(const void* in, void* out, void* codes, void* scales, long long rows,
                long long D, long long is, int dt, hipStream_t st) {
  if (rows < 0 || D < 1 || is < 0 || dt < 0 || dt > 2) return (int)hipErrorInvalidValue;
  if (rows == 0) return 0;
  // whole blocks and no gaps: one long row (no division)
  if (D % 32 == 0 && (is == D || rows == 1)) {
    D *= rows;
    is = D;
    rows = 1;
  }
  A8Args a{in, out, (int8_t*)codes, (uint8_t*)scales, rows, D, is, (D + 31) / 32 * 4, 0};
  a.total = rows * a.nv;
  long long blocks = (a.total + kNT - 1) / kNT;
  if (blocks > (1 << 20)) blocks = 1 << 20;
  const dim3 g((unsigned)blocks);
  if (dt == 0) hipLaunchKernelGGL((act8_kernel<0, OP>), g, dim3(kNT), 0, st, a);
  if (dt == 1) hipLaunchKernelGGL((act8_kernel<1, OP>), g, dim3(kNT), 0, st, a);
  if (dt == 2) hipLaunchKernelGGL((act8_kernel<2, OP>), g, dim3(kNT), 0, st, a);
  return (int)hipGetLastError();
}

// ===========================================================================
// Weight gradient of a dense layer from its kept input:
//   dW[n][k] = sum_m dy[m][n] x8[m][k],   db[n] = sum_m dy[m][n]
// A matrix product whose reduction runs over the rows of both operands.  A
// block owns a 128 x 128 tile of dW and walks 32 rows a step: dy and the decoded
// codes go through registers into LDS as [m][column] bf16 rows (256 B, swizzled
// by tr_swz so that the transposed reads have no bank conflicts), the fragments
// (8 consecutive m of a column) come from ds_read_b64_tr_b16.
//
// dy in fp16 / fp32 is cut into 2 / 3 bf16 terms by truncation (8 significant
// bits each: 11 and 24 bits are exact), one matrix product per term into the same
// accumulators; x8 is exact in bf16 and needs one.  So fp32 gradients keep fp32
// products at a third of the bf16 rate.
//
// db comes from the same fragments times a column of ones; the k-tiles of one
// n-tile share the rows' steps for it.
//
// Few tiles: the rows are split, every split writes its partial tile and a
// second launch adds them in order (no atomics).
//
// This kernel serves the smaller sizes (1024 x 1024 x 1024 bf16 26 us, 256 x 1024 x
// 1024 17 us: the start and end of a block and the partial sums); at large ones it is
// bound by its own staging (16384 x 4096 x 4096 1448 us, 0.38 PFLOP/s).
// ===========================================================================
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kT = 128;       // tile edge, n and k
constexpr int kMS = 32;       // rows a step
constexpr int kPlane = kMS * kT * 2;

struct D8Args {
  const void* dy;         // [M][dys]
  const int8_t* codes;    // [M][K]
  const uint8_t* scales;  // [M][kb]
  float* dw;              // [N][K]
  float* db;              // [N] or null
  float* slab;            // [splits][N][K] (several splits)
  float* part;            // [splits * ktiles][N]: db's parts
  long long dys;
  long long M;
  int N, K, kb, ntiles, ktiles, splits, add;
  long long mps;          // rows of a split (multiple of kMS)
};

__device__ __forceinline__ f32x4 mma16(const uint4& a, const uint4& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// 8 consecutive m of column c0 + (lane & 15) from a swizzled [m][RB / 2] bf16 plane:
// lane l: m = 8 (l >> 4) ..
template <int RB>
__device__ __forceinline__ uint4 col_frag(const unsigned char* plane, int c0, int lane) {
  const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
  const int r0 = 8 * g + q, r1 = r0 + 4;
  const int slot = (c0 >> 3) | (p >> 1), inner = (p & 1) * 8;
  const int o0 = r0 * RB + ((slot ^ tr_swz<RB>(r0)) << 4) + inner;
  const int o1 = r1 * RB + ((slot ^ tr_swz<RB>(r1)) << 4) + inner;
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_s16x4*)(uintptr_t)(const __attribute__((address_space(3))) void*)(plane + o0));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (lds_s16x4*)(uintptr_t)(const __attribute__((address_space(3))) void*)(plane + o1));
  const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(uint4, v);
}

// The first bf16 term of f (8 leading bits, never an overflow) and the exact rest;
// an infinity or NaN has no rest.
__device__ __forceinline__ uint32_t cut_term(float& f) {
  const uint32_t u = __float_as_uint(f);
  uint32_t h = u & 0xffff0000u;
  if ((u & 0x7f800000u) == 0x7f800000u) {
    if (u & 0x007fffffu) h |= 0x00400000u;  // NaN stays one
    f = 0.f;
  } else {
    f -= __uint_as_float(h);
  }
  return h >> 16;
}

template <int DT>
__global__ __launch_bounds__(kNT, 2) void dense8_wgrad_kernel(D8Args a) {
  typedef typename Elem<DT>::raw raw;
  constexpr int TERMS = DT == 1 ? 1 : DT == 2 ? 2 : 3;
  constexpr int BUF = (TERMS + 1) * kPlane;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * BUF];
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int wn = wave >> 1, wk = wave & 1;
  const int L = xcd_linear(blockIdx.x, gridDim.x);
  const int tiles = a.ntiles * a.ktiles;
  const int split = L / tiles, tile = L - split * tiles;
  const int kt = tile % a.ktiles, nt = tile / a.ktiles;
  const int n0 = nt * kT, k0 = kt * kT;
  const long long m0 = split * a.mps, m1 = min(a.M, m0 + a.mps);
  const int steps = (int)((m1 - m0 + kMS - 1) / kMS);

  // staging: dy rows tid / 16 and + 16, columns 8 (tid % 16); codes row tid / 8,
  // columns 16 (tid % 8)
  const int dr = tid >> 4, dc = (tid & 15) * 8, xr = tid >> 3, xc = (tid & 7) * 16;
  const int dn = a.N - n0 - dc, xn = a.K - k0 - xc;
  const raw* dyp = reinterpret_cast<const raw*>(a.dy) + n0 + dc;
  const int8_t* cp = a.codes + k0 + xc;
  const uint8_t* sp = a.scales + ((k0 + xc) >> 5);
  float dreg[2][8];
  uint32_t creg[4], ereg;
  auto load = [&](int s) {
    const long long m = m0 + (long long)s * kMS;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long r = m + dr + 16 * i;
      load8_n<DT>(dyp + r * a.dys, r < m1 ? dn : 0, 0.f, dreg[i]);
    }
    const long long r = m + xr;
    const int n = r < m1 ? xn : 0;
    creg[0] = creg[1] = creg[2] = creg[3] = 0u;
    ereg = 7u;
    if (n > 0) {
      const int8_t* p = cp + r * a.K;
      ereg = sp[r * a.kb];
      if (n >= 16) {
        const Bytes16 b = *reinterpret_cast<const Bytes16*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) creg[i] = b[i];
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (i < n) creg[i >> 2] |= (uint32_t)(uint8_t)p[i] << (8 * (i & 3));
      }
    }
  };
  auto store = [&](int s) {
    unsigned char* buf = smem + (s & 1) * BUF;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = dr + 16 * i;
      const int o = r * 256 + (((tid & 15) ^ tr_swz<256>(r)) << 4);
      if constexpr (TERMS == 1) {
        uint4 w;
        w.x = bf16_pair(dreg[i][0], dreg[i][1]);
        w.y = bf16_pair(dreg[i][2], dreg[i][3]);
        w.z = bf16_pair(dreg[i][4], dreg[i][5]);
        w.w = bf16_pair(dreg[i][6], dreg[i][7]);
        *reinterpret_cast<uint4*>(buf + o) = w;
      } else {
#pragma unroll
        for (int t = 0; t < TERMS; ++t) {
          uint32_t h[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) h[j] = cut_term(dreg[i][j]);
          const uint4 w = {h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16),
                           h[6] | (h[7] << 16)};
          *reinterpret_cast<uint4*>(buf + t * kPlane + o) = w;
        }
      }
    }
    const float step = step_of(ereg);
    unsigned char* xb = buf + TERMS * kPlane;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t c = creg[2 * h + (j >> 1)];
        w[j] = bf16_pair(code_at(c, 2 * (j & 1)) * step, code_at(c, 2 * (j & 1) + 1) * step);
      }
      *reinterpret_cast<uint4*>(xb + xr * 256 +
                                ((((tid & 7) * 2 + h) ^ tr_swz<256>(xr)) << 4)) =
          uint4{w[0], w[1], w[2], w[3]};
    }
  };

  f32x4 acc[4][4], bacc[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    bacc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const uint4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};

  if (steps > 0) load(0);
  for (int s = 0; s < steps; ++s) {
    store(s);
    __syncthreads();
    if (s + 1 < steps) load(s + 1);
    const unsigned char* buf = smem + (s & 1) * BUF;
    uint4 x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = col_frag<256>(buf + TERMS * kPlane, wk * 64 + j * 16, lane);
    const bool sum = a.db && wk == 0 && s % a.ktiles == kt;
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      uint4 d[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = col_frag<256>(buf + t * kPlane, wn * 64 + i * 16, lane);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mma16(d[i], x[j], acc[i][j]);
      if (sum)
#pragma unroll
        for (int i = 0; i < 4; ++i) bacc[i] = mma16(d[i], ones, bacc[i]);
    }
    // the next store goes to the other buffer: its readers passed the barrier above
  }

  const bool direct = a.splits == 1;
  float* out = direct ? a.dw : a.slab + (long long)split * a.N * a.K;
  const bool add = direct && (a.add & 1);
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + wn * 64 + i * 16 + 4 * (lane >> 4) + e;
      if (n >= a.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + wk * 64 + j * 16 + (lane & 15);
        if (k < a.K) {
          float* o = out + (long long)n * a.K + k;
          *o = add ? *o + acc[i][j][e] : acc[i][j][e];
        }
      }
    }
  if (a.db && wk == 0 && (lane & 15) == 0) {
    float* part = a.part + ((long long)split * a.ktiles + kt) * a.N;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn * 64 + i * 16 + 4 * (lane >> 4) + e;
        if (n < a.N) part[n] = bacc[i][e];
      }
  }
}

// ---------------------------------------------------------------------------
// The same product for large sizes: a block of 8 waves owns a 256 x 256 tile and
// walks 64 rows a step in two halves of 32.  dy rows go to LDS by LDS-DMA, two
// steps ahead into three buffers; codes go through registers, are decoded between
// the matrix instructions of the step before their use and stored as bf16 rows into
// two buffers.  One wave holds 128 x 64 of the tile, 32 accumulators of 16 x 16.
//
// One barrier per step, before its last quarter of products: behind it the first
// fragments of the next step are read while those products run, and nothing reads
// this step's buffers any more.  (With two dy buffers and two barriers a step took
// 4800 cycles whatever the load; the products are 2048 and the transposed LDS
// reads, at the measured 133 B per cycle, 1500.)  Each quarter's fragments are read a
// quarter ahead, six to eight at a time.  The barrier waits for the wave's own LDS
// reads and writes.  Loads return in order: the explicit vmcnt wait counts the
// instructions behind the dy rows that are needed (4 and 4 for the next codes, 4 for
// the dy rows after them).  Behind the last row both kinds read valid stand-ins, so
// the counts never change.
//
// The rows of a term are padded to whole steps (Mp = M rounded up to 64): dy rows
// behind M are zeros, so the kept rows beside them may be any that exist.  (A NaN
// block among those makes its columns of dW NaN, which they are anyway: the row is
// part of the sum.)
//
// dy needs whole 16-byte chunks (N and the row stride multiples of 8, 16-byte
// base).  Any other dy, and fp16 / fp32, is first cut into its bf16 terms,
// [term][Mp][N8], and the product runs over the terms one after the other (virtual
// row r: kept row r mod Mp).
//
// Measured: 16384 x 4096 x 4096 bf16 500 - 548 us over several machines (1.0 - 1.1
// PFLOP/s; the library's product of the same shape with a bf16 input 460, 555 on its
// first calls), fp16 1033 - 1093, fp32 1592 - 1602.
// ---------------------------------------------------------------------------
constexpr int kW = 256;                 // tile edge
constexpr int kWNT = 512;               // threads
constexpr int kWPiece = 32 * kW * 2;    // a half: 32 rows of 512 B
constexpr int kWBuf = 2 * kWPiece;      // a step's dy or x
constexpr int kWX = 3 * kWBuf;          // x behind three dy buffers
constexpr int kWLds = 5 * kWBuf;        // all 160 KB of a CU

__device__ __attribute__((aligned(512))) uint4 g_a8_zero[32];  // 512 B of zeros

struct D8WideArgs {
  const uint16_t* dy;     // [dyrows][dys] bf16
  const int8_t* codes;    // [M][K]
  const uint8_t* scales;  // [M][kb]
  float* dw;
  float* db;
  float* slab;
  float* part;
  long long dys;
  int rps;                // virtual rows of a split (multiple of 64)
  int dyrows;             // rows that exist: M, or all R of the terms
  int M, Mp, R, N, K, kb, ntiles, ktiles, splits, add;
};

// 16 bytes per lane to LDS address lds (wave-uniform) + 16 * lane, from a uniform
// base and 32-bit lane offsets, or from an address per lane (s_nop: the wait state
// between a scalar write of M0 and a load to LDS)
__device__ __forceinline__ void dma16(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off),
               "s"(base), "s"(lds)
               : "m0", "memory");
}
__device__ __forceinline__ void dma16_any(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src),
               "s"(lds)
               : "m0", "memory");
}

__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// KCUT: K is no multiple of 8.  All LDS is dynamic and addressed by byte from 0.
template <bool KCUT>
__global__ __launch_bounds__(kWNT, 2) void dense8_wide_kernel(D8WideArgs a) {
  typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) u32x4 lds_u128;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wn = wave >> 2, wk = wave & 3;
  const int L = xcd_linear(blockIdx.x, gridDim.x);
  const int tiles = a.ntiles * a.ktiles;
  const int split = L / tiles, tile = L - split * tiles;
  const int kt = tile % a.ktiles, nt = tile / a.ktiles;
  const int n0 = nt * kW, k0 = kt * kW;
  // R < 2^31 - 256: the steps that run ahead of the last row fit too
  const int r0 = split * a.rps, r1 = min(a.R, r0 + a.rps);
  const int steps = (r1 - r0) >> 6;

  // dy: instruction i of wave w fills piece rows (8 i + w) * 2 + (lane >> 5); LDS slot
  // lane & 31 holds the row's 16-byte chunk (lane & 31) ^ tr_swz(row).  Chunks behind N
  // are the tile's first one (their rows of dW are not stored).
  const int arow = wave * 2 + (lane >> 5);  // i = 1: + 16, the same swizzle
  const int chunk = (lane & 31) ^ tr_swz<512>(arow);
  const int acol = n0 + chunk * 8 < a.N ? chunk * 16 : 0;
  const unsigned char* dyb = reinterpret_cast<const unsigned char*>(a.dy) + n0 * 2LL;
  const long long dyrow = a.dys * 2;
  const uint32_t aoff = (uint32_t)(arow * (int)dyrow + acol);
  auto issue = [&](int s, int h, uint32_t buf) {
    const uint32_t dst = buf + h * kWPiece + wave * 1024;
    const int rb = r0 + s * 64 + h * 32;  // uniform
    if (rb + 32 <= a.dyrows) {
      const unsigned char* base = dyb + rb * dyrow;
      dma16(base, aoff, dst);
      dma16(base + 16 * dyrow, aoff, dst + 8192);
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = rb + arow + 16 * i;
        const unsigned char* src = reinterpret_cast<const unsigned char*>(g_a8_zero) + chunk * 16;
        if (r < a.dyrows) src = dyb + r * dyrow + acol;
        dma16_any(src, dst + i * 8192);
      }
    }
  };

  // codes: 8 of columns 8 (tid & 31) of rows tid >> 5 and + 16 of a half.  A chunk that K
  // cuts is read from the row's last 8 and moved down; columns behind K: any valid place.
  const int crow = tid >> 5, col = k0 + (tid & 31) * 8;
  const int cc = col >= a.K ? 0 : KCUT ? min(col, a.K - 8) : col;
  const int back = col >= a.K ? 0 : 8 * (col - cc);
  const int sc = (col >= a.K ? 0 : col) >> 5;
  const uint32_t coff = (uint32_t)(crow * a.K + cc), eoff = (uint32_t)(crow * a.kb + sc);
  struct Codes {
    Bytes8 w[2];
    uint32_t e[2];
  };
  auto fetch = [&](Codes& c, int s, int h) {
    int mb = r0 + s * 64 + h * 32;  // uniform; row in its term
#pragma unroll
    for (int i = 0; i < 3; ++i) mb = mb >= a.Mp ? mb - a.Mp : mb;  // past the last: any row
    mb = mb >= a.Mp ? 0 : mb;
    const int m0 = min(mb, a.M - 1);
    const int8_t* p = a.codes + (long long)m0 * a.K;
    const uint8_t* q = a.scales + (long long)m0 * a.kb;
    uint32_t oa = coff, ob = coff + 16 * a.K, ea = eoff, eb = eoff + 16 * a.kb;
    if (mb + 32 > a.M) {  // uniform; rows behind M: the last one
      const int ra = min(crow, a.M - 1 - m0), rb = min(crow + 16, a.M - 1 - m0);
      oa = (uint32_t)(ra * a.K + cc);
      ob = (uint32_t)(rb * a.K + cc);
      ea = (uint32_t)(ra * a.kb + sc);
      eb = (uint32_t)(rb * a.kb + sc);
    }
    c.w[0] = *reinterpret_cast<const Bytes8*>(p + oa);
    c.e[0] = q[ea];
    c.w[1] = *reinterpret_cast<const Bytes8*>(p + ob);
    c.e[1] = q[eb];
  };
  // the other 16 rows of a half have the same swizzle
  const uint32_t xput = crow * 512 + (((tid & 31) ^ tr_swz<512>(crow)) << 4);
  auto put = [&](const Codes& c, int s, int h) {
    const uint32_t at = xput + kWX + (s & 1) * kWBuf + h * kWPiece;
    // NaN blocks, the largest steps (E >= 254) and subnormal ones (E < 7, which wraps)
    const bool far_end = __any(max(c.e[0] - 7u, c.e[1] - 7u) >= 247u);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint32_t b[2] = {c.w[i][0], c.w[i][1]};
      if constexpr (KCUT) {
        const u64_t v = (((u64_t)b[1] << 32) | b[0]) >> back;
        b[0] = (uint32_t)v;
        b[1] = (uint32_t)(v >> 32);
      }
      u32x4 o;
      if (far_end) {
        const float st = step_of(c.e[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          o[j] = bf16_pair(code_at(b[j >> 1], 2 * (j & 1)) * st,
                           code_at(b[j >> 1], 2 * (j & 1) + 1) * st);
      } else {
        // code + 128 as an unsigned byte, which the conversion picks itself, and one
        // fma (538 us at 16384 x 4096 x 4096; signed bytes, v_cvt_f32_i32 with a byte
        // operand, 570).  At E = 254 the 128 steps to take off would overflow.
        const float st = __uint_as_float((c.e[i] - 6u) << 23), off = -128.f * st;
        b[0] ^= 0x80808080u;
        b[1] ^= 0x80808080u;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t w = b[j >> 1];
          const float x = (float)((w >> (16 * (j & 1))) & 0xffu);
          const float y = (float)((w >> (16 * (j & 1) + 8)) & 0xffu);
          o[j] = bf16_pair(__builtin_fmaf(x, st, off), __builtin_fmaf(y, st, off));
        }
      }
      *(lds_u128*)(uintptr_t)(at + i * 8192) = o;
    }
  };

  f32x4 acc[8][4], bacc[2];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  bacc[0] = bacc[1] = f32x4{0.f, 0.f, 0.f, 0.f};
  const uint4 ones = {0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
  uint4 d1[4], d2[4], x1[4], x2[4];
  // A fragment's byte address is (lane part) ^ (column block part): row, swizzled
  // chunk and buffer occupy separate bits.  Rows + 4: + 2048 and the chunk's lowest bit
  // flipped.  Recomputed at each read (one xor): kept in registers the 48
  // addresses would spill.
  const int q4 = (lane & 15) >> 2, p4 = lane & 3, frow = 8 * (lane >> 4) + q4;
  const uint32_t f0 = frow * 512 + (((p4 >> 1) ^ tr_swz<512>(frow)) << 4) + (p4 & 1) * 8;
  const uint32_t fd = f0 ^ (wn * 256), fx = f0 ^ (wk * 128);
  auto frag = [&](uint32_t l, uint32_t block, uint32_t piece) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(uintptr_t)((l ^ block) + piece));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_s16x4*)(uintptr_t)((l ^ (block | 16u)) + (piece + 2048)));
    const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(uint4, v);
  };
  auto readD = [&](uint4 (&d)[4], uint32_t buf, int h, int mh) {
    uint32_t l = fd + buf;
    asm volatile("" : "+v"(l));
#pragma unroll
    for (int i = 0; i < 4; ++i) d[i] = frag(l, mh * 128 + i * 32, h * kWPiece);
  };
  auto readX = [&](uint4& d0, uint4& d1, int s, int h, int j) {  // fragments j and j + 1
    uint32_t l = fx + kWX + (s & 1) * kWBuf;
    asm volatile("" : "+v"(l));
    d0 = frag(l, j * 32, h * kWPiece);
    d1 = frag(l, j * 32 + 32, h * kWPiece);
  };
  auto mma = [&](const uint4 (&d)[4], const uint4 (&x)[4], int mh) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[mh * 4 + i][j] = mma16(d[i], x[j], acc[mh * 4 + i][j]);
  };
  // db: the four waves with the same dy columns take a quarter of their fragments each
  auto sums = [&](const uint4 (&d)[4], int mh) {
    if ((wk >> 1) != mh) return;
    if (wk & 1) {
      bacc[0] = mma16(d[2], ones, bacc[0]);
      bacc[1] = mma16(d[3], ones, bacc[1]);
    } else {
      bacc[0] = mma16(d[0], ones, bacc[0]);
      bacc[1] = mma16(d[1], ones, bacc[1]);
    }
  };

  Codes c0, c1;
  uint32_t cur = 0, nxt = kWBuf, far = 2 * kWBuf;  // dy buffers of steps s, s + 1, s + 2
  issue(0, 0, cur);
  issue(0, 1, cur);
  fetch(c0, 0, 0);
  fetch(c1, 0, 1);
  put(c0, 0, 0);
  put(c1, 0, 1);
  fetch(c0, 1, 0);
  fetch(c1, 1, 1);
  issue(1, 0, nxt);
  issue(1, 1, nxt);
  wait_vmcnt<12>();  // dy of step 0
  lds_barrier();
  readD(d1, cur, 0, 0);
  readX(x1[0], x1[1], 0, 0, 0);
  readX(x1[2], x1[3], 0, 0, 2);
  for (int s = 0; s < steps; ++s) {
    const bool sum = a.db && s % a.ktiles == kt;  // uniform
    // half 0, the first 64 of the wave's dy columns
    readD(d2, cur, 0, 1);
    readX(x2[0], x2[1], s, 1, 0);
    __builtin_amdgcn_sched_barrier(0);
    put(c0, s + 1, 0);
    mma(d1, x1, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (sum) sums(d1, 0);
    fetch(c0, s + 2, 0);
    __builtin_amdgcn_sched_barrier(0);
    // ... the second
    readD(d1, cur, 1, 0);
    readX(x2[2], x2[3], s, 1, 2);
    __builtin_amdgcn_sched_barrier(0);
    mma(d2, x1, 1);
    if (sum) sums(d2, 1);
    __builtin_amdgcn_sched_barrier(0);
    // half 1
    readD(d2, cur, 1, 1);
    __builtin_amdgcn_sched_barrier(0);
    put(c1, s + 1, 1);
    mma(d1, x2, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (sum) sums(d1, 0);
    fetch(c1, s + 2, 1);
    issue(s + 2, 0, far);
    issue(s + 2, 1, far);
    __builtin_amdgcn_sched_barrier(0);
    wait_vmcnt<12>();  // dy of the next step
    lds_barrier();
    readD(d1, nxt, 0, 0);
    readX(x1[0], x1[1], s + 1, 0, 0);
    readX(x1[2], x1[3], s + 1, 0, 2);
    __builtin_amdgcn_sched_barrier(0);
    mma(d2, x2, 1);
    if (sum) sums(d2, 1);
    __builtin_amdgcn_sched_barrier(0);
    const uint32_t old = cur;
    cur = nxt;
    nxt = far;
    far = old;
  }
  wait_vmcnt<0>();  // no LDS-DMA may outlive the block

  const bool direct = a.splits == 1;
  float* out = direct ? a.dw : a.slab + (long long)split * a.N * a.K;
  const bool add = direct && (a.add & 1);
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = n0 + wn * 128 + i * 16 + 4 * (lane >> 4) + e;
      if (n >= a.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + wk * 64 + j * 16 + (lane & 15);
        if (k < a.K) {
          float* o = out + (long long)n * a.K + k;
          *o = add ? *o + acc[i][j][e] : acc[i][j][e];
        }
      }
    }
  if (a.db && (lane & 15) == 0) {
    float* part = a.part + ((long long)split * a.ktiles + kt) * a.N;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int n = n0 + wn * 128 + (2 * wk + i) * 16 + 4 * (lane >> 4) + e;
        if (n < a.N) part[n] = bacc[i][e];
      }
  }
}

// dy [M][dys] -> its bf16 terms [TERMS][Mp][N8]; columns behind N and rows behind M zero
template <int DT>
__global__ __launch_bounds__(kNT) void dense8_terms_kernel(const void* dy, long long dys,
                                                           long long M, long long Mp, int N,
                                                           int N8, uint16_t* out) {
  constexpr int TERMS = DT == 1 ? 1 : DT == 2 ? 2 : 3;
  typedef typename Elem<DT>::raw raw;
  const int chunks = N8 >> 3;
  const long long total = Mp * chunks, step = (long long)gridDim.x * kNT;
  for (long long id = (long long)blockIdx.x * kNT + threadIdx.x; id < total; id += step) {
    const long long m = total < (1LL << 31) ? (uint32_t)id / (uint32_t)chunks : id / chunks;
    const int c = (int)(id - m * chunks) * 8;
    float f[8];
    load8_n<DT>(reinterpret_cast<const raw*>(dy) + m * dys + c, m < M ? N - c : 0, 0.f, f);
#pragma unroll
    for (int t = 0; t < TERMS; ++t) {
      uint32_t h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = cut_term(f[j]);
      *reinterpret_cast<uint4*>(out + (t * Mp + m) * N8 + c) =
          uint4{h[0] | (h[1] << 16), h[2] | (h[3] << 16), h[4] | (h[5] << 16), h[6] | (h[7] << 16)};
    }
  }
}

// out[i] (+)= sum over p of part[p][i], in a fixed order, for dW and db in one launch.
struct D8Sum {
  const float* part;
  float* out;
  long long n;
  int parts, add;
  int blocks;  // of this sum
  bool wide;   // 4 values per thread, the parts in order; else sliced
};
constexpr int kSumNT = 1024;

__device__ __forceinline__ void sum_wide(const D8Sum& a, long long block) {
  typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // odd sizes
  const long long i = (block * kSumNT + threadIdx.x) * 4;
  if (i >= a.n) return;
  const float* q = a.part + i;
  if (i + 4 <= a.n) {
    f32x4 s = *reinterpret_cast<const f32x4u*>(q);
    int p = 1;
    for (; p + 4 <= a.parts; p += 4) {  // four loads in flight
      f32x4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const f32x4u*>(q + (p + j) * a.n);
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[j];
    }
    for (; p < a.parts; ++p) s += *reinterpret_cast<const f32x4u*>(q + p * a.n);
    if (a.add) s += *reinterpret_cast<const f32x4u*>(a.out + i);
    *reinterpret_cast<f32x4u*>(a.out + i) = s;
  } else {
    for (long long j = i; j < a.n; ++j) {
      float s = a.part[j];
      for (int p = 1; p < a.parts; ++p) s += a.part[p * a.n + j];
      a.out[j] = a.add ? s + a.out[j] : s;
    }
  }
}

// many parts of few values: 16 slices of the parts side by side, each in order, joined
// in order
__device__ __forceinline__ void sum_sliced(const D8Sum& a, long long block, float (&red)[16][64]) {
  const int col = threadIdx.x & 63, sl = threadIdx.x >> 6;
  const long long i = block * 64 + col;
  float s = 0.f;
  if (i < a.n) {
    const float* q = a.part + sl * a.n + i;
    int p = sl;
    for (; p + 48 < a.parts; p += 64, q += 64 * a.n) {  // four loads in flight
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = q[16 * j * a.n];
#pragma unroll
      for (int j = 0; j < 4; ++j) s += v[j];
    }
    for (; p < a.parts; p += 16, q += 16 * a.n) s += *q;
  }
  red[sl][col] = s;
  __syncthreads();
  if (sl == 0 && i < a.n) {
#pragma unroll
    for (int o = 1; o < 16; ++o) s += red[o][col];
    a.out[i] = a.add ? a.out[i] + s : s;
  }
}

__global__ __launch_bounds__(kSumNT) void dense8_sum_kernel(D8Sum dw, D8Sum db) {
  __shared__ float red[16][64];
  const bool first = (int)blockIdx.x < dw.blocks;
  const D8Sum& a = first ? dw : db;
  const long long block = first ? blockIdx.x : blockIdx.x - dw.blocks;
  if (a.wide) {
    sum_wide(a, block);
  } else {
    sum_sliced(a, block, red);
  }
}

D8Sum dense8_sum(const float* part, int parts, long long n, float* out, int add) {
  const bool wide = parts <= 8 || n >= (1 << 18);
  const long long per = wide ? 4LL * kSumNT : 64;
  return D8Sum{part, out, n, parts, add, (int)((n + per - 1) / per), wide};
}

// Sizes and workspace of one call.  wide: the 256 x 256 kernel.
struct D8Plan {
  bool wide, terms;       // terms: dy is cut into its bf16 terms first
  int ntiles, ktiles, splits, N8;
  long long rps;          // rows (wide: virtual rows) of a split
  long long slab, parts;  // floats
  long long bytes;
};

D8Plan dense8_plan(long long M, int N, int K, int dt, long long dys, bool aligned, int variant) {
  D8Plan p{};
  // us per call, 128 / 256 kernel (rows x outputs x inputs, bf16): 1024 x 1024 x 1024
  // 26 / 42, 4096 x 512 x 512 30 / 32, 16384 x 1024 x 128 30 / 36, 32768 x 256 x 512
  // 39 / 43, 512 x 2048 x 2048 31 / 30, 4096 x 768 x 768 45 / 37, 16384 x 1024 x 1024
  // 99 / 64, 16384 x 4096 x 4096 1448 / 498.
  p.wide = variant == 1 || (variant < 0 && M >= 64 && N >= 192 && K >= 192 &&
                            (long long)N * K >= (1 << 18) &&
                            (double)M * N * K >= 2147483648.0);
  const int T = p.wide ? kW : kT;
  p.ntiles = (N + T - 1) / T;
  p.ktiles = (K + T - 1) / T;
  const long long tiles = (long long)p.ntiles * p.ktiles;
  p.N8 = (N + 7) & ~7;
  p.terms = p.wide && (dt != 1 || !aligned || N != p.N8 || (dys & 7));
  const int terms = dt == 1 ? 1 : dt == 2 ? 2 : 3;
  long long s = 1;
  if (p.wide) {
    // one block per CU and about a microsecond per step: the split that takes the fewest
    // rounds of steps (12 more per block for its start and end) and slab bytes
    const long long R = terms * ((M + 63) / 64 * 64);
    double best = 1e30;
    for (long long c = 1; c <= 64 && (c == 1 || R / c >= 512); ++c) {
      const double rounds = (double)((tiles * c + 255) / 256);
      const double cost = rounds * ((double)(R / c) / 64 + 12) +
                          (c > 1 ? 8e-6 / 5 * (double)c * N * K + 5 : 0);
      if (cost < best) {
        best = cost;
        s = c;
      }
    }
    p.rps = ((R + s - 1) / s + 63) / 64 * 64;
    p.splits = (int)((R + p.rps - 1) / p.rps);
  } else {
    // two blocks per CU, at least 256 rows per split
    s = (512 + tiles - 1) / tiles;
    const long long most = (M + 255) / 256;
    if (s > most) s = most;
    if (s < 1) s = 1;
    p.rps = ((M + s - 1) / s + kMS - 1) / kMS * kMS;
    p.splits = (int)((M + p.rps - 1) / p.rps);
  }
  p.slab = p.splits > 1 ? (long long)p.splits * N * K : 0;
  p.parts = (long long)p.splits * p.ktiles * N;
  p.slab = (p.slab + 3) & ~3LL;
  p.parts = (p.parts + 3) & ~3LL;  // the terms start 16-byte aligned
  p.bytes = 4 * (p.slab + p.parts) + (p.terms ? 2LL * terms * ((M + 63) / 64 * 64) * p.N8 : 0);
  return p;
}

bool dense8_ok(long long M, int N, int K, long long dys) {
  return M >= 1 && N >= 1 && K >= 1 && M < (1LL << 29) && N < (1 << 24) && K < (1 << 24) &&
         dys >= 0 && dys < (1 << 24) &&
         ((N + kT - 1LL) / kT) * ((K + kT - 1LL) / kT) < (1 << 20);
}

int dense8_wide_launch(const D8WideArgs& a, hipStream_t st) {
  // by device: over 64 KB of LDS are allowed per kernel and device (twice does no harm)
  static std::atomic<bool> ready[64];
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return (int)e;
  if (dev < 0 || dev >= 64 || !ready[dev].load(std::memory_order_acquire)) {
    for (const void* f :
         {(const void*)dense8_wide_kernel<false>, (const void*)dense8_wide_kernel<true>}) {
      e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, kWLds);
      if (e != hipSuccess) return (int)e;
    }
    if (dev >= 0 && dev < 64) ready[dev].store(true, std::memory_order_release);
  }
  const dim3 g((unsigned)(a.ntiles * a.ktiles * a.splits));
  if (a.K & 7)
    hipLaunchKernelGGL(dense8_wide_kernel<true>, g, dim3(kWNT), kWLds, st, a);
  else
    hipLaunchKernelGGL(dense8_wide_kernel<false>, g, dim3(kWNT), kWLds, st, a);
  return (int)hipGetLastError();
}

}  // namespace

// x [rows][xs] -> codes [rows][D], scales [rows][ceil(D / 32)]; dt: 0 fp32, 1
// bf16, 2 fp16.
ZK_EXPORT int zk_pack8(const void* x, void* codes, void* scales, long long rows, long long D,
                       long long xs, int dt, hipStream_t st) {
  return act8_launch<kPack>(x, nullptr, codes, scales, rows, D, xs, dt, st);
}

ZK_EXPORT int zk_unpack8(const void* codes, const void* scales, void* out, long long rows,
                         long long D, int dt, hipStream_t st) {
  return act8_launch<kUnpack>(nullptr, out, const_cast<void*>(codes), const_cast<void*>(scales),
                              rows, D, D, dt, st);
}

// y = x Phi(x); codes / scales (both or neither): the 8-bit form of x.
ZK_EXPORT int zk_gelu8_fwd(const void* x, void* y, void* codes, void* scales, long long rows,
                           long long D, long long xs, int dt, hipStream_t st) {
  return codes ? act8_launch<kGeluKeep>(x, y, codes, scales, rows, D, xs, dt, st)
               : act8_launch<kGeluFwd>(x, y, nullptr, nullptr, rows, D, xs, dt, st);
}

// dx = dy (Phi(x8) + x8 phi(x8))
ZK_EXPORT int zk_gelu8_bwd(const void* dy, const void* codes, const void* scales, void* dx,
                           long long rows, long long D, long long dys, int dt, hipStream_t st) {
  return act8_launch<kGeluBwd>(dy, dx, const_cast<void*>(codes), const_cast<void*>(scales), rows, D,
                               dys, dt, st);
}

// Workspace bytes of zk_dense8_wgrad for the same arguments (aligned: dy starts on
// 16 bytes), or -1 for sizes it does not take.
ZK_EXPORT long long zk_dense8_wgrad_ws_bytes(long long M, int N, int K, long long dys, int dt,
                                             int aligned, int variant) {
  if (!dense8_ok(M, N, K, dys) || dt < 0 || dt > 2 || variant > 1 ||
      (variant == 1 && (M < 64 || K < 64)))
    return -1;
  return dense8_plan(M, N, K, dt, dys, aligned != 0, variant).bytes;
}

// dw [N][K] and db [N] (or null), fp32, from dy [M][dys] and the kept input
// [M][K].  add: bit 0 dw, bit 1 db are accumulated into instead of written.
// variant: 0 the 128 x 128 kernel, 1 the 256 x 256 one (M, K >= 64), -1 by size.
ZK_EXPORT int zk_dense8_wgrad(const void* dy, const void* codes, const void* scales, void* dw,
                              void* db, void* ws, long long ws_bytes, long long M, int N, int K,
                              long long dys, int dt, int add, int variant, hipStream_t st) {
  const bool aligned = ((uintptr_t)dy & 15) == 0;
  const long long need = zk_dense8_wgrad_ws_bytes(M, N, K, dys, dt, aligned, variant);
  if (need < 0 || (need > 0 && !ws) || ws_bytes < need || ((uintptr_t)ws & 15))
    return (int)hipErrorInvalidValue;
  const D8Plan p = dense8_plan(M, N, K, dt, dys, aligned, variant);
  const int kb = (K + 31) / 32;
  float* const slab = (float*)ws;
  if (p.wide) {
    const int terms = dt == 1 ? 1 : dt == 2 ? 2 : 3;
    const int Mp = (int)((M + 63) / 64 * 64);
    D8WideArgs a{(const uint16_t*)dy, (const int8_t*)codes, (const uint8_t*)scales, (float*)dw,
                 (float*)db, slab, slab + p.slab, dys, (int)p.rps, (int)M, (int)M, Mp,
                 terms * Mp, N, K, kb, p.ntiles, p.ktiles, p.splits, add};
    if (p.terms) {
      uint16_t* t = (uint16_t*)(slab + p.slab + p.parts);
      const long long blocks = ((long long)Mp * (p.N8 >> 3) + kNT - 1) / kNT;
      const dim3 g((unsigned)(blocks < (1 << 16) ? blocks : (1 << 16)));
      if (dt == 0)
        hipLaunchKernelGGL(dense8_terms_kernel<0>, g, dim3(kNT), 0, st, dy, dys, M, Mp, N, p.N8, t);
      if (dt == 1)
        hipLaunchKernelGGL(dense8_terms_kernel<1>, g, dim3(kNT), 0, st, dy, dys, M, Mp, N, p.N8, t);
      if (dt == 2)
        hipLaunchKernelGGL(dense8_terms_kernel<2>, g, dim3(kNT), 0, st, dy, dys, M, Mp, N, p.N8, t);
      ZK_CHECK_LAUNCH();
      a.dy = t;
      a.dys = p.N8;
      a.dyrows = a.R;
    }
    const int e = dense8_wide_launch(a, st);
    if (e) return e;
  } else {
    D8Args a{dy, (const int8_t*)codes, (const uint8_t*)scales, (float*)dw, (float*)db, slab,
             slab + p.slab, dys, M, N, K, kb, p.ntiles, p.ktiles, p.splits, add, p.rps};
    const dim3 g((unsigned)((long long)p.ntiles * p.ktiles * p.splits));
    if (dt == 0) hipLaunchKernelGGL(dense8_wgrad_kernel<0>, g, dim3(kNT), 0, st, a);
    if (dt == 1) hipLaunchKernelGGL(dense8_wgrad_kernel<1>, g, dim3(kNT), 0, st, a);
    if (dt == 2) hipLaunchKernelGGL(dense8_wgrad_kernel<2>, g, dim3(kNT), 0, st, a);
    ZK_CHECK_LAUNCH();
  }
  D8Sum sw{}, sb{};
  if (p.splits > 1) sw = dense8_sum(slab, p.splits, (long long)N * K, (float*)dw, add & 1);
  if (db) sb = dense8_sum(slab + p.slab, p.splits * p.ktiles, N, (float*)db, (add >> 1) & 1);
  if (sw.blocks + sb.blocks > 0)
    hipLaunchKernelGGL(dense8_sum_kernel, dim3((unsigned)(sw.blocks + sb.blocks)), dim3(kSumNT), 0,
                       st, sw, sb);
  ZK_CHECK_LAUNCH();
  return 0;
}
